"""The row operators of a language model's training step and of its scoring, as
measurable cases.

Each case is one pass through an operator of `jules_amd.ops`: dropout from a
counter-based generator (with the residual's addition or without), the residual's
addition with dropout and layer norm, their backward pass with the gradients of
the norm's weight and bias, log probabilities of given tokens with the entropy and
the most likely alternatives, and their gradient with respect to the logits.

Dropout: element (i, j) of [M, N] is dropped where its 16 random bits are below
t = round(65536 p), and otherwise multiplied by 65536 / (65536 - t).  The bits are
half word j % 8 (the low half of each word first) of Philox4x32 with 10 rounds
(Salmon, Moraes, Dror and Shaw, 2011) at the counter (j / 8, i, low and high word
of rng[1] + offset) and the key (low and high word of rng[0]).
"""
import math
import random

import torch

DEV = "cuda:0"
own = False  # False: the plain forms; True: the calls of the framework's operators

EPS = 1e-5
SITE = 7  # which of a step's masks
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2, "none": 0}


def listed():
    return [
        # a short sequence through a small model's embedding: latency counts
        dict(name="dropout_small", kind="dropout", rows=128, width=768, x="bf16", residual="none", p=0.1),
        # activations of an odd shape in fp32
        dict(name="dropout_ragged", kind="dropout", rows=1999, width=5001, x="f32", residual="none", p=0.25),
        # the end of a sublayer, a training step of the benchmark's attention shape:
        # 8 sequences of 4096 tokens, 32 heads of 128
        dict(name="dropout_add_step", kind="dropout", rows=32768, width=4096, x="bf16", residual="f32", p=0.1),
        # the norm of a few tokens, and its way back
        dict(name="norm_small", kind="norm", rows=64, width=1024, x="bf16", residual="bf16", p=0.1),
        dict(name="norm_grad_small", kind="norm_grad", rows=64, width=1024, x="bf16", h="bf16", dh=True, p=0.1),
        # a sublayer's dropout, addition and norm in that training step, and its way back
        dict(name="norm_step", kind="norm", rows=32768, width=4096, x="bf16", residual="bf16", p=0.1),
        dict(name="norm_grad_step", kind="norm_grad", rows=32768, width=4096, x="bf16", h="bf16", dh=True, p=0.1),
        # fine-tuning without dropout, an fp32 stream of odd width
        dict(name="norm_grad_ragged", kind="norm_grad", rows=1999, width=5001, x="f32", h="f32", dh=False, p=0.0),
        # one decoding step of 8 sequences that report 20 alternatives
        dict(name="logp_decode", kind="logp", rows=8, vocab=128256, pad=0, x="f32", scale=1.0, top=20, masked=False),
        # a prompt's tokens scored, with 5 alternatives each
        dict(name="logp_prompt", kind="logp", rows=2048, vocab=50257, pad=0, x="f32", scale=1.0, top=5, masked=False),
        # a policy's log probabilities and entropy over sampled texts, the rows of
        # a padded output layer, and the gradient of its objective
        dict(name="logp_policy", kind="logp", rows=4096, vocab=50257, pad=47, x="bf16", scale=1.25, top=0, masked=False),
        dict(name="logp_grad_policy", kind="logp_grad", rows=4096, vocab=50257, pad=47, x="bf16", scale=1.25, entropy=True,
             masked=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["dropout", "norm", "norm_grad", "logp", "logp", "logp_grad"])
    x = rng.choice(["bf16", "f32"])
    if kind in ("logp", "logp_grad"):
        vocab = _log(rng, 200, 260000)
        case = dict(kind=kind, rows=_log(rng, 1, min(16384, (1 << 26) // vocab)), vocab=vocab, pad=rng.choice([0, 0, -vocab % 64]),
                    x=x, scale=rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)]), masked=rng.random() < 0.25)
        if kind == "logp":
            return dict(case, top=rng.choice([0, 1, 5, 20, rng.randint(2, 64)]))
        return dict(case, entropy=rng.random() < 0.5)
    width = _log(rng, 64, 16384)
    p = rng.choice([0.0, 0.05, 0.1, 0.1, 0.25, 0.5])
    case = dict(kind=kind, rows=_log(rng, 1, min(32768, (1 << 25) // width)), width=width, x=x)
    if kind == "norm_grad":
        return dict(case, h=rng.choice(["bf16", "f32"]), dh=rng.random() < 0.7, p=p)
    if kind == "norm":
        return dict(case, residual=rng.choice(["bf16", "f32", "none"]), p=p)
    return dict(case, residual=rng.choice(["bf16", "f32", "none"]), p=p or 0.1)


def work(case):
    kind, x = case["kind"], _SIZE[case["x"]]
    if kind in ("logp", "logp_grad"):
        n = case["rows"] * case["vocab"]
        if kind == "logp":
            # logits and tokens in; three numbers and the alternatives out
            return {"bytes": n * x + case["rows"] * (4 + 12 + 8 * case["top"]), "flops": 6 * n}
        # logits, token, log-sum-exp and the loss's gradients in; the logits' out
        return {"bytes": 2 * n * x + case["rows"] * (12 + 8 * case["entropy"]), "flops": 8 * n}
    n = case["rows"] * case["width"]
    if kind == "dropout":
        r = _SIZE[case["residual"]]
        return {"bytes": n * (x + (2 * r if r else x)), "flops": 2 * n}
    if kind == "norm":
        r = _SIZE[case["residual"]]
        # without a residual the norm's input is kept only where dropout changed it
        kept = 2 * r if r else x if case["p"] else 0
        return {"bytes": n * (2 * x + kept) + 8 * case["width"] + 8 * case["rows"], "flops": 10 * n}
    h = _SIZE[case["h"]]
    # the output's gradient, h and what else reaches h's gradient in; h's gradient out, x's
    # apart from it where dropout or its type makes it another
    apart = x if case["p"] or x != h else 0
    return {"bytes": n * (x + h + h * case["dh"] + h + apart) + 12 * case["width"] + 8 * case["rows"], "flops": 14 * n}


# ---- inputs ------------------------------------------------------------------


def _moments(h):
    d = h.double()
    mean = d.mean(-1)
    return mean.float(), torch.rsqrt((d - mean[:, None]).square().mean(-1) + EPS).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    state = dict(case=case)
    x = _TYPES[case["x"]]
    if case["kind"] in ("logp", "logp_grad"):
        rows, vocab = case["rows"], case["vocab"]
        # some words are likely everywhere, and each place has likely words of its own
        whole = (2.0 * normal(vocab + case["pad"]) + 2.5 * normal(rows, vocab + case["pad"])).to(x)
        logits = whole[:, :vocab]
        if case["masked"]:  # what a grammar forbids
            logits.masked_fill_(torch.rand(rows, vocab, generator=gen, device=DEV) < 0.4, float("-inf"))
        # the likeliest token of most places, some other one elsewhere
        other = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
        tokens = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.7, logits.float().argmax(-1), other)
        state.update(logits=logits, tokens=tokens.to(torch.int32))
        if case["kind"] == "logp_grad":
            z = logits.double() * case["scale"]
            lse = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[:, None])
            state["lse"] = lse.float()
            state["entropy"] = (lse - (p * z.clamp(min=-1e30)).sum(-1)).float() if case["entropy"] else None
            state["dlogp"] = -normal(rows) / rows
            state["dentropy"] = torch.full((rows,), -0.01 / rows, device=DEV) if case["entropy"] else None
        return state
    shape = (case["rows"], case["width"])
    state["rng"] = torch.tensor([0x1234567 * (seed + 1), 1000 * seed], dtype=torch.int64, device=DEV)
    if case["kind"] == "norm_grad":
        h = (normal(*shape) * torch.exp(0.3 * normal(shape[1])) + 0.2 * normal(shape[1])).to(_TYPES[case["h"]])
        mean, rstd = _moments(h)
        state.update(h=h, mean=mean, rstd=rstd, dy=(0.01 * normal(*shape)).to(x), gamma=1.0 + 0.2 * normal(shape[1]),
                     dh=(0.01 * normal(*shape)).to(h.dtype) if case["dh"] else None)
        return state
    state["x"] = normal(*shape).to(x)
    # a residual stream: some channels larger than the others
    state["r"] = None if case["residual"] == "none" else (
        2.0 * torch.exp(0.5 * normal(shape[1])).clamp_(max=4.0) * normal(*shape)).to(_TYPES[case["residual"]])
    if case["kind"] == "norm":
        state.update(gamma=1.0 + 0.2 * normal(shape[1]), beta=0.1 * normal(shape[1]))
    return state


# ---- one pass ------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)(state, state["case"])


def _own(s, case):
    from jules_amd import ops

    if case["kind"] == "dropout":
        return dict(y=ops.dropout(s["x"], case["p"], s["rng"], offset=SITE, residual=s["r"]))
    if case["kind"] == "norm":
        y, h, mean, rstd = ops.add_layernorm(s["x"], s["r"], s["gamma"], s["beta"], EPS, p=case["p"], rng=s["rng"], offset=SITE)
        return dict(y=y, h=h, mean=mean, rstd=rstd)
    if case["kind"] == "norm_grad":
        dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(s["dy"], s["h"], s["mean"], s["rstd"], s["gamma"], dh=s["dh"], p=case["p"],
                                                      rng=s["rng"], offset=SITE)
        return dict(dx=dx, dr=dr, dgamma=dgamma, dbeta=dbeta)
    if case["kind"] == "logp":
        out = ops.token_logprobs(s["logits"], s["tokens"], scale=case["scale"], top=case["top"])
        return dict(logp=out.logp, lse=out.lse, entropy=out.entropy, ids=out.top_ids, top=out.top_logp)
    return dict(dx=ops.token_logprobs_bwd(s["logits"], s["tokens"], s["lse"], s["dlogp"], entropy=s["entropy"],
                                          dentropy=s["dentropy"], scale=case["scale"]))


def _plain(s, case):
    return {"dropout": _plain_dropout, "norm": _plain_norm, "norm_grad": _plain_norm_grad, "logp": _plain_logp,
            "logp_grad": _plain_logp_grad}[case["kind"]](s, case)


def _factors(s, rows, width, p):
    """What each element is multiplied by, fp32 [rows, width]."""
    t = round(65536 * p)
    low = 0xFFFFFFFF
    seed, at = s["rng"][0], s["rng"][1] + SITE
    k = [seed & low, seed >> 32 & low]
    blocks = (width + 7) // 8
    c = [torch.arange(blocks, device=DEV).expand(rows, blocks), torch.arange(rows, device=DEV)[:, None].expand(rows, blocks),
         (at & low).expand(rows, blocks), (at >> 32 & low).expand(rows, blocks)]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # 64 bits, wrapping
        c = [(b >> 32 & low) ^ c[1] ^ k[0], b & low, (a >> 32 & low) ^ c[3] ^ k[1], a & low]
        k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
    words = torch.stack(c, -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, 8 * blocks)[:, :width]
    return (bits >= t).float() * (65536.0 / (65536 - t))


def _plain_dropout(s, case):
    y = s["x"].float() * _factors(s, case["rows"], case["width"], case["p"])
    if s["r"] is None:
        return dict(y=y.to(s["x"].dtype))
    return dict(y=(s["r"].float() + y).to(s["r"].dtype))


def _plain_norm(s, case):
    x, r = s["x"], s["r"]
    h = x.float()
    if case["p"]:
        h = h * _factors(s, case["rows"], case["width"], case["p"])
    if r is not None:
        h = r.float() + h
    mean = h.mean(-1, keepdim=True)
    d = h - mean
    rstd = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
    y = d * rstd * s["gamma"] + s["beta"]
    return dict(y=y.to(x.dtype), h=h.to(x.dtype if r is None else r.dtype), mean=mean[:, 0], rstd=rstd[:, 0])


def _plain_norm_grad(s, case):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    n = (s["h"].float() - s["mean"][:, None]) * rstd
    a = dy * s["gamma"]
    dr = rstd * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    if s["dh"] is not None:
        dr = dr + s["dh"].float()
    dx = dr * _factors(s, case["rows"], case["width"], case["p"]) if case["p"] else dr
    return dict(dx=dx.to(s["dy"].dtype), dr=dr.to(s["h"].dtype), dgamma=(dy * n).sum(0), dbeta=dy.sum(0))


def _plain_logp(s, case):
    x = s["logits"].float()
    z = x * case["scale"]
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log = torch.log(total)
    entropy = log - (e * d.clamp(min=-1e30)).sum(-1, keepdim=True) / total
    out = dict(logp=(d.gather(1, s["tokens"].long()[:, None]) - log)[:, 0], lse=(z.amax(-1, keepdim=True) + log)[:, 0],
               entropy=entropy[:, 0], ids=None, top=None)
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        out["ids"], out["top"] = ids.to(torch.int32), d.gather(1, ids) - log
    return out


def _plain_logp_grad(s, case):
    log = s["logits"].float() * case["scale"] - s["lse"][:, None]
    p = torch.exp(log)
    g = -p * s["dlogp"][:, None]
    if s["entropy"] is not None:
        g = g - p * (log.clamp(min=-1e30) + s["entropy"][:, None]) * s["dentropy"][:, None]
    g.scatter_add_(1, s["tokens"].long()[:, None], s["dlogp"][:, None])
    return dict(dx=(g * case["scale"]).to(s["logits"].dtype))


# ---- the definitions, in 64 bits ----------------------------------------------


def _exact_factors(s, case):
    """The factors from the generator in numpy's 64-bit unsigned numbers, some rows at a time."""
    import numpy as np

    t = round(65536 * case["p"])
    seed, at = (int(v) for v in s["rng"])
    at = (at + SITE) % 2**64
    blocks = -(-case["width"] // 8)
    parts = []
    for first in range(0, case["rows"], 4096):
        rows = min(4096, case["rows"] - first)
        c = [np.arange(blocks, dtype=np.uint32), np.arange(first, first + rows, dtype=np.uint32)[:, None],
             np.uint32(at % 2**32), np.uint32(at // 2**32)]
        c = [np.broadcast_to(v, (rows, blocks)) for v in c]
        for i in range(10):
            wide = [np.multiply(c[j], m, dtype=np.uint64) for j, m in ((0, 0xD2511F53), (2, 0xCD9E8D57))]
            halves = [w.view(np.uint32).reshape(rows, blocks, 2) for w in wide]  # low, high
            key = [np.uint32((seed % 2**32 + i * 0x9E3779B9) % 2**32), np.uint32((seed // 2**32 + i * 0xBB67AE85) % 2**32)]
            c = [halves[1][..., 1] ^ c[1] ^ key[0], halves[1][..., 0], halves[0][..., 1] ^ c[3] ^ key[1], halves[0][..., 0]]
        bits = np.stack(c, -1).view(np.uint16).reshape(rows, 8 * blocks)[:, :case["width"]]
        parts.append(torch.from_numpy(bits >= t).to(DEV))
    return torch.cat(parts).double() * (65536 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logp":
        return _exact_logp(s, case)
    if case["kind"] == "logp_grad":
        log = torch.log_softmax(s["logits"].double() * case["scale"], -1)
        p = torch.exp(log)
        g = -s["dlogp"].double()[:, None] * p
        g[torch.arange(case["rows"], device=DEV), s["tokens"].long()] += s["dlogp"].double()
        if s["dentropy"] is not None:
            entropy = -(p * log.clamp(min=-1e300)).sum(-1, keepdim=True)
            g -= s["dentropy"].double()[:, None] * p * (log.clamp(min=-1e300) + entropy)
        return dict(dx=case["scale"] * g)
    f = _exact_factors(s, case) if case["p"] else 1.0
    if case["kind"] == "dropout":
        y = f * s["x"].double()
        return dict(y=y if s["r"] is None else y + s["r"].double())
    if case["kind"] == "norm":
        h = f * s["x"].double()
        if s["r"] is not None:
            h = h + s["r"].double()
        var, mean = torch.var_mean(h, -1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        return dict(y=(h - mean[:, None]) * rstd[:, None] * s["gamma"].double() + s["beta"].double(), h=h, mean=mean, rstd=rstd)
    # the norm's gradient by the projection off the constant and the normalised row
    dy, width = s["dy"].double(), case["width"]
    var, mean = torch.var_mean(s["h"].double(), -1, correction=0, keepdim=True)
    n = (s["h"].double() - mean) / torch.sqrt(var + EPS)
    a = dy * s["gamma"].double()
    a = a - (a.sum(-1, keepdim=True) + n * (a * n).sum(-1, keepdim=True)) / width
    dr = a / torch.sqrt(var + EPS)
    if s["dh"] is not None:
        dr = dr + s["dh"].double()
    return dict(dx=f * dr, dr=dr, dgamma=(n * dy).sum(0), dbeta=dy.sum(0))


def _exact_logp(s, case):
    x = s["logits"].double()
    log = torch.log_softmax(x * case["scale"], -1)
    at = torch.arange(case["rows"], device=DEV)
    out = dict(logp=log[at, s["tokens"].long()], lse=torch.logsumexp(x * case["scale"], -1),
               entropy=-(torch.exp(log) * log.clamp(min=-1e300)).sum(-1), ids=None, top=None)
    if case["top"]:
        ids, left = [], x.clone()
        for _ in range(case["top"]):  # the lowest index of the largest that is left
            here = (left == left.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)
            ids.append(here)
            left[at, here] = -math.inf
        ids = torch.stack(ids, -1)
        out["ids"], out["top"] = ids.to(torch.int32), log.gather(1, ids)
    return out
