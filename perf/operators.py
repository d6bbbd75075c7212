"""The operators around a quantised decoder's products, as measurable cases.

Each case is one pass through an operator of `jules_amd.ops`, as a decoder calls
it between its matrix products: the residual's addition with the
root-mean-square norm (int8 rows and per-token scales for `matmul_w8a8`, or
rows of the input's type), rotary positions of one or several axes and their
backward pass, rows written into and read back from a paged key/value cache
held in 4 bits, and attention over that cache for single tokens, for drafts
and for chunks of a prompt.

The 4-bit cache: a row is the D values of one token and key/value head.  It is
held as (scale s, minimum m), both bf16, and D codes of 4 bits; code c stands
for m + s * c.  Pages of `page` tokens:
  k       uint8 [pages, heads, page, D/2]; of 8 neighbouring elements e = 0..7,
          the four bytes hold (e0, e2), (e4, e6), (e1, e3), (e5, e7), the first
          of each two in the low half of its byte
  v       uint8 [pages, heads, page/4, 2*D]; of 4 tokens t = 0..3 and 4
          neighbouring elements e = 0..3, the eight bytes hold (e0, e1), (e2, e3)
          of t0, then of t1, t2 and t3
  k_meta, v_meta  bf16 [pages, heads, page, 2]: s and m of each row
"""
import math
import random

import torch

DEV = "cuda:0"
own = False  # False: the plain forms; True: the calls of the framework's operators

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}


def listed():
    return [
        # one decoding step of 8 sequences at the width of the W8A16 decode
        # configuration: int8 rows for the next product
        dict(name="norm_int8_decode", kind="norm", rows=8, width=8192, x="bf16", residual="f32", out="i8"),
        # a prompt's rows between two int8 products
        dict(name="norm_int8_prompt", kind="norm", rows=8192, width=8192, x="bf16", residual="bf16", out="i8"),
        # an fp32 residual stream of odd width, rows as they are
        dict(name="norm_ragged", kind="norm", rows=1999, width=5001, x="f32", residual="f32", out="f32"),
        # one decoding step far into its text: query and key heads of one fused
        # projection, in fp32 as the int8 product leaves them
        dict(name="rotary_decode", kind="rotary", batch=1, tokens=8, heads=40, gap=8, dim=128, rotated=128, axes=1,
             pairing="half", inverse=False, x="f32", out="bf16", last=1000000),
        # a video's tokens: time, height and width
        dict(name="rotary_video", kind="rotary", batch=2, tokens=8000, heads=40, gap=8, dim=128, rotated=128, axes=3,
             pairing="half", inverse=False, x="bf16", out="bf16", last=4000),
        # the gradient's way back through the heads of a training step of the
        # benchmark's attention shape, half of each head rotated
        dict(name="rotary_backward", kind="rotary", batch=8, tokens=4096, heads=32, gap=0, dim=128, rotated=64, axes=2,
             pairing="adjacent", inverse=True, x="bf16", out="bf16", last=4096),
        # the rows of one decoding step into the cache, and back
        dict(name="append_decode", kind="append", batch=64, new=1, ragged=False, length=4096, kv_heads=8, head_dim=128,
             page=64, x="bf16"),
        # a batch of prompts into the cache, and back
        dict(name="append_prompt", kind="append", batch=16, new=2048, ragged=True, length=4096, kv_heads=8, head_dim=128,
             page=64, x="f32"),
        # one token of one sequence: latency counts
        dict(name="attend_one", kind="attend", batch=1, new=1, ragged=False, length=1000, kv_heads=8, group=4,
             head_dim=128, page=64),
        # a serving batch of unequal lengths
        dict(name="attend_batch", kind="attend", batch=64, new=1, ragged=True, length=8192, kv_heads=8, group=8,
             head_dim=128, page=64),
        # drafted tokens of one very long text
        dict(name="attend_long", kind="attend", batch=1, new=5, ragged=False, length=131072, kv_heads=4, group=8,
             head_dim=64, page=256),
        # chunks of prompts over what the cache holds of them
        dict(name="attend_chunk", kind="attend", batch=4, new=1024, ragged=True, length=8192, kv_heads=8, group=4,
             head_dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "append", "attend", "attend"])
    if kind == "norm":
        width = _log(rng, 64, 16384)
        x = rng.choice(["bf16", "f32"])
        return dict(kind=kind, rows=_log(rng, 1, min(16384, (1 << 25) // width)), width=width, x=x,
                    residual=rng.choice(["bf16", "f32", "none"]), out=rng.choice(["i8", "i8", x]))
    if kind == "rotary":
        axes = rng.choice([1, 1, 2, 3])
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        heads = _log(rng, 1, 64)
        batch = rng.choice([1, 1, 2, 3])
        tokens = _log(rng, 1, (1 << 26) // (batch * heads * dim))
        x = rng.choice(["bf16", "f32"])
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, gap=rng.choice([0, heads]), dim=dim,
                    rotated=rng.choice([dim, dim // 2]), axes=axes, pairing=rng.choice(["half", "adjacent"]),
                    inverse=rng.random() < 0.3, x=x, out=rng.choice([x, "bf16"]),
                    last=_log(rng, 100, 1000000) if axes == 1 else _log(rng, 100, 10000))
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    head_dim = rng.choice([64, 128, 128])
    batch = _log(rng, 1, 64)
    if kind == "append":
        new = _log(rng, 1, 16384 // batch)
        return dict(kind=kind, batch=batch, new=new, ragged=rng.random() < 0.7, length=new + _log(rng, 1, 4096),
                    kv_heads=min(kv_heads, 8), head_dim=head_dim, page=page, x=rng.choice(["bf16", "f32"]))
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    new = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 512)])
    # no more keys to lay out, and no more scores, than the largest listed case
    most = min(131072, (1 << 18) // batch * 8 // kv_heads, (1 << 28) // (batch * kv_heads * group * new))
    return dict(kind=kind, batch=batch, new=new, ragged=rng.random() < 0.7, length=new + _log(rng, 1, max(1, most - new)),
                kv_heads=kv_heads, group=group, head_dim=head_dim, page=page)


# ---- what a case says of its sequences -------------------------------------


def _sequences(case):
    """(lengths with the new tokens, numbers of new tokens) of the sequences:
    the longest of each at full size, the others of a ragged batch anywhere
    between a token (a sixteenth of the length) and that."""
    rng = random.Random(case["batch"] * 1000003 + case["new"] * 1009 + case["length"])
    new = [case["new"]] * case["batch"]
    lens = [case["length"]] * case["batch"]
    if case["ragged"]:
        for b in range(1, case["batch"]):
            new[b] = rng.randint(1, case["new"])
            lens[b] = rng.randint(max(new[b], case["length"] // 16), case["length"])
    return lens, new


def work(case):
    if case["kind"] == "norm":
        n, size = case["rows"] * case["width"], {"f32": 4, "bf16": 2, "i8": 1, "none": 0}
        r = size[case["residual"]]
        b = n * (size[case["x"]] + 2 * r + size[case["out"]]) + 4 * case["width"]
        return {"bytes": b + (4 * case["rows"] if case["out"] == "i8" else 0), "flops": 6 * n}
    if case["kind"] == "rotary":
        t = case["batch"] * case["tokens"]
        n, size = t * case["heads"] * case["dim"], {"f32": 4, "bf16": 2}
        return {"bytes": n * (size[case["x"]] + size[case["out"]]) + 4 * t * case["axes"] + 6 * case["rotated"],
                "flops": 3 * t * case["heads"] * case["rotated"]}
    lens, new = _sequences(case)
    row = case["head_dim"] + 8  # codes, scale and minimum of a key row and a value row
    if case["kind"] == "append":
        n = 2 * sum(new) * case["kv_heads"] * case["head_dim"]
        # rows in, codes out, codes in, values out
        return {"bytes": n * ({"f32": 4, "bf16": 2}[case["x"]] + 2) + 2 * sum(new) * case["kv_heads"] * row, "flops": 6 * n}
    heads = case["kv_heads"] * case["group"]
    seen = sum(n * (l - n) + n * (n + 1) // 2 for l, n in zip(lens, new))
    return {"bytes": sum(lens) * case["kv_heads"] * row + sum(new) * heads * (4 * case["head_dim"] + 4),
            "flops": 4 * seen * heads * case["head_dim"]}


# ---- inputs ------------------------------------------------------------------


def _quantise(x):
    """Rows of fp32 values -> (codes int32, scale and minimum bf16 [..., 2])."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, m = ((hi - lo) / 15.0).to(torch.bfloat16), lo.to(torch.bfloat16)
    c = torch.where(s > 0, torch.round((x - m.float()) / s.float()), torch.zeros_like(x)).clamp_(0, 15)
    return c.to(torch.int32), torch.cat([s, m], -1)


def _k_bytes(c):
    """Codes [..., D] -> the bytes of key rows [..., D/2]."""
    c = c.reshape(*c.shape[:-1], c.shape[-1] // 8, 4, 2).transpose(-1, -2)  # e = 2 * j + half -> [half, j]
    c = c.reshape(*c.shape[:-2], 4, 2)
    return (c[..., 0] | c[..., 1] << 4).to(torch.uint8).flatten(-2)


def _v_bytes(c):
    """Codes [..., D] -> the bytes of a token's value row [..., D/4, 2]."""
    c = c.reshape(*c.shape[:-1], c.shape[-1] // 4, 2, 2)
    return (c[..., 0] | c[..., 1] << 4).to(torch.uint8)


def _cache(case, gen, lens, filled):
    """A pool with the sequences' pages in random places, a few pages more."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    need = [-(-l // page) for l in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV, dtype=torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    state = dict(table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if filled:
        # some channels of keys are much larger than the rest
        wide = 1.0 + 3.0 * (torch.rand(dim, generator=gen, device=DEV) > 0.95)
        c, state["k_meta"] = _quantise(torch.randn(pages, heads, page, dim, generator=gen, device=DEV) * wide)
        state["k"] = _k_bytes(c)
        c, state["v_meta"] = _quantise(torch.randn(pages, heads, page, dim, generator=gen, device=DEV))
        c = _v_bytes(c).reshape(pages, heads, page // 4, 4, dim // 4, 2)
        state["v"] = c.transpose(-2, -3).reshape(pages, heads, page // 4, 2 * dim).contiguous()
    else:
        state["k"] = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device=DEV)
        state["v"] = torch.zeros(pages, heads, page // 4, 2 * dim, dtype=torch.uint8, device=DEV)
        for n in ("k_meta", "v_meta"):
            state[n] = torch.zeros(pages, heads, page, 2, dtype=torch.bfloat16, device=DEV)
    return state


def _rotary_case(case, gen):
    pairs = case["rotated"] // 2
    p = torch.arange(pairs, dtype=torch.float64, device=DEV)
    axis = torch.arange(pairs, device=DEV) * case["axes"] // pairs  # neighbouring pairs share an axis
    t = case["batch"] * case["tokens"]
    if case["axes"] == 1:  # the last tokens of a long text, or all of a shorter one
        first = max(0, case["last"] - case["tokens"])
        pos = (first + torch.arange(t, device=DEV) % case["tokens"]).reshape(1, t)
    else:
        pos = torch.randint(0, case["last"], (case["axes"], t), generator=gen, device=DEV)
    # heads of a fused projection: `gap` more of them between two tokens
    x = torch.randn(case["batch"], case["tokens"], case["heads"] + case["gap"], case["dim"], generator=gen, device=DEV)
    x = x.to(_TYPES[case["x"]])[:, :, :case["heads"]].transpose(1, 2)
    return dict(x=x, pos=pos.to(torch.int32).reshape(case["axes"], case["batch"], case["tokens"]).contiguous(),
                freq=torch.pow(10000.0, -p / pairs), axis=axis.to(torch.int32))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case)
    if case["kind"] == "norm":
        shape = (case["rows"], case["width"])
        # a residual stream: a few channels and tokens much larger than the rest, a padded row
        size = torch.exp(0.5 * torch.randn(case["width"], generator=gen, device=DEV)).clamp_(max=4.0)
        x = torch.randn(shape, generator=gen, device=DEV)
        r = 2.0 * size * torch.randn(shape, generator=gen, device=DEV)
        if case["rows"] > 4:
            x[3], r[3] = 0.0, 0.0
        state.update(x=x.to(_TYPES[case["x"]]), w=1.0 + 0.2 * torch.randn(case["width"], generator=gen, device=DEV),
                     r=None if case["residual"] == "none" else r.to(_TYPES[case["residual"]]))
    elif case["kind"] == "rotary":
        state.update(_rotary_case(case, gen))
    else:
        lens, new = _sequences(case)
        state.update(_cache(case, gen, lens, case["kind"] == "attend"))
        ends = [0]
        for n in new:
            ends.append(ends[-1] + n)
        # equal numbers of new tokens need no list of where each sequence's begin
        state["cu"] = torch.tensor(ends, dtype=torch.int32, device=DEV) if case["ragged"] else None
        if case["kind"] == "append":
            rows = torch.randn(2, ends[-1], case["kv_heads"], case["head_dim"], generator=gen, device=DEV)
            state["k_new"], state["v_new"] = rows.to(_TYPES[case["x"]])
        else:
            q = torch.randn(ends[-1], case["kv_heads"] * case["group"], case["head_dim"], generator=gen, device=DEV)
            state["q"] = q.to(torch.bfloat16)
    return state


# ---- one pass ------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)(state, state["case"])


def _own(s, case):
    from jules_amd import ops

    if case["kind"] == "norm":
        if case["out"] == "i8":
            q, scale, r = ops.add_rmsnorm_int8(s["x"], s["r"], s["w"], 1e-5)
            y = torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))
            return dict(y=y, scale=scale, r=r)
        y, r = ops.add_rmsnorm(s["x"], s["r"], s["w"], 1e-5)
        return dict(y=y, r=r)
    if case["kind"] == "rotary":
        return dict(y=ops.rotary(s["x"], s["pos"], s["freq"], s["axis"], pairing=case["pairing"], inverse=case["inverse"],
                                 dtype=_TYPES[case["out"]]))
    cache = ops.KV4Cache(s["k"], s["v"], s["k_meta"], s["v_meta"])
    if case["kind"] == "append":
        ops.kv4_append(cache, s["k_new"], s["v_new"], s["table"], s["lens"], cu_q=s["cu"], max_q=case["new"])
        k, v = ops.kv4_read(cache, s["table"], s["lens"], s["k_new"].shape[0], cu_q=s["cu"], max_q=case["new"])
        return dict(k=k, v=v)
    o, lse = ops.kv4_attention(s["q"], cache, s["table"], s["lens"], cu_q=s["cu"], max_q=case["new"],
                               max_len=case["length"], return_lse=True)
    return dict(o=o, lse=lse)


def _plain(s, case):
    if case["kind"] == "norm":
        return _plain_norm(s, case)
    if case["kind"] == "rotary":
        return _plain_rotary(s, case)
    return _plain_append(s, case) if case["kind"] == "append" else _plain_attend(s, case)


def _plain_norm(s, case):
    x, r = s["x"], s["r"]
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * s["w"]
    kept = None if r is None else h.to(r.dtype)
    if case["out"] != "i8":
        return dict(y=y.to(x.dtype), r=kept)
    scale = y.abs().amax(-1, keepdim=True) / 127.0
    q = torch.where(scale > 0, torch.round(y / scale), torch.zeros_like(y)).to(torch.int8)
    return dict(y=(q * scale).to(torch.bfloat16), scale=scale[:, 0], r=kept)


def _plain_rotary(s, case):
    x, rot = s["x"].float(), case["rotated"]
    # far positions: the angle in 64 bits
    a = s["pos"].double()[s["axis"].long()] * s["freq"][:, None, None]  # [pairs, batch, tokens]
    a = a.permute(1, 2, 0)[:, None]
    cos, sin = torch.cos(a).float(), torch.sin(a).float()
    if case["inverse"]:
        sin = -sin
    if case["pairing"] == "half":
        u, w = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([u * cos - w * sin, u * sin + w * cos, x[..., rot:]], -1)
    else:
        u, w = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.cat([torch.stack([u * cos - w * sin, u * sin + w * cos], -1).flatten(-2), x[..., rot:]], -1)
    return dict(y=y.to(_TYPES[case["out"]]))


def _new_tokens(s, tokens):
    """(sequence, position in it) of each new token."""
    n, dev = s["lens"].numel(), s["lens"].device
    cu = s["cu"] if s["cu"] is not None else torch.arange(n + 1, dtype=torch.int32, device=dev) * (tokens // n)
    t = torch.arange(tokens, device=dev)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    return b, s["lens"][b] - cu[b + 1] + t


def _nibbles(x):
    return torch.stack([x & 15, x >> 4], -1)


def _k_values(k, meta):
    """Bytes [..., D/2] and (s, m) [..., 2] of key rows -> their values [..., D]."""
    c = _nibbles(k.reshape(*k.shape[:-1], k.shape[-1] // 4, 2, 2)).flatten(-2)  # [half, j]
    return meta[..., 1:].float() + meta[..., :1].float() * c.transpose(-1, -2).flatten(-3).float()


def _v_values(v, meta):
    """Bytes [..., page/4, 2*D] and (s, m) [..., page, 2] of a page's value rows -> [..., page, D]."""
    c = v.reshape(*v.shape[:-1], v.shape[-1] // 8, 4, 2).transpose(-2, -3)
    c = _nibbles(c).flatten(-3).flatten(-3, -2)
    return meta[..., 1:].float() + meta[..., :1].float() * c.float()


def _plain_append(s, case):
    k, v, page = s["k_new"].float(), s["v_new"].float(), case["page"]
    b, at = _new_tokens(s, k.shape[0])
    pages, off = s["table"][b, at // page].long(), at % page
    c, m = _quantise(k)
    s["k"][pages, :, off] = _k_bytes(c)
    s["k_meta"][pages, :, off] = m
    c, m = _quantise(v)
    held = s["v"].view(*s["v"].shape[:-1], case["head_dim"] // 4, 4, 2)
    held[pages, :, off // 4, :, off % 4] = _v_bytes(c)
    s["v_meta"][pages, :, off] = m
    k = _k_values(s["k"][pages, :, off], s["k_meta"][pages, :, off])
    c = _nibbles(held[pages, :, off // 4, :, off % 4]).flatten(-3).float()
    m = s["v_meta"][pages, :, off].float()
    return dict(k=k.to(torch.bfloat16), v=(m[..., 1:] + m[..., :1] * c).to(torch.bfloat16))


def _plain_attend(s, case):
    q, table, lens = s["q"], s["table"].clamp(min=0).long(), s["lens"].long()
    heads, group, dim, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    batch, new, longest = case["batch"], case["new"], table.shape[1] * page
    k = _k_values(s["k"][table], s["k_meta"][table]).transpose(1, 2).reshape(batch, heads, longest, dim)
    v = _v_values(s["v"][table], s["v_meta"][table]).transpose(1, 2).reshape(batch, heads, longest, dim)
    b, at = _new_tokens(s, q.shape[0])
    place = b * new + at - (lens[b] - new)  # the last new token of each sequence is its last row
    rows = torch.zeros(batch * new, heads * group, dim, device=q.device)
    rows[place] = q.float()
    rows = rows.reshape(batch, new, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, heads, new * group, dim)
    scores = torch.matmul(rows, k.transpose(2, 3)).mul_(dim ** -0.5)
    key = torch.arange(longest, device=q.device)
    last = lens[:, None] - new + torch.arange(new, device=q.device)  # rows before the first new token are dropped below
    hidden = key > last.clamp(min=0)[:, :, None]
    scores.view(batch, heads, new, group, longest).masked_fill_(hidden[:, None, :, None], float("-inf"))
    # what a page holds behind its sequence's end is not read
    v = torch.where((key < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp_(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total
    o = o.reshape(batch, heads, new, group, dim).permute(0, 2, 1, 3, 4).reshape(batch * new, heads * group, dim)
    lse = (top + torch.log(total)).reshape(batch, heads, new, group).permute(0, 2, 1, 3).reshape(batch * new, heads * group)
    return dict(o=o[place].to(torch.bfloat16), lse=lse[place])


# ---- the definitions, in 64 bits ----------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double()
        h = h if s["r"] is None else h + s["r"].double()
        y = s["w"].double() * h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["width"] + 1e-5)
        out = dict(y=y, r=None if s["r"] is None else h)
        if case["out"] == "i8":
            out["scale"] = y.abs().max(-1).values / 127
            step = out["scale"].clamp(min=1e-300)[:, None]
            out["y"] = torch.round(y / step) * step
        return out
    if case["kind"] == "rotary":
        return _exact_rotary(s, case)
    return _exact_append(s, case) if case["kind"] == "append" else _exact_attend(s, case)


def _exact_rotary(s, case):
    # a pair as a complex number, times exp(i * angle)
    x, rot = s["x"].double(), case["rotated"]
    sign = -1.0 if case["inverse"] else 1.0
    out = x.clone()
    for p in range(rot // 2):
        i, j = (p, p + rot // 2) if case["pairing"] == "half" else (2 * p, 2 * p + 1)
        a = sign * s["freq"][p] * s["pos"][int(s["axis"][p])].double()
        z = torch.complex(x[..., i], x[..., j]) * torch.polar(torch.ones_like(a), a)[:, None]
        out[..., i], out[..., j] = z.real, z.imag
    return dict(y=out)


def _exact_append(s, case):
    out = {}
    for n in ("k", "v"):
        x = s[n + "_new"].double()
        low = x.min(-1, keepdim=True).values
        step = ((x.max(-1, keepdim=True).values - low) / 15).to(torch.bfloat16).double()
        low = low.to(torch.bfloat16).double()
        out[n] = low + step * torch.round((x - low) / step.clamp(min=1e-300)).clamp(0, 15)
    return out


def _exact_attend(s, case):
    dim, page, group = case["head_dim"], case["page"], case["group"]
    d = torch.arange(dim, device=DEV)
    t = torch.arange(page, device=DEV)
    # where element d of token t lies within a page of one head: byte and half
    k_byte = t[:, None] * (dim // 2) + d // 8 * 4 + d % 2 * 2 + d % 8 // 4
    k_half = (d % 8 // 2 % 2).expand(page, dim)
    v_byte = t[:, None] // 4 * (2 * dim) + d // 4 * 8 + t[:, None] % 4 * 2 + d % 4 // 2
    v_half = (d % 2).expand(page, dim)

    def rows(held, meta, byte, half, pages, h, length):
        flat = held[pages, h].reshape(pages.numel(), -1)[:, byte].to(torch.int64)
        c = (flat >> (4 * half)) % 16
        m = meta[pages, h].double()
        return (m[..., 1:] + m[..., :1] * c).reshape(-1, dim)[:length]

    lens, new = _sequences(case)
    o = torch.empty(sum(new), case["kv_heads"] * group, dim, dtype=torch.float64, device=DEV)
    lse = torch.empty(o.shape[:2], dtype=torch.float64, device=DEV)
    first = 0
    for b, (length, n) in enumerate(zip(lens, new)):
        pages = s["table"][b, :-(-length // page)].long()
        hidden = torch.arange(length, device=DEV) > torch.arange(length - n, length, device=DEV)[:, None]
        for h in range(case["kv_heads"]):
            k = rows(s["k"], s["k_meta"], k_byte, k_half, pages, h, length)
            v = rows(s["v"], s["v_meta"], v_byte, v_half, pages, h, length)
            at = (slice(first, first + n), slice(h * group, (h + 1) * group))
            scores = torch.matmul(s["q"][at].double(), k.t()) / math.sqrt(dim)
            scores = scores.masked_fill(hidden[:, None], -math.inf)
            lse[at] = torch.logsumexp(scores, -1)
            o[at] = torch.matmul(torch.softmax(scores, -1), v)
        first += n
    return dict(o=o, lse=lse)
