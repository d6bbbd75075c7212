"""Plain 64-bit versions of a training step's row operators (dropout, layer norm
with its gradients, token log probabilities with theirs), in numpy, with bounds on
how far the kernels' roundings may be from them.  A rounding to a type is off by
at most half a step: 2^-24 of the value in fp32, 2^-8 in bf16."""
import numpy as np
import torch

from tests.decoder64 import BF16, F32, f64

SLACK = 1.01  # for products of roundings


def step(dtype):
    """Of a value rounded to `dtype` from fp32."""
    return BF16 if dtype == torch.bfloat16 else 0.0


# ---- dropout -------------------------------------------------------------------


def philox(counter, key):
    """Philox4x32 with 10 rounds: 4 arrays of uint32 and 2 numbers -> 4 arrays."""
    c = [np.asarray(v, np.uint64) for v in counter]
    low = np.uint64(0xFFFFFFFF)
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    return [v.astype(np.uint32) for v in c]


def kept(M, N, p, rng, offset, rows=None):
    """bool [M, N]: which elements are kept."""
    rows = np.arange(M) if rows is None else np.asarray(rows)
    seed, at = rng[0] % 2**64, (rng[1] + offset) % 2**64
    blocks = -(-N // 8)
    c = np.broadcast_arrays(np.arange(blocks)[None], rows[:, None], at % 2**32, at // 2**32)
    words = np.stack(philox(c, (seed % 2**32, seed // 2**32)), -1)
    bits = np.stack([words & 0xFFFF, words >> 16], -1).reshape(len(rows), 8 * blocks)[:, :N]
    return bits >= threshold(p)


def threshold(p):
    return int(np.rint(float(np.float32(p)) * 65536))


def drop32(x, p, rng, offset):
    """Dropout of x [M, N] as float32, the one rounding of the product included."""
    x = x.float().cpu().numpy()
    if not threshold(p):
        return x
    factor = np.float32(65536 / (65536 - threshold(p)))
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(kept(*x.shape, p, rng, offset), x * factor, np.float32(0.0))


# ---- layer norm ------------------------------------------------------------------


def layernorm64(h, gamma, beta, eps):
    """h float32 [M, N] -> (y, mean, rstd) in 64 bits, and how far the kernel's y may be."""
    h = h.astype(np.float64)
    mean = h.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(np.square(h - mean).mean(-1, keepdims=True) + eps)
    g = 1.0 if gamma is None else f64(gamma)
    n = (h - mean) * rstd * g
    y = n + (0.0 if beta is None else f64(beta))
    # the mean's rounding; the distance's, rstd's and their product's; the sum's
    bound = SLACK * F32 * (np.abs(mean) * rstd * np.abs(g) + 3 * np.abs(n) + np.abs(y))
    return y, mean[:, 0], rstd[:, 0], bound


def layernorm_bwd64(dy, h, mean, rstd, gamma, dh, rows_added):
    """(dr, dgamma, dbeta) in 64 bits from the kernel's inputs, and how far its sums in
    fp32 may be: a thread adds at most 32 elements of a row one after another (N / 1024
    in rows over 16384), then up to 22 parts; a column's sum has `rows_added` rows in
    a chain at most, then the parts."""
    M, N = dy.shape
    dy, h, mean, rstd = f64(dy), f64(h), f64(mean)[:, None], f64(rstd)[:, None]
    g = np.ones(N) if gamma is None else f64(gamma)
    a, n = dy * g, (h - mean) * rstd
    c1, c2 = a.mean(-1, keepdims=True), (a * n).mean(-1, keepdims=True)
    chain = (32 if N <= 16384 else N / 1024 + 8) + 22
    e1 = (chain + 2) * F32 * np.abs(a).mean(-1, keepdims=True)
    e2 = (chain + 5) * F32 * np.abs(a * n).mean(-1, keepdims=True)
    core = rstd * (a - c1 - n * c2)
    dr = core + (0.0 if dh is None else f64(dh))
    bound = SLACK * (rstd * (e1 + np.abs(n) * e2 + F32 * (2 * np.abs(a) + 2 * np.abs(c1) + 5 * np.abs(n * c2)))
                     + F32 * (2 * np.abs(core) + np.abs(dr)))
    chain = rows_added + 150
    return (dr, (dy * n).sum(0), dy.sum(0), bound, SLACK * (chain + 3) * F32 * np.abs(dy * n).sum(0),
            SLACK * chain * F32 * np.abs(dy).sum(0))


# ---- log probabilities -----------------------------------------------------------


def logprobs64(x, tokens, scale):
    """Of rows of numbers and -infinity: dict of lse, entropy, log [M, N] and logp in 64 bits, with
    bounds.  Distances z from the row's maximum carry 4 roundings into the exponents (the
    difference, the product, the factor's two), e^z 2 more, and the distance between two
    maxima the same; 110 joins of 3 roundings and chains of 64 additions at most.  The
    entry point takes scale as fp32."""
    x, scale = f64(x), float(np.float32(scale))
    with np.errstate(divide="ignore", invalid="ignore"):
        z = (x - np.where(np.isfinite(x), x, -np.inf).max(-1, keepdims=True)) * scale
        none = ~np.isfinite(x).any(-1)
        z[none] = -np.inf
        e = np.exp(z)
        s = e.sum(-1, keepdims=True)
        log = np.where(none[:, None], -np.inf, z - np.log(s))
        p = np.where(none[:, None], 0.0, e / np.where(s > 0, s, 1.0))
        far = np.where(p > 0, np.abs(np.where(p > 0, z, 0.0)), 0.0)
        mean, square = (p * far).sum(-1), (p * far * far).sum(-1)
        ln_s = np.where(none, 0.0, np.log(s[:, 0]))
        lse = np.where(none, -np.inf, np.where(np.isfinite(x), x, -np.inf).max(-1) * scale + ln_s)
    chain = 3 * 110 + 70
    e_s = F32 * (8 * mean + chain + 2) + 4 * F32 * np.abs(ln_s)
    entropy = np.where(none, 0.0, ln_s + mean)
    out = dict(lse=lse, entropy=entropy, log=log, none=none)
    out["e_lse"] = SLACK * (e_s + 2 * F32 * np.abs(np.where(none, 0.0, lse)))
    out["e_entropy"] = SLACK * (e_s * (1 + mean) + F32 * (8 * square + (chain + 6) * mean + 2 * np.abs(ln_s)))
    out["e_log"] = SLACK * (e_s[:, None] + F32 * (3 * np.abs(np.where(np.isfinite(z), z, 0.0)) + 2 * np.abs(ln_s[:, None])))
    if tokens is not None:
        at = np.arange(len(x)), np.clip(tokens.cpu().numpy().reshape(-1), 0, x.shape[1] - 1)
        out["logp"], out["e_logp"] = log[at], out["e_log"][at]
    return out


def top64(x, top):
    """Indices of the largest, falling, equal ones by rising index."""
    return np.argsort(-f64(x), -1, kind="stable")[:, :top]


def logprobs_bwd64(x, tokens, lse, entropy, dlogp, dentropy, scale):
    """The gradient in 64 bits from the kernel's inputs, lse, entropy and scale as fp32 among
    them, and its bound."""
    scale = float(np.float32(scale))
    x, lse, g = f64(x), f64(lse)[:, None], f64(dlogp)[:, None]
    with np.errstate(invalid="ignore"):
        log = np.where(np.isfinite(lse), x * scale - lse, -np.inf)
    p = np.exp(log)
    far = np.where(p > 0, np.abs(np.where(p > 0, log, 0.0)), 0.0)
    t = tokens.cpu().numpy().reshape(-1)
    g = np.where((t < 0)[:, None] | ~np.isfinite(lse), 0.0, g)
    gh = np.zeros_like(g) if dentropy is None else np.where(np.isfinite(lse), f64(dentropy)[:, None], 0.0)
    H = np.zeros_like(g) if dentropy is None else f64(entropy)[:, None]
    y = -p * (g + gh * (np.where(p > 0, log, 0.0) + H))
    bound = np.abs(y) * F32 * (3 * far + 8) + p * F32 * (5 * np.abs(gh) * (far + np.abs(H)) + 3 * np.abs(g))
    rows = np.nonzero(t >= 0)[0]
    y[rows, t[rows]] += g[rows, 0]
    bound[rows, t[rows]] += 2 * F32 * np.abs(g[rows, 0])
    return scale * y, SLACK * scale * (bound + 2 * F32 * np.abs(y))
