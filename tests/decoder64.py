"""Plain 64-bit versions of the operators between a quantised decoder's products
(norm, rotary positions, 4-bit key/value cache, attention over it), in numpy,
with bounds on how far the kernels' roundings may be from them.  A rounding to a
type is off by at most half a step: 2^-24 of the value in fp32, 2^-8 in bf16."""
import numpy as np
import torch

F32, BF16 = 2.0**-24, 2.0**-8


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def bf16(x):
    """x rounded to bf16 (ties to even), as float32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()


# ---- norm --------------------------------------------------------------------


def norm64(x, r, w, eps):
    """(h, y, s, y / s): h = x + r, y its norm, s = max|y| / 127."""
    h = f64(x) + (0.0 if r is None else f64(r))
    w = f64(w)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w
    s = np.abs(y).max(-1) / 127.0
    t = np.divide(y, s[..., None], out=np.zeros_like(y), where=s[..., None] > 0)
    return h, y, s, t


# ---- rotary --------------------------------------------------------------------


def rotary64(x, pos, freq, axis, pairing, inverse):
    """x [B,H,S,D] float64, pos [axes,B,S], freq [P], axis [P] or None."""
    P = len(freq)
    axis = np.zeros(P, int) if axis is None else axis
    # in longdouble: the product of a far position and a frequency keeps its fraction
    a = pos[axis].astype(np.longdouble) * freq[:, None, None].astype(np.longdouble)
    a = np.moveaxis(a, 0, -1)[:, None]
    if inverse:
        a = -a
    c, s = np.cos(a).astype(np.float64), np.sin(a).astype(np.float64)
    out = x.copy()
    i = np.arange(P) if pairing == "half" else 2 * np.arange(P)
    j = i + P if pairing == "half" else i + 1
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., i] * s + x[..., j] * c
    return out


def rotary_bound(x, P, pairing, out_bf16):
    """Per element: cos and sin off by at most 3 * 2^-23 (the angle's fraction of a
    turn rounded to fp32, at most 2 pi 2^-26; sincospi within 2 ulp), two
    products and a sum in fp32, the output's rounding."""
    i = np.arange(P) if pairing == "half" else 2 * np.arange(P)
    j = i + P if pairing == "half" else i + 1
    b = np.zeros_like(x)
    size = np.abs(x[..., i]) + np.abs(x[..., j])
    b[..., i] = b[..., j] = size * (3 * 2.0**-23 + 3 * F32)
    return b


# ---- 4-bit rows --------------------------------------------------------------------


def quantise(x):
    """The stored form of rows of float32: (codes int, s, m as float32 holding
    bf16).  The same fp32 operations as the definition names, so exact."""
    x = np.asarray(x, np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        rng = ((hi - lo) * (np.float32(1.0) / np.float32(15.0))).astype(np.float32)
        s, m = bf16(rng), bf16(lo)
        bad = ~np.isfinite(x).all(-1, keepdims=True) | ~np.isfinite(rng) | ~np.isfinite(m)
        c = np.rint(((x - m) / s).astype(np.float32))
    c = np.where((s > 0) & ~bad, np.clip(np.nan_to_num(c), 0, 15), 0).astype(np.int64)
    s, m = np.where(bad, np.nan, s), np.where(bad, np.nan, m)
    return c, s[..., 0].astype(np.float32), m[..., 0].astype(np.float32)


class Pool:
    """A cache in numpy: codes [pages, heads, page, D], s and m [pages, heads, page]."""

    def __init__(self, pages, heads, page, D, rng):
        self.c = rng.integers(0, 16, (pages, heads, page, D))
        self.s = bf16(rng.uniform(0.1, 0.4, (pages, heads, page)))
        self.m = bf16(-7.5 * self.s + rng.normal(0, 0.3, (pages, heads, page)))

    def packed(self, dev):
        """k, v, meta tensors in the library's layout: the pool as keys and as values."""
        c, (pages, heads, page, D) = self.c, self.c.shape
        e = c.reshape(pages, heads, page, D // 8, 8)
        k = np.stack([e[..., 0] | e[..., 2] << 4, e[..., 4] | e[..., 6] << 4, e[..., 1] | e[..., 3] << 4,
                      e[..., 5] | e[..., 7] << 4], -1).reshape(pages, heads, page, D // 2)
        e = c.reshape(pages, heads, page // 4, 4, D // 4, 4)
        v = np.stack([e[..., 0] | e[..., 1] << 4, e[..., 2] | e[..., 3] << 4], -1)  # [.., token, D/4, 2]
        v = v.swapaxes(-2, -3).reshape(pages, heads, page // 4, 2 * D)
        meta = torch.from_numpy(np.stack([self.s, self.m], -1)).to(torch.bfloat16)
        return (torch.from_numpy(k.astype(np.uint8)).to(dev), torch.from_numpy(np.ascontiguousarray(v).astype(np.uint8)).to(dev),
                meta.to(dev))


def unpack_k(k):
    """uint8 [..., D/2] -> codes [..., D]."""
    b = k.cpu().numpy().astype(np.int64)
    b = b.reshape(*b.shape[:-1], -1, 4)
    out = np.empty((*b.shape[:-1], 8), np.int64)
    for byte, (lo, hi) in enumerate([(0, 2), (4, 6), (1, 3), (5, 7)]):
        out[..., lo], out[..., hi] = b[..., byte] & 15, b[..., byte] >> 4
    return out.reshape(*out.shape[:-2], -1)


def unpack_v(v):
    """uint8 [..., page/4, 2D] -> codes [..., page, D]."""
    b = v.cpu().numpy().astype(np.int64)
    lead, quads, D = b.shape[:-2], b.shape[-2], b.shape[-1] // 2
    b = b.reshape(*lead, quads, D // 4, 4, 2).swapaxes(-2, -3)  # [.., quads, token, D/4, 2]
    out = np.stack([b & 15, b >> 4], -1).reshape(*lead, quads * 4, D)
    return out


# ---- attention ---------------------------------------------------------------------


def attention64(q, kc, ks, km, vc, vs, vm, group, scale, first):
    """One sequence: q [n, heads*group, D] float64, codes [heads, L, D], s and m
    [heads, L]; token i sees keys 0 .. first + i.  Returns o, lse and how far the
    kernel's may be from them.

    Scores: keys are exact, products and sums fp32 from -sum(q) up, of numbers
    that add to at most 3 sum|q|: D/8 + 8 roundings of 16 s times that (the
    matrix instruction rounds at most once for 8 products), times the scale.
    Output: each probability times its scale is rounded to bf16 and weighs the
    code's distance from 7.5; a score's error e makes 2 e of the output's size;
    then the output's own rounding."""
    n, hq, D = q.shape
    o, lse = np.zeros((n, hq, D)), np.full((n, hq), -np.inf)
    bo, bl = np.zeros((n, hq, D)), np.zeros((n, hq))
    for h in range(hq):
        j = h // group
        k = km[j][:, None].astype(np.float64) + ks[j][:, None].astype(np.float64) * kc[j]
        v = vm[j][:, None].astype(np.float64) + vs[j][:, None].astype(np.float64) * vc[j]
        far = vs[j][:, None].astype(np.float64) * np.abs(vc[j] - 7.5)
        for i in range(n):
            e = first + i + 1
            if e <= 0:
                continue
            with np.errstate(invalid="ignore"):
                x = scale * (k[:e] @ q[i, h])
            if not np.isfinite(x).all() or not np.isfinite(v[:e]).all():
                o[i, h], lse[i, h] = np.nan, np.nan
                continue
            top = x.max()
            p = np.exp(x - top)
            total = p.sum()
            o[i, h] = p @ v[:e] / total
            lse[i, h] = top + np.log(total)
            err = ((D / 8 + 8) * F32 * scale * 3 * np.abs(q[i, h]).sum()
                   * (16 * ks[j][:e] + np.abs(km[j][:e])).max() + 8 * F32 * np.abs(x).max())
            bo[i, h] = (BF16 * (p @ far[:e]) / total + 2 * (err + e * F32) * (p @ (np.abs(v[:e]) + 25 * far[:e].max()) / total)
                        + (BF16 + 4 * F32) * np.abs(o[i, h]))
            bl[i, h] = err + 4 * F32 * (1 + abs(lse[i, h])) + 64 * F32
    return o, lse, bo, bl
