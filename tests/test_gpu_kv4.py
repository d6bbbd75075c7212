"""GPU tests of the 4-bit key/value cache (ops.KV4Cache): jules_hip_kv4_append bit
for bit against the stored form's definition, jules_hip_kv4_read, and
jules_hip_kv4_attention against softmax in 64 bits: one token and many, grouped
heads, lengths of zero and around every tile and page, splits, pages in any
order, what lies behind a sequence's end, rows that hold NaN, bad pages, views,
streams, captured graphs, offsets past 32 bits."""
import numpy as np
import pytest
import torch

from jules_amd import ops
from tests.decoder64 import BF16, Pool, attention64, bf16, f64, quantise, unpack_k, unpack_v
from tests.helpers import case

pytestmark = pytest.mark.gpu

f32, b16, i32 = torch.float32, torch.bfloat16, torch.int32


def _int(dev, a):
    return torch.tensor(np.asarray(a), dtype=i32, device=dev)


def _table(rng, lens, page, pages, width=None):
    """Each sequence's pages in random places, -1 behind them."""
    need = [-(-n // page) for n in lens]
    order = rng.permutation(pages)
    t = np.full((len(lens), max(1, max(need)) if width is None else width), -1)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return t


def _state(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.k_meta, cache.v_meta)]


def _fill(cache, seed=0):
    """Anything in every byte, as an allocation may hold."""
    g = torch.Generator(cache.k.device).manual_seed(seed)
    for t in (cache.k, cache.v, cache.k_meta.view(torch.uint8), cache.v_meta.view(torch.uint8)):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=t.device, dtype=torch.uint8))


# ---- rows in and out -----------------------------------------------------------------


@pytest.mark.parametrize("D,page,heads,t", [(64, 16, 1, f32), (64, 64, 3, b16), (128, 32, 2, f32), (128, 256, 1, b16),
                                            (128, 16, 5, b16), (64, 128, 8, f32)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_and_read(dev, D, page, heads, t, ragged):
    rng = np.random.default_rng(D + page + heads)
    new = [3] * 4 if not ragged else [1, 0, 37, 6, 300, 2]
    before = [0, 5, 15, 16, 61, 200][:len(new)]
    lens = [a + b for a, b in zip(before, new)]
    case(f"kv4 append D={D} page={page} heads={heads} {t} {new}")
    pages = sum(-(-n // page) for n in lens) + 2
    table = _table(rng, lens, page, pages)
    cache = ops.KV4Cache.empty(pages, heads, D, page, dev)
    _fill(cache)
    was = _state(cache)
    tokens = sum(new) + (5 if ragged else 0)  # rows 2 .. are the sequences', 3 behind them
    first = 2 if ragged else 0
    x = torch.from_numpy(rng.standard_normal((2, tokens, heads, D)).astype(np.float32) * 3).to(t)
    x[:, first, 0, 0] = 40.0
    k, v = x.to(dev)
    cu = _int(dev, first + np.concatenate([[0], np.cumsum(new)])) if ragged else None
    tab, ln = _int(dev, table), _int(dev, lens)
    ops.kv4_append(cache, k, v, tab, ln, cu_q=cu, max_q=max(new) if ragged else None)
    torch.cuda.synchronize()
    # every byte: the rows' and, as they were, all others
    want = [unpack_k(was[0]), unpack_v(was[1]), was[2].cpu(), was[3].cpu()]
    values = np.zeros((2, tokens, heads, D), np.float32)
    row = first
    for b, n in enumerate(new):
        for i in range(n):
            at = lens[b] - n + i
            p, off = table[b][at // page], at % page
            for j in range(2):
                c, s, m = quantise(x[j, row].float().numpy())
                want[j][p, :, off] = c
                want[2 + j][p, :, off] = torch.from_numpy(np.stack([s, m], -1)).to(b16)
                values[j, row] = m[:, None] + s[:, None] * c
            row += 1
    assert np.array_equal(unpack_k(cache.k), want[0]) and np.array_equal(unpack_v(cache.v), want[1])
    for got, w in ((cache.k_meta, want[2]), (cache.v_meta, want[3])):
        assert torch.equal(got.cpu().view(torch.int16), w.view(torch.int16))
    for ot in (f32, b16):
        kr = torch.full((tokens, heads, D), 7.0, dtype=ot, device=dev)
        vr = kr.clone()
        ops.kv4_read(cache, tab, ln, tokens, cu_q=cu, max_q=max(new), dtype=ot, k=kr, v=vr)
        own = slice(first, first + sum(new))
        for got, w in ((kr, values[0]), (vr, values[1])):
            assert torch.equal(got[own].cpu(), torch.from_numpy(w[own]).to(ot))
            assert (got[:first] == 7.0).all() and (got[first + sum(new):] == 7.0).all()
    # and the values are the rows to half a step, and what s and m were rounded by
    own = slice(first, first + sum(new))
    for j in range(2):
        xs = x[j, own].double().numpy()
        size = xs.max(-1, keepdims=True) - xs.min(-1, keepdims=True)
        bound = size / 30 * (1 + BF16) + BF16 * (size + np.abs(xs.min(-1, keepdims=True))) + 1e-5
        assert (np.abs(values[j, own] - xs) <= bound).all()


def test_append_special_rows(dev):
    """Constant rows, NaN, infinities, the types' ends, tiny ranges."""
    D, page = 128, 16
    rows = np.random.default_rng(1).standard_normal((12, 1, D)).astype(np.float32)
    rows[0] = 0.0
    rows[1] = 1.7
    rows[2, 0, 5] = np.nan
    rows[3, 0, 127] = np.inf
    rows[4, 0, 0] = -np.inf
    rows[5] = np.finfo(np.float32).min
    rows[6, 0, :64], rows[6, 0, 64:] = 3e38, -3e38  # the range passes fp32
    rows[7] *= 1e-38
    rows[8] = 1e30 * rows[8]
    rows[9] = 1000.0 + 1e-3 * rows[9]
    rows[10, 0, 3] = 1e4
    x = torch.from_numpy(rows).to(dev)
    cache = ops.KV4Cache.empty(1, 1, D, page, dev)
    tab, ln = _int(dev, [[0]]), _int(dev, [12])
    ops.kv4_append(cache, x, x, tab, ln)
    c, s, m = quantise(rows[:, 0])
    c[7] = unpack_k(cache.k)[0, 0, 7]  # below the smallest normal number: see the values
    assert np.array_equal(unpack_k(cache.k)[0, 0, :12], c)
    assert np.array_equal(unpack_k(cache.k)[:, :, :12], unpack_v(cache.v)[:, :, :12])
    k, v = ops.kv4_read(cache, tab, ln, 12, dtype=f32)
    assert torch.equal(k.view(i32), v.view(i32))
    for i in (2, 3, 4, 5, 6):
        assert torch.isnan(k[i]).all()
    for i in (0, 1, 8, 9, 10, 11):
        assert np.array_equal(k[i, 0].cpu().numpy(), (m[i].astype(np.float64) + s[i].astype(np.float64) * c[i]).astype(np.float32))
    assert not k[0].any()
    assert (np.abs(f64(k[7, 0]) - rows[7, 0]) <= 1e-38).all()


def test_append_outside(dev):
    """Rows before position 0, on no page, past the table; cu_q that says nonsense."""
    D, page = 64, 16
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 2, D, generator=g).to(dev)
    cache = ops.KV4Cache.empty(4, 2, D, page, dev)
    _fill(cache)

    def rows_changed(table, lens, cu, n=40):
        was = _state(cache)
        ops.kv4_append(cache, x[:n], x[:n], _int(dev, table), _int(dev, lens), cu_q=None if cu is None else _int(dev, cu),
                       max_q=n if cu is not None else None)
        torch.cuda.synchronize()
        moved = (cache.k_meta.view(torch.int16) != was[2].view(torch.int16)).any(-1).any(1)
        return int(moved.sum())

    assert rows_changed([[0, 1]], [10], None) == 10        # 30 of 40 are before position 0
    assert rows_changed([[2, -1]], [40], None) == 16       # page 2's; the second page is none, 8 rows past it
    assert rows_changed([[7, 3]], [32], [0, 32]) == 16     # 7 is not a page of the pool
    assert rows_changed([[0, 1]], [-5], None) == 0
    assert rows_changed([[0, 1]], [2**31 - 1], None) == 0
    was = _state(cache)
    ops.kv4_append(cache, x, x, _int(dev, [[0, 1]]), _int(dev, [20]), cu_q=_int(dev, [0, 20]), max_q=0)
    ops.kv4_append(cache, -x, -x, _int(dev, [[2, 3]]), _int(dev, [32]), cu_q=_int(dev, [0, 32]), max_q=2**31 - 1)
    torch.cuda.synchronize()
    assert int((cache.k != was[0]).flatten(2).any(-1).any(-1).sum()) == 4  # a hint costs time only
    assert rows_changed([[0], [1]], [8, 8], [30, 20, 50]) == 8  # none, then rows 20 .. 39 of which 8 fit
    assert rows_changed([[0, 1], [2, 3]], [20, 20], [-7, 5, 5]) == 5
    k, v = ops.kv4_read(cache, _int(dev, [[0, 9]]), _int(dev, [30]), 40)
    assert not k[:10].any() and torch.isfinite(k[10:26]).all() and torch.isnan(k[26:]).all() and torch.isnan(v[26:]).all()


def test_append_views(dev):
    """Rows of a fused projection, at any 2-byte address."""
    D, page = 128, 32
    qkv = torch.randn(50, 9, D + 1, device=dev).to(b16)
    k, v = qkv[:, 2:5, 1:], qkv[:, 6:9, :D]
    tab, ln = _int(dev, [[1, 0]]), _int(dev, [50])
    one, two = (ops.KV4Cache.empty(2, 3, D, page, dev) for _ in "12")
    for c in (one, two):
        for t in (c.k, c.v, c.k_meta, c.v_meta):
            t.zero_()
    ops.kv4_append(one, k, v, tab, ln)
    ops.kv4_append(two, k.contiguous(), v.contiguous(), tab, ln)
    assert all(torch.equal(a, b) for a, b in zip(_state(one), _state(two)))


# ---- attention ------------------------------------------------------------------------


def _problem(dev, D, page, heads, group, lens, new, seed=0, pages=None, cu=True, scale_q=1.0, width=None):
    rng = np.random.default_rng(seed)
    pages = pages or sum(-(-n // page) for n in lens) + 2
    K, V = Pool(pages, heads, page, D, rng), Pool(pages, heads, page, D, rng)
    k, _, km = K.packed(dev)
    _, v, vm = V.packed(dev)
    table = _table(rng, lens, page, pages, width)
    q = bf16(scale_q * rng.standard_normal((sum(new), heads * group, D)))
    ends = np.concatenate([[0], np.cumsum(new)])
    return dict(K=K, V=V, cache=ops.KV4Cache(k, v, km, vm), table=table, lens=lens, new=new, q=q, ends=ends, D=D, page=page,
                group=group, args=dict(table=_int(dev, table), lens=_int(dev, lens), cu_q=_int(dev, ends) if cu else None),
                qd=torch.from_numpy(q).to(b16).to(dev))


def _want(p, b, scale):
    """Sequence b of problem p in 64 bits."""
    L, n, page = p["lens"][b], p["new"][b], p["page"]
    at = np.arange(max(L, 0))
    rows = [p["table"][b][at // page], at % page]
    take = lambda a: np.moveaxis(a[rows[0], :, rows[1]], 0, 1)  # noqa: E731  [heads, L, ...]
    K, V = p["K"], p["V"]
    return attention64(p["q"][p["ends"][b]:p["ends"][b + 1]].astype(np.float64), take(K.c), take(K.s), take(K.m), take(V.c),
                       take(V.s), take(V.m), p["group"], scale, L - n)


def _compare(p, o, lse, scale):
    o, lse = f64(o), f64(lse)
    for b in range(len(p["lens"])):
        own = slice(p["ends"][b], p["ends"][b + 1])
        w, wl, bo, bl = _want(p, b, scale)
        nan = np.isnan(w).any(-1)
        assert np.array_equal(np.isnan(o[own]).all(-1), nan), b
        assert np.array_equal(np.isnan(lse[own]), nan), b
        off = np.abs(o[own] - w) - 1.01 * bo
        assert (off[~nan] <= 0).all(), (b, off[~nan].max())
        none = np.isneginf(wl)
        assert np.array_equal(np.isneginf(lse[own]), none)
        assert (np.abs(lse[own] - wl) <= 1.01 * bl)[~nan & ~none].all(), b


def _run(p, scale=None, **kw):
    scale = ops.default_scale(p["D"]) if scale is None else scale
    o, lse = ops.kv4_attention(p["qd"], p["cache"], **p["args"], scale=scale, return_lse=True, **kw)
    torch.cuda.synchronize()
    _compare(p, o, lse, scale)
    return o, lse


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,heads,group", [(16, 2, 4), (64, 1, 1), (256, 3, 8), (32, 2, 16), (128, 1, 17)])
def test_one_token(dev, D, page, heads, group):
    """Decoding: lengths around every tile, page and split."""
    lens = [1, 2, 3, 4, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 512, 513, 777]
    case(f"kv4 attention one token D={D} page={page} heads={heads} group={group}")
    p = _problem(dev, D, page, heads, group, lens, [1] * len(lens), seed=D + group, cu=False)
    _run(p, max_len=max(lens))
    _run(p, max_len=1)  # a hint that is too small costs time only


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads,group,new", [
    (2, 4, [2, 3, 1, 4, 0, 5]),            # drafts: up to 20 rows
    (1, 5, [7, 1, 6, 0, 3]),               # 35 rows
    (2, 8, [8, 2, 5]),                     # 64 rows
    (1, 3, [23, 1, 40, 0, 64]),            # more than 64 rows: waves of their own
    (2, 1, [200, 130, 1]), (1, 16, [33, 20]), (1, 64, [2, 1])])
def test_many_tokens(dev, D, heads, group, new):
    page = 32
    lens = [n + b for n, b in zip(new, [0, 300, 15, 1, 64, 500])]
    case(f"kv4 attention D={D} heads={heads} group={group} new={new} lens={lens}")
    p = _problem(dev, D, page, heads, group, lens, new, seed=D + sum(new))
    _run(p, max_q=max(new), max_len=max(lens))
    _run(p)                      # no hints
    _run(p, max_q=1, max_len=1)  # hints that are too small
    _run(p, max_q=0, max_len=0)
    _run(p, max_q=2**31 - 1, max_len=2**31 - 1)  # and much too large


@pytest.mark.parametrize("scale_q,scale", [(1.0, 0.01), (8.0, 1.0), (0.02, 1.0), (30.0, 0.5)])
def test_scales(dev, scale_q, scale):
    """Flat and sharp softmaxes: the reference moves often, or once."""
    p = _problem(dev, 128, 64, 2, 4, [400, 64, 33], [1, 9, 33], seed=5, scale_q=scale_q)
    case(f"kv4 attention scale_q={scale_q} scale={scale}")
    _run(p, scale=scale)


@pytest.mark.parametrize("power", [90, 16, -60])
@pytest.mark.parametrize("D,lens,new", [(128, [400, 64, 33], [1, 1, 1]), (64, [5000], [2]), (128, [300, 90], [40, 33])])
def test_scaled_values(dev, D, lens, new, power):
    """Values times a power of two: each sum and rounding scales with them, bit for bit.
    5000 keys leave 2^103 for the largest, and with scores of unit variance no
    probability is below 2^-30."""
    case(f"kv4 attention values times 2^{power} D={D} lens={lens}")
    p = _problem(dev, D, 64, 2, 4, lens, new, seed=15)
    hints = dict(max_q=max(new), max_len=max(lens))
    o, lse = _run(p, **hints)
    p["V"].m[:], p["V"].s[:] = p["V"].m * 2.0**power, p["V"].s * 2.0**power
    _, v, vm = p["V"].packed(dev)
    p["cache"] = ops.KV4Cache(p["cache"].k, v, p["cache"].k_meta, vm)
    o2, lse2 = _run(p, **hints)
    assert torch.equal(o2.float(), o.float() * 2.0**power) and torch.equal(lse2, lse)


def test_growing_scores(dev):
    """Keys whose scores rise from first to last: the reference moves at every step;
    and scores far below zero."""
    for sign in (1.0, -1.0):
        p = _problem(dev, 64, 16, 1, 4, [500], [3], seed=6)
        p["q"][:] = bf16(np.abs(p["q"]))
        p["K"].m[:] = 0.0
        for at in range(500):
            pg, off = p["table"][0][at // 16], at % 16
            p["K"].m[pg, 0, off] = bf16([sign * at / 10.0])[0]
        k, _, km = p["K"].packed(dev)
        p["cache"] = ops.KV4Cache(k, p["cache"].v, km, p["cache"].v_meta)
        p["qd"] = torch.from_numpy(p["q"]).to(b16).to(dev)
        _run(p, scale=0.25, max_len=500)
        _run(p, scale=0.25, max_len=1)


def test_empty_sequences(dev):
    """A token that sees no key: 0 and -infinity."""
    p = _problem(dev, 128, 16, 2, 3, [0, 5, 0, 3, 40], [1, 9, 0, 60, 30], seed=7)
    o, lse = _run(p)
    assert not o[0].any() and torch.isneginf(lse[0]).all()      # length 0
    assert not o[1:5].any() and o[6:10].any(-1).all()           # 4 of 9 before position 0
    # negative lengths are empty
    p["args"]["lens"] = _int(dev, [-3, 0, 0, 0, 0])
    o, lse = ops.kv4_attention(p["qd"], p["cache"], **p["args"], return_lse=True)
    assert not o.any() and torch.isneginf(lse).all()


def test_rows_outside_are_left(dev):
    p = _problem(dev, 64, 32, 1, 4, [70, 33], [5, 2], seed=8)
    q = torch.cat([p["qd"][:3], p["qd"], p["qd"][:4]])
    args = dict(p["args"], cu_q=p["args"]["cu_q"] + 3)
    for max_len in (70, 5000):  # whole and split
        out = torch.full(q.shape, 7.0, dtype=b16, device=dev)
        lse = torch.full(q.shape[:2], 7.0, device=dev)
        ops.kv4_attention(q, p["cache"], **args, out=out, lse=lse, max_len=max_len)
        _compare(p, out[3:10], lse[3:10], ops.default_scale(64))
        for t in (out, lse):
            assert (t[:3] == 7.0).all() and (t[10:] == 7.0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_behind_the_end(dev, new):
    """What pages hold behind a sequence's end, NaN included, does not count."""
    lens = [1 + new, 37 + new, 64 + new, 17 + new]
    p = _problem(dev, 128, 64, 2, 4, lens, [new] * 4, seed=9)
    want = _run(p)
    nan = torch.tensor(float("nan"), dtype=b16, device=dev)
    for b, n in enumerate(lens):
        pg, off = p["table"][b][n // 64] if n % 64 else -1, n % 64
        if pg >= 0:
            for t in (p["cache"].k_meta, p["cache"].v_meta):
                t[pg, :, off:] = nan
                t[pg, :, off::2] = float("inf")
            p["cache"].k[pg, :, off:] = 255
    got = ops.kv4_attention(p["qd"], p["cache"], **p["args"], return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("which", ["K", "V"])
@pytest.mark.parametrize("new", [6, 50])
def test_nan_rows_reach_those_that_see_them(dev, which, new):
    """A row held as NaN makes NaN of the tokens at and after it, of its head."""
    p = _problem(dev, 64, 16, 2, 2, [120, 90], [new, new], seed=10)
    pool, at = p[which], 120 - new + 3  # the fourth new token of sequence 0
    pg, off = p["table"][0][at // 16], at % 16
    pool.s[pg, 1, off] = pool.m[pg, 1, off] = np.nan
    meta = p["cache"].k_meta if which == "K" else p["cache"].v_meta
    meta[pg, 1, off] = float("nan")
    o, lse = ops.kv4_attention(p["qd"], p["cache"], **p["args"], return_lse=True)
    ref = attention_rows = p["ends"][0] + 3
    assert torch.isnan(o[ref:new, 2:]).all() and not torch.isnan(o[:ref]).any()
    assert not torch.isnan(o[attention_rows:new, :2]).any() and not torch.isnan(o[new:]).any()


def test_bad_pages(dev):
    """Pages outside the pool and positions past the table: NaN for the tokens that
    see them, nothing for the others, and no read outside."""
    p = _problem(dev, 128, 16, 1, 4, [100, 100, 40], [60, 1, 1], seed=11, width=7)
    base, _ = _run(p)
    for bad in (-1, 10**6, -2**31, 2**31 - 1, p["cache"].pages):
        table = p["args"]["table"].clone()
        table[0, 4] = bad  # positions 64 .. 79: new tokens 24 .. see them
        o, lse = ops.kv4_attention(p["qd"], p["cache"], table, p["args"]["lens"], p["args"]["cu_q"], return_lse=True)
        assert torch.isnan(o[24:60]).all() and torch.isnan(lse[24:60]).all()
        assert torch.equal(o[:24], base[:24]) and torch.equal(o[60:], base[60:])
    for long in (113, 5000, 2**31 - 1):  # the table has room for 112
        lens = p["args"]["lens"].clone()
        lens[1] = long
        for max_len in (100, 2**31 - 1):
            o, lse = ops.kv4_attention(p["qd"], p["cache"], p["args"]["table"], lens, p["args"]["cu_q"], return_lse=True,
                                       max_len=max_len)
            assert torch.isnan(o[60]).all() and torch.isnan(lse[60]).all()
            assert torch.isfinite(o[61]).all() and torch.isfinite(o[:60]).all()


def test_views_and_shared_pages(dev):
    """Queries of a fused projection; two sequences with the same beginning."""
    p = _problem(dev, 128, 16, 2, 4, [50, 50], [1, 1], seed=12)
    want, _ = _run(p)
    wide = torch.zeros(2, 14, 136, dtype=b16, device=dev)
    wide[:, 3:11, 8:] = p["qd"]
    view = wide[:, 3:11, 8:]
    assert torch.equal(ops.kv4_attention(view, p["cache"], **p["args"]), want)
    table = p["args"]["table"].clone()
    table[1] = table[0]
    q = p["qd"].clone()
    q[1] = q[0]
    o = ops.kv4_attention(q, p["cache"], table, p["args"]["lens"])
    assert torch.equal(o[0], want[0]) and torch.equal(o[1], o[0])


def test_deterministic_and_overlapping(dev):
    """The same bits every time, also with another call on another stream."""
    p = _problem(dev, 128, 64, 2, 8, [3000, 777, 2500], [1, 1, 1], seed=13, cu=False)
    want = _run(p, max_len=3000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = ops.kv4_attention(p["qd"], p["cache"], **p["args"], max_len=3000, return_lse=True)
        with torch.cuda.stream(side):
            other = ops.kv4_attention(p["qd"], p["cache"], **p["args"], max_len=3000, return_lse=True)
        torch.cuda.synchronize()
        for r in (got, other):
            assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])


def test_graph(dev):
    """A decoding step captured once, replayed as the sequences grow; two graphs with
    a workspace each."""
    D, page, heads, group = 128, 16, 2, 4
    p = _problem(dev, D, page, heads, group, [300, 41], [1, 1], seed=14, cu=False, width=20)
    table = torch.arange(40, dtype=i32, device=dev).view(2, 20)
    cache = ops.KV4Cache.empty(40, heads, D, page, dev)
    _fill(cache)
    lens = _int(dev, [0, 0])
    twin = ops.KV4Cache.empty(40, heads, D, page, dev)
    kv = torch.randn(2, 300, heads, D, device=dev)
    start = _int(dev, [280, 20])
    for c in (cache, twin):
        ops.kv4_append(c, kv[0], kv[1], table, start, cu_q=_int(dev, [0, 280, 300]))
    lens.copy_(start)
    k, v, q = kv[0, :2].clone(), kv[1, :2].clone(), p["qd"]
    graphs = []
    for _ in range(2):
        out, g = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.kv4_append(cache, k, v, table, lens)
            ops.kv4_attention(q, cache, table, lens, out=out, max_len=320)
        graphs.append((g, out))
    for i in range(6):
        lens += 1
        k.copy_(torch.randn_like(k))
        v.copy_(torch.randn_like(v))
        q.copy_(torch.randn_like(q.float()))
        ops.kv4_append(twin, k, v, table, lens)
        want = ops.kv4_attention(q, twin, table, lens, max_len=320)
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_graph_with_splits(dev):
    """Keys enough for several ranges: each captured graph has its own workspace,
    and eager calls go on beside them."""
    p = _problem(dev, 128, 64, 2, 4, [5000, 4097], [1, 1], seed=15, cu=False)
    q, args = p["qd"], dict(p["args"], max_len=5000)
    assert ops.lib().jules_hip_kv4_attention_workspace_size(2, 2, 8, 2, 128, 1, 5000) > 0
    graphs = []
    for _ in range(2):
        out, lse, g = torch.empty_like(q), torch.empty(2, 8, device=dev), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.kv4_attention(q, p["cache"], out=out, lse=lse, **args)
        graphs.append((g, out, lse))
    for i in range(5):
        q.copy_(torch.randn_like(q.float()))
        p["args"]["lens"].copy_(_int(dev, [5000 - 600 * i, 4097 - 1000 * i]))
        want = ops.kv4_attention(q, p["cache"], return_lse=True, **args)
        torch.cuda.synchronize()
        for g, out, lse in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out, lse in graphs:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_offsets_past_32_bits(dev):
    """Pages whose bytes, and whose rows times their size, lie past 2^32."""
    D, page, heads, pages = 128, 256, 8, 33000
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 10 GB of device memory")
    case("kv4 pool of 4.3 GB of keys")
    cache = ops.KV4Cache.empty(pages, heads, D, page, dev)
    small = ops.KV4Cache.empty(2, heads, D, page, dev)
    kv = torch.randn(2, 300, heads, D, device=dev)
    q = torch.randn(1, 16, D, device=dev).to(b16)
    ln = _int(dev, [300])
    got = []
    for c, last in ((cache, pages - 1), (small, 1)):
        tab = _int(dev, [[last, last - 1]])
        ops.kv4_append(c, kv[0], kv[1], tab, ln)
        got.append((*ops.kv4_read(c, tab, ln, 300), ops.kv4_attention(q, c, tab, ln)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_hints_that_disagree(dev):
    """A prompt's rows with the hints of one token over a long text: more splits
    would not fit the workspace than are taken."""
    p = _problem(dev, 64, 32, 2, 4, [1500], [1000], seed=16)
    case("kv4 attention of 1000 tokens, max_q=1 max_len=131072")
    assert 0 < ops.lib().jules_hip_kv4_attention_workspace_size(1, 1000, 8, 2, 64, 1, 131072) <= 256 << 20
    _run(p, max_q=1, max_len=131072)


# ---- together ----------------------------------------------------------------------------


def test_decoding_steps(dev):
    """A decoder layer's steps as a user runs them: norm to int8, the int8 product,
    positions, cache, attention, the W8A16 product; a prompt first, then tokens one by
    one.  The attention of each step equals that of a whole pass over what the cache
    holds, in 64 bits."""
    hidden, heads, hq, D, page, B = 256, 2, 4, 64, 16, 2
    g = torch.Generator().manual_seed(20)
    proj = torch.randint(-127, 128, (hidden, (hq + 2 * heads) * D), generator=g, dtype=torch.int8).to(dev)
    ps = (torch.rand((hq + 2 * heads) * D, generator=g) * 2e-3).to(dev)
    back = torch.randint(-127, 128, (hq * D, hidden), generator=g, dtype=torch.int8).to(dev)
    bs = (torch.rand(hidden, generator=g) * 1e-3).to(dev)
    norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(dev)
    freq, _ = ops.rotary_frequencies(D, device=dev)
    cache = ops.KV4Cache.empty(16, heads, D, page, dev)
    _fill(cache)
    table = torch.arange(16, dtype=i32, device=dev).view(2, 8)
    lens = [0, 0]
    seen = [[], []]

    def step(x, residual, new):
        nonlocal lens
        lens = [a + n for a, n in zip(lens, new)]
        ln, cu = _int(dev, lens), _int(dev, np.concatenate([[0], np.cumsum(new)]))
        q8, s8, residual = ops.add_rmsnorm_int8(x, residual, norm)
        qkv = ops.matmul_w8a8(q8, proj, s8, ps).view(-1, hq + 2 * heads, D)
        pos = torch.cat([torch.arange(a - n, a) for a, n in zip(lens, new)]).to(i32).to(dev)
        qk = ops.rotary(qkv[:, :hq + heads].transpose(0, 1), pos, freq, dtype=f32).transpose(0, 1)
        q = qk[:, :hq].to(b16)
        ops.kv4_append(cache, qk[:, hq:], qkv[:, hq + heads:], table, ln, cu_q=cu, max_q=max(new))
        o = ops.kv4_attention(q, cache, table, ln, cu_q=cu, max_q=max(new))
        at = 0
        for b, n in enumerate(new):
            kc, ks, km = quantise(qk[at:at + n, hq:].cpu().numpy())
            vc, vs, vm = quantise(qkv[at:at + n, hq + heads:].cpu().numpy())
            seen[b].append([np.moveaxis(a, 1, 0) for a in (kc, ks, km, vc, vs, vm)])
            held = [np.concatenate(a, 1) for a in zip(*seen[b])]
            w, _, bo, _ = attention64(f64(q[at:at + n]), *held, hq // heads, ops.default_scale(D), lens[b] - n)
            assert (np.abs(f64(o[at:at + n]) - w) <= 1.01 * bo).all()
            at += n
        rows = o.reshape(o.shape[0], hq * D)
        parts = [ops.w8a16_gemm(rows[i:i + 16].contiguous(), back, bs, act="none") for i in range(0, rows.shape[0], 16)]
        return torch.cat(parts), residual

    new = [37, 20]
    y, r = step(torch.randn(57, hidden, generator=g).to(b16).to(dev), torch.randn(57, hidden, generator=g).to(dev), new)
    y, r = y[[36, 56]].contiguous(), r[[36, 56]].contiguous()
    for _ in range(20):
        y, r = step(y, r, [1, 1])
        assert torch.isfinite(y).all() and torch.isfinite(r).all()
