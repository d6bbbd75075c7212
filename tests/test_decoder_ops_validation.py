"""CPU tests of the argument checks of the norm, rotary and 4-bit cache operators:
the statuses of the C ABI, and the ValueErrors of the torch front end.  Every call
here is refused, or has nothing to do, before a device is touched."""
import ctypes

import pytest
import torch

from jules_amd import _lib, ops

OK, NULL, SHAPE, DTYPE, ALIGN, ACT, WS, HIP, UNSUP, NOTFOUND, ARG = range(11)
P = 0x10000  # a non-null, aligned address that is never dereferenced
F32, BF16, I8, I32 = 0, 1, 2, 3
f32, bf16, i8, i32, u8, f64 = torch.float32, torch.bfloat16, torch.int8, torch.int32, torch.uint8, torch.float64


def _t(shape, dtype=f32):
    return torch.zeros(shape, dtype=dtype)


def _raises(fn, *args, match, exc=ValueError, **kw):
    with pytest.raises(exc, match=match):
        fn(*args, **kw)


# ---- C ABI ---------------------------------------------------------------------


@pytest.mark.parametrize("change,status", [
    (dict(x_dtype=2), DTYPE), (dict(r_dtype=3), DTYPE), (dict(out_dtype=3), DTYPE), (dict(out_dtype=-1), DTYPE),
    (dict(M=-1), SHAPE), (dict(N=-1), SHAPE), (dict(M=1 << 21, N=1 << 21), SHAPE),
    (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(eps=float("inf")), ARG),
    (dict(r=None), ARG), (dict(out_dtype=F32), ARG),
    (dict(x=None), NULL), (dict(w=None), NULL), (dict(out=None), NULL), (dict(scale=None), NULL),
    (dict(x=P + 2), ALIGN), (dict(r=P + 1), ALIGN), (dict(w=P + 2), ALIGN), (dict(r_out=P + 1), ALIGN), (dict(scale=P + 2), ALIGN),
    (dict(M=0, x=None, w=None, out=None, scale=None), OK), (dict(N=0, x=None), OK),
])
def test_add_rmsnorm_statuses(change, status):
    a = dict(x_dtype=F32, r_dtype=BF16, out_dtype=I8, x=P, r=P, w=P, r_out=P, out=P, scale=P, M=4, N=8, eps=1e-5)
    a.update(change)
    assert _lib.lib().jules_hip_add_rmsnorm(*a.values(), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_dtype=2), DTYPE), (dict(out_dtype=7), DTYPE), (dict(pairing=2), ARG), (dict(inverse=-1), ARG),
    (dict(B=-1), SHAPE), (dict(H=65536), SHAPE), (dict(B=1 << 14, S=(1 << 13) + 1), SHAPE), (dict(D=1), SHAPE),
    (dict(D=1026, R=64), SHAPE), (dict(R=63), SHAPE), (dict(R=0), SHAPE), (dict(R=130), SHAPE), (dict(axes=0), SHAPE),
    (dict(axes=17), SHAPE), (dict(x=None), NULL), (dict(xs=None), NULL), (dict(pos=None), NULL), (dict(freq=None), NULL),
    (dict(x=P + 2), ALIGN), (dict(out=P + 1), ALIGN), (dict(freq=P + 4), ALIGN), (dict(axis=P + 2), ALIGN),
    (dict(xs=(-1, 128, 128)), ARG), (dict(xs=(1 << 41, 0, 0)), ARG),
    (dict(os=(5120, 64, 640)), ARG),      # heads overlap
    (dict(os=(0, 128, 640)), ARG),        # batches overlap
    (dict(os=(1000, 128, 640)), ARG),     # a batch within the one before
    (dict(out=P), ARG),                   # in place with another dtype
    (dict(out=P, out_dtype=F32, os=(640, 1280, 128)), ARG),  # in place with other strides
    (dict(B=0, x=None, out=None), OK), (dict(S=0, x=None), OK), (dict(H=0), OK),
])
def test_rotary_statuses(change, status):
    a = dict(x_dtype=F32, out_dtype=BF16, pairing=0, inverse=0, x=P, xs=(5120, 128, 640), out=2 * P, os=(5120, 128, 640),
             pos=P, freq=P, axis=P, axes=2, B=2, H=5, S=8, D=128, R=128)
    a.update(change)
    for k in ("xs", "os"):
        if a[k] is not None:
            a[k] = (ctypes.c_int64 * 3)(*a[k])
    assert _lib.lib().jules_hip_rotary(*a.values(), None) == status


def _cache(**change):
    c = dict(k=P, v=P, k_meta=P, v_meta=P, num_pages=8, page_size=64, heads=4, head_dim=128)
    c.update(change)
    return ctypes.byref(_lib.JhKV4Cache(*c.values()))


_SHARED = [
    (dict(cache=None), NULL), (dict(cache=_cache(k=None)), NULL), (dict(cache=_cache(v_meta=None)), NULL),
    (dict(cache=_cache(num_pages=0)), SHAPE), (dict(cache=_cache(heads=0)), SHAPE), (dict(cache=_cache(heads=65536)), SHAPE),
    (dict(cache=_cache(head_dim=96)), UNSUP), (dict(cache=_cache(page_size=48)), UNSUP), (dict(cache=_cache(page_size=512)), UNSUP),
    (dict(cache=_cache(page_size=8)), UNSUP), (dict(cache=_cache(num_pages=2**31 - 1, heads=65535)), SHAPE),
    (dict(cache=_cache(v=P + 8)), ALIGN), (dict(cache=_cache(k_meta=P + 4)), ALIGN),
    (dict(table=None), NULL), (dict(lens=None), NULL), (dict(table=P + 2), ALIGN), (dict(cu_q=P + 1), ALIGN),
    (dict(batch=-1), SHAPE), (dict(batch=65536), SHAPE), (dict(tokens=-1), SHAPE), (dict(max_q=-1), SHAPE), (dict(max_pages=-1), SHAPE),
    (dict(cu_q=None, tokens=7), SHAPE), (dict(batch=0, table=None, lens=None), OK), (dict(tokens=0, lens=None), OK),
]


@pytest.mark.parametrize("change,status", _SHARED + [
    (dict(dtype=2), DTYPE), (dict(k=None), NULL), (dict(v=P + 1), ALIGN), (dict(dtype=F32, k=P + 2), ALIGN),
    (dict(kt=-1), ARG), (dict(vh=1 << 41), ARG)])
def test_kv4_append_statuses(change, status):
    a = dict(dtype=BF16, cache=_cache(), k=P, kt=512, kh=128, v=P, vt=512, vh=128, table=P, max_pages=4, lens=P, cu_q=P, batch=2,
             tokens=6, max_q=3)
    a.update(change)
    assert _lib.lib().jules_hip_kv4_append(*a.values(), None) == status


@pytest.mark.parametrize("change,status", _SHARED + [(dict(dtype=3), DTYPE), (dict(v=None), NULL), (dict(k=P + 8), ALIGN)])
def test_kv4_read_statuses(change, status):
    a = dict(dtype=BF16, cache=_cache(), k=P, v=P, table=P, max_pages=4, lens=P, cu_q=P, batch=2, tokens=6, max_q=3)
    a.update(change)
    assert _lib.lib().jules_hip_kv4_read(*a.values(), None) == status


@pytest.mark.parametrize("change,status", _SHARED + [
    (dict(scale=0.0), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG), (dict(heads_q=6), SHAPE),
    (dict(heads_q=0), SHAPE), (dict(max_len=-1), SHAPE), (dict(tokens=1 << 28), SHAPE), (dict(q=None), NULL),
    (dict(out=None), NULL), (dict(q=P + 8), ALIGN), (dict(qt=1028), ALIGN), (dict(qh=132), ALIGN), (dict(out=P + 2), ALIGN),
    (dict(lse=P + 2), ALIGN), (dict(qt=-8), ARG), (dict(max_len=100000), WS), (dict(max_len=100000, ws=P, ws_bytes=64), WS),
    (dict(ws=P + 8), ALIGN)])
def test_kv4_attention_statuses(change, status):
    a = dict(scale=0.1, cache=_cache(), q=P, qt=1024, qh=128, out=P, lse=P, heads_q=8, table=P, max_pages=4, lens=P, cu_q=P, batch=2,
             tokens=6, max_q=3, max_len=100, ws=None, ws_bytes=0)
    a.update(change)
    assert _lib.lib().jules_hip_kv4_attention(*a.values(), None) == status


def test_kv4_workspace_size():
    f = _lib.lib().jules_hip_kv4_attention_workspace_size
    assert f(1, 1, 32, 8, 128, 1, 64) == 0                # one range of keys
    assert f(1, 1, 32, 8, 128, 1, 100000) > 0
    for bad in ((0, 1, 32, 8, 128, 1, 99999), (65536, 1, 32, 8, 128, 1, 99999), (1, 0, 32, 8, 128, 1, 99999), (1, 1, 30, 8, 128, 1, 99999),
                (1, 1, 32, 8, 96, 1, 99999), (1, 1, 32, 0, 128, 1, 99999), (1, 1 << 28, 32, 8, 128, 1, 99999),
                (1, 1, 32, 8, 128, -1, 99999), (1, 1, 32, 8, 128, 1, -1)):
        assert f(*bad) == 0
    # whatever the sizes, the sums of all splits fit what a row may have
    for batch in (1, 3, 64, 65535):
        for max_q in (0, 1, 7, 16, 1000, 2**31 - 1):
            for max_len in (0, 1, 1000, 10**6, 2**31 - 1):
                n = f(batch, 16, 16, 4, 128, max_q, max_len)
                assert n % (16 * 16 * 130 * 4) == 0 and n // (16 * 16 * 130 * 4) <= 4096


# ---- torch front end --------------------------------------------------------------


def test_add_rmsnorm_checks():
    x, r, w = _t((4, 10), bf16), _t((4, 10)), _t((10,))
    for fn in (ops.add_rmsnorm, ops.add_rmsnorm_int8):
        _raises(fn, x, r, w, match="GPU tensor")
        _raises(fn, x.half(), r, w, match="dtype")
        _raises(fn, x, _t((4, 11)), w, match="shape")
        _raises(fn, x, r, _t((11,)), match="elements")
        _raises(fn, x, r, w.double(), match="dtype")
        _raises(fn, x.t(), None, w, match="contiguous")
        _raises(fn, x, r, w, residual_out=_t((4, 10), bf16), match="dtype")
        _raises(fn, x, None, w, residual_out=_t((4, 10)), match="without residual")
        _raises(fn, x, r, w, out=_t((4, 9), i8 if fn is ops.add_rmsnorm_int8 else f32), match="shape")
    _raises(ops.add_rmsnorm, x, r, w, out=_t((4, 10), i8), match="dtype")
    _raises(ops.add_rmsnorm_int8, x, r, w, out=_t((4, 10)), match="dtype")
    _raises(ops.add_rmsnorm_int8, x, r, w, scale=_t((5,)), match="elements")


def test_rotary_checks():
    x, pos, freq, axis = _t((2, 3, 5, 64)), _t((2, 2, 5), i32), _t((32,), f64), _t((32,), i32)
    ok = dict(x=x, positions=pos, inv_freq=freq, pair_axis=axis)
    _raises(ops.rotary, **ok, match="GPU tensor")
    for change, match in [(dict(x=_t((5, 64))), "dimensions"), (dict(x=x.double()), "fp32 or bf16"),
                          (dict(x=x.transpose(2, 3)), "last stride"), (dict(positions=pos.long()), "dtype"),
                          (dict(positions=_t((2, 2, 6), i32)), "elements|shape"), (dict(positions=_t((2, 5, 2), i32)), "shape"),
                          (dict(positions=pos[0, 0]), "positions"), (dict(inv_freq=freq.float()), "dtype"),
                          (dict(inv_freq=_t((33,), f64)), "pairs"), (dict(inv_freq=_t((0,), f64)), "pairs"),
                          (dict(pair_axis=axis.long()), "dtype"), (dict(pair_axis=_t((31,), i32)), "elements"),
                          (dict(pairing="both"), "pairing"), (dict(out=_t((2, 3, 5, 63))), "shape"),
                          (dict(out=_t((2, 3, 5, 64)), dtype=bf16), "dtype"), (dict(dtype=f64), "dtype"),
                          (dict(positions=pos.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous")]:
        _raises(ops.rotary, **{**ok, **change}, match=match)


def test_rotary_frequencies():
    freq, axis = ops.rotary_frequencies(8, device="cpu")
    assert axis is None and freq.dtype == f64 and torch.allclose(freq, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=f64))
    freq, axis = ops.rotary_frequencies(12, (1, 0, 5), base=100.0, device="cpu")
    assert axis.tolist() == [0, 2, 2, 2, 2, 2] and axis.dtype == i32
    for bad in ((7, None), (0, None), (8, (1, 2)), (8, (5, -1))):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(*bad, device="cpu")


def _pool(pages=4, heads=2, D=64, page=32):
    return ops.KV4Cache.empty(pages, heads, D, page, device="cpu")


def test_kv4_cache_checks():
    c = _pool()
    assert (c.pages, c.heads, c.head_dim, c.page_size) == (4, 2, 64, 32)
    good = [c.k, c.v, c.k_meta, c.v_meta]
    for i, t, match in [(0, c.k[0], "dimensions"), (0, c.k.to(i8), "dtype"), (1, c.v[:3], "shape"), (1, c.v.transpose(0, 1), "contiguous"),
                        (2, c.k_meta.float(), "dtype"), (3, c.v_meta[:, :, :16], "contiguous|shape")]:
        bad = list(good)
        bad[i] = t
        _raises(ops.KV4Cache, *bad, match=match)


def test_kv4_checks():
    c, table, lens, cu = _pool(), _t((3, 5), i32), _t((3,), i32), _t((4,), i32)
    k, q = _t((6, 2, 64), bf16), _t((6, 8, 64), bf16)
    _raises(ops.kv4_append, c, k, k, table, lens, match="GPU tensor")
    _raises(ops.kv4_read, c, table, lens, 6, match="GPU tensor")
    _raises(ops.kv4_attention, q, c, table, lens, match="GPU tensor")
    _raises(ops.kv4_append, (c.k,), k, k, table, lens, exc=TypeError, match="KV4Cache")
    _raises(ops.kv4_read, None, table, lens, 6, exc=TypeError, match="KV4Cache")
    _raises(ops.kv4_attention, q, None, table, lens, exc=TypeError, match="KV4Cache")
    for change, match in [(dict(table=table.long()), "dtype"), (dict(table=table[0]), "dimensions"), (dict(table=table.t()), "contiguous"),
                          (dict(lens=_t((2,), i32)), "elements"), (dict(lens=lens.long()), "dtype"),
                          (dict(cu_q=_t((3,), i32)), "elements"), (dict(cu_q=cu.long()), "dtype"), (dict(max_q=3), "unequal")]:
        a = {**dict(table=table, lens=lens), **change}
        _raises(ops.kv4_append, c, k, k, **a, match=match)
        _raises(ops.kv4_read, c, tokens=6, **a, match=match)
        _raises(ops.kv4_attention, q, c, **a, match=match)
    _raises(ops.kv4_append, c, k[:5], k[:5], table, lens, match="unequal")
    _raises(ops.kv4_append, c, k, k.float(), table, lens, match="dtype")
    _raises(ops.kv4_append, c, k, k[:5], table, lens, match="shape")
    _raises(ops.kv4_append, c, k.half(), k.half(), table, lens, match="dtype")
    _raises(ops.kv4_append, c, _t((6, 3, 64)), _t((6, 3, 64)), table, lens, match="shape")
    _raises(ops.kv4_append, c, _t((6, 64, 2)).transpose(1, 2), k, table, lens, match="last stride")
    _raises(ops.kv4_read, c, table, lens, 6, dtype=f64, match="dtype")
    _raises(ops.kv4_read, c, table, lens, 6, k=_t((6, 2, 64)), match="dtype")
    _raises(ops.kv4_read, c, table, lens, 6, v=_t((5, 2, 64), bf16), match="shape")
    _raises(ops.kv4_attention, q.float(), c, table, lens, match="dtype")
    _raises(ops.kv4_attention, q[0], c, table, lens, match="dimensions")
    _raises(ops.kv4_attention, q[:, :7], c, table, lens, match="heads")
    _raises(ops.kv4_attention, _t((6, 8, 128), bf16), c, table, lens, match="shape")
    _raises(ops.kv4_attention, q, c, table, lens, out=q.float(), match="dtype")
    _raises(ops.kv4_attention, q, c, table, lens, lse=_t((6, 7)), match="elements")
    _raises(ops.kv4_attention, q, c, table, lens, workspace=_t((8, 8)).t()[:3], match="contiguous")


def test_kv4_cache_tensors_are_fixed():
    """Assigning another tensor (a larger pool), or the sizes, would leave the calls
    with the old one's address: refused."""
    c = _pool()
    for name, value in dict(k=c.k.clone(), v=c.v.clone(), k_meta=c.k_meta.clone(), v_meta=c.v_meta.clone(), pages=9, heads=1,
                            page_size=16, head_dim=128).items():
        _raises(setattr, c, name, value, exc=AttributeError, match="new KV4Cache")
        assert getattr(c, name) is not value


def test_kv4_cache_takes_attributes_of_its_user():
    class Layer(ops.KV4Cache):
        def __init__(self, *tensors, index):
            self.index = index
            super().__init__(*tensors)

    c = _pool()
    c.owner = "layer 3"
    layer = Layer(c.k, c.v, c.k_meta, c.v_meta, index=3)
    assert c.owner == "layer 3" and layer.index == 3 and layer.pages == 4


@pytest.mark.parametrize("name", ["k", "v", "k_meta", "v_meta"])
def test_kv4_cache_addresses_are_the_tensors(monkeypatch, name):
    """A tensor whose memory has moved is passed where it now lies; one whose size
    is another is refused."""
    c, table, lens = _pool(), _t((3, 5), i32), _t((3,), i32)
    k, q = _t((6, 2, 64), bf16), _t((6, 8, 64), bf16)
    passed = []

    def call(t, fn, *args):
        passed.extend(a._obj for a in args if isinstance(getattr(a, "_obj", None), _lib.JhKV4Cache))

    monkeypatch.setattr(ops, "_one_device", lambda *a: None)
    monkeypatch.setattr(ops, "_call", call)
    calls = [lambda: ops.kv4_append(c, k, k, table, lens), lambda: ops.kv4_read(c, table, lens, 6),
             lambda: ops.kv4_attention(q, c, table, lens)]
    t = getattr(c, name)
    held = [t.data]  # the old memory stays, so that the new is elsewhere
    for fn in calls:
        t.data = t.data.clone()
        held.append(t.data)
        fn()
        assert getattr(passed.pop(), name) == t.data_ptr() and not passed
    t.data = t.data[:3].clone()
    for fn in calls:
        _raises(fn, match="size")
    assert not passed


def test_kv4_workspace_of_wrong_hints():
    """A max_q that is too small asks for many splits of many rows: bounded, and of
    what right hints ask for nothing is taken."""
    f = _lib.lib().jules_hip_kv4_attention_workspace_size
    most = 256 << 20
    assert f(1, 8192, 32, 8, 128, 1, 131072) <= most
    for batch in (1, 2, 7, 64, 1000):
        for tokens in (batch, 100 * batch, 1 << 20, (1 << 30) // 64):
            for heads_q, heads, D in ((64, 8, 128), (8, 8, 64), (64, 1, 64)):
                for max_q in (0, 1, 5, 20, 1000, tokens):
                    for max_len in (1, 5000, 131072, 2**31 - 1):
                        assert f(batch, tokens, heads_q, heads, D, max_q, max_len) <= most
    # single tokens of 64 sequences of 8 heads of 8 in 4 splits, 5 drafted of one in 64
    assert f(64, 64, 64, 8, 128, 1, 8192) == 64 * 64 * 4 * 130 * 4
    assert f(1, 5, 32, 4, 64, 5, 131072) == 5 * 32 * 64 * 66 * 4
