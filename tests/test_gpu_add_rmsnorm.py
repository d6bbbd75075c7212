"""GPU tests of jules_hip_add_rmsnorm (ops.add_rmsnorm, ops.add_rmsnorm_int8)
against the formula in 64 bits: every row length's kernel and its borders, rows
at any address, each combination of types, in place, rows of zeros, NaN,
infinities, tiny and huge values, another stream, a captured graph, and the int8
product that takes the rows."""
import numpy as np
import pytest
import torch

from jules_amd import ops
from tests.decoder64 import BF16, F32, f64, norm64
from tests.helpers import case

pytestmark = pytest.mark.gpu

f32, bf16 = torch.float32, torch.bfloat16
EPS = 1e-5
WIDTHS = [1, 2, 7, 8, 9, 63, 511, 512, 513, 2040, 2048, 2049, 5001, 8191, 8192, 8193, 16384, 20003, 32768, 32769, 70001]


def _operands(dev, M, N, xt, rt, seed=0, shift=0):
    """x, residual (None without type) and weight; `shift` elements past an
    allocation's begin, so that rows are not 16-byte aligned."""
    g = torch.Generator().manual_seed(seed)

    def make(scale, t):
        flat = torch.empty(M * N + shift, dtype=t, device=dev)
        flat[shift:] = (scale * torch.randn(M * N, generator=g)).to(dev)
        return flat[shift:].view(M, N)

    return (make(1.0, xt), None if rt is None else make(2.0, rt),
            (1.0 + 0.3 * torch.randn(N, generator=g)).to(dev))


def _check(x, r, w, y, q, s, h, eps=EPS):
    h64, y64, s64, t64 = norm64(x, r, w, eps)
    if r is not None:
        # x + r in fp32, then the residual's type
        step = F32 + (BF16 if r.dtype == bf16 else 0)
        assert (np.abs(f64(h) - h64) <= 1.01 * step * np.abs(h64)).all()
    if y is not None:
        # h, the factor (whose sum of squares takes rounded h), two products: 6
        # roundings in fp32, then the type's
        step = 6 * F32 + (BF16 if y.dtype == bf16 else 0)
        assert (np.abs(f64(y) - y64) <= 1.01 * step * np.abs(y64)).all()
    if q is not None:
        assert (np.abs(f64(s) - s64) <= 8 * F32 * s64).all()
        # h, h w, 127 / max, the product with it: under 8 roundings of a number up to 127
        assert (np.abs(f64(q) - t64) <= 0.5 + 8 * 127 * F32).all()


@pytest.mark.parametrize("N", WIDTHS)
def test_widths(dev, N):
    for M, xt, rt, shift in ((3, f32, f32, 0), (5, bf16, bf16, 1), (2, bf16, f32, 0), (1, f32, bf16, 3), (3, bf16, None, 1),
                             (2, f32, None, 0)):
        case(f"add_rmsnorm {M}x{N} {xt} {rt} shift {shift}")
        x, r, w = _operands(dev, M, N, xt, rt, N, shift)
        y, h = ops.add_rmsnorm(x, r, w, EPS)
        q, s, h2 = ops.add_rmsnorm_int8(x, r, w, EPS)
        torch.cuda.synchronize()
        assert y.dtype == xt and (h is None) == (r is None)
        if r is not None:
            assert h.dtype == rt and torch.equal(h, h2)
        _check(x, r, w, y, q, s, h)


def test_many_rows(dev):
    case("add_rmsnorm 5000 rows")
    x, r, w = _operands(dev, 5000, 264, bf16, f32, 3)
    q, s, h = ops.add_rmsnorm_int8(x, r, w, EPS)
    y, _ = ops.add_rmsnorm(x, r, w, EPS, out=torch.empty(5000, 264, device=dev))
    _check(x, r, w, y, q, s, h)


@pytest.mark.parametrize("N", [500, 2000, 8000, 20001, 40001])
def test_in_place(dev, N):
    """residual_out = residual and out = x give the same bits."""
    x, r, w = _operands(dev, 4, N, bf16, bf16, 5)
    y, h = ops.add_rmsnorm(x, r, w, EPS)
    q, s, _ = ops.add_rmsnorm_int8(x, r, w, EPS)
    r2 = r.clone()
    q2, s2, h2 = ops.add_rmsnorm_int8(x, r2, w, EPS, residual_out=r2)
    assert h2 is r2 and torch.equal(r2, h) and torch.equal(q2, q) and torch.equal(s2, s)
    x3, r3 = x.clone(), r.clone()
    ops.add_rmsnorm(x3, r3, w, EPS, out=x3, residual_out=r3)
    assert torch.equal(x3, y) and torch.equal(r3, h)


@pytest.mark.parametrize("N", [40, 1000, 3000, 10000, 33000])
def test_extreme_rows(dev, N):
    """Zeros, NaN, infinities, tiny and huge values; rows beside them are theirs alone."""
    case(f"add_rmsnorm extreme rows of {N}")
    x, r, w = _operands(dev, 9, N, f32, f32, 7)
    x[0] = r[0] = 0.0
    x[1, N // 2] = float("nan")
    r[2, N - 1] = float("inf")
    x[3] *= 1e-37
    r[3] *= 1e-37
    x[4] *= 1e29
    r[4] *= 1e29
    x[5], r[5] = 3e38, 3e38  # x + r passes fp32
    x[6] *= 1e-30
    r[6] *= 1e-30
    x[7, 0], r[7, 0] = float("inf"), float("-inf")
    q, s, h = ops.add_rmsnorm_int8(x, r, w, EPS)
    y, _ = ops.add_rmsnorm(x, r, w, EPS)
    for i in (1, 2, 5, 7):
        assert torch.isnan(s[i]) and not q[i].any()
    assert s[0] == 0 and not q[0].any() and not y[0].any()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, N - 1]) and torch.isnan(y[5]).all()
    keep = [0, 4, 6, 8]
    _check(x[keep], r[keep], w, y[keep], q[keep], s[keep], h[keep])
    # row 3: h near the smallest normal number keeps its codes
    _, _, _, t = norm64(x[3:4], r[3:4], w, EPS)
    assert (np.abs(f64(q[3:4]) - t) <= 0.5 + 1e-3).all()


def test_empty(dev):
    x, r, w = _operands(dev, 0, 16, f32, f32)
    y, h = ops.add_rmsnorm(x, r, w)
    assert y.shape == (0, 16) and h.shape == (0, 16)


def test_feeds_the_int8_product(dev):
    """q and scale are the A and scale_a of matmul_w8a8: the product is that of the
    dequantised rows to fp32 rounding; a NaN row is NaN, and no other."""
    M, N, K = 20, 96, 1024
    x, r, w = _operands(dev, M, K, bf16, f32, 11)
    x[4, 7] = float("nan")
    B = torch.randint(-127, 128, (K, N), dtype=torch.int8, device=dev, generator=torch.Generator(dev).manual_seed(1))
    sb = torch.rand(N, device=dev) * 0.01
    q, s, _ = ops.add_rmsnorm_int8(x, r, w)
    C = f64(ops.matmul_w8a8(q, B, s, sb))
    want = (f64(q) @ f64(B)) * f64(s)[:, None] * f64(sb)
    assert np.isnan(C[4]).all()
    rows = [i for i in range(M) if i != 4]
    assert (np.abs(C[rows] - want[rows]) <= 4 * F32 * np.abs(want[rows])).all()


def test_stream_and_graph(dev):
    x, r, w = _operands(dev, 64, 4096, bf16, bf16, 13)
    want = ops.add_rmsnorm_int8(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rmsnorm_int8(x, r, w)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out, scale, kept = (torch.empty_like(t) for t in want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.add_rmsnorm_int8(x, r, w, out=out, scale=scale, residual_out=kept)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        want = ops.add_rmsnorm_int8(x, r, w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(scale, want[1]) and torch.equal(kept, want[2])


# a row count and width for each kernel: one and 4 waves a row, 1024 threads of 8,
# 256 of 16 and of 32, 512 and 1024 of 32, and rows that are read twice
KERNELS = [(5, 40), (5, 1000), (5, 3000), (600, 3001), (600, 5001), (5, 10000), (5, 20001), (3, 33000)]


@pytest.mark.parametrize("M,N", KERNELS)
@pytest.mark.parametrize("what", ["one NaN", "the last NaN", "all NaN", "infinite over zeros", "minus infinite"])
def test_weights_that_are_no_numbers(dev, M, N, what):
    """y is NaN or infinite somewhere, so int8 rows have no scale: NaN and codes 0, as
    with a NaN in x.  fp32 rows are NaN or infinite in the weight's columns alone; the residual is as ever."""
    case(f"add_rmsnorm {M}x{N} weight: {what}")
    x, r, w = _operands(dev, M, N, f32, f32, 17)
    j = {"one NaN": N // 2, "the last NaN": N - 1, "all NaN": slice(None), "infinite over zeros": N // 3, "minus infinite": 1}[what]
    x[:, j], r[:, j] = (0.0, 0.0) if what == "infinite over zeros" else (x[:, j], r[:, j])
    plain, h0 = ops.add_rmsnorm(x, r, w, EPS)
    w[j] = float("inf") if "over" in what else float("-inf") if "minus" in what else float("nan")
    q, s, h = ops.add_rmsnorm_int8(x, r, w, EPS)
    y, h2 = ops.add_rmsnorm(x, r, w, EPS)
    torch.cuda.synchronize()
    assert torch.equal(h, h0) and torch.equal(h2, h0)
    assert torch.isnan(s).all() and not q.any()
    own = torch.zeros(N, dtype=torch.bool, device=dev)
    own[j] = True
    assert torch.equal(y[:, ~own], plain[:, ~own])
    assert not torch.isfinite(y[:, own]).any()
    assert torch.isnan(y[:, own]).all() == ("minus" not in what)


def _check_on(x, r, w, y, q, s, h):
    """_check with the formula on the device, for many rows, a block of them at a time."""
    for i in range(0, x.shape[0], 512):
        at = slice(i, i + 512)
        h64 = x[at].double() + (0.0 if r is None else r[at].double())
        y64 = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + EPS) * w.double()
        s64 = y64.abs().amax(-1) / 127.0
        if r is not None:
            step = F32 + (BF16 if r.dtype == bf16 else 0)
            assert ((h[at].double() - h64).abs() <= 1.01 * step * h64.abs()).all(), i
        step = 6 * F32 + (BF16 if y.dtype == bf16 else 0)
        assert ((y[at].double() - y64).abs() <= 1.01 * step * y64.abs()).all(), i
        assert ((s[at].double() - s64).abs() <= 8 * F32 * s64).all(), i
        assert ((q[at].double() - y64 / s64[:, None]).abs() <= 0.5 + 8 * 127 * F32).all(), i


@pytest.mark.parametrize("M,N,xt,rt", [
    # widths at the borders of the kernels for more than 512 rows
    (513, 2049, bf16, bf16), (513, 4096, f32, f32), (513, 4097, bf16, f32), (513, 5001, f32, bf16), (513, 8192, bf16, bf16),
    (512, 8192, f32, bf16),
    # more rows than are resident: each block goes on to a third and a fourth
    (33000, 200, bf16, f32), (6200, 513, f32, f32), (3100, 2050, bf16, bf16), (3100, 5001, f32, None), (1550, 8193, bf16, f32),
    (1550, 16385, bf16, None), (4100, 32769, bf16, None)])
def test_rows_beyond_the_blocks(dev, M, N, xt, rt):
    """Rows of sizes a million apart side by side: what a row is scaled by is its own."""
    case(f"add_rmsnorm {M}x{N} {xt} {rt}")
    g = torch.Generator(dev).manual_seed(M + N)
    size = 10.0 ** (6.0 * torch.rand(M, 1, generator=g, device=dev) - 3.0)
    x = (size * torch.randn(M, N, generator=g, device=dev)).to(xt)
    r = None if rt is None else (2.0 * size * torch.randn(M, N, generator=g, device=dev)).to(rt)
    w = 1.0 + 0.3 * torch.randn(N, generator=g, device=dev)
    y, h = ops.add_rmsnorm(x, r, w, EPS)
    q, s, h2 = ops.add_rmsnorm_int8(x, r, w, EPS)
    torch.cuda.synchronize()
    assert r is None or torch.equal(h, h2)
    _check_on(x, r, w, y, q, s, h)
