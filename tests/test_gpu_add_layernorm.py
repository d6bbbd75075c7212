"""GPU tests of jules_hip_add_layernorm and jules_hip_add_layernorm_bwd
(ops.add_layernorm, ops.add_layernorm_bwd) against the formulas in 64 bits: every
row length's kernel and its borders, rows at any address, each combination of
types, dropout, what may be left out, in place, rows of equal elements, NaN,
infinities, tiny, huge and far-off values, more rows than blocks, differences of
the loss, other streams, shared workspaces and a replayed graph."""
import numpy as np
import pytest
import torch

from jules_amd import _lib, ops
from tests.decoder64 import F32, f64
from tests.helpers import case
from tests.training64 import SLACK, drop32, kept, layernorm64, layernorm_bwd64, step, threshold

pytestmark = pytest.mark.gpu

f32, bf16 = torch.float32, torch.bfloat16
EPS = 1e-5
TINY = 2.0**-126
RNG = (0x0123456789ABCDEF, 77)
WIDTHS = [1, 2, 7, 8, 9, 63, 127, 128, 129, 511, 512, 513, 2047, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 20003, 40001]


def _rng(dev):
    return torch.tensor(RNG, dtype=torch.int64, device=dev)


def _rows(dev, M, N, dtype, seed, shift=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(M * N + shift, dtype=dtype, device=dev)
    flat[shift:] = (scale * torch.randn(M * N, generator=g)).to(dev)
    return flat[shift:].view(M, N)


def _weights(dev, N, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    return (1.0 + 0.3 * torch.randn(N, generator=g)).to(dev), (0.2 * torch.randn(N, generator=g)).to(dev)


def _h32(x, r, p, offset=0):
    """h as the kernel has it in fp32."""
    h = drop32(x, p, RNG, offset)
    return h if r is None else r.float().cpu().numpy() + h


def _check_forward(x, r, gamma, beta, p, y, h, mean, rstd, eps=EPS, offset=0):
    h32 = _h32(x, r, p, offset)
    want, m64, s64, bound = layernorm64(h32, gamma, beta, eps)
    assert torch.equal(h.cpu(), torch.from_numpy(h32).to(h.dtype))
    assert (np.abs(f64(y) - want) <= bound + SLACK * step(y.dtype) * np.abs(want) + TINY).all()
    assert (np.abs(f64(mean).reshape(-1) - m64) <= SLACK * F32 * np.abs(m64) + 2.0**-45 * np.abs(h32).mean(-1)).all()
    assert (np.abs(f64(rstd).reshape(-1) - s64) <= 2 * F32 * s64).all()


def _check_backward(dy, h, mean, rstd, gamma, dh, p, grads, offset=0, rows_added=None):
    dx, dr, dgamma, dbeta = grads
    M, N = dy.shape
    want, wg, wb, bound, bg, bb = layernorm_bwd64(dy, h, mean, rstd, gamma, dh, M if rows_added is None else rows_added)
    if dr is not None:
        assert (np.abs(f64(dr) - want) <= bound + SLACK * step(dr.dtype) * np.abs(want) + TINY).all()
    if dx is not None:
        f = kept(M, N, p, RNG, offset) * (65536.0 / (65536 - threshold(p))) if threshold(p) else 1.0
        assert (np.abs(f64(dx) - f * want) <= f * bound * (1 + F32) + SLACK * (2 * F32 + step(dx.dtype)) * np.abs(f * want) + TINY).all()
        if threshold(p):
            assert (f64(dx)[f == 0] == 0).all()
    if dgamma is not None:
        assert (np.abs(f64(dgamma) - wg) <= bg + TINY).all()
    if dbeta is not None:
        assert (np.abs(f64(dbeta) - wb) <= bb + TINY).all()


@pytest.mark.parametrize("N", WIDTHS)
def test_forward_widths(dev, N):
    gamma, beta = _weights(dev, N, N)
    for M, xt, rt, p, shift in ((3, f32, f32, 0.1, 0), (5, bf16, bf16, 0.5, 1), (2, bf16, f32, 0.0, 0), (1, f32, bf16, 0.3, 3),
                                (3, bf16, None, 0.25, 1), (2, f32, None, 0.0, 0), (37, bf16, bf16, 0.1, 0)):
        case(f"add_layernorm {M}x{N} {xt} {rt} p={p} shift {shift}")
        x = _rows(dev, M, N, xt, N, shift)
        r = None if rt is None else _rows(dev, M, N, rt, N + 1, shift, 2.0)
        out = ops.add_layernorm(x, r, gamma, beta, EPS, p=p, rng=_rng(dev), offset=4)
        torch.cuda.synchronize()
        assert out[0].dtype == xt and out[1].dtype == (rt or xt) and (out[1] is x) == (rt is None and p == 0.0)
        _check_forward(x, r, gamma, beta, p, *out, offset=4)


@pytest.mark.parametrize("N", WIDTHS)
def test_backward_widths(dev, N):
    gamma, _ = _weights(dev, N, N)
    for M, xt, ht, more, p, shift in ((3, f32, f32, True, 0.1, 0), (5, bf16, bf16, True, 0.5, 1), (2, bf16, f32, False, 0.0, 0),
                                      (1, f32, bf16, True, 0.3, 3), (3, bf16, bf16, False, 0.0, 1), (37, bf16, bf16, True, 0.1, 0)):
        case(f"add_layernorm_bwd {M}x{N} {xt} {ht} dh {more} p={p} shift {shift}")
        h = _rows(dev, M, N, ht, N, shift, 2.0)
        dy = _rows(dev, M, N, xt, N + 1, shift)
        dh = _rows(dev, M, N, ht, N + 2, shift) if more else None
        _, _, mean, rstd = ops.add_layernorm(h, None, gamma)
        grads = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=p, rng=_rng(dev), offset=4)
        torch.cuda.synchronize()
        assert grads[0].dtype == xt and grads[1].dtype == ht and (grads[0] is grads[1]) == (p == 0.0 and xt == ht)
        _check_backward(dy, h, mean, rstd, gamma, dh, p, grads, offset=4)


@pytest.mark.parametrize("M,N", [(70000, 64), (70001, 100), (20000, 264), (9000, 1000), (5000, 2050), (3100, 5001), (1300, 8200),
                                 (2100, 16400)])
def test_rows_beyond_the_blocks(dev, M, N):
    """Rows of sizes a million apart side by side: what a row is scaled by is its own."""
    case(f"add_layernorm {M}x{N}")
    g = torch.Generator(dev).manual_seed(M + N)
    size = 10.0 ** (6.0 * torch.rand(M, 1, generator=g, device=dev) - 3.0)
    x = (size * torch.randn(M, N, generator=g, device=dev)).to(bf16)
    r = (2.0 * size * torch.randn(M, N, generator=g, device=dev)).to(bf16)
    dy, dh = (torch.randn(M, N, generator=g, device=dev).to(bf16) for _ in range(2))
    gamma, beta = _weights(dev, N, 3)
    y, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta, EPS, p=0.1, rng=_rng(dev))
    dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.1, rng=_rng(dev))
    torch.cuda.synchronize()
    sums = np.zeros((2, N)), np.zeros((2, N))
    for i in range(0, M, 4096):
        at = slice(i, min(i + 4096, M))
        rows = np.arange(at.start, at.stop)
        keep = kept(M, N, 0.1, RNG, 0, rows)
        f = np.float32(65536 / (65536 - threshold(0.1)))
        h32 = r[at].float().cpu().numpy() + np.where(keep, x[at].float().cpu().numpy() * f, np.float32(0))
        want, m64, s64, bound = layernorm64(h32, gamma, beta, EPS)
        assert torch.equal(h[at].cpu(), torch.from_numpy(h32).to(bf16)), i
        assert (np.abs(f64(y[at]) - want) <= bound + SLACK * step(bf16) * np.abs(want) + TINY).all(), i
        assert (np.abs(f64(rstd[at]) - s64) <= 2 * F32 * s64).all(), i
        want, wg, wb, bound, bg, bb = layernorm_bwd64(dy[at], h[at], mean[at], rstd[at], gamma, dh[at], M)
        assert (np.abs(f64(dr[at]) - want) <= bound + SLACK * step(bf16) * np.abs(want) + TINY).all(), i
        want, bound = want * keep * float(f), bound * keep * float(f)
        assert (np.abs(f64(dx[at]) - want) <= bound * (1 + F32) + SLACK * (2 * F32 + step(bf16)) * np.abs(want) + TINY).all(), i
        sums[0][:] += wg, wb
        sums[1][:] += bg, bb
    assert (np.abs(f64(dgamma) - sums[0][0]) <= sums[1][0]).all() and (np.abs(f64(dbeta) - sums[0][1]) <= sums[1][1]).all()
    # a chain of all the rows is what the bound allows; in truth a thread adds few of them
    assert np.linalg.norm(f64(dgamma) - sums[0][0]) <= 1e-6 * np.linalg.norm(sums[0][0])


@pytest.mark.parametrize("N", [100, 500, 2000, 8000, 12000, 20001])
def test_what_may_be_left_out(dev, N):
    x, r, dy, dh = (_rows(dev, 6, N, f32, i) for i in range(4))
    gamma, beta = _weights(dev, N, 1)
    for g, b in ((None, None), (gamma, None), (None, beta)):
        out = ops.add_layernorm(x, r, g, b)
        _check_forward(x, r, g, b, 0.0, *out)
        _check_backward(dy, out[1], out[2], out[3], g, None, 0.0, ops.add_layernorm_bwd(dy, out[1], out[2], out[3], g))
    _, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta)
    all_ = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.2, rng=_rng(dev))
    some = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.2, rng=_rng(dev), weight_grads=False)
    assert torch.equal(some[0], all_[0]) and torch.equal(some[1], all_[1]) and some[2] is None and some[3] is None


@pytest.mark.parametrize("N", [100, 500, 2000, 8000, 12000, 20001])
def test_in_place(dev, N):
    """out = x, h = residual; dx = dy, dresidual = dh: the same bits."""
    x, r, dy, dh = (_rows(dev, 6, N, bf16, i) for i in range(4))
    gamma, beta = _weights(dev, N, 1)
    rng = _rng(dev)
    y, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta, p=0.1, rng=rng)
    x2, r2 = x.clone(), r.clone()
    got = ops.add_layernorm(x2, r2, gamma, beta, p=0.1, rng=rng, out=x2, h=r2)
    assert got[0] is x2 and got[1] is r2 and torch.equal(x2, y) and torch.equal(r2, h)
    want = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.1, rng=rng)
    dy2, dh2 = dy.clone(), dh.clone()
    got = ops.add_layernorm_bwd(dy2, h, mean, rstd, gamma, dh2, p=0.1, rng=rng, dx=dy2, dresidual=dh2)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is dy2 and got[1] is dh2


@pytest.mark.parametrize("M,N", [(6, 100), (700, 2000), (6, 20001)])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_in_place_without_a_residual(dev, M, N, dtype):
    """out = x where h would be x: h is what x was, and the gradients are those of the call beside it."""
    x, dy = _rows(dev, M, N, dtype, 1), _rows(dev, M, N, dtype, 2)
    gamma, beta = _weights(dev, N, 1)
    want = ops.add_layernorm(x, None, gamma, beta)
    assert want[1] is x
    grads = ops.add_layernorm_bwd(dy, *want[1:], gamma)
    for out in (lambda t: t, lambda t: t.view(M, N)):  # x itself, and another tensor of the same place
        mine = x.clone()
        got = ops.add_layernorm(mine, None, gamma, beta, out=out(mine))
        assert torch.equal(mine, want[0]) and torch.equal(got[1], x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(ops.add_layernorm_bwd(dy, *got[1:], gamma), grads))


@pytest.mark.parametrize("M,N", [(5000, 300), (3000, 2000), (700, 3000), (1500, 8000), (600, 12000)])
def test_in_place_of_many_rows(dev, M, N):
    """Rows whose columns' sums are left in the workspace."""
    dy, h, dh = (_rows(dev, M, N, bf16, i) for i in range(3))
    gamma, _ = _weights(dev, N, 1)
    rng = _rng(dev)
    _, _, mean, rstd = ops.add_layernorm(h, None, gamma)
    want = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.1, rng=rng)
    got = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh, p=0.1, rng=rng, dx=dy, dresidual=dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is dy and got[1] is dh


@pytest.mark.parametrize("N", [100, 1000, 3000, 20001])
def test_outputs_of_other_types(dev, N):
    """y in fp32 of bf16 rows and the reverse; h of x where there is no residual, x's own place among them."""
    x, r = _rows(dev, 5, N, bf16, 1), _rows(dev, 5, N, f32, 2)
    gamma, beta = _weights(dev, N, 1)
    for p in (0.0, 0.3):
        out = ops.add_layernorm(x, r, gamma, beta, p=p, rng=_rng(dev), out=torch.empty(5, N, device=dev))
        _check_forward(x, r, gamma, beta, p, *out)
        out = ops.add_layernorm(r, x, gamma, beta, p=p, rng=_rng(dev), out=torch.empty(5, N, dtype=bf16, device=dev))
        _check_forward(r, x, gamma, beta, p, *out)
        out = ops.add_layernorm(x, None, gamma, beta, p=p, rng=_rng(dev), h=torch.empty(5, N, device=dev))
        _check_forward(x, None, gamma, beta, p, *out)
        want = ops.add_layernorm(x, None, gamma, beta, p=p, rng=_rng(dev))
        mine = x.clone()
        got = ops.add_layernorm(mine, None, gamma, beta, p=p, rng=_rng(dev), h=mine)
        assert got[1] is mine and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M,N", [(6, 100), (6, 5000), (900, 2000), (6, 20001)])
def test_outputs_that_are_not_wanted(dev, M, N):
    """Through the C ABI: each output alone has the bits that it has beside the others."""
    dy, h = _rows(dev, M, N, bf16, 1), _rows(dev, M, N, bf16, 2)
    gamma, _ = _weights(dev, N, 1)
    _, _, mean, rstd = ops.add_layernorm(h, None, gamma)
    want = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, p=0.2, rng=_rng(dev))
    rng, ws = _rng(dev), ops.add_layernorm_bwd_workspace(M, N, dev)
    for i in range(4):
        out = [torch.zeros_like(t) if k == i else None for k, t in enumerate(want)]
        st = _lib.lib().jules_hip_add_layernorm_bwd(
            1, 1, 0.2, rng.data_ptr(), 0, dy.data_ptr(), h.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), gamma.data_ptr(),
            *(None if t is None else t.data_ptr() for t in out), M, N, ws.data_ptr(), ws.numel() * 4,
            torch.cuda.current_stream().cuda_stream)
        assert st == 0 and torch.equal(out[i], want[i]), i


def test_offsets_past_32_bits(dev):
    """2.3 * 10^9 elements: the first and the last rows, and the columns' sums of rows that are 0 but for the last."""
    M, N = 140000, 16384
    case(f"add_layernorm {M}x{N}")
    rows = torch.tensor([0, 1, M - 2, M - 1], device=dev)
    x = torch.zeros(M, N, dtype=bf16, device=dev)
    x[rows] = _rows(dev, 4, N, bf16, 1)
    y, h, mean, rstd = ops.add_layernorm(x, None, p=0.3, rng=_rng(dev))
    keep = kept(M, N, 0.3, RNG, 0, rows.cpu().numpy())
    h32 = np.where(keep, x[rows].float().cpu().numpy() * np.float32(65536 / (65536 - threshold(0.3))), np.float32(0))
    want, _, _, bound = layernorm64(h32, None, None, EPS)
    assert torch.equal(h[rows].cpu(), torch.from_numpy(h32).to(bf16)) and not y[2:M - 2].any()
    assert (np.abs(f64(y[rows]) - want) <= bound + SLACK * step(bf16) * np.abs(want) + TINY).all()
    del y
    dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(x, h, mean, rstd, p=0.3, rng=_rng(dev))
    _check_backward(x[rows], h[rows], mean[rows], rstd[rows], None, None, 0.0, (None, dr[rows], dgamma, dbeta), rows_added=M)
    assert not dr[2:M - 2].any() and (dx[rows].cpu()[~torch.from_numpy(keep)] == 0).all()


def test_longest_row(dev):
    """A row of 2^31 - 1 elements: grids formed near the end of 32 bits, every column's own sums,
    and the rest at the row's ends and in its middle."""
    N = 2**31 - 1
    case(f"add_layernorm 1x{N}")
    g = torch.Generator(dev).manual_seed(4)
    h, dy = (torch.empty(1, N, dtype=bf16, device=dev).normal_(generator=g) for _ in range(2))
    y, _, mean, rstd = ops.add_layernorm(h)
    dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(dy, h, mean, rstd)
    torch.cuda.synchronize()
    total, square, c1, c2, size1, size2 = (0.0,) * 6
    for i in range(0, N, 1 << 28):
        part, grad = h[0, i:i + (1 << 28)].double(), dy[0, i:i + (1 << 28)].double()
        total, square = total + part.sum().item(), square + part.square().sum().item()
        n = (part - mean.double()) * rstd.double()
        c1, size1 = c1 + grad.sum().item(), size1 + grad.abs().sum().item()
        c2, size2 = c2 + (grad * n).sum().item(), size2 + (grad * n).abs().sum().item()
    assert abs(mean.item() - total / N) <= F32 * abs(total / N) + 2.0**-45
    var = square / N - (total / N) ** 2
    assert abs(rstd.item() - (var + EPS) ** -0.5) <= 2 * F32 * (var + EPS) ** -0.5
    # one row: the columns' sums are its products, rounded as often
    for i in range(0, N, 1 << 28):
        at = slice(i, min(i + (1 << 28), N))
        assert torch.equal(dbeta[at], dy[0, at].float()), i
        assert torch.equal(dgamma[at], dy[0, at].float() * ((h[0, at].float() - mean) * rstd)), i
    chain = (N / 1024 + 30) * F32  # as in layernorm_bwd64
    for at in (slice(0, 5000), slice(2**30 - 2500, 2**30 + 2500), slice(N - 5000, N)):
        n, grad = (h[0, at].double() - mean.double()) * rstd.double(), dy[0, at].double()
        assert ((y[0, at].double() - n).abs() <= step(bf16) * SLACK * n.abs() + 4 * F32 * (1 + n.abs())).all()
        want = rstd.double() * (grad - c1 / N - n * c2 / N)
        bound = rstd.double() * (chain * size1 / N + n.abs() * chain * size2 / N) + SLACK * step(bf16) * want.abs() + 8 * F32 * (1 + want.abs() + n.abs())
        assert ((dr[0, at].double() - want).abs() <= bound).all() and dx is dr


@pytest.mark.parametrize("M,N", [(3, 1), (3, 100), (3, 513), (3, 2047), (3, 5001), (3, 12001), (3, 16387), (20, 40001), (2100, 100),
                                 (2100, 1001), (600, 2047), (600, 3001), (600, 5001), (600, 12001)])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_equal_elements_far_from_zero(dev, M, N, dtype):
    """Rows of 1e37 everywhere: a distance of 0 from the mean, where 0 less the mean times rstd is
    past fp32's range, as it would be for elements behind the row's end."""
    h = torch.full((M, N), 1e37, device=dev).to(dtype)
    h[1] = -h[1]
    dy, dh = _rows(dev, M, N, dtype, 1), _rows(dev, M, N, dtype, 2)
    gamma, _ = _weights(dev, N, 1)
    y, _, mean, rstd = ops.add_layernorm(h, None, gamma)
    assert not y.any()
    grads = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, dh)
    assert all(torch.isfinite(t).all() for t in grads) and not grads[2].any()
    _check_backward(dy, h, mean, rstd, gamma, dh, 0.0, grads)


@pytest.mark.parametrize("N", [100, 500, 2000, 8000, 12000, 20001])
def test_extreme_rows(dev, N):
    """Equal elements, NaN, infinities, tiny, huge and far-off values; rows beside them are theirs alone."""
    case(f"add_layernorm extreme rows of {N}")
    x, r = _rows(dev, 9, N, f32, 5), _rows(dev, 9, N, f32, 6)
    gamma, beta = _weights(dev, N, 2)
    x[0], r[0] = 0.0, 3.7
    x[1, N // 2] = float("nan")
    r[2, N - 1] = float("inf")
    x[3] *= 1e-30
    r[3] *= 1e-30
    x[4] *= 1e18
    r[4] *= 1e18
    x[5], r[5] = 3e38, 3e38
    r[6] += 1e6  # far from zero
    x[7, 0], r[7, 0] = float("inf"), float("-inf")
    y, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta)
    for i in (1, 2, 5, 7):
        assert torch.isnan(y[i]).all() and torch.isnan(rstd[i]), i
    assert torch.equal(y[0], beta)
    keep = [0, 3, 4, 6, 8]
    _check_forward(x[keep], r[keep], gamma, beta, 0.0, y[keep], h[keep], mean[keep], rstd[keep])
    dy = _rows(dev, 9, N, f32, 7)
    dx, dr, dgamma, _ = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma)
    _check_backward(dy[keep], h[keep], mean[keep], rstd[keep], gamma, None, 0.0, (dx[keep], dr[keep], None, None))
    for i in (1, 2, 5, 7):
        assert torch.isnan(dr[i]).all(), i
    dy[[1, 2, 5, 7]], h[[1, 2, 5, 7]], mean[[1, 2, 5, 7]], rstd[[1, 2, 5, 7]] = 0.0, 0.0, 0.0, 1.0
    _, _, dgamma, dbeta = ops.add_layernorm_bwd(dy, h, mean, rstd, gamma)
    _check_backward(dy, h, mean, rstd, gamma, None, 0.0, (None, None, dgamma, dbeta))


def test_empty(dev):
    x = torch.empty(0, 16, device=dev)
    y, h, mean, rstd = ops.add_layernorm(x, x)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(x, x, mean, rstd)
    assert dx.shape == (0, 16) and torch.equal(dgamma, torch.zeros(16, device=dev)) and torch.equal(dbeta, dgamma)


def test_leading_dimensions(dev):
    x, r = _rows(dev, 24, 72, bf16, 1).view(2, 3, 4, 72), _rows(dev, 24, 72, bf16, 2).view(2, 3, 4, 72)
    y, h, mean, rstd = ops.add_layernorm(x, r, p=0.1, rng=_rng(dev))
    assert mean.shape == (2, 3, 4) and y.shape == x.shape
    flat = ops.add_layernorm(x.view(24, 72), r.view(24, 72), p=0.1, rng=_rng(dev))
    assert all(torch.equal(a.reshape(-1), b.reshape(-1)) for a, b in zip((y, h, mean, rstd), flat))
    assert ops.add_layernorm_bwd(y, h, mean, rstd)[1].shape == x.shape


def test_differences(dev):
    """The gradients against differences of the loss sum(w y) + sum(v h), in 64 bits from the
    kernel's own outputs: central, steps of 2^-6, third derivatives of the loss below 50, so
    their own error is below 50 * 2^-12 / 6 a unit of direction; y is rounded to fp32,
    2^-24 of sums below 4000, over the step."""
    M, N, e = 4, 24, 2.0**-6
    x, r, w, v = (_rows(dev, M, N, f32, i) for i in range(4))
    gamma, beta = _weights(dev, N, 1)
    rng = _rng(dev)

    def loss(x, r, gamma, beta):
        y, h, _, _ = ops.add_layernorm(x, r, gamma, beta, EPS, p=0.25, rng=rng)
        return ((w.double() * y.double()).sum() + (v.double() * h.double()).sum()).item()

    _, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta, EPS, p=0.25, rng=rng)
    dx, dr, dgamma, dbeta = ops.add_layernorm_bwd(w, h, mean, rstd, gamma, v, p=0.25, rng=rng)
    at = [x, r, gamma, beta]
    for i, grad in enumerate((dx, dr, dgamma, dbeta)):
        for k in range(6):
            d = _rows(dev, 1, at[i].numel(), f32, 50 + 10 * i + k).view(at[i].shape)
            d = d / d.norm()
            plus, minus = list(at), list(at)
            plus[i], minus[i] = at[i] + e * d, at[i] - e * d
            slope = (loss(*plus) - loss(*minus)) / (2 * e)
            assert abs(slope - (grad.double() * d.double()).sum().item()) <= 50 * e * e / 6 + 2 * 4000 * F32 / e, (i, k)


def test_streams_and_workspaces(dev):
    """Calls that overlap in time, each with a workspace of its own."""
    sets = []
    for i in range(2):
        dy, h = _rows(dev, 700, 2048, bf16, i), _rows(dev, 700, 2048, bf16, i + 9)
        _, _, mean, rstd = ops.add_layernorm(h)
        sets.append((dy, h, mean, rstd))
    want = [ops.add_layernorm_bwd(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    spaces = [ops.add_layernorm_bwd_workspace(700, 2048, dev) for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.add_layernorm_bwd(*sets[i], workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


@pytest.mark.parametrize("M,N", [(300, 1500), (1200, 1500), (600, 5000)])
def test_graph(dev, M, N):
    """Forward and backward in one graph, the position moved on between the replays, eager
    calls between them."""
    x, r, dy = (_rows(dev, M, N, bf16, i) for i in range(3))
    gamma, beta = _weights(dev, N, 1)
    rng = _rng(dev)

    def run():
        y, h, mean, rstd = ops.add_layernorm(x, r, gamma, beta, p=0.1, rng=rng, offset=3)
        return (y, h, mean, rstd, *ops.add_layernorm_bwd(dy, h, mean, rstd, gamma, y, p=0.1, rng=rng, offset=3))

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        rng[1] += 8
        want = run()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
