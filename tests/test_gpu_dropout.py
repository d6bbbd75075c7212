"""GPU tests of jules_hip_dropout (ops.dropout): bit for bit what the generator and
two fp32 operations give, at widths that end inside a piece of 8, at any address, in
each combination of types, with the residual and in place, over many rows; NaN and
infinity in dropped places; the mask's independence of everything but its numbers;
the share that is dropped; another stream and a replayed graph."""
import numpy as np
import pytest
import torch

from jules_amd import _lib, ops
from tests.helpers import case
from tests.training64 import drop32, kept, threshold

pytestmark = pytest.mark.gpu

f32, bf16 = torch.float32, torch.bfloat16
SEED, AT = -0x123456789ABCDEF, 2**40 + 5


def _rng(dev, seed=SEED, at=AT):
    return torch.tensor([seed, at], dtype=torch.int64, device=dev)


def _rows(dev, M, N, dtype, seed=0, shift=0):
    """[M, N] that begins `shift` elements past an allocation's begin."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(M * N + shift, dtype=dtype, device=dev)
    flat[shift:] = torch.randn(M * N, generator=g).to(dev)
    return flat[shift:].view(M, N)


def _want(x, r, p, dtype, offset=0, seed=SEED, at=AT):
    y = drop32(x, p, (seed, at), offset)
    if r is not None:
        y = r.float().cpu().numpy() + y
    return torch.from_numpy(np.ascontiguousarray(y, np.float32)).to(dtype)


def _same(got, want):
    return torch.equal(got.cpu(), want) or bool(((got.cpu() == want) | (got.cpu().isnan() & want.isnan())).all())


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 15, 64, 127, 1000, 4096, 5001, 70001])
def test_widths(dev, N):
    for M, xt, rt, ot, p, shift in ((3, f32, None, f32, 0.5, 0), (5, bf16, None, bf16, 0.1, 1), (2, bf16, f32, f32, 0.3, 3),
                                    (4, f32, bf16, bf16, 0.9, 1), (1, bf16, bf16, bf16, 0.25, 0), (2, f32, None, bf16, 0.0, 0),
                                    (2, bf16, None, f32, 0.75, 0), (3, f32, f32, f32, 0.125, 1)):
        case(f"dropout {M}x{N} {xt} {rt} {ot} p={p} shift {shift}")
        x = _rows(dev, M, N, xt, N, shift)
        r = None if rt is None else _rows(dev, M, N, rt, N + 1, shift)
        y = ops.dropout(x, p, _rng(dev), offset=11, residual=r, dtype=None if rt else ot)
        torch.cuda.synchronize()
        assert y.dtype == ot and _same(y, _want(x, r, p, ot, 11)), (M, N, p)


@pytest.mark.parametrize("N", [1, 8, 13, 768, 5001])
def test_nothing_dropped_without_rng(dev, N):
    """p = 0, or one that rounds to it, takes no rng (evaluation): x, or its sum with the residual, in each
    combination of types, through the front end and the C ABI."""
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for xt, rt, ot in ((f32, None, f32), (bf16, None, bf16), (f32, None, bf16), (bf16, None, f32), (f32, f32, f32), (bf16, bf16, bf16),
                       (bf16, f32, f32), (f32, bf16, bf16)):
        case(f"dropout 33x{N} {xt} {rt} {ot} p=0 without rng")
        x = _rows(dev, 33, N, xt, N)
        x[0, 0], x[32, N - 1] = float("nan"), float("inf")
        r = None if rt is None else _rows(dev, 33, N, rt, N + 1)
        want = _want(x, r, 0.0, ot)
        y = ops.dropout(x, 0.0, residual=r, dtype=None if rt else ot)
        torch.cuda.synchronize()
        assert y.dtype == ot and _same(y, want), (xt, rt, ot)
        for p in (0.0, 2.0**-18):
            out = torch.empty_like(want, device=dev)
            st = lib.jules_hip_dropout(int(xt == bf16), int(ot == bf16), p, None, 5, x.data_ptr(), None if r is None else r.data_ptr(),
                                       out.data_ptr(), 33, N, stream)
            torch.cuda.synchronize()
            assert st == 0 and _same(out, want), (xt, rt, ot, p)
    assert torch.equal(ops.dropout(x[1:3], 0.0, out=x[1:3]).cpu(), x[1:3].cpu())


@pytest.mark.parametrize("M,N", [(70000, 40), (70000, 33), (9000, 520), (1, 3000001)])
def test_more_than_one_turn_of_the_blocks(dev, M, N):
    case(f"dropout {M}x{N}")
    x = _rows(dev, M, N, bf16, 3)
    y = ops.dropout(x, 0.2, _rng(dev))
    assert _same(y, _want(x, None, 0.2, bf16))


def test_offsets_past_32_bits(dev):
    """2.3 * 10^9 elements: the first and the last rows."""
    M, N = 70001, 32767
    case(f"dropout {M}x{N}")
    rows = np.array([0, 1, M - 2, M - 1])
    y = ops.dropout(torch.ones(M, N, dtype=bf16, device=dev), 0.5, _rng(dev))
    assert torch.equal(y[torch.from_numpy(rows).to(dev)].cpu() != 0, torch.from_numpy(kept(M, N, 0.5, (SEED, AT), 0, rows)))


@pytest.mark.parametrize("N", [37, 1024])
def test_in_place(dev, N):
    x, r = _rows(dev, 50, N, f32, 1), _rows(dev, 50, N, f32, 2)
    rng = _rng(dev)
    want, sum_ = ops.dropout(x, 0.3, rng), ops.dropout(x, 0.3, rng, residual=r)
    a, b, c = x.clone(), r.clone(), x.clone()
    assert ops.dropout(a, 0.3, rng, out=a) is a and torch.equal(a, want)
    ops.dropout(x, 0.3, rng, residual=b, out=b)
    ops.dropout(c, 0.3, rng, residual=r, out=c)
    assert torch.equal(b, sum_) and torch.equal(c, sum_)


def test_dropped_nan_and_infinity(dev):
    x = torch.full((64, 100), float("nan"), device=dev)
    x[:, ::3] = float("inf")
    y = ops.dropout(x, 0.5, _rng(dev)).cpu()
    keep = torch.from_numpy(kept(64, 100, 0.5, (SEED, AT), 0))
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    r = torch.ones(64, 100, device=dev)
    assert (ops.dropout(x, 0.5, _rng(dev), residual=r).cpu()[~keep] == 1).all()


def test_what_the_mask_depends_on(dev):
    """On the place, the seed, and the position with the offset; not on types, or on
    rows behind or in front; a shape with as many elements is another mask."""
    x = torch.ones(40, 96, device=dev)

    def mask(x, p=0.5, rng=_rng(dev), **kw):
        return ops.dropout(x, p, rng, **kw).float().reshape(-1) != 0

    base = mask(x)
    assert torch.equal(base, mask(x.bfloat16())) and torch.equal(base, mask(x.view(5, 8, 96)))
    assert torch.equal(base[:20 * 96], mask(x[:20]))
    assert torch.equal(base, mask(x, rng=_rng(dev, at=AT - 3), offset=3))
    assert torch.equal(base, mask(x, rng=_rng(dev, at=-1), offset=AT + 1))  # 64 bits, wrapping
    for other in (mask(x, offset=1), mask(x, rng=_rng(dev, SEED + 1)), mask(x, rng=_rng(dev, SEED + 2**32)),
                  mask(x, offset=2**32), mask(x.view(80, 48))):
        assert 0.4 < (base != other).float().mean() < 0.6
    # a larger p drops what a smaller one drops
    assert not (mask(x, 0.7) & ~mask(x, 0.2)).any()


@pytest.mark.parametrize("p", [2.0**-16, 0.1, 0.5, 0.9, 1.0 - 2.0**-16])
def test_share(dev, p):
    """What is dropped of 2^24 elements: within 6 standard deviations of t / 65536."""
    n = 1 << 24
    y = ops.dropout(torch.ones(4096, 4096, device=dev), p, _rng(dev))
    t = threshold(p) / 65536
    share = (y == 0).double().mean().item()
    assert abs(share - t) <= 6 * (t * (1 - t) / n) ** 0.5
    assert (y[y != 0] == np.float32(65536 / (65536 - threshold(p)))).all()


def test_gradient(dev):
    """sum(g * dropout(x)) is linear in x: its gradient is the same call on g."""
    x, g, v = (_rows(dev, 30, 77, f32, i) for i in range(3))
    rng = _rng(dev)
    grad = ops.dropout(g, 0.4, rng).double()
    change = (g.double() * (ops.dropout(x + v, 0.4, rng).double() - ops.dropout(x, 0.4, rng).double())).sum()
    # x + v and the two products round once each: 3 half steps of values below 20, 2310 elements, weights below 6
    assert abs(change - (grad * v.double()).sum()) <= 3 * 20 * 2.0**-24 * (g.double().abs().sum() * 2)


def test_empty(dev):
    assert ops.dropout(torch.empty(0, 8, device=dev), 0.5, _rng(dev)).shape == (0, 8)
    assert ops.dropout(torch.empty(3, 0, device=dev), 0.5, _rng(dev)).shape == (3, 0)


def test_stream_and_graph(dev):
    """A captured call drops other elements when the position has moved on."""
    x = _rows(dev, 128, 1000, bf16, 5)
    rng = _rng(dev)
    want = ops.dropout(x, 0.1, rng, offset=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.dropout(x, 0.1, rng, offset=2)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.dropout(x, 0.1, rng, offset=2, out=out)
    seen = []
    for i in range(4):
        rng[1] += 16
        x.copy_(torch.randn_like(x))
        want = ops.dropout(x, 0.1, rng, offset=2)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        seen.append(out != 0)
    assert not torch.equal(seen[0], seen[1])
