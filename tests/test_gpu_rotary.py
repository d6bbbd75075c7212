"""GPU tests of jules_hip_rotary (ops.rotary) against the rotation in extended
precision: one and several axes, both pairings, part of a head rotated, far and
negative positions, strided views, in place, both types in and out, and the
inverse as the gradient: against the formula, and against differences."""
import numpy as np
import pytest
import torch

from jules_amd import ops
from tests.decoder64 import BF16, F32, f64, rotary64, rotary_bound
from tests.helpers import case

pytestmark = pytest.mark.gpu

f32, bf16 = torch.float32, torch.bfloat16


def _check(x, y, pos, freq, axis, pairing, inverse):
    x64 = f64(x)
    pos, freq = pos.cpu().numpy(), freq.cpu().numpy()
    want = rotary64(x64, pos, freq, None if axis is None else axis.cpu().numpy(), pairing, inverse)
    bound = rotary_bound(x64, len(freq), pairing, y.dtype == bf16)
    step = BF16 if y.dtype == bf16 else F32
    assert (np.abs(f64(y) - want) <= 1.01 * (bound + step * (np.abs(want) + bound))).all()
    # what is not rotated is copied
    rest = y[..., 2 * len(freq):]
    assert torch.equal(rest, x[..., 2 * len(freq):].to(y.dtype))


def _x(dev, shape, t, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dev).to(t)


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("B,H,S,D,R,sections", [
    (1, 1, 1, 2, 2, None), (1, 3, 1, 64, 64, None), (2, 5, 7, 80, 80, None), (1, 40, 8, 128, 128, None),
    (2, 3, 33, 128, 64, (8, 12, 12)), (1, 4, 50, 96, 48, (3, 0, 21)), (3, 2, 17, 128, 128, (16, 24, 24)),
    (1, 2, 5, 12, 10, (2, 3)), (1, 1, 3, 7, 6, None), (1, 2, 300, 256, 256, (64, 64)), (1, 3, 2, 1024, 1024, None),
    (2, 64, 200, 128, 128, None), (1, 1, 4, 1023, 1022, None), (1, 2, 9, 1024, 2, None)])
def test_shapes(dev, B, H, S, D, R, sections, pairing):
    axes = 1 if sections is None else len(sections)
    freq, axis = ops.rotary_frequencies(R, sections, device=dev)
    g = torch.Generator().manual_seed(S)
    pos = torch.randint(0, 5000, (axes, B, S), generator=g, dtype=torch.int32).to(dev)
    for xt, ot, inverse in ((f32, f32, False), (bf16, bf16, True), (f32, bf16, False), (bf16, f32, False)):
        case(f"rotary {B}x{H}x{S}x{D} R={R} {sections} {pairing} {xt}->{ot} inverse={inverse}")
        x = _x(dev, (B, H, S, D), xt, D)
        y = ops.rotary(x, pos, freq, axis, pairing=pairing, inverse=inverse, dtype=ot)
        assert y.dtype == ot and y.is_contiguous()
        _check(x, y, pos, freq, axis, pairing, inverse)


def test_far_and_negative_positions(dev):
    freq, _ = ops.rotary_frequencies(128, device=dev)
    pos = torch.tensor([[[0, 1, -1, 999999, 16777217, 2**31 - 1, -2**31, -123456789]]], dtype=torch.int32, device=dev)
    x = _x(dev, (1, 2, 8, 128), f32, 1)
    y = ops.rotary(x, pos, freq)
    # the turns are three roundings of 2^-53 off, of up to 2^31 radians: 2^-20 of pairs below 8
    want = rotary64(f64(x), pos.cpu().numpy(), freq.cpu().numpy(), None, "half", False)
    bound = rotary_bound(f64(x), 64, "half", False)
    assert (np.abs(f64(y) - want) <= 1.01 * (bound + F32 * np.abs(want)) + 2.0**-20 * 8).all()
    near = [0, 1, 2, 3, 4]
    _check(x[:, :, near], y[:, :, near], pos[:, :, near], freq, None, "half", False)


def test_views(dev):
    """Heads of a fused projection, token-major memory, broadcast batches, three
    dimensions, outputs into such views; what lies between is left alone."""
    freq, axis = ops.rotary_frequencies(64, (16, 16), device=dev)
    qkv = _x(dev, (2, 30, 12, 64), bf16, 2)  # [B, S, heads, D]
    pos = torch.randint(0, 900, (2, 2, 30), dtype=torch.int32, device=dev)
    x = qkv[:, :, 2:7].transpose(1, 2)
    want = ops.rotary(x.contiguous(), pos, freq, axis)
    assert torch.equal(ops.rotary(x, pos, freq, axis), want)
    hold = torch.full((2, 30, 9, 66), 7.0, dtype=bf16, device=dev)
    view = hold[:, :, 1:6, 1:65].transpose(1, 2)  # 2-byte aligned rows
    assert ops.rotary(x, pos, freq, axis, out=view) is view
    assert torch.equal(view, want)
    hold[:, :, 1:6, 1:65] = 7.0
    assert (hold == 7.0).all()
    # in place, the neighbours untouched
    kept = qkv.clone()
    ops.rotary(x, pos, freq, axis, out=x)
    assert torch.equal(x, want)
    qkv[:, :, 2:7] = kept[:, :, 2:7]
    assert torch.equal(qkv, kept)
    # [H, S, D], and one batch for all positions' batches
    one = x[0]
    assert torch.equal(ops.rotary(one, pos[:, 0].contiguous(), freq, axis), ops.rotary(x[:1], pos[:, :1].contiguous(), freq, axis)[0])
    wide = x[:1].expand(2, -1, -1, -1)
    got = ops.rotary(wide, pos, freq, axis)
    assert torch.equal(got[1], ops.rotary(x[:1], pos[:, 1:].contiguous(), freq, axis)[0])


def test_an_axis_that_is_none(dev):
    freq, axis = ops.rotary_frequencies(32, (8, 8), device=dev)
    axis[3], axis[9] = 2, -1
    x = _x(dev, (1, 2, 4, 40), f32, 3)
    pos = torch.ones(2, 1, 4, dtype=torch.int32, device=dev)
    y = ops.rotary(x, pos, freq, axis)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 19, 9, 25]] = True
    assert torch.isnan(y[..., bad]).all() and not torch.isnan(y[..., ~bad]).any()


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_gradient(dev, pairing):
    """d/dx of sum(rotary(x) * g) is rotary(g, inverse): by the formula's transpose,
    and by differences (the map is linear: exact but for fp32 rounding)."""
    freq, axis = ops.rotary_frequencies(24, (5, 7), device=dev)
    x, g = _x(dev, (1, 2, 6, 32), f32, 4), _x(dev, (1, 2, 6, 32), f32, 5)
    pos = torch.randint(-50, 5000, (2, 1, 6), dtype=torch.int32, device=dev)
    grad = ops.rotary(g, pos, freq, axis, pairing=pairing, inverse=True)
    _check(g, grad, pos, freq, axis, pairing, True)
    base = f64(ops.rotary(x, pos, freq, axis, pairing=pairing))
    rng = np.random.default_rng(6)
    for _ in range(24):
        i = tuple(int(rng.integers(0, n)) for n in x.shape)
        moved = x.clone()
        moved[i] += 1.0
        step = f64(moved)[i] - f64(x)[i]
        diff = ((f64(ops.rotary(moved, pos, freq, axis, pairing=pairing)) - base) * f64(g)).sum() / step
        # two outputs change, each rounded a few times at a size below 8
        assert abs(diff - f64(grad)[i]) <= 8 * 2 * 8 * F32 * 8
    # there and back
    back = ops.rotary(ops.rotary(x, pos, freq, axis, pairing=pairing), pos, freq, axis, pairing=pairing, inverse=True)
    assert (np.abs(f64(back) - f64(x)) <= 2e-6 * 8).all()


def test_autograd_user(dev):
    """As a training program uses it: a function whose backward is the inverse."""
    freq, _ = ops.rotary_frequencies(64, device=dev)
    pos = torch.arange(16, dtype=torch.int32, device=dev).view(1, 1, 16)

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return ops.rotary(x, pos, freq)

        @staticmethod
        def backward(ctx, g):
            return ops.rotary(g, pos, freq, inverse=True)

    x = _x(dev, (1, 2, 16, 64), f32, 8).requires_grad_()
    w = _x(dev, (1, 2, 16, 64), f32, 9)
    (Rotary.apply(x) * w).sum().backward()
    _check(w, x.grad, pos, freq, None, "half", True)


def test_stream_and_graph(dev):
    freq, axis = ops.rotary_frequencies(128, (32, 32), device=dev)
    x = _x(dev, (1, 8, 64, 128), bf16, 10)
    pos = torch.randint(0, 4000, (2, 1, 64), dtype=torch.int32, device=dev)
    want = ops.rotary(x, pos, freq, axis)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(x, pos, freq, axis)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rotary(x, pos, freq, axis, out=out)
    for _ in range(3):
        pos += 17
        x.copy_(torch.randn_like(x))
        want = ops.rotary(x, pos, freq, axis)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_empty(dev):
    freq, _ = ops.rotary_frequencies(64, device=dev)
    pos = torch.zeros(1, 0, dtype=torch.int32, device=dev)
    assert ops.rotary(torch.empty(3, 0, 64, device=dev), pos, freq).shape == (3, 0, 64)


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("B,S,H,D,R,axes", [
    (2, 33001, 1, 128, 128, 1), (2, 8003, 3, 128, 64, 2), (2, 1003, 40, 128, 128, 3), (3, 9001, 5, 7, 6, 1),
    (2, 4101, 1, 1024, 1024, 2), (5, 701, 8, 256, 128, 1)])
def test_large(dev, B, S, H, D, R, axes, pairing):
    """Enough work for several tokens a block: numbers of tokens that do not divide
    by a block's, so that blocks cross from one batch to the next and the last is
    ragged; out of place from a fused projection, and in place."""
    case(f"rotary {B}x{H}x{S}x{D} R={R} {pairing}")
    g = torch.Generator(dev).manual_seed(S)
    freq, axis = ops.rotary_frequencies(R, None if axes == 1 else (R // 2 - axes + 1,) + (1,) * (axes - 1), device=dev)
    pos = torch.randint(0, 5000, (axes, B, S), generator=g, device=dev).to(torch.int32)
    x = torch.randn(B, S, H + 1, D, generator=g, device=dev).to(bf16)[:, :, :H].transpose(1, 2)
    a = pos.double()[axis.long()] if axis is not None else pos.double().expand(R // 2, B, S)
    a = (a * freq[:, None, None]).permute(1, 2, 0)[:, None]
    i = torch.arange(R // 2, device=dev) * (1 if pairing == "half" else 2)
    j = i + (R // 2 if pairing == "half" else 1)
    u, v = x[..., i].double(), x[..., j].double()
    want, bound = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=dev)
    want[..., i], want[..., j] = u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()
    # as rotary_bound; the angle here, of up to 5000 radians, is 2^-40 off
    bound[..., i] = bound[..., j] = (u.abs() + v.abs()) * (3 * 2.0**-23 + 3 * F32 + 2.0**-40)

    def check(y, step):
        assert ((y.double() - want).abs() <= 1.01 * (bound + step * (want.abs() + bound))).all()
        assert torch.equal(y[..., R:], x[..., R:].to(y.dtype))

    y = ops.rotary(x, pos, freq, axis, pairing=pairing)
    check(y, BF16)
    check(ops.rotary(x, pos, freq, axis, pairing=pairing, dtype=f32), F32)
    kept = x.clone(memory_format=torch.preserve_format)
    ops.rotary(kept, pos, freq, axis, pairing=pairing, out=kept)
    assert torch.equal(kept, y)
