"""GPU tests of jules_hip_token_logprobs and jules_hip_token_logprobs_bwd
(ops.token_logprobs, ops.token_logprobs_bwd) against the formulas in 64 bits: every
row length's kernel and its borders, rows split over blocks, padded rows at any
address, both types, masks that leave some, one and no element, equal logits,
alternatives that lie together, NaN and infinities, tokens that are none, in place,
differences, other streams and a replayed graph."""
import numpy as np
import pytest
import torch

from jules_amd import ops
from tests.decoder64 import f64
from tests.helpers import case
from tests.training64 import SLACK, logprobs64, logprobs_bwd64, step, top64

pytestmark = pytest.mark.gpu

f32, bf16, i32 = torch.float32, torch.bfloat16, torch.int32
INF = float("inf")
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 500, 2047, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769, 50257, 65536, 65537,
          128256, 200001]


def _logits(dev, M, N, dtype, seed=0, shift=0, pad=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(M * (N + pad) + shift, dtype=dtype, device=dev)
    flat[shift:] = (scale * torch.randn(M * (N + pad), generator=g)).to(dev)
    return flat[shift:].view(M, N + pad)[:, :N]


def _tokens(dev, M, N, seed=0):
    return torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(seed), dtype=i32).to(dev)


def _normal(dev, M, seed=0):
    return torch.randn(M, generator=torch.Generator().manual_seed(seed + 500)).to(dev)


@np.errstate(invalid="ignore")  # -infinity less itself, in places that are compared apart
def _check(x, tokens, scale, out, top):
    want = logprobs64(x, tokens, scale)
    rows = ~want["none"]
    for name in ("lse", "entropy"):
        got, w = f64(getattr(out, name)).reshape(-1), want[name]
        assert (np.abs(got - w)[rows] <= want["e_" + name][rows]).all(), name
        assert (got[~rows] == w[~rows]).all(), name
    finite = np.isfinite(want["logp"])
    got = f64(out.logp).reshape(-1)
    assert (np.abs(got - want["logp"])[finite] <= want["e_logp"][finite]).all()
    assert (got[~finite] == want["logp"][~finite]).all()
    if top:
        ids = top64(x, top)
        assert (out.top_ids.cpu().numpy().reshape(ids.shape) == ids).all()
        at = np.arange(len(ids))[:, None], ids
        got, w, e = f64(out.top_logp).reshape(ids.shape), want["log"][at], want["e_log"][at]
        finite = np.isfinite(w)
        assert (np.abs(got - w)[finite] <= e[finite]).all() and (got[~finite] == w[~finite]).all()


@pytest.mark.parametrize("N", WIDTHS)
def test_widths(dev, N):
    for M, t, top, scale, pad, shift in ((3, f32, 5, 1.0, 0, 0), (5, bf16, 20, 0.7, 3, 1), (300, bf16, 0, 1.0, 0, 0),
                                         (2, f32, 64, 1.3, 5, 3), (260, f32, 2, 1.0, 0, 1), (1, bf16, 1, 2.0, 0, 0)):
        if M * N > 20_000_000:
            continue
        top = min(top, N)
        case(f"token_logprobs {M}x{N} {t} top {top} scale {scale} pad {pad} shift {shift}")
        x, tokens = _logits(dev, M, N, t, N, shift, pad), _tokens(dev, M, N)
        out = ops.token_logprobs(x, tokens, scale=scale, top=top)
        torch.cuda.synchronize()
        assert (out.top_ids is None) == (top == 0)
        _check(x, tokens, scale, out, top)


@pytest.mark.parametrize("N", [70, 3000, 9000, 20000, 50257, 131072])
@pytest.mark.parametrize("M", [2, 257])
def test_equal_logits(dev, M, N):
    """All equal, and few values: the lowest indices come first, however many are equal."""
    if M * N > 13_000_000:
        M = 40
    tokens = _tokens(dev, M, N)
    for fill in (lambda x: x.fill_(2.5), lambda x: x.fill_(-0.0), lambda x: x.copy_(torch.round(x / 4) * 0.0),
                 lambda x: x.copy_(torch.round(x / 4)), lambda x: x.copy_(torch.where(x > 0, 0.0, -torch.finfo(f32).max))):
        x = _logits(dev, M, N, f32, 3)
        fill(x)
        for top in (1, 20, 64):
            _check(x, tokens, 1.0, ops.token_logprobs(x, tokens, top=top), top)


@pytest.mark.parametrize("N,split", [(300, False), (16384, False), (50257, False), (65536, True), (128256, True)])
def test_alternatives_that_lie_together(dev, N, split):
    """The largest of a row side by side, far apart, rising, falling, all of one thread's."""
    M = 260 if not split else 4
    x = _logits(dev, M, N, f32, 5, scale=1.0)
    for i in range(M):
        if i % 5 == 0:
            at = torch.arange(min(N, 512)) + (i * 37) % max(1, N - 512)
        elif i % 5 == 1:
            at = torch.arange(0, N, max(1, N // 70))[:70]
        elif i % 5 == 2:  # pieces of 8 every 8 * 256 and 8 * 1024 elements
            at = (torch.arange(0, N, 8 * (256 if i % 2 else 1024))[:, None] + torch.arange(8)).reshape(-1)
            at = at[at < N]
        elif i % 5 == 3:
            at = torch.arange(N)
        else:
            at = torch.arange(N - 1, -1, -1)
        x[i, at.to(dev)] = torch.linspace(5.0, 9.0, len(at), device=dev)
    tokens = _tokens(dev, M, N)
    for top in (1, 7, 64):
        case(f"alternatives together {M}x{N} top {top}")
        _check(x, tokens, 1.0, ops.token_logprobs(x, tokens, top=top), top)


@pytest.mark.parametrize("N", [9, 1000, 9000, 50257, 128256])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_masked(dev, N, dtype):
    """What a mask leaves: some, few, one, nothing; masks of the type's lowest value; the token masked."""
    M = 9
    x, tokens = _logits(dev, M, N, dtype, 7), _tokens(dev, M, N)
    few = torch.arange(0, N, max(1, N // 5), device=dev)
    x[0, N // 3:] = -INF
    for row, low in ((1, -INF), (2, torch.finfo(dtype).min)):
        keep = x[row, few].clone()
        x[row] = low
        x[row, few] = keep
    x[3] = -INF
    x[3, N - 1] = 1.5
    x[4] = -INF
    x[5] = torch.finfo(dtype).min
    x[6] = -INF
    x[6, 0] = torch.finfo(dtype).min
    x[7, int(tokens[7])] = -INF
    for top in (0, 1, 6):
        out = ops.token_logprobs(x, tokens, top=top)
        torch.cuda.synchronize()
        _check(x, tokens, 1.0, out, top)
    assert out.lse[4] == -INF and out.logp[4] == -INF and out.entropy[4] == 0 and (out.top_logp[4] == -INF).all()
    assert out.entropy[3] == 0 and out.top_logp[3, 0] == 0 and out.entropy[6] == 0 and out.logp[7] == -INF
    g = _normal(dev, M)
    g[4] = float("nan")  # what a loss makes of -infinity
    dx = ops.token_logprobs_bwd(x, tokens, out.lse, g, out.entropy, -g)
    assert torch.equal(dx[4], torch.zeros_like(dx[4]))
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    _check_bwd(x[keep], tokens[keep], out.lse[keep], out.entropy[keep], g[keep], -g[keep], 1.0, dx[keep])


@pytest.mark.parametrize("N", [9, 1000, 9000, 50257])
def test_masked_with_large_gradients(dev, N):
    """What a scaled loss makes of the entropy's gradient: a masked place has none, however large it is."""
    M = 6
    x, tokens = _logits(dev, M, N, f32, 13), _tokens(dev, M, N)
    keep = x[torch.arange(M, device=dev), tokens.long()]
    for low in (-INF, torch.finfo(f32).min, -1e30):
        x[:, N // 2:] = low
        x[torch.arange(M, device=dev), tokens.long()] = keep
        x[5] = -INF
        out = ops.token_logprobs(x, tokens)
        for size in (1e6, 1e9, 1e20, 1e30):
            g, h = size * _normal(dev, M, 1), size * _normal(dev, M, 2)
            dx = ops.token_logprobs_bwd(x, tokens, out.lse, g, out.entropy, h)
            assert torch.isfinite(dx).all() and (dx[x <= -1e30] == 0).all(), (low, size)
            _check_bwd(x, tokens, out.lse, out.entropy, g, h, 1.0, dx)


@pytest.mark.parametrize("N", [9, 1000, 9000, 50257, 128256])
def test_nan_and_infinity(dev, N):
    """A row with one is NaN everywhere, and no other row."""
    M, top = 7, 5
    x, tokens = _logits(dev, M, N, f32, 9), _tokens(dev, M, N)
    x[0, N - 1] = float("nan")
    x[2, N // 2] = INF
    x[4] = float("nan")
    x[5, 0], x[5, 1:] = float("nan"), -INF
    out = ops.token_logprobs(x, tokens, top=top)
    torch.cuda.synchronize()
    for i in (0, 2, 4, 5):
        assert all(torch.isnan(v[i]).all() for v in (out.lse, out.logp, out.entropy, out.top_logp)), i
        assert (out.top_ids[i] == -1).all()
    rows = [1, 3, 6]
    _check(x[rows], tokens[rows], 1.0, ops.TokenLogprobs(*(v[rows] for v in out)), top)
    dx = ops.token_logprobs_bwd(x, tokens, out.lse, torch.ones(M, device=dev))
    assert torch.isnan(dx[[0, 2, 4, 5]]).all() and torch.isfinite(dx[rows]).all()


@pytest.mark.parametrize("N", [50, 5000, 50257, 70000])
def test_tokens_that_are_none(dev, N):
    x = _logits(dev, 5, N, bf16, 2)
    tokens = torch.tensor([-1, -100, N, 2**31 - 1, N - 1], dtype=i32, device=dev)
    out = ops.token_logprobs(x, tokens)
    assert (out.logp[:2] == 0).all() and torch.isnan(out.logp[2:4]).all() and torch.isfinite(out.logp[4])
    assert torch.isfinite(out.lse).all() and torch.isfinite(out.entropy).all()
    g = torch.tensor([float("nan"), 1.0, 1.0, 1.0, 1.0], device=dev)
    h = torch.full((5,), 0.5, device=dev)
    assert torch.equal(ops.token_logprobs_bwd(x, tokens, out.lse, g)[:2], torch.zeros(2, N, dtype=bf16, device=dev))
    dx = ops.token_logprobs_bwd(x, tokens, out.lse, g, out.entropy, h)
    assert torch.isnan(dx[2:4]).all()
    rows = [0, 1, 4]
    _check_bwd(x[rows], tokens[rows], out.lse[rows], out.entropy[rows], torch.nan_to_num(g[rows]), h[rows], 1.0, dx[rows])


@pytest.mark.parametrize("N", [50, 5000, 50257])
def test_padding_rows(dev, N):
    """A negative token takes the log probability's gradient away, whatever it holds, and leaves the
    entropy's: 0 where that is 0, and else what the row has with a dlogp of 0."""
    x = _logits(dev, 4, N, f32, 2)
    x[3, 1] = float("nan")
    tokens = torch.tensor([-1, -7, -(2**31), -1], dtype=i32, device=dev)
    out = ops.token_logprobs(x, tokens, top=2)
    assert (out.logp == 0).all() and (out.top_ids[3] == -1).all() and torch.isnan(out.lse[3]) and torch.isnan(out.entropy[3])
    g = torch.tensor([float("nan"), INF, 3.0, 1.0], device=dev)
    h = torch.tensor([0.0, 0.5, -0.25, 0.0], device=dev)
    dx = ops.token_logprobs_bwd(x, tokens, out.lse, g, out.entropy, h)
    zero = ops.token_logprobs_bwd(x, _tokens(dev, 4, N), out.lse, torch.zeros(4, device=dev), out.entropy, h)
    assert not dx[0].any() and dx[1:3].any() and torch.equal(dx[:3], zero[:3]) and torch.isnan(dx[3]).all()
    assert not ops.token_logprobs_bwd(x, tokens, out.lse, g)[:3].any()


def _check_bwd(x, tokens, lse, entropy, g, h, scale, dx):
    want, bound = logprobs_bwd64(x, tokens, lse, entropy, g, h, scale)
    assert (np.abs(f64(dx) - want) <= bound + SLACK * step(dx.dtype) * np.abs(want) + 2.0**-120).all()


@pytest.mark.parametrize("N", WIDTHS)
def test_backward_widths(dev, N):
    for M, t, more, scale, pad, shift in ((3, f32, True, 1.0, 0, 0), (5, bf16, True, 0.7, 3, 1), (70, bf16, False, 1.0, 0, 0),
                                          (2, f32, False, 1.3, 5, 3)):
        case(f"token_logprobs_bwd {M}x{N} {t} entropy {more} scale {scale} pad {pad} shift {shift}")
        x, tokens = _logits(dev, M, N, t, N, shift, pad), _tokens(dev, M, N)
        g, h = _normal(dev, M, N), _normal(dev, M, N + 1) if more else None
        out = ops.token_logprobs(x, tokens, scale=scale)
        dx = ops.token_logprobs_bwd(x, tokens, out.lse, g, out.entropy, h, scale=scale)
        torch.cuda.synchronize()
        assert dx.dtype == t and dx.is_contiguous()
        _check_bwd(x, tokens, out.lse, out.entropy, g, h, scale, dx)


@pytest.mark.parametrize("N,pad", [(1000, 0), (5001, 7)])
def test_in_place_and_padding(dev, N, pad):
    """dlogits = logits: the same bits, and what lies between the rows is left as it was."""
    x, tokens = _logits(dev, 20, N, bf16, 4, 0, pad), _tokens(dev, 20, N)
    whole = x._base.view(20, N + pad) if pad else x
    out = ops.token_logprobs(x, tokens)
    g = _normal(dev, 20)
    want = ops.token_logprobs_bwd(x, tokens, out.lse, g)
    behind = whole[:, N:].clone()
    assert ops.token_logprobs_bwd(x, tokens, out.lse, g, out=x) is x
    assert torch.equal(x, want) and torch.equal(whole[:, N:], behind)


@pytest.mark.parametrize("N,top", [(2**21, 64), (2**21, 0), (122881, 64), (600001, 33)])
def test_longest_rows(dev, N, top):
    """Rows split by what the keys of many alternatives take."""
    case(f"token_logprobs 3x{N} top {top}")
    x, tokens = _logits(dev, 3, N, bf16, 11, 1), _tokens(dev, 3, N)
    _check(x, tokens, 1.0, ops.token_logprobs(x, tokens, top=top), top)


def test_rows_beyond_the_blocks(dev):
    """More items than the grid takes at once, and rows of one element to a few."""
    for M, N, top in ((1_100_000, 5, 3), (1_050_000, 1, 1)):
        case(f"token_logprobs {M}x{N}")
        x, tokens = _logits(dev, M, N, f32, 1), _tokens(dev, M, N)
        out = ops.token_logprobs(x, tokens, top=top)
        log = torch.log_softmax(x.double(), -1)
        # bounds as in logprobs64 of 5 elements at most 40 apart
        assert ((out.logp.double() - log.gather(1, tokens.long()[:, None])[:, 0]).abs() <= 800 * 2.0**-24).all()
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(out.top_ids.long(), order)
        dx = ops.token_logprobs_bwd(x, tokens, out.lse, torch.ones(M, device=dev))
        want = -torch.exp(log)
        want.scatter_add_(1, tokens.long()[:, None], torch.ones(M, 1, device=dev, dtype=torch.float64))
        assert ((dx.double() - want).abs() <= 1000 * 2.0**-24).all()


def test_offsets_past_32_bits(dev):
    """2.3 * 10^9 elements: the first and the last rows; every other row of them."""
    M, N = 45700, 50257
    case(f"token_logprobs {M}x{N}")
    x = torch.zeros(M, N, dtype=bf16, device=dev)
    rows = torch.tensor([0, 2, M - 4, M - 2], device=dev)
    x[rows] = _logits(dev, 4, N, bf16, 3)
    tokens, g = _tokens(dev, M, N), _normal(dev, M)
    out = ops.token_logprobs(x, tokens, top=5)
    part = lambda o, r: ops.TokenLogprobs(*(v[r] for v in o))  # noqa: E731
    _check(x[rows], tokens[rows], 1.0, part(out, rows), 5)
    half = ops.token_logprobs(x[::2], tokens[::2].contiguous(), top=5)
    assert all(torch.equal(a[::2], b) for a, b in zip(out, half))
    dx = ops.token_logprobs_bwd(x, tokens, out.lse, g)
    _check_bwd(x[rows], tokens[rows], out.lse[rows], None, g[rows], None, 1.0, dx[rows])
    ops.token_logprobs_bwd(x[::2], tokens[::2].contiguous(), half.lse, g[::2].contiguous(), out=x[::2])
    assert torch.equal(x[::2], dx[::2])


def test_leading_dimensions_and_out(dev):
    x = _logits(dev, 12, 600, bf16, 1, 0, 8)
    x3 = x._base.view(3, 4, 608)[..., :600]
    tokens = _tokens(dev, 12, 600)
    a, b = ops.token_logprobs(x, tokens, top=4), ops.token_logprobs(x3, tokens.view(3, 4), top=4)
    assert b.logp.shape == (3, 4) and b.top_ids.shape == (3, 4, 4)
    assert all(torch.equal(u.reshape(-1), v.reshape(-1)) for u, v in zip(a, b))
    one = ops.TokenLogprobs(lse=torch.empty(12, device=dev))
    assert ops.token_logprobs(x, out=one) is one and torch.equal(one.lse, a.lse)
    none = ops.token_logprobs(x, top=2)
    assert none.logp is None and torch.equal(none.top_ids, a.top_ids[:, :2]) and torch.equal(none.entropy, a.entropy)
    row = ops.token_logprobs(x[0], tokens[:1], top=4)
    assert row.logp.shape == () and torch.equal(row.top_ids, a.top_ids[0])
    g = _normal(dev, 12)
    assert torch.equal(ops.token_logprobs_bwd(x3, tokens, a.lse, g).view(12, 600), ops.token_logprobs_bwd(x, tokens, a.lse, g))


def test_outputs_are_tensors_of_their_own(dev):
    """What an autograd function returns of them can be changed in place, and a change of one leaves
    what was saved of another."""
    x, tokens = _logits(dev, 6, 600, f32, 1).requires_grad_(), _tokens(dev, 6, 600)

    class Logprob(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            out = ops.token_logprobs(x, tokens, top=2)
            ctx.save_for_backward(x, out.lse, out.entropy)
            return out.logp, out.entropy

        @staticmethod
        def backward(ctx, g, h):
            x, lse, entropy = ctx.saved_tensors
            return ops.token_logprobs_bwd(x, tokens, lse, g.contiguous(), entropy, h.contiguous())

    logp, entropy = Logprob.apply(x)
    logp.mul_(0.5)  # a mask, say
    (logp.sum() + 2.0 * entropy.sum()).backward()
    o = ops.token_logprobs(x.detach(), tokens)
    assert torch.equal(logp, 0.5 * o.logp)
    want = ops.token_logprobs_bwd(x.detach(), tokens, o.lse, torch.full((6,), 0.5, device=dev), o.entropy, torch.full((6,), 2.0, device=dev))
    assert torch.equal(x.grad, want)
    for out in (ops.token_logprobs(x.detach(), tokens, top=2), ops.token_logprobs(x.detach(), top=2)):
        versions = [t._version for t in out if t is not None]
        out.lse.zero_()
        assert [t._version for t in out if t is not None] == [v + (t is out.lse) for v, t in zip(versions, (t for t in out if t is not None))]
        assert all(t._base is None for t in out if t is not None)


def test_empty(dev):
    out = ops.token_logprobs(torch.empty(0, 9, device=dev), torch.empty(0, dtype=i32, device=dev), top=2)
    assert out.logp.shape == (0,) and out.top_ids.shape == (0, 2)
    e = torch.empty(0, device=dev)
    assert ops.token_logprobs_bwd(torch.empty(0, 9, device=dev), torch.empty(0, dtype=i32, device=dev), e, e).shape == (0, 9)


def test_differences(dev):
    """The gradient against differences of sum(g logp + h entropy): central, steps of 2^-5 along
    unit directions.  Third derivatives of both are below 10 (moments of a distribution
    over unit directions, times distances below 10), so 10 * 12 * 3 * 2^-10 / 6 at most; the
    outputs' bounds over the step."""
    M, N, e = 12, 40, 2.0**-5
    x, tokens = _logits(dev, M, N, f32, 6, scale=1.5), _tokens(dev, M, N)
    g, h = _normal(dev, M, 1), _normal(dev, M, 2)

    def loss(x):
        o = ops.token_logprobs(x, tokens, scale=0.8)
        return (g.double() * o.logp.double() + h.double() * o.entropy.double()).sum().item()

    o = ops.token_logprobs(x, tokens, scale=0.8)
    dx = ops.token_logprobs_bwd(x, tokens, o.lse, g, o.entropy, h, scale=0.8)
    w = logprobs64(x, tokens, 0.8)
    rounding = (f64(g.abs()) * w["e_logp"] + f64(h.abs()) * w["e_entropy"]).sum()
    for k in range(8):
        d = torch.randn(M, N, generator=torch.Generator().manual_seed(10 + k)).to(dev)
        d = d / d.norm()
        slope = (loss(x + e * d) - loss(x - e * d)) / (2 * e)
        assert abs(slope - (dx.double() * d.double()).sum().item()) <= 10 * 12 * 3 * e * e / 6 + 2 * rounding / e


def test_streams_and_graph(dev):
    """Split rows: overlapping calls with workspaces of their own; a graph replayed between eager calls."""
    sets = [(_logits(dev, 4, 100000, f32, i), _tokens(dev, 4, 100000, i)) for i in range(2)]
    want = [ops.token_logprobs(*s, top=9) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    spaces = [ops.token_logprobs_workspace(4, 100000, 9, dev) for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.token_logprobs(*sets[i], top=9, workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))
    x, tokens = sets[0]
    g = torch.ones(4, device=dev)

    def run():
        o = ops.token_logprobs(x, tokens, top=9)
        return (*o, ops.token_logprobs_bwd(x, tokens, o.lse, g, o.entropy, g))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        w = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, w))
