"""GPU test of a training step's row operators together, as they are used: two
sublayers' dropout, addition and layer norm around a product, an output layer,
policy log probabilities with entropy, and all of it backwards, against autograd in
64 bits on the CPU over the same masks."""
import numpy as np
import pytest
import torch

from jules_amd import ops
from tests.helpers import case
from tests.training64 import kept, threshold

pytestmark = pytest.mark.gpu

RNG = (4242, 10)


def _step(w, x, tokens, advantage, rng, p, eps=1e-5):
    """One step's loss and gradients through the framework's operators, fp32."""
    g = {}
    e = ops.dropout(x, p, rng, offset=0)
    y1, h1, m1, s1 = ops.add_layernorm(e, None, w["g1"], w["b1"], eps)
    a = ops.gemm_bias_act(y1, w["W1"])
    y2, h2, m2, s2 = ops.add_layernorm(a, h1, w["g2"], w["b2"], eps, p=p, rng=rng, offset=1)
    logits = ops.gemm_bias_act(y2, w["W2"])
    vocab = logits.shape[1] - 3  # the output layer is padded to a round width
    o = ops.token_logprobs(logits[:, :vocab], tokens, scale=0.9, top=3)
    loss = -(advantage * o.logp).sum() - 0.01 * o.entropy.sum()

    dlogits = torch.zeros_like(logits)
    ops.token_logprobs_bwd(logits[:, :vocab], tokens, o.lse, -advantage, o.entropy, torch.full_like(advantage, -0.01), scale=0.9,
                           out=dlogits[:, :vocab])
    g["W2"] = ops.gemm_bias_act(y2.t().contiguous(), dlogits)
    dy2 = ops.gemm_bias_act(dlogits, w["W2"].t().contiguous())
    da, dh1, g["g2"], g["b2"] = ops.add_layernorm_bwd(dy2, h2, m2, s2, w["g2"], p=p, rng=rng, offset=1)
    g["W1"] = ops.gemm_bias_act(y1.t().contiguous(), da)
    dy1 = ops.gemm_bias_act(da, w["W1"].t().contiguous())
    de, _, g["g1"], g["b1"] = ops.add_layernorm_bwd(dy1, h1, m1, s1, w["g1"], dh=dh1)
    g["x"] = ops.dropout(de, p, rng, offset=0)
    return loss, o, g


def _step64(w, x, tokens, advantage, p, at, eps=1e-5):
    w = {k: v.double().cpu().requires_grad_() for k, v in w.items()}
    x = x.double().cpu().requires_grad_()
    M, N = x.shape
    f = 65536 / (65536 - threshold(p))

    def mask(offset):
        return torch.from_numpy(kept(M, N, p, (RNG[0], at), offset) * f)

    def norm(h, g, b):
        d = h - h.mean(-1, keepdim=True)
        return d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * g + b

    h1 = x * mask(0)
    h2 = h1 + (norm(h1, w["g1"], w["b1"]) @ w["W1"]) * mask(1)
    logits = (norm(h2, w["g2"], w["b2"]) @ w["W2"])[:, :-3] * 0.9
    log = torch.log_softmax(logits, -1)
    logp = log.gather(1, tokens.cpu().long()[:, None])[:, 0]
    entropy = -(log.exp() * log).sum(-1)
    loss = -(advantage.cpu().double() * logp).sum() - 0.01 * entropy.sum()
    loss.backward()
    return loss, logp, {k: v.grad for k, v in (*w.items(), ("x", x))}


def _operands(dev, M=96, N=200, V=643):
    g = torch.Generator().manual_seed(3)

    def normal(*s, scale=1.0):
        return (scale * torch.randn(*s, generator=g)).to(dev)

    w = dict(W1=normal(N, N, scale=N**-0.5), W2=normal(N, V, scale=N**-0.5), g1=1 + normal(N, scale=0.2), b1=normal(N, scale=0.1),
             g2=1 + normal(N, scale=0.2), b2=normal(N, scale=0.1))
    tokens = torch.randint(0, V - 3, (M,), generator=g, dtype=torch.int32).to(dev)
    return w, normal(M, N), tokens, normal(M) / M


def _near(got, want):
    """fp32 of chains of products 200 to 640 deep: each about 2^-24 sqrt(depth) of its norm, and the
    norms' and softmax's gradients take differences of such sums; 2^-24 * 640 bounds one product's
    chain against its terms' norm, of which the longest path here has five."""
    far = (got.double().cpu() - want).norm() / want.norm()
    assert far <= 5 * 640 * 2.0**-24, far


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
def test_step(dev, p):
    case(f"training step p={p}")
    w, x, tokens, advantage = _operands(dev)
    rng = torch.tensor(RNG, dtype=torch.int64, device=dev)
    loss, o, g = _step(w, x, tokens, advantage, rng, p)
    loss64, logp, want = _step64(w, x, tokens, advantage, p, RNG[1])
    _near(o.logp, logp.detach())
    assert abs(loss.item() - loss64.item()) <= 5 * 640 * 2.0**-24 * (advantage.double().abs().sum().item() * 20 + 10)
    assert set(g) == set(want)
    for k in want:
        _near(g[k], want[k])


def test_step_in_a_graph(dev):
    """The step captured, replayed with the position moved on, eager steps between the replays."""
    w, x, tokens, advantage = _operands(dev)
    rng = torch.tensor(RNG, dtype=torch.int64, device=dev)

    def run():
        _, o, g = _step(w, x, tokens, advantage, rng, 0.1)
        return [*o, *g.values()]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        rng[1] += 2
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert not np.array_equal(kept(4, 40, 0.1, (RNG[0], RNG[1] + 2), 0), kept(4, 40, 0.1, (RNG[0], RNG[1] + 4), 0))
