"""CPU tests of dropout, layer norm with gradients and token log probabilities: the
generator against its published vectors, the statuses of the C ABI, and the
ValueErrors of the torch front end.  Every call here is refused, or has nothing to
do, before a device is touched."""
import numpy as np
import pytest
import torch

from jules_amd import _lib, ops
from tests.training64 import philox

OK, NULL, SHAPE, DTYPE, ALIGN, ACT, WS, HIP, UNSUP, NOTFOUND, ARG = range(11)
P = 0x10000  # a non-null, aligned address that is never dereferenced
F32, BF16 = 0, 1
f32, bf16, i32, i64 = torch.float32, torch.bfloat16, torch.int32, torch.int64
NAN, INF = float("nan"), float("inf")


def _raises(fn, *args, match, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_generator_vectors():
    """The known answers that come with the generator's paper (philox4x32, 10 rounds)."""
    for c, k, want in (((0,) * 4, (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                       ((2**32 - 1,) * 4, (2**32 - 1,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                       ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                        "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join("%08x" % v for v in philox(c, k)) == want


# ---- C ABI ---------------------------------------------------------------------


@pytest.mark.parametrize("change,status", [
    (dict(x_dtype=2), DTYPE), (dict(out_dtype=3), DTYPE), (dict(M=-1), SHAPE), (dict(N=-1), SHAPE), (dict(M=1 << 21, N=1 << 21), SHAPE),
    (dict(p=-0.1), ARG), (dict(p=1.0), ARG), (dict(p=NAN), ARG), (dict(p=1.0 - 2.0**-18), ARG),
    (dict(rng=None), NULL), (dict(x=None), NULL), (dict(out=None), NULL), (dict(rng=P + 4), ALIGN), (dict(x=P + 2), ALIGN),
    (dict(out=P + 1), ALIGN), (dict(res=P + 1), ALIGN), (dict(M=0, x=None, out=None, rng=None), OK), (dict(N=0, x=None), OK),
    (dict(out=P), ARG),  # in place with another dtype
])
def test_dropout_statuses(change, status):
    a = dict(x_dtype=F32, out_dtype=BF16, p=0.1, rng=P, offset=0, x=P, res=2 * P, out=3 * P, M=4, N=8)
    a.update(change)
    assert _lib.lib().jules_hip_dropout(*a.values(), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_dtype=2), DTYPE), (dict(h_dtype=2), DTYPE), (dict(out_dtype=-1), DTYPE), (dict(M=-1), SHAPE), (dict(M=1 << 21, N=1 << 21), SHAPE),
    (dict(eps=-1.0), ARG), (dict(eps=NAN), ARG), (dict(eps=INF), ARG), (dict(p=1.0), ARG), (dict(p=NAN), ARG),
    (dict(rng=None), NULL), (dict(x=None), NULL), (dict(out=None), NULL), (dict(x=P + 2), ALIGN), (dict(res=P + 1), ALIGN),
    (dict(h=P + 1), ALIGN), (dict(gamma=P + 2), ALIGN), (dict(beta=P + 1), ALIGN), (dict(mean=P + 2), ALIGN), (dict(rstd=P + 2), ALIGN),
    (dict(out=P + 1), ALIGN), (dict(rng=P + 4), ALIGN), (dict(M=0, x=None), OK), (dict(N=0, out=None), OK),
    (dict(h=P), ARG), (dict(out=P, out_dtype=BF16), ARG),  # in place with another dtype
    (dict(out=3 * P), ARG), (dict(out=2 * P, out_dtype=BF16), ARG),  # out is h, or the residual
])
def test_add_layernorm_statuses(change, status):
    a = dict(x_dtype=F32, h_dtype=BF16, out_dtype=F32, p=0.1, rng=P, offset=0, x=P, res=2 * P, gamma=P, beta=P, h=3 * P, out=4 * P, mean=P, rstd=P,
             M=4, N=8, eps=1e-5)
    a.update(change)
    assert _lib.lib().jules_hip_add_layernorm(*a.values(), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_dtype=2), DTYPE), (dict(h_dtype=2), DTYPE), (dict(M=-1), SHAPE), (dict(M=1 << 21, N=1 << 21), SHAPE), (dict(p=1.5), ARG),
    (dict(rng=None), NULL), (dict(dy=None), NULL), (dict(h=None), NULL), (dict(mean=None), NULL), (dict(rstd=None), NULL),
    (dict(dy=P + 2), ALIGN), (dict(h=P + 1), ALIGN), (dict(dh=P + 1), ALIGN), (dict(dx=P + 2), ALIGN), (dict(dr=P + 1), ALIGN),
    (dict(dgamma=P + 2), ALIGN), (dict(dbeta=P + 2), ALIGN), (dict(gamma=P + 2), ALIGN), (dict(ws=P + 2), ALIGN),
    (dict(ws=None), WS), (dict(ws_bytes=255), WS), (dict(N=0, dy=None), OK),
    (dict(dx=2 * P), ARG), (dict(dx=3 * P), ARG), (dict(dx=5 * P), ARG), (dict(dr=2 * P), ARG), (dict(dr=P), ARG), (dict(dbeta=6 * P), ARG),
])
def test_add_layernorm_bwd_statuses(change, status):
    a = dict(x_dtype=F32, h_dtype=BF16, p=0.1, rng=P, offset=0, dy=P, h=2 * P, dh=3 * P, mean=P, rstd=P, gamma=P, dx=4 * P, dr=5 * P, dgamma=6 * P, dbeta=7 * P,
             M=4000, N=8, ws=P, ws_bytes=1 << 20)
    a.update(change)
    if "ws_bytes" in change:
        a["ws_bytes"] = _lib.lib().jules_hip_add_layernorm_bwd_workspace_size(a["M"], a["N"]) - 1
    assert _lib.lib().jules_hip_add_layernorm_bwd(*a.values(), None) == status


def test_layernorm_workspace_size():
    f = _lib.lib().jules_hip_add_layernorm_bwd_workspace_size
    for M, N in ((1, 1), (7, 64), (64, 1024), (512, 16384), (2048, 512)):  # few rows
        assert f(M, N) == 0
    for M, N in ((513, 2048), (2049, 1), (64, 16385), (32768, 4096), (1 << 20, 128), (5000, 16384), (5000, 100000)):
        assert 8 * N <= f(M, N) <= 8 * 1024 * N
    assert f(0, 8) == 0 and f(8, 0) == 0 and f(-1, 8) == 0 and f(1 << 21, 1 << 21) == 0


_LOGPROB = [(dict(dtype=2), DTYPE), (dict(M=-1), SHAPE), (dict(N=0), SHAPE), (dict(N=(1 << 21) + 1, stride=1 << 23), SHAPE),
            (dict(M=1 << 30, N=1 << 20, stride=1 << 20), SHAPE), (dict(stride=99), ARG), (dict(stride=1 << 41), ARG), (dict(stride=-100), ARG),
            (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=NAN), ARG), (dict(scale=INF), ARG), (dict(logits=None), NULL),
            (dict(tokens=None), NULL), (dict(logits=P + 1), ALIGN), (dict(tokens=P + 2), ALIGN), (dict(lse=P + 2), ALIGN),
            (dict(entropy=P + 1), ALIGN), (dict(M=0, logits=None), OK)]


@pytest.mark.parametrize("change,status", _LOGPROB + [
    (dict(top=-1), ARG), (dict(top=65), ARG), (dict(N=3, stride=3), ARG), (dict(ids=None), NULL), (dict(top_logp=None), NULL),
    (dict(ids=P + 2), ALIGN), (dict(top_logp=P + 2), ALIGN), (dict(logp=P + 2), ALIGN),
    (dict(N=100000, stride=100000, ws=None), WS), (dict(N=100000, stride=100000, ws_bytes=15), WS), (dict(N=100000, stride=100000, ws=P + 4), ALIGN)])
def test_token_logprobs_statuses(change, status):
    a = dict(dtype=BF16, logits=P, stride=100, scale=1.0, tokens=P, logp=P, lse=P, entropy=P, top=4, ids=P, top_logp=P, M=8, N=100, ws=P,
             ws_bytes=1 << 20)
    a.update(change)
    assert _lib.lib().jules_hip_token_logprobs(*a.values(), None) == status


@pytest.mark.parametrize("change,status", _LOGPROB + [
    (dict(lse=None), NULL), (dict(dlogp=None), NULL), (dict(out=None), NULL), (dict(entropy=None), NULL), (dict(out=P + 1), ALIGN),
    (dict(dlogp=P + 2), ALIGN), (dict(dentropy=P + 2), ALIGN), (dict(out_stride=99), ARG), (dict(out=P, out_stride=101), ARG)])
def test_token_logprobs_bwd_statuses(change, status):
    a = dict(dtype=BF16, logits=P, stride=100, scale=1.0, tokens=P, lse=P, entropy=P, dlogp=P, dentropy=P, out=2 * P, out_stride=100, M=8, N=100)
    a.update(change)
    if "stride" in change and "out_stride" not in change and status == SHAPE:
        a["out_stride"] = a["stride"]
    assert _lib.lib().jules_hip_token_logprobs_bwd(*a.values(), None) == status


def test_logprobs_workspace_size():
    f = _lib.lib().jules_hip_token_logprobs_workspace_size
    assert f(4096, 50257, 20) == 0            # a block a row
    assert f(4096, 128256, 0) == 0 and f(4096, 128256, 20) == 0
    assert f(1, 128256, 20) > 0 and f(8, 128256, 0) > 0 and f(4096, 400000, 64) > 0
    assert f(8, 1000, 5) == 0
    for bad in ((0, 100, 1), (1, 0, 1), (1, (1 << 21) + 1, 1), (1, 100000, 65), (1, 100000, -1), (-1, 100000, 1)):
        assert f(*bad) == 0


# ---- torch front end --------------------------------------------------------------


def test_dropout_refusals():
    x, rng = torch.zeros(4, 8), torch.zeros(2, dtype=i64)
    _raises(ops.dropout, x, 0.1, rng, match="GPU tensor")
    _raises(ops.dropout, x, 0.1, match="rng")
    _raises(ops.dropout, x, 0.1, torch.zeros(3, dtype=i64), match="elements")
    _raises(ops.dropout, x, 0.1, torch.zeros(2), match="dtype")
    for p in (-0.1, 1.0, NAN, 2.0):
        _raises(ops.dropout, x, p, rng, match="p ")
    for offset in (-1, 2**64):
        _raises(ops.dropout, x, 0.1, rng, offset=offset, match="offset")
    _raises(ops.dropout, x.half(), 0.1, rng, match="dtype")
    _raises(ops.dropout, x.t(), 0.1, rng, match="contiguous")
    _raises(ops.dropout, x, 0.1, rng, residual=torch.zeros(4, 9), match="shape")
    _raises(ops.dropout, x, 0.1, rng, residual=x, dtype=bf16, match="dtype")
    _raises(ops.dropout, x, 0.1, rng, dtype=i32, match="dtype")
    _raises(ops.dropout, x, 0.1, rng, dtype=bf16, out=x, match="dtype")
    _raises(ops.dropout, x, 0.1, rng, out=torch.zeros(8, 4), match="shape")


def test_add_layernorm_refusals():
    x, g, rng = torch.zeros(4, 8), torch.zeros(8), torch.zeros(2, dtype=i64)
    _raises(ops.add_layernorm, x, match="GPU tensor")
    _raises(ops.add_layernorm, x.half(), match="dtype")
    _raises(ops.add_layernorm, x.t(), match="contiguous")
    _raises(ops.add_layernorm, x, x.bfloat16()[:2], match="shape")
    _raises(ops.add_layernorm, x, x, g[:7], match="elements")
    _raises(ops.add_layernorm, x, x, g, g.bfloat16(), match="dtype")
    _raises(ops.add_layernorm, x, p=0.5, match="rng")
    _raises(ops.add_layernorm, x, x, h=x.bfloat16(), match="dtype")
    _raises(ops.add_layernorm, x, x, out=torch.zeros(8, 4), match="shape")
    _raises(ops.add_layernorm, x, x, mean=torch.zeros(5), match="elements")
    _raises(ops.add_layernorm, x, x, rstd=torch.zeros(4, dtype=bf16), match="dtype")
    m = torch.zeros(4)
    f = ops.add_layernorm_bwd
    _raises(f, x, x, m, m, match="GPU tensor")
    _raises(f, x, x[:3], m, m, match="shape")
    _raises(f, x, x, m[:3], m, match="elements")
    _raises(f, x, x, m, m.double(), match="dtype")
    _raises(f, x, x, m, m, g[:7], match="elements")
    _raises(f, x, x, m, m, g, dh=x.bfloat16(), match="dtype")
    _raises(f, x, x, m, m, g, dx=x.bfloat16(), match="dtype")
    _raises(f, x, x, m, m, g, dresidual=torch.zeros(8, 4), match="shape")
    _raises(f, x, x, m, m, g, dgamma=g[:7], match="elements")
    _raises(f, x, x, m, m, g, dbeta=g, weight_grads=False, match="weight_grads")
    _raises(f, x, x, m, m, g, p=0.1, match="rng")
    _raises(f, x, x, m, m, g, p=0.1, rng=rng[:1], match="elements")
    _raises(f, x, x, m, m, g, workspace=torch.zeros(8, 4).t(), match="workspace")


def test_token_logprobs_refusals():
    x, t, v = torch.zeros(4, 8), torch.zeros(4, dtype=i32), torch.zeros(4)
    f = ops.token_logprobs
    _raises(f, x, t, match="GPU tensor")
    _raises(f, x.half(), t, match="fp32 or bf16")
    _raises(f, torch.zeros(()), t, match="dimension")
    _raises(f, x.t(), t, match="last stride")
    _raises(f, torch.zeros(4, 16)[:, ::2], t, match="last stride")
    _raises(f, torch.zeros(1, 8).expand(4, 8), t, match="overlap")
    _raises(f, torch.zeros(3, 4, 8)[:, :2], torch.zeros(6, dtype=i32), match="equally far")
    _raises(f, x, t.long(), match="dtype")
    _raises(f, x, t[:3], match="elements")
    for top in (-1, 9, 65):
        _raises(f, x, t, top=top, match="top")
    o = ops.TokenLogprobs
    _raises(f, x, None, out=o(logp=v), match="without tokens")
    _raises(f, x, t, out=o(lse=v[:3]), match="elements")
    _raises(f, x, t, top=2, out=o(lse=v), match="top_ids")
    _raises(f, x, t, out=o(top_ids=t), match="top is 0")
    _raises(f, x, t, top=2, out=o(top_ids=torch.zeros(4, 2, dtype=i32), top_logp=torch.zeros(4, 3)), match="elements")
    f = ops.token_logprobs_bwd
    _raises(f, x, t, v, v, match="GPU tensor")
    _raises(f, x, t, v[:3], v, match="elements")
    _raises(f, x, t, v, v.double(), match="dtype")
    _raises(f, x, t, v, v, dentropy=v, match="entropy")
    _raises(f, x, t, v, v, entropy=v, dentropy=v[:2], match="elements")
    _raises(f, x, t, v, v, out=x.bfloat16(), match="out")
    _raises(f, x, t, v, v, out=torch.zeros(4, 9), match="out")
    _raises(f, x, t, v, v, out=x.t().contiguous().t(), match="last stride")


def test_row_strides():
    s = ops._row_stride
    assert s(torch.zeros(4, 8), "x") == 8 and s(torch.zeros(4, 9)[:, :8], "x") == 9 and s(torch.zeros(2, 3, 9)[..., :8], "x") == 9
    assert s(torch.zeros(2, 1, 9)[..., :8], "x") == 9 and s(torch.zeros(1, 9)[:, :8], "x") == 8 and s(torch.zeros(6, 8)[::2], "x") == 16
    assert s(torch.zeros(8), "x") == 8 and s(torch.zeros(5, 1), "x") == 1 and s(torch.zeros(4, 2)[:, :1], "x") == 2


@pytest.mark.parametrize("shape", [(2**32 + 8,), (2**31,), (2**31, 1), (2**32 + 5, 2)])
def test_sizes_past_32_bits(shape):
    """More rows, or elements a row, than the C ABI's int holds are refused, not cut off."""
    x, rng = torch.empty(shape, dtype=bf16, device="meta"), torch.empty(2, dtype=i64, device="meta")
    rows = torch.empty(shape[:-1], device="meta")
    _raises(ops.dropout, x, 0.5, rng, match="32 bits")
    _raises(ops.dropout, x, 0.0, match="32 bits")
    _raises(ops.add_layernorm, x, match="32 bits")
    _raises(ops.add_layernorm_bwd, x, x, rows, rows, match="32 bits")
    _raises(ops.token_logprobs, x, match="32 bits")
    _raises(ops.token_logprobs_bwd, x, rows, rows, rows, match="32 bits")
    _raises(ops.add_rmsnorm, x, None, rows, match="32 bits")
    M, N = (1, *shape) if len(shape) == 1 else shape
    _raises(ops.add_layernorm_bwd_workspace, M, N, "cpu", match="32 bits")
    _raises(ops.token_logprobs_workspace, M, N, 0, "cpu", match="32 bits")


def test_rows_of_no_elements():
    """They have no mean to return; without rows there is nothing to return."""
    for x in (torch.zeros(3, 0), torch.zeros(2, 3, 0, dtype=bf16)):
        _raises(ops.add_layernorm, x, match="no elements")
        _raises(ops.add_layernorm, x, x, match="no elements")
    _raises(ops.add_layernorm, torch.zeros(0, 8), match="GPU tensor")


@pytest.mark.parametrize("N", [65536, 128256, 1 << 20])
def test_which_rows_are_split(N):
    """For the chip's sake, up to 512 of 65536 elements and more."""
    f = _lib.lib().jules_hip_token_logprobs_workspace_size
    for M in (1, 64, 511, 512):
        assert f(M, N, 0) > 0, M
    for M in (513, 768, 1023, 1024, 5000):
        assert f(M, N, 0) == 0, M
    assert f(512, 65535, 0) == 0 and f(1, 65535, 1) == 0
