"""torch-tensor front end of the C ABI.

Each function checks every tensor it is given (inputs, outputs, workspaces):
first dtype, contiguity and shape, then, for all of them together, that they
are GPU tensors on one device; only then does it call the corresponding
jules_hip_* entry point on torch's current HIP stream.  The C ABI sees raw
pointers only, so these checks are what keep a wrongly shaped tensor from
becoming an out-of-bounds GPU access.  torch provides device memory and the
stream only; all arithmetic happens in libjules_hip.so.  Names follow the
reference's jules::kernel functions (include/jules/Kernel/FusedKernels.h,
FlashAttention.h).
"""
import ctypes
from typing import NamedTuple, Optional

import numpy as np

import torch

from ._lib import ACT, BF16, F32, I8, JhKV4Cache, check, lib

_DT = {torch.float32: F32, torch.bfloat16: BF16}
_REAL = (torch.float32, torch.bfloat16)


def _stream(t):
    # the raw handle of torch.cuda.current_stream(t.device), without building
    # the Stream object around it
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(t, name, dtypes, shape=None, numel=None):
    """Structural check of one tensor argument: dtype, contiguity and shape
    (or element count).  Raises ValueError."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: {t.numel()} elements, expected {numel}")


def _rank(t, name, rank):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.dim() != rank:
        raise ValueError(f"{name} must have {rank} dimensions, got {t.dim()}")


def _workspace(ws, name):
    """A caller-supplied workspace: any dtype, contiguous; returns its size
    in bytes (the C ABI checks it against what the call needs)."""
    if not isinstance(ws, torch.Tensor) or not ws.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor")
    return ws.numel() * ws.element_size()


def _on_device(**tensors):
    """Every given tensor (None entries skipped) is a GPU tensor on the device
    of the first one; returns that device."""
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a GPU tensor")
        if first is None:
            first, index = t, t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    return None if first is None else first.device


def _act(act):
    return ACT[act] if isinstance(act, str) else int(act)


def gemm_bias_act(A, B, bias=None, act="none", out=None):
    """C = act(A @ B + bias).  fp32 (bit-exact with the reference's fma chain) or
    bf16 (MFMA, fp32 accumulate).  Mirrors tiledMatmulWithActivation /
    fusedMatmulBiasRelu (FusedKernels.h:378, :265)."""
    _rank(A, "A", 2)
    _rank(B, "B", 2)
    _need(A, "A", (torch.float32, torch.bfloat16))
    _need(B, "B", (A.dtype,))
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if bias is not None:
        _need(bias, "bias", (torch.float32,), numel=N)
    if out is not None:
        _need(out, "out", (A.dtype,), shape=(M, N))
    _on_device(A=A, B=B, bias=bias, out=out)
    if out is None:
        out = torch.empty((M, N), dtype=A.dtype, device=A.device)
    check(lib().jules_hip_gemm_bias_act(_DT[A.dtype], _act(act), _ptr(A), _ptr(B), _ptr(bias),
                                        _ptr(out), M, N, K, _stream(A)))
    return out


def activation(x, act="gelu", out=None):
    """out = act(x), fp32; act='gelu' is fusedGelu (FusedKernels.h:606)."""
    _need(x, "x", (torch.float32,))
    if out is not None:
        _need(out, "out", (torch.float32,), numel=x.numel())
    _on_device(x=x, out=out)
    if out is None:
        out = torch.empty_like(x)
    check(lib().jules_hip_activation(_act(act), _ptr(out), _ptr(x), x.numel(), _stream(x)))
    return out


def default_scale(D):
    """1.0f / sqrtf((float)D) evaluated in fp32, as FlashAttention.h:135 does."""
    return float(np.float32(1.0) / np.sqrt(np.float32(D)))


def flash_attention(Q, K, V, causal=False, scale=None, out=None, lse=None):
    """Flash-attention forward, [B,H,S,D]; scale defaults to 1/sqrtf(D) as in
    flashAttention (FlashAttention.h:135)."""
    _rank(Q, "Q", 4)
    _need(Q, "Q", (torch.float32, torch.bfloat16))
    _need(K, "K", (Q.dtype,), shape=Q.shape)
    _need(V, "V", (Q.dtype,), shape=Q.shape)
    B, H, S, D = Q.shape
    if out is not None:
        _need(out, "out", (Q.dtype,), shape=Q.shape)
    if lse is not None:
        _need(lse, "lse", (torch.float32,), numel=B * H * S)
    _on_device(Q=Q, K=K, V=V, out=out, lse=lse)
    if scale is None:
        scale = default_scale(D)
    if out is None:
        out = torch.empty_like(Q)
    check(lib().jules_hip_flash_attn_fwd(_DT[Q.dtype], int(bool(causal)), float(scale), _ptr(Q),
                                         _ptr(K), _ptr(V), _ptr(out), _ptr(lse), B, H, S, D,
                                         _stream(Q)))
    return out


def flash_attention_bwd(Q, K, V, O, dO, lse, causal=False, scale=None, dQ=None, dK=None, dV=None,
                        workspace=None):
    """Flash-attention backward (jules_hip_flash_attn_bwd; no reference
    counterpart): (dQ, dK, dV) for the forward O = flash_attention(Q, K, V,
    causal, scale, lse=lse).  bf16 [B,H,S,D]; lse fp32 [B,H,S]."""
    _rank(Q, "Q", 4)
    _need(Q, "Q", (torch.bfloat16,))
    for t, n in ((K, "K"), (V, "V"), (O, "O"), (dO, "dO")):
        _need(t, n, (Q.dtype,), shape=Q.shape)
    B, H, S, D = Q.shape
    _need(lse, "lse", (torch.float32,), numel=B * H * S)
    for t, n in ((dQ, "dQ"), (dK, "dK"), (dV, "dV")):
        if t is not None:
            _need(t, n, (Q.dtype,), shape=Q.shape)
    ws_bytes = None if workspace is None else _workspace(workspace, "workspace")
    _on_device(Q=Q, K=K, V=V, O=O, dO=dO, lse=lse, dQ=dQ, dK=dK, dV=dV, workspace=workspace)
    if scale is None:
        scale = default_scale(D)
    dQ = torch.empty_like(Q) if dQ is None else dQ
    dK = torch.empty_like(Q) if dK is None else dK
    dV = torch.empty_like(Q) if dV is None else dV
    if workspace is None:
        nbytes = lib().jules_hip_flash_attn_bwd_workspace_size(B, H, S)
        workspace = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=Q.device)
        ws_bytes = workspace.numel()
    check(lib().jules_hip_flash_attn_bwd(_DT[Q.dtype], int(bool(causal)), float(scale), _ptr(Q),
                                         _ptr(K), _ptr(V), _ptr(O), _ptr(dO), _ptr(lse), _ptr(dQ),
                                         _ptr(dK), _ptr(dV), B, H, S, D, _ptr(workspace),
                                         ws_bytes, _stream(Q)))
    return dQ, dK, dV


def w8a16_workspace(M, N, K, device):
    n = lib().jules_hip_w8a16_workspace_size(M, N, K)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def w8a16_gemm(x, W, scale, bias=None, act="silu", out=None, workspace=None):
    """y = act(scale * (x @ W) + bias); x bf16 [M,K], W int8 [K,N]."""
    _rank(x, "x", 2)
    _rank(W, "W", 2)
    _need(x, "x", (torch.bfloat16,))
    _need(W, "W", (torch.int8,))
    M, K = x.shape
    K2, N = W.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    _need(scale, "scale", (torch.float32,), numel=N)
    if bias is not None:
        _need(bias, "bias", (torch.float32,), numel=N)
    if out is not None:
        _need(out, "out", (torch.bfloat16,), shape=(M, N))
    ws_bytes = None if workspace is None else _workspace(workspace, "workspace")
    _on_device(x=x, W=W, scale=scale, bias=bias, out=out, workspace=workspace)
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    if workspace is None:
        workspace = w8a16_workspace(M, N, K, x.device)
        ws_bytes = workspace.numel()
    check(lib().jules_hip_w8a16_gemm_bias_act(_act(act), _ptr(x), _ptr(W), _ptr(scale),
                                              _ptr(bias), _ptr(out), M, N, K, _ptr(workspace),
                                              ws_bytes, _stream(x)))
    return out


class PackedW8:
    """int8 weights [K,N] repacked for jules_hip_w8a16_packed_gemm_bias_act:
    `data` is the packed uint8 array, K and N the logical shape."""

    def __init__(self, data, K, N):
        self.data, self.K, self.N = data, K, N


def w8a16_pack(W):
    """Repack int8 W [K,N] (row-major) into the packed W8A16 layout (done
    once, at weight-load time)."""
    _rank(W, "W", 2)
    _need(W, "W", (torch.int8,))
    _on_device(W=W)
    K, N = W.shape
    n = lib().jules_hip_w8a16_packed_size(K, N)
    if n == 0:
        raise ValueError(f"w8a16_pack: unsupported shape {tuple(W.shape)}")
    Wp = torch.empty((n,), dtype=torch.uint8, device=W.device)
    check(lib().jules_hip_w8a16_pack(_ptr(W), K, N, _ptr(Wp), n, _stream(W)))
    return PackedW8(Wp, K, N)


def w8a16_gemm_packed(x, Wp, scale, bias=None, act="silu", out=None):
    """y = act(scale * (x @ W) + bias) with W given packed (w8a16_pack);
    x bf16 [M,K]."""
    if not isinstance(Wp, PackedW8):
        raise TypeError("Wp must come from w8a16_pack")
    _rank(x, "x", 2)
    _need(x, "x", (torch.bfloat16,))
    M, K = x.shape
    N = Wp.N
    if K != Wp.K:
        raise ValueError("inner dimensions differ")
    _need(Wp.data, "Wp", (torch.uint8,), numel=lib().jules_hip_w8a16_packed_size(K, N))
    _need(scale, "scale", (torch.float32,), numel=N)
    if bias is not None:
        _need(bias, "bias", (torch.float32,), numel=N)
    if out is not None:
        _need(out, "out", (torch.bfloat16,), shape=(M, N))
    _on_device(x=x, Wp=Wp.data, scale=scale, bias=bias, out=out)
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    check(lib().jules_hip_w8a16_packed_gemm_bias_act(_act(act), _ptr(x), _ptr(Wp.data), _ptr(scale),
                                                     _ptr(bias), _ptr(out), M, N, K, _stream(x)))
    return out


def _int8_operands(A, B, bias, out):
    _rank(A, "A", 2)
    _rank(B, "B", 2)
    _need(A, "A", (torch.int8,))
    _need(B, "B", (torch.int8,))
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if bias is not None:
        _need(bias, "bias", (torch.float32,), numel=N)
    if out is not None:
        _need(out, "out", (torch.float32,), shape=(M, N))
    return M, N, K


def matmul_int8(A, B, scale_a, scale_b, bias=None, out=None):
    """matmulInt8 (FusedKernels.h:867) with the scalar path's semantics."""
    M, N, K = _int8_operands(A, B, bias, out)
    _on_device(A=A, B=B, bias=bias, out=out)
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    check(lib().jules_hip_matmul_int8(_ptr(A), _ptr(B), _ptr(out), M, N, K, float(scale_a),
                                      float(scale_b), _ptr(bias), _stream(A)))
    return out


def matmul_w8a8(A, B, scale_a, scale_b, bias=None, out=None):
    """C = float(A @ B) * (scale_a[i] * scale_b[j]) [+ bias] with exact int32
    accumulation (jules_hip_matmul_w8a8): int8 A [M,K], B [K,N], fp32
    per-token scale_a [M] (or None) and per-channel scale_b [N]."""
    M, N, K = _int8_operands(A, B, bias, out)
    if scale_a is not None:
        _need(scale_a, "scale_a", (torch.float32,), numel=M)
    _need(scale_b, "scale_b", (torch.float32,), numel=N)
    _on_device(A=A, B=B, scale_a=scale_a, scale_b=scale_b, bias=bias, out=out)
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    check(lib().jules_hip_matmul_w8a8(_ptr(A), _ptr(B), _ptr(out), M, N, K, _ptr(scale_a),
                                      _ptr(scale_b), _ptr(bias), _stream(A)))
    return out


def _c_int(n, name):
    """A count as the C ABI's int takes it: ctypes would cut a larger one off."""
    n = int(n)
    if not -2**31 <= n < 2**31:
        raise ValueError(f"{name} {n} is not within 32 bits")
    return n


def _rows(x):
    shape = x.shape
    N = shape[-1] if shape else 1
    M = x.numel() // N if N else 0
    if M >= 2**31 or N >= 2**31:
        raise ValueError(f"{M} rows of {N} elements: the number of each must be within 32 bits")
    return M, N


def softmax(x, out=None):
    """fusedSoftmax (FusedKernels.h:464) over the last dimension of fp32 x."""
    _need(x, "x", (torch.float32,))
    if out is not None:
        _need(out, "out", (torch.float32,), shape=x.shape)
    _on_device(x=x, out=out)
    if out is None:
        out = torch.empty_like(x)
    M, N = _rows(x)
    check(lib().jules_hip_softmax(_ptr(out), _ptr(x), M, N, _stream(x)))
    return out


def layernorm(x, gamma, beta, eps=1e-5, out=None):
    """fusedLayerNorm (FusedKernels.h:532) over the last dimension of fp32 x."""
    _need(x, "x", (torch.float32,))
    M, N = _rows(x)
    _need(gamma, "gamma", (torch.float32,), numel=N)
    _need(beta, "beta", (torch.float32,), numel=N)
    if out is not None:
        _need(out, "out", (torch.float32,), shape=x.shape)
    _on_device(x=x, gamma=gamma, beta=beta, out=out)
    if out is None:
        out = torch.empty_like(x)
    check(lib().jules_hip_layernorm(_ptr(out), _ptr(x), _ptr(gamma), _ptr(beta), M, N,
                                    float(eps), _stream(x)))
    return out


def _one_device(names, *tensors):
    """_on_device without a dictionary where all is well: for calls short enough
    that its cost shows."""
    index = tensors[0].get_device()
    if index >= 0:
        for t in tensors:
            if t is not None and t.get_device() != index:
                break
        else:
            return
    _on_device(**dict(zip(names, tensors)))


def _call(t, fn, *args):
    """check(fn(*args, stream)) on t's device and torch's current stream there,
    whichever device is the current one."""
    index = t.get_device()
    if torch._C._cuda_getDevice() == index:
        check(fn(*args, _stream(t)))
    else:
        with torch.cuda.device(index):
            check(fn(*args, _stream(t)))


def _add_rmsnorm(x, residual, weight, eps, out, out_types, scale, residual_out):
    _need(x, "x", _REAL)
    M, N = _rows(x)
    _need(weight, "weight", (torch.float32,), numel=N)
    if residual is not None:
        _need(residual, "residual", _REAL, shape=x.shape)
        if residual_out is not None:
            _need(residual_out, "residual_out", (residual.dtype,), shape=x.shape)
    elif residual_out is not None:
        raise ValueError("residual_out without residual")
    if out is not None:
        _need(out, "out", out_types, shape=x.shape)
    if scale is not None:
        _need(scale, "scale", (torch.float32,), numel=M)
    _one_device(("x", "weight", "residual", "out", "scale", "residual_out"), x, weight, residual, out, scale, residual_out)
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(residual)
    if out is None:
        out = torch.empty_like(x, dtype=out_types[0])
    int8 = out.dtype == torch.int8
    if int8 and scale is None:
        scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _call(x, lib().jules_hip_add_rmsnorm, _DT[x.dtype], F32 if residual is None else _DT[residual.dtype],
          I8 if int8 else _DT[out.dtype], x.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(residual_out),
          out.data_ptr(), _ptr(scale), M, N, float(eps))
    return out, scale, residual_out


def add_rmsnorm(x, residual, weight, eps=1e-5, out=None, residual_out=None):
    """h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight over the last
    dimension (jules_hip_add_rmsnorm; no counterpart in the reference).  x and
    residual fp32 or bf16, each by itself, residual or None; weight fp32.
    Returns (y, h): y of x's dtype (or of out's, fp32 or bf16), h of the
    residual's dtype, None without one.  residual_out may be residual."""
    y, _, h = _add_rmsnorm(x, residual, weight, eps, out, (x.dtype, *_REAL) if isinstance(x, torch.Tensor) else _REAL,
                           None, residual_out)
    return y, h


def add_rmsnorm_int8(x, residual, weight, eps=1e-5, out=None, scale=None, residual_out=None):
    """add_rmsnorm with int8 rows and a scale for each: returns (q, scale, h)
    with y = q * scale to half a step, q and scale being the A and scale_a of
    matmul_w8a8."""
    return _add_rmsnorm(x, residual, weight, eps, out, (torch.int8,), scale, residual_out)


def _drop_args(p, rng, offset):
    """Dropout's p, rng and offset as the C ABI takes them."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"p {p} must be at least 0 and below 1")
    if p > 0.0 or rng is not None:
        _need(rng, "rng", (torch.int64,), numel=2)
    if not 0 <= offset < 2**64:
        raise ValueError(f"offset {offset} must be within 64 bits")
    return p, _ptr(rng), int(offset)


def dropout(x, p, rng=None, offset=0, residual=None, dtype=None, out=None):
    """[residual +] x with each element dropped with probability p and the others
    scaled by 1 / (1 - p) (jules_hip_dropout; no counterpart in the reference).  No
    mask is stored: which elements are dropped follows from their place in
    [M, N] (N the last dimension), p, rng (int64 [2] on the device: seed and position,
    read when the kernel runs) and offset, so the gradient is
    dropout(grad, p, rng, offset) with rng as it was.  p is rounded to a multiple of
    2^-16.  x fp32 or bf16; the result of `dtype` (x's), or of residual's and of
    its shape.  out may be x or residual."""
    _need(x, "x", _REAL)
    M, N = _rows(x)
    p, rng_ptr, offset = _drop_args(p, rng, offset)
    if residual is not None:
        _need(residual, "residual", _REAL if dtype is None else (dtype,), shape=x.shape)
        dtype = residual.dtype
    elif dtype is None:
        dtype = x.dtype if out is None else out.dtype
    if dtype not in _DT:
        raise ValueError(f"dtype {dtype} not in {tuple(_DT)}")
    if out is not None:
        _need(out, "out", (dtype,), shape=x.shape)
    _one_device(("x", "rng", "residual", "out"), x, rng, residual, out)
    if out is None:
        out = torch.empty_like(x, dtype=dtype)
    _call(x, lib().jules_hip_dropout, _DT[x.dtype], _DT[dtype], p, rng_ptr, offset, x.data_ptr(), _ptr(residual), out.data_ptr(),
          M, N)
    return out


def add_layernorm(x, residual=None, gamma=None, beta=None, eps=1e-5, p=0.0, rng=None, offset=0, out=None, h=None, mean=None,
                  rstd=None):
    """h = residual + dropout(x), y = (h - mean(h)) / sqrt(var(h) + eps) * gamma +
    beta over the last dimension (jules_hip_add_layernorm; no counterpart in the
    reference, whose fusedLayerNorm is layernorm above).  x and residual fp32 or bf16, each by
    itself, residual or None; gamma, beta fp32 or None (ones, zeros); p, rng,
    offset: dropout's.  Returns (y, h, mean, rstd), what add_layernorm_bwd takes: y of x's dtype (or of
    out's), h of residual's, or of x's without one (x itself where p is 0 and out is not
    x), mean and rstd fp32.  out may be x, h may be residual."""
    _need(x, "x", _REAL)
    M, N = _rows(x)
    if not N:
        raise ValueError("x: rows of no elements have no mean")
    p, rng_ptr, offset = _drop_args(p, rng, offset)
    if gamma is not None:
        _need(gamma, "gamma", (torch.float32,), numel=N)
    if beta is not None:
        _need(beta, "beta", (torch.float32,), numel=N)
    if residual is not None:
        _need(residual, "residual", _REAL, shape=x.shape)
    if h is not None:
        _need(h, "h", _REAL if residual is None else (residual.dtype,), shape=x.shape)
    if out is not None:
        _need(out, "out", _REAL, shape=x.shape)
    if mean is not None:
        _need(mean, "mean", (torch.float32,), numel=M)
    if rstd is not None:
        _need(rstd, "rstd", (torch.float32,), numel=M)
    _one_device(("x", "residual", "gamma", "beta", "rng", "out", "h", "mean", "rstd"), x, residual, gamma, beta, rng, out, h, mean,
                rstd)
    # without a residual and dropout h is x, unless y takes its place
    if h is None and (residual is not None or p > 0.0 or (out is not None and out.data_ptr() == x.data_ptr())):
        h = torch.empty_like(x if residual is None else residual)
    if out is None:
        out = torch.empty_like(x)
    if mean is None:
        mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    if rstd is None:
        rstd = torch.empty_like(mean)
    _call(x, lib().jules_hip_add_layernorm, _DT[x.dtype], F32 if h is None else _DT[h.dtype], _DT[out.dtype], p, rng_ptr, offset,
          x.data_ptr(), _ptr(residual), _ptr(gamma), _ptr(beta), _ptr(h), out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), M, N,
          float(eps))
    return out, x if h is None else h, mean, rstd


def add_layernorm_bwd_workspace(M, N, device):
    nbytes = lib().jules_hip_add_layernorm_bwd_workspace_size(_c_int(M, "M"), _c_int(N, "N"))
    return torch.empty((max(nbytes, 4) // 4,), dtype=torch.float32, device=device)


def add_layernorm_bwd(dy, h, mean, rstd, gamma=None, dh=None, p=0.0, rng=None, offset=0, dx=None, dresidual=None, dgamma=None,
                      dbeta=None, weight_grads=True, workspace=None):
    """Gradients of add_layernorm (jules_hip_add_layernorm_bwd): dy of y's dtype, h,
    mean and rstd as it returned them, gamma, p, rng (as it was) and offset those
    that it was given, dh (of h's dtype) what reaches h past the norm.  Returns
    (dx, dresidual, dgamma, dbeta): dresidual, of h's dtype, is the gradient of h;
    dx, of dy's, that of x, which is dresidual itself where p is 0, the types are
    the same and neither was passed; dgamma, dbeta fp32 [N], None where
    weight_grads is false.  dx may be dy, dresidual may be dh."""
    _need(dy, "dy", _REAL)
    M, N = _rows(dy)
    _need(h, "h", _REAL, shape=dy.shape)
    _need(mean, "mean", (torch.float32,), numel=M)
    _need(rstd, "rstd", (torch.float32,), numel=M)
    p, rng_ptr, offset = _drop_args(p, rng, offset)
    if gamma is not None:
        _need(gamma, "gamma", (torch.float32,), numel=N)
    if dh is not None:
        _need(dh, "dh", (h.dtype,), shape=h.shape)
    if dx is not None:
        _need(dx, "dx", (dy.dtype,), shape=dy.shape)
    if dresidual is not None:
        _need(dresidual, "dresidual", (h.dtype,), shape=h.shape)
    if not weight_grads and (dgamma is not None or dbeta is not None):
        raise ValueError("dgamma or dbeta without weight_grads")
    if dgamma is not None:
        _need(dgamma, "dgamma", (torch.float32,), numel=N)
    if dbeta is not None:
        _need(dbeta, "dbeta", (torch.float32,), numel=N)
    ws_bytes = 0 if workspace is None else _workspace(workspace, "workspace")
    _one_device(("dy", "h", "mean", "rstd", "gamma", "dh", "rng", "dx", "dresidual", "dgamma", "dbeta", "workspace"), dy, h, mean,
                rstd, gamma, dh, rng, dx, dresidual, dgamma, dbeta, workspace)
    one = p == 0.0 and dy.dtype == h.dtype and dx is None and dresidual is None
    if dresidual is None:
        dresidual = torch.empty_like(h)
    if dx is None and not one:
        dx = torch.empty_like(dy)
    if weight_grads:
        if dgamma is None:
            dgamma = dy.new_empty((N,), dtype=torch.float32)
        if dbeta is None:
            dbeta = torch.empty_like(dgamma)
        if workspace is None:
            ws_bytes = lib().jules_hip_add_layernorm_bwd_workspace_size(M, N)
            if ws_bytes:
                workspace = dy.new_empty((ws_bytes,), dtype=torch.uint8)
    _call(dy, lib().jules_hip_add_layernorm_bwd, _DT[dy.dtype], _DT[h.dtype], p, rng_ptr, offset, dy.data_ptr(), h.data_ptr(), _ptr(dh),
          mean.data_ptr(), rstd.data_ptr(), _ptr(gamma), _ptr(dx), dresidual.data_ptr(), _ptr(dgamma), _ptr(dbeta), M, N,
          _ptr(workspace), ws_bytes)
    return dresidual if one else dx, dresidual, dgamma, dbeta


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns, or writes into."""
    logp: Optional[torch.Tensor] = None
    lse: Optional[torch.Tensor] = None
    entropy: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None
    top_logp: Optional[torch.Tensor] = None


_LOGPROBS_NAMES = ("logits", "tokens", "workspace", *TokenLogprobs._fields)


def _row_stride(t, name):
    """Elements between two rows of a tensor whose last dimension is dense and whose
    others lie as those of a dense one would, rows of a padded width among them."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DT:
        raise ValueError(f"{name}: fp32 or bf16 tensor expected")
    shape = t.shape
    if not shape:
        raise ValueError(f"{name} must have at least one dimension")
    N = shape[-1]
    if t.is_contiguous():
        return N
    if N > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last stride must be 1")
    step = span = None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != span:
            raise ValueError(f"{name}: rows must be equally far apart")
        span = stride * size
    if step is None:
        return N
    if step < N:
        raise ValueError(f"{name}: rows overlap")
    return step


def token_logprobs_workspace(M, N, top, device):
    nbytes = lib().jules_hip_token_logprobs_workspace_size(_c_int(M, "M"), _c_int(N, "N"), _c_int(top, "top"))
    return torch.empty((max(nbytes, 8) // 8 + 1,), dtype=torch.int64, device=device)


def token_logprobs(logits, tokens=None, scale=1.0, top=0, out=None, workspace=None):
    """Log probabilities of `tokens` under softmax(scale * logits) over the last
    dimension, with the log-sum-exp, the entropy and the `top` likeliest tokens of
    each row (jules_hip_token_logprobs; no counterpart in the reference, whose
    fusedCrossEntropyLoss is cross_entropy).  logits fp32 or bf16 [..., N], N up to
    2^21, rows equally far apart (logits[..., :N] of a padded width); tokens
    int32, one a row, a negative one for none (logp 0, the rest as ever), or None; top at most 64.
    Returns TokenLogprobs(logp, lse, entropy, top_ids, top_logp): fp32 of logits' leading shape, the last two
    [..., top] int32 and fp32 (None where top is 0), by falling logit and rising index.  out: a
    TokenLogprobs to write into, whose entries that are None are not wanted."""
    stride = _row_stride(logits, "logits")
    M, N = _rows(logits)
    top = int(top)
    if top < 0 or top > 64 or top > N:
        raise ValueError(f"top {top} must be at most 64 and {N}")
    if tokens is not None:
        _need(tokens, "tokens", (torch.int32,), numel=M)
    if out is not None:
        if out.logp is not None and tokens is None:
            raise ValueError("logp without tokens")
        for name, t in (("logp", out.logp), ("lse", out.lse), ("entropy", out.entropy)):
            if t is not None:
                _need(t, name, (torch.float32,), numel=M)
        if (out.top_ids is not None or out.top_logp is not None) and not top:
            raise ValueError("top_ids or top_logp where top is 0")
        if top:
            _need(out.top_ids, "top_ids", (torch.int32,), numel=M * top)
            _need(out.top_logp, "top_logp", (torch.float32,), numel=M * top)
    ws_bytes = 0 if workspace is None else _workspace(workspace, "workspace")
    _one_device(_LOGPROBS_NAMES, logits, tokens, workspace, *(out or ()))
    if out is None:
        lead = logits.shape[:-1]
        # tensors of their own: views of one would count each other's changes in place, which autograd looks at
        lse = logits.new_empty(lead, dtype=torch.float32)
        top_logp = logits.new_empty((*lead, top), dtype=torch.float32) if top else None
        out = TokenLogprobs(None if tokens is None else torch.empty_like(lse), lse, torch.empty_like(lse),
                            torch.empty_like(top_logp, dtype=torch.int32) if top else None, top_logp)
    if workspace is None:
        ws_bytes = lib().jules_hip_token_logprobs_workspace_size(M, N, top)
        if ws_bytes:
            workspace = logits.new_empty((ws_bytes,), dtype=torch.uint8)
    _call(logits, lib().jules_hip_token_logprobs, _DT[logits.dtype], logits.data_ptr(), stride, float(scale), _ptr(tokens),
          _ptr(out.logp), _ptr(out.lse), _ptr(out.entropy), top, _ptr(out.top_ids), _ptr(out.top_logp), M, N, _ptr(workspace),
          ws_bytes)
    return out


def token_logprobs_bwd(logits, tokens, lse, dlogp, entropy=None, dentropy=None, scale=1.0, out=None):
    """The gradient of token_logprobs' logp and entropy with respect to the logits
    (jules_hip_token_logprobs_bwd), in their dtype: logits, tokens and scale as they were, lse and
    entropy as it returned them, dlogp and dentropy (or None) fp32, one a row.  dlogp is not looked at
    where the token is negative; dentropy is, so that it has to be 0 in a padding row.  out may be logits."""
    stride = _row_stride(logits, "logits")
    M, N = _rows(logits)
    _need(tokens, "tokens", (torch.int32,), numel=M)
    _need(lse, "lse", (torch.float32,), numel=M)
    _need(dlogp, "dlogp", (torch.float32,), numel=M)
    if dentropy is not None:
        _need(dentropy, "dentropy", (torch.float32,), numel=M)
        _need(entropy, "entropy", (torch.float32,), numel=M)
    elif entropy is not None:
        _need(entropy, "entropy", (torch.float32,), numel=M)
    if out is not None:
        out_stride = _row_stride(out, "out")
        if out.shape != logits.shape or out.dtype != logits.dtype:
            raise ValueError(f"out: {out.dtype} {tuple(out.shape)}, expected {logits.dtype} {tuple(logits.shape)}")
    _one_device(("logits", "tokens", "lse", "dlogp", "entropy", "dentropy", "out"), logits, tokens, lse, dlogp, entropy, dentropy, out)
    if out is None:
        out, out_stride = torch.empty_like(logits, memory_format=torch.contiguous_format), N
    _call(logits, lib().jules_hip_token_logprobs_bwd, _DT[logits.dtype], logits.data_ptr(), stride, float(scale), tokens.data_ptr(),
          lse.data_ptr(), _ptr(entropy), dlogp.data_ptr(), _ptr(dentropy), out.data_ptr(), out_stride, M, N)
    return out


def rotary_frequencies(rotary_dim, sections=None, base=10000.0, device="cuda"):
    """(inv_freq fp64 [rotary_dim/2], pair_axis int32 or None) of rotary:
    inv_freq[p] = base^(-2p / rotary_dim).  sections: numbers of pairs of each
    axis, in order (they sum to rotary_dim/2); None for a single axis."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and at least 2")
    pairs = rotary_dim // 2
    p = torch.arange(pairs, dtype=torch.float64)
    inv_freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -p / pairs).to(device)
    if sections is None:
        return inv_freq, None
    if any(n < 0 for n in sections) or sum(sections) != pairs:
        raise ValueError(f"sections {tuple(sections)} must sum to {pairs}")
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(list(sections)))
    return inv_freq, axis.to(torch.int32).to(device)


_PAIRING = {"half": 0, "adjacent": 1}


_I64x3 = ctypes.c_int64 * 3


def _rotary_strides(t, name):
    """Strides of batch, head and token of [B,H,S,D], or of [H,S,D], which is one batch."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DT:
        raise ValueError(f"{name}: fp32 or bf16 tensor expected")
    *outer, last = t.stride()
    if last != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the last stride must be 1")
    return _I64x3(*outer) if len(outer) == 3 else _I64x3(0, *outer)


def rotary(x, positions, inv_freq, pair_axis=None, pairing="half", inverse=False, dtype=None, out=None):
    """Rotary positions of one or several axes (jules_hip_rotary; no counterpart
    in the reference) on x [B,H,S,D] or [H,S,D], fp32 or bf16, of any strides
    whose last is 1 (a transposed [tokens, heads, D], heads of a fused
    projection).  positions int32 [axes, B, S], [axes, S] for [H,S,D]; a single
    axis may be left out.  inv_freq fp64 [R/2], pair_axis int32 [R/2] or None:
    rotary_frequencies.  pairing "half": elements p and p + R/2, "adjacent": 2p
    and 2p + 1.  inverse: the other way, which takes the gradient of the output
    to that of x.  out: of x's shape, any such strides (x itself: in place); if
    None, dense of `dtype` (x's)."""
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError("x must be a tensor of 3 or 4 dimensions")
    strides = _rotary_strides(x, "x")
    B, H, S, D = x.shape if x.dim() == 4 else (1, *x.shape)
    where = (S,) if x.dim() == 3 else (B, S)
    if not isinstance(positions, torch.Tensor) or positions.dim() not in (len(where), len(where) + 1):
        raise ValueError("positions must be a tensor [axes, *tokens] or [*tokens]")
    axes = 1 if positions.dim() == len(where) else positions.shape[0]
    _need(positions, "positions", (torch.int32,), numel=axes * B * S)
    if positions.shape[-len(where):] != where:
        raise ValueError(f"positions: shape {tuple(positions.shape)}, expected [axes, *{where}]")
    _need(inv_freq, "inv_freq", (torch.float64,))
    R = 2 * inv_freq.numel()
    if R < 2 or R > D:
        raise ValueError(f"inv_freq: {R // 2} pairs for {D} elements")
    if pair_axis is not None:
        _need(pair_axis, "pair_axis", (torch.int32,), numel=R // 2)
    if pairing not in _PAIRING:
        raise ValueError(f"pairing {pairing!r} not in {tuple(_PAIRING)}")
    if dtype is None:
        dtype = x.dtype if out is None else out.dtype
    elif dtype not in _DT:
        raise ValueError(f"dtype {dtype} not in {tuple(_DT)}")
    if out is not None:
        out_strides = _rotary_strides(out, "out")
        if out.shape != x.shape:
            raise ValueError(f"out: shape {tuple(out.shape)}, expected {tuple(x.shape)}")
        if out.dtype != dtype:
            raise ValueError(f"out: dtype {out.dtype}, expected {dtype}")
    _one_device(("x", "positions", "inv_freq", "pair_axis", "out"), x, positions, inv_freq, pair_axis, out)
    if out is None:
        out = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
        out_strides = _I64x3(H * S * D, S * D, D)
    _call(x, lib().jules_hip_rotary, _DT[x.dtype], _DT[dtype], _PAIRING[pairing], int(bool(inverse)), x.data_ptr(),
          strides, out.data_ptr(), out_strides, positions.data_ptr(), inv_freq.data_ptr(), _ptr(pair_axis), axes, B, H, S,
          D, R)
    return out


class KV4Cache:
    """A paged key/value cache held in 4 bits (jh_kv4_cache; layout in
    include/jules_hip.h): k uint8 [pages, heads, page_size, D/2], v uint8
    [pages, heads, page_size/4, 2*D], k_meta and v_meta bf16 [pages, heads,
    page_size, 2] with each row's scale and minimum.  These and the sizes
    cannot be assigned: a larger pool is a new KV4Cache."""

    def __init__(self, k, v, k_meta, v_meta):
        _rank(k, "k", 4)
        _need(k, "k", (torch.uint8,))
        pages, heads, page_size, half = k.shape
        _need(v, "v", (torch.uint8,), shape=(pages, heads, page_size // 4, 4 * half))
        meta = (pages, heads, page_size, 2)
        _need(k_meta, "k_meta", (torch.bfloat16,), shape=meta)
        _need(v_meta, "v_meta", (torch.bfloat16,), shape=meta)
        c = JhKV4Cache(None, None, None, None, pages, page_size, heads, 2 * half)
        self.__dict__.update(k=k, v=v, k_meta=k_meta, v_meta=v_meta, pages=pages, heads=heads, page_size=page_size,
                             head_dim=2 * half)
        self._struct, self._ref = c, ctypes.byref(c)
        self._numels = (k.numel(), v.numel(), k_meta.numel(), v_meta.numel())

    _FIXED = frozenset(("k", "v", "k_meta", "v_meta", "pages", "heads", "page_size", "head_dim"))

    def __setattr__(self, name, value):
        if name in self._FIXED:
            raise AttributeError(f"{name} of a KV4Cache cannot be assigned: make a new KV4Cache")
        super().__setattr__(name, value)

    def _at(self):
        """jh_kv4_cache of the tensors where they lie now."""
        k, v, k_meta, v_meta, c = self.k, self.v, self.k_meta, self.v_meta, self._struct
        if (k.numel(), v.numel(), k_meta.numel(), v_meta.numel()) != self._numels:
            raise ValueError("cache: the size of a tensor has changed")
        c.k, c.v, c.k_meta, c.v_meta = k.data_ptr(), v.data_ptr(), k_meta.data_ptr(), v_meta.data_ptr()
        return self._ref

    @classmethod
    def empty(cls, pages, heads, head_dim, page_size=64, device="cuda"):
        """A pool of `pages` pages; what they hold is not set."""
        return cls(torch.empty(pages, heads, page_size, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.empty(pages, heads, page_size // 4, 2 * head_dim, dtype=torch.uint8, device=device),
                   *(torch.empty(pages, heads, page_size, 2, dtype=torch.bfloat16, device=device) for _ in "kv"))


_KV4_SCALE = {D: default_scale(D) for D in (64, 128)}


def _kv4_batch(cache, table, lens, cu_q, max_q, tokens):
    """Checks of what the calls on a KV4Cache share; returns (batch, max_q)."""
    if not isinstance(cache, KV4Cache):
        raise TypeError("cache must be a KV4Cache")
    _rank(table, "table", 2)
    _need(table, "table", (torch.int32,))
    batch = table.shape[0]
    _need(lens, "lens", (torch.int32,), numel=batch)
    if cu_q is None:
        each = tokens // batch if batch else 0
        if each * batch != tokens or max_q not in (None, each):
            raise ValueError(f"{tokens} tokens for {batch} sequences, max_q {max_q}: unequal numbers need cu_q")
        return batch, each
    _need(cu_q, "cu_q", (torch.int32,), numel=batch + 1)
    return batch, tokens if max_q is None else int(max_q)


def _kv4_rows(t, name, dtypes, tail):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must have 3 dimensions")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if t.shape[1:] != tail:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [tokens, {tail[0]}, {tail[1]}]")
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last stride must be 1")


def kv4_append(cache, k, v, table, lens, cu_q=None, max_q=None):
    """Writes new rows into the cache (jules_hip_kv4_append; no counterpart in
    the reference): k, v [tokens, heads, D], fp32 or bf16, of any strides whose
    last is 1.  table int32 [batch, max_pages]: the pages of each sequence;
    lens int32 [batch]: tokens of each, the new ones among them; rows cu_q[b]
    .. cu_q[b+1] - 1 are the last ones of sequence b (None: the same number
    each).  max_q: the largest number of new rows of a sequence, where the caller
    knows it; left out beside cu_q it counts as all of them, and the call starts
    that many workgroups for every sequence."""
    tail = (cache.heads, cache.head_dim) if isinstance(cache, KV4Cache) else (0, 0)
    if tail != (0, 0):
        _kv4_rows(k, "k", _REAL, tail)
        _kv4_rows(v, "v", (k.dtype,), tail)
        if v.shape != k.shape:
            raise ValueError(f"v: shape {tuple(v.shape)}, expected {tuple(k.shape)}")
    tokens = k.shape[0]
    batch, max_q = _kv4_batch(cache, table, lens, cu_q, max_q, tokens)
    _one_device(("k", "v", "cache.k", "cache.v", "cache.k_meta", "cache.v_meta", "table", "lens", "cu_q"), k, v, cache.k,
                cache.v, cache.k_meta, cache.v_meta, table, lens, cu_q)
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    _call(k, lib().jules_hip_kv4_append, _DT[k.dtype], cache._at(), k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
          table.data_ptr(), table.shape[1], lens.data_ptr(), _ptr(cu_q), batch, tokens, max_q)


def kv4_read(cache, table, lens, tokens, cu_q=None, max_q=None, dtype=torch.bfloat16, k=None, v=None):
    """The rows that kv4_append with the same arguments writes, as values
    (jules_hip_kv4_read): (k, v) [tokens, heads, D] of dtype.  With lens and
    cu_q of whole sequences it lays a cache out for flash_attention."""
    batch, max_q = _kv4_batch(cache, table, lens, cu_q, max_q, tokens)
    shape = (tokens, cache.heads, cache.head_dim)
    if dtype not in _DT:
        raise ValueError(f"dtype {dtype} not in {tuple(_DT)}")
    for t, n in ((k, "k"), (v, "v")):
        if t is not None:
            _need(t, n, (dtype,), shape=shape)
    _one_device(("lens", "table", "cache.k", "cache.v", "cache.k_meta", "cache.v_meta", "cu_q", "k", "v"), lens, table,
                cache.k, cache.v, cache.k_meta, cache.v_meta, cu_q, k, v)
    k = lens.new_empty(shape, dtype=dtype) if k is None else k
    v = lens.new_empty(shape, dtype=dtype) if v is None else v
    _call(lens, lib().jules_hip_kv4_read, _DT[dtype], cache._at(), k.data_ptr(), v.data_ptr(), table.data_ptr(),
          table.shape[1], lens.data_ptr(), _ptr(cu_q), batch, tokens, max_q)
    return k, v


def kv4_attention(q, cache, table, lens, cu_q=None, max_q=None, max_len=None, scale=None, out=None, lse=None,
                  return_lse=False, workspace=None):
    """Attention of new tokens over the cache (jules_hip_kv4_attention; no
    counterpart in the reference): q bf16 [tokens, heads_q, D], heads_q a
    multiple of the cache's heads, each token over its sequence's keys up to
    its own position; table, lens, cu_q and max_q as in kv4_append, which comes
    before (max_q also decides the tile, one for the batch).  max_len: the largest
    of lens, where the caller knows it (None: what the table has room for).  scale defaults to 1/sqrtf(D).  Returns out
    [tokens, heads_q, D], or (out, lse [tokens, heads_q]) with return_lse."""
    if isinstance(cache, KV4Cache):
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must have 3 dimensions")
        if q.shape[1] < 1 or q.shape[1] % cache.heads:
            raise ValueError(f"q: {q.shape[1]} heads, the cache has {cache.heads}")
        _kv4_rows(q, "q", (torch.bfloat16,), (q.shape[1], cache.head_dim))
    tokens, heads_q = q.shape[:2]
    batch, max_q = _kv4_batch(cache, table, lens, cu_q, max_q, tokens)
    if out is not None:
        _need(out, "out", (torch.bfloat16,), shape=q.shape)
    if lse is not None:
        _need(lse, "lse", (torch.float32,), numel=tokens * heads_q)
    ws_bytes = 0 if workspace is None else _workspace(workspace, "workspace")
    _one_device(("q", "cache.k", "cache.v", "cache.k_meta", "cache.v_meta", "table", "lens", "cu_q", "out", "lse",
                 "workspace"), q, cache.k, cache.v, cache.k_meta, cache.v_meta, table, lens, cu_q, out, lse, workspace)
    if max_len is None:
        max_len = min(table.shape[1] * cache.page_size, 2**31 - 1)
    if scale is None:
        scale = _KV4_SCALE[cache.head_dim] if cache.head_dim in _KV4_SCALE else default_scale(cache.head_dim)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if lse is None and return_lse:
        lse = q.new_empty((tokens, heads_q), dtype=torch.float32)
    if workspace is None:
        ws_bytes = lib().jules_hip_kv4_attention_workspace_size(batch, tokens, heads_q, cache.heads, cache.head_dim,
                                                                max_q, max_len)
        if ws_bytes:
            workspace = q.new_empty((ws_bytes,), dtype=torch.uint8)
    qt, qh, _ = q.stride()
    _call(q, lib().jules_hip_kv4_attention, float(scale), cache._at(), q.data_ptr(), qt, qh, out.data_ptr(), _ptr(lse),
          heads_q, table.data_ptr(), table.shape[1], lens.data_ptr(), _ptr(cu_q), batch, tokens, max_q, int(max_len),
          _ptr(workspace), ws_bytes)
    return (out, lse) if return_lse else out


def cross_entropy_workspace(M, device):
    nbytes = lib().jules_hip_cross_entropy_workspace_size(int(M))
    return torch.empty(((nbytes + 3) // 4,), dtype=torch.float32, device=device)


def cross_entropy(logits, targets, grad=None, loss=None, workspace=None):
    """fusedCrossEntropyLoss (FusedKernels.h:766): returns (loss[1], grad) on the device."""
    _need(logits, "logits", (torch.float32,))
    M, N = _rows(logits)
    _need(targets, "targets", (torch.int32,), numel=M)
    if grad is not None:
        _need(grad, "grad", (torch.float32,), shape=logits.shape)
    if loss is not None:
        _need(loss, "loss", (torch.float32,), numel=1)
    ws_bytes = None if workspace is None else _workspace(workspace, "workspace")
    _on_device(logits=logits, targets=targets, grad=grad, loss=loss, workspace=workspace)
    if grad is None:
        grad = torch.empty_like(logits)
    if loss is None:
        loss = torch.empty((1,), dtype=torch.float32, device=logits.device)
    if workspace is None:
        workspace = cross_entropy_workspace(M, logits.device)
        ws_bytes = workspace.numel() * 4
    check(lib().jules_hip_cross_entropy(_ptr(logits), _ptr(targets), _ptr(grad), _ptr(loss), M, N,
                                        _ptr(workspace), ws_bytes, _stream(logits)))
    return loss, grad


def _mlp_operands(X, W1, b1, W2, b2):
    for t, n in ((X, "X"), (W1, "W1"), (W2, "W2")):
        _rank(t, n, 2)
    for t, n in ((X, "X"), (W1, "W1"), (b1, "b1"), (W2, "W2"), (b2, "b2")):
        _need(t, n, (torch.float32,))
    M, K1 = X.shape
    K1b, N1 = W1.shape
    N1b, N2 = W2.shape
    if K1b != K1 or N1b != N1 or b1.numel() != N1 or b2.numel() != N2:
        raise ValueError("mlp: operand shapes disagree")
    return M, K1, N1, N2


def mlp_forward(X, W1, b1, W2, b2, out=None, workspace=None):
    """fusedMLPForward (FusedKernels.h:659): relu(X W1 + b1) W2 + b2, fp32."""
    M, K1, N1, N2 = _mlp_operands(X, W1, b1, W2, b2)
    if out is not None:
        _need(out, "out", (torch.float32,), shape=(M, N2))
    ws_bytes = None if workspace is None else _workspace(workspace, "workspace")
    _on_device(X=X, W1=W1, b1=b1, W2=W2, b2=b2, out=out, workspace=workspace)
    if out is None:
        out = torch.empty((M, N2), dtype=torch.float32, device=X.device)
    if workspace is None:
        nbytes = lib().jules_hip_mlp_forward_workspace_size(M, K1, N1, N2)
        workspace = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=X.device)
        ws_bytes = workspace.numel()
    check(lib().jules_hip_mlp_forward(_ptr(X), _ptr(W1), _ptr(b1), _ptr(W2), _ptr(b2), _ptr(out),
                                      M, K1, N1, N2, _ptr(workspace), ws_bytes, _stream(X)))
    return out


def mlp_workspace(M, K1, N1, N2, device):
    nbytes = lib().jules_hip_mlp_workspace_size(int(M), int(K1), int(N1), int(N2))
    return torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=device)


def mlp_forward_backward(X, W1, b1, W2, b2, targets, with_dX=False, workspace=None, out=None):
    """interleavedMLPForwardBackward (InterleavedAutodiff.h:55): fp32 2-layer
    MLP, softmax cross entropy against int32 targets, and the gradients.
    Returns a dict with output, loss (1 element), dW1, db1, dW2, db2 and
    dX (None unless with_dX), all on X's device; `out`, a dict returned by an
    earlier call with the same shapes, is reused instead of allocating."""
    M, K1, N1, N2 = _mlp_operands(X, W1, b1, W2, b2)
    _need(targets, "targets", (torch.int32,), numel=M)
    shapes = {"output": (M, N2), "loss": (1,), "dW1": (K1, N1), "db1": (N1,), "dW2": (N1, N2),
              "db2": (N2,), "dX": (M, K1)}
    if out is not None:
        with_dX = out["dX"] is not None
        for k, shp in shapes.items():
            if out[k] is not None:
                _need(out[k], f"out[{k!r}]", (torch.float32,), shape=shp)
    ws_bytes = None if workspace is None else _workspace(workspace, "workspace")
    outs = {} if out is None else {f"out[{k!r}]": v for k, v in out.items()}
    dev = _on_device(X=X, W1=W1, b1=b1, W2=W2, b2=b2, targets=targets, workspace=workspace, **outs)
    if out is None:
        out = {k: torch.empty(shp, dtype=torch.float32, device=dev)
               if k != "dX" or with_dX else None for k, shp in shapes.items()}
    if workspace is None:
        workspace = mlp_workspace(M, K1, N1, N2, dev)
        ws_bytes = workspace.numel()
    check(lib().jules_hip_mlp_forward_backward(
        _ptr(X), _ptr(W1), _ptr(b1), _ptr(W2), _ptr(b2), _ptr(targets), _ptr(out["output"]),
        _ptr(out["dW1"]), _ptr(out["db1"]), _ptr(out["dW2"]), _ptr(out["db2"]), _ptr(out["dX"]),
        M, K1, N1, N2, _ptr(out["loss"]), _ptr(workspace), ws_bytes, _stream(X)))
    return out


def mfma_ceiling(out, workgroups, iters):
    """Launch the MFMA calibration kernel (jules_hip_mfma_ceiling; no
    counterpart in the reference) on torch's current stream: `workgroups` x 4
    waves, each issuing 16 * iters v_mfma_f32_32x32x16_bf16 on random
    operands.  out: fp32 GPU tensor of workgroups * 256 elements.  Returns
    the FLOP count of the launch."""
    _need(out, "out", (torch.float32,))
    if out.numel() < workgroups * 256:
        raise ValueError("out must hold workgroups * 256 floats")
    _on_device(out=out)
    check(lib().jules_hip_mfma_ceiling(_ptr(out), int(workgroups), int(iters), _stream(out)))
    return 32768.0 * 16 * iters * 4 * workgroups


def hbm_read_floor(buf, out, workgroups=256):
    """Launch the HBM read calibration (jules_hip_hbm_read_floor; no
    counterpart in the reference) on torch's current stream: one streaming
    read of `buf` (contiguous, a multiple of 16 bytes).  out: int32 GPU tensor
    of workgroups * 256 elements.  Returns the bytes read."""
    if not isinstance(buf, torch.Tensor) or not buf.is_contiguous():
        raise ValueError("buf must be a contiguous tensor")
    _need(out, "out", (torch.int32,))
    if out.numel() < workgroups * 256:
        raise ValueError("out must hold workgroups * 256 int32")
    _on_device(buf=buf, out=out)
    nbytes = buf.numel() * buf.element_size()
    check(lib().jules_hip_hbm_read_floor(_ptr(buf), nbytes, _ptr(out), int(workgroups), _stream(buf)))
    return nbytes
