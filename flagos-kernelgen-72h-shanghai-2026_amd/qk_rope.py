"""RMS norm of each query and key head with the rotation by position in the same
pass, and its gradients.

``qk_norm_rope`` computes, for every head row x of q and k,

    y = rotate(x / sqrt(mean(x^2) + eps) * weight, position)

in fp32 with one rounding, from the views of a fused projection as they are;
``qk_norm_rope_bwd`` the gradients of q, k and both weights.  The kernels are
libfagq.so's ``fagq_qk_norm_rope_launch`` and ``fagq_qk_norm_rope_bwd_launch``
(include/fagq_rope.h); there is no fallback.  Neither records anything for autograd: their results
carry no gradient, and a training program calls the backward from a ``torch.autograd.Function``
of its own.

No counterpart in the reference repository: its RMSNorm
(src/task01_fused_add_rmsnorm_group_quant.py:88-100) is over hidden rows.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mla_bwd import check_workspace

_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
IDX_I32, IDX_I64 = 0, 1
MAX_D = 512


def index_code(t: torch.Tensor, name: str) -> int:
    if t.dtype == torch.int32:
        return IDX_I32
    if t.dtype == torch.int64:
        return IDX_I64
    raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")


def _heads(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype,
           dev: torch.device) -> list[int]:
    """The token and head strides of a [T, H, D] tensor with contiguous rows."""
    if t.device != dev or t.dtype != dtype or tuple(t.shape) != shape or t.stride(2) != 1:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {shape} on {dev} with "
                         f"contiguous rows, got {t.dtype} {tuple(t.shape)} strides {t.stride()} "
                         f"on {t.device}")
    # A dimension of one element is never stepped over.
    return [t.stride(i) if t.shape[i] > 1 else 0 for i in (0, 1)]


def _check(q, k, q_weight, k_weight, cos, sin, positions):
    """Checks what both directions take; returns (T, Hq, Hk, D, R, table rows, index code)."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [T, H, D], got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"q must be bfloat16, float16 or float32, got {q.dtype}")
    dev = q.device
    if dev.type != "cuda":
        raise ValueError("q must be a GPU (HIP) tensor; this operator has no CPU path")
    T, Hq, D = (int(s) for s in q.shape)
    Hk = int(k.shape[1])
    if D % 16 or not 16 <= D <= MAX_D:
        raise ValueError(f"head dim must be a multiple of 16 up to {MAX_D}, got {D}")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t.device != dev or t.dtype != q.dtype or tuple(t.shape) != (D,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {q.dtype} tensor of shape ({D},) on {dev}")
    if cos.dim() != 2 or tuple(sin.shape) != tuple(cos.shape):
        raise ValueError(f"cos and sin must share a shape [positions, R / 2], got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.device != dev or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 tensor on {dev}")
    R = 2 * int(cos.shape[1])
    if R % 16 or not 16 <= R <= D:
        raise ValueError(f"cos and sin must cover a multiple of 16 dims up to {D}, got {R}")
    idx = index_code(positions, "positions")
    if positions.device != dev or tuple(positions.shape) != (T,) or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous tensor of shape ({T},) on {dev}")
    return T, Hq, Hk, D, R, int(cos.shape[0]), idx


def _ptr(t: torch.Tensor):
    return ctypes.c_void_p(t.data_ptr())


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                 interleaved: bool = False, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
    """q [T, Hq, D], k [T, Hk, D]: bfloat16, float16 or float32 with contiguous rows at any
    16-byte aligned token and head strides (views of a fused projection); q_weight, k_weight
    [D] of the same type; cos, sin: float32 [positions, R / 2] tables, the first R dims are
    rotated in pairs (i, i + R / 2), or (2 i, 2 i + 1) if ``interleaved``; positions [T]:
    int32 or int64.  D and R are multiples of 16.  A token with a position outside the tables
    is padding and gets zeros.  Returns ``(q_out, k_out)``, allocated unless given; they may be
    q and k themselves.  Autograd does not see the call (``qk_norm_rope_bwd`` has the
    gradients).  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(q)
    if mod is not None:
        r = mod.rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, q_out, k_out,
                     fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_qk_norm_rope_launch")
        # An argument the binding leaves to the checks below.
    T, Hq, Hk, D, R, table, idx = _check(q, k, q_weight, k_weight, cos, sin, positions)
    dev = q.device
    if q_out is None:
        q_out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    if k_out is None:
        k_out = torch.empty(T, Hk, D, dtype=q.dtype, device=dev)
    strides = (_heads(q, "q", (T, Hq, D), q.dtype, dev) + _heads(k, "k", (T, Hk, D), q.dtype, dev)
               + _heads(q_out, "q_out", (T, Hq, D), q.dtype, dev)
               + _heads(k_out, "k_out", (T, Hk, D), q.dtype, dev))
    if T == 0:                      # empty tensors have no address to pass
        return q_out, k_out
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.fagq_qk_norm_rope_launch(
            _ptr(q), _ptr(k), _ptr(q_weight), _ptr(k_weight), _ptr(cos), _ptr(sin),
            _ptr(positions), _ptr(q_out), _ptr(k_out), (ctypes.c_int64 * 8)(*strides), T, Hq, Hk,
            D, R, table, float(eps), int(bool(interleaved)), _DTYPES[q.dtype], idx,
            ctypes.c_void_p(stream))
    _lib.check(st, "fagq_qk_norm_rope_launch")
    return q_out, k_out


def bwd_workspace_bytes(T: int, Hq: int, Hk: int, D: int) -> int:
    n = _lib.load().fagq_qk_norm_rope_bwd_workspace_bytes(T, Hq, Hk, D)
    if n < 0:
        raise ValueError(f"no workspace size for T={T}, Hq={Hq}, Hk={Hk}, D={D}")
    return n


def qk_norm_rope_bwd(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                     q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                     sin: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                     interleaved: bool = False, dq: torch.Tensor | None = None,
                     dk: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """Gradients of ``qk_norm_rope``: dq_out [T, Hq, D] and dk_out [T, Hk, D] are those of its
    outputs, the other arguments its inputs.  Returns ``(dq, dk, dq_weight, dk_weight)``: dq and
    dk of q's type (allocated unless given, views of a fused gradient included), the weights'
    float32 [D].  ``workspace`` (optional): a uint8 GPU tensor of at least
    ``bwd_workspace_bytes(T, Hq, Hk, D)`` bytes, which calls that may overlap do not share.
    Padding rows get zeros."""
    mod, fast_stream = _lib.fast_module(q) if workspace is None else (None, None)
    if mod is not None:
        r = mod.rope_bwd(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, dq_out,
                         dk_out, dq, dk, fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_qk_norm_rope_bwd_launch")
        # An argument the binding leaves to the checks below.
    T, Hq, Hk, D, R, table, idx = _check(q, k, q_weight, k_weight, cos, sin, positions)
    dev = q.device
    if dq is None:
        dq = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    if dk is None:
        dk = torch.empty(T, Hk, D, dtype=q.dtype, device=dev)
    strides = []
    for name, t, H in (("dq_out", dq_out, Hq), ("dk_out", dk_out, Hk), ("q", q, Hq), ("k", k, Hk),
                       ("dq", dq, Hq), ("dk", dk, Hk)):
        strides += _heads(t, name, (T, H, D), q.dtype, dev)
    need = bwd_workspace_bytes(T, Hq, Hk, D)
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    else:
        check_workspace(workspace, need, dev)
    if T == 0:
        return dq, dk, *torch.zeros(2, D, dtype=torch.float32, device=dev)
    dweights = torch.empty(2, D, dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.fagq_qk_norm_rope_bwd_launch(
            _ptr(dq_out), _ptr(dk_out), _ptr(q), _ptr(k), _ptr(q_weight), _ptr(k_weight),
            _ptr(cos), _ptr(sin), _ptr(positions), _ptr(dq), _ptr(dk), _ptr(dweights[0]),
            _ptr(dweights[1]), _ptr(workspace), workspace.numel() * workspace.element_size(),
            (ctypes.c_int64 * 12)(*strides), T, Hq, Hk, D, R, table, float(eps),
            int(bool(interleaved)), _DTYPES[q.dtype], idx, ctypes.c_void_p(stream))
    _lib.check(st, "fagq_qk_norm_rope_bwd_launch")
    return dq, dk, dweights[0], dweights[1]
