"""Causal attention of whole prompts, packed one behind the other, and its gradients.

``prompt_attention`` takes q, k and v as they leave ``qk_norm_rope`` (or as views of a fused
projection), or keys and values that ``kv_cache_read`` gathered for a prefill that continues its
contexts; ``prompt_attention_bwd`` the gradients.  The kernels are libfagq.so's
(include/fagq_prompt.h); there is no fallback.  Neither records anything for autograd: their
results carry no gradient, and a training program calls the backward from a
``torch.autograd.Function`` of its own.

No counterpart in the reference repository: its MLA backward
(src/task03_mla_bwd_nope_dkdv.py:453-480) is of one shared latent.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mla_bwd import check_workspace
from .qk_rope import _heads

_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
HEAD_DIMS = (64, 128, 256)
FILL_OUT, FILL_LSE = 1, 2
FILL_DQ, FILL_DK, FILL_DV = 1, 2, 4


def _ptr(t: torch.Tensor | None):
    return None if t is None or t.numel() == 0 else ctypes.c_void_p(t.data_ptr())


def _check_lengths(t: torch.Tensor, name: str, dev: torch.device, count: int | None = None) -> int:
    if t.device != dev or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() \
            or t.shape[0] < 1 or count not in (None, t.shape[0]):
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape "
                         f"({'B + 1' if count is None else count},) on {dev}")
    return int(t.shape[0]) - 1


def _check(q, k, v, cu_seqlens, cu_seqlens_k):
    """Checks what both directions take; returns (B, T, Tk, Hq, H, D)."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q must be [T, Hq, D] and k [Tk, H, D], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    dev = q.device
    if dev.type != "cuda":
        raise ValueError("q must be a GPU (HIP) tensor; this operator has no CPU path")
    T, Hq, D = (int(s) for s in q.shape)
    Tk, H = int(k.shape[0]), int(k.shape[1])
    if D not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS}, got {D}")
    if H < 1 or Hq < 1 or Hq % H:
        raise ValueError(f"{Hq} query heads do not share {H} heads of k evenly")
    B = _check_lengths(cu_seqlens, "cu_seqlens", dev)
    if cu_seqlens_k is not None:
        _check_lengths(cu_seqlens_k, "cu_seqlens_k", dev, B + 1)
    elif T != Tk:
        raise ValueError(f"without cu_seqlens_k, k must have q's {T} rows, got {Tk}")
    return B, T, Tk, Hq, H, D


def workspace_bytes(B: int, T: int, Tk: int, Hq: int, H: int, D: int) -> int:
    """Workspace bytes of a ``prompt_attention`` of exactly these sizes (not monotone: see
    ``bwd_workspace_bytes``)."""
    n = _lib.load().fagq_prompt_attention_workspace_bytes(B, T, Tk, Hq, H, D)
    if n < 0:
        raise ValueError(f"no workspace size for B={B}, T={T}, Tk={Tk}, Hq={Hq}, H={H}, D={D}")
    return n


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     sm_scale: float, cu_seqlens_k: torch.Tensor | None = None,
                     return_lse: bool = False, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None):
    """Causal attention of B packed sequences.

    q [T, Hq, D], k, v [Tk, H, D]: bfloat16 or float16 with contiguous rows at any 16-byte aligned
    token and head strides; D is 64, 128 or 256, Hq a multiple of H (query head h reads head
    ``h // (Hq // H)``).  cu_seqlens: int32 [B + 1], ascending from 0: sequence b is the rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` of q, and of k and v those of ``cu_seqlens_k``
    (default: the same).  With n queries and m keys, query i sees the keys up to ``i + m - n``, so
    that a chunk of new tokens continues its context; a query that sees none gets zeros.

    Returns ``out`` [T, Hq, D] (contiguous, allocated unless given), with ``return_lse`` also the
    float32 [Hq, T] log-sum-exp of each query's scores (-inf for one without keys).  Rows behind
    the last sequence are left as they were in a given ``out``, zeros (lse: -inf) otherwise.
    ``workspace`` (optional): a uint8 GPU tensor of at least ``workspace_bytes(...)`` bytes, which
    calls that may overlap do not share.  The rows that sequences name are finite; others are not
    read.  Autograd does not see the call.  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(q) if workspace is None else (None, None)
    if mod is not None:
        r = mod.prompt(q, k, v, cu_seqlens, cu_seqlens_k, sm_scale, return_lse, out, fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_prompt_attention_launch")
        # An argument the binding leaves to the checks below.
    B, T, Tk, Hq, H, D = _check(q, k, v, cu_seqlens, cu_seqlens_k)
    dev = q.device
    strides = (_heads(q, "q", (T, Hq, D), q.dtype, dev) + _heads(k, "k", (Tk, H, D), q.dtype, dev)
               + _heads(v, "v", (Tk, H, D), q.dtype, dev))
    fill = FILL_LSE
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
        fill |= FILL_OUT
    elif out.dtype != q.dtype or tuple(out.shape) != (T, Hq, D) or not out.is_contiguous() \
            or out.device != dev:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of shape {(T, Hq, D)} on {dev}")
    lse = torch.empty(Hq, T, dtype=torch.float32, device=dev) if return_lse else None
    need = workspace_bytes(B, T, Tk, Hq, H, D)
    if workspace is not None:
        check_workspace(workspace, need, dev)
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if T > 0:
        lib = _lib.load()
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream(dev).cuda_stream
            st = lib.fagq_prompt_attention_launch(
                _ptr(q), _ptr(k), _ptr(v), _ptr(cu_seqlens), _ptr(cu_seqlens_k), _ptr(out),
                _ptr(lse), _ptr(workspace) if need else None,
                workspace.numel() * workspace.element_size() if need else 0,
                (ctypes.c_int64 * 6)(*strides), B, T, Tk, Hq, H, D, float(sm_scale),
                _DTYPES[q.dtype], fill, ctypes.c_void_p(stream))
        _lib.check(st, "fagq_prompt_attention_launch")
    return (out, lse) if return_lse else out


def bwd_workspace_bytes(B: int, T: int, Tk: int, Hq: int, H: int, D: int) -> int:
    """Workspace bytes of a ``prompt_attention_bwd`` of exactly these sizes.  Not monotone: a smaller
    call is cut into more parts and may need more, so a workspace that serves several calls is as
    large as the largest of theirs."""
    n = _lib.load().fagq_prompt_attention_bwd_workspace_bytes(B, T, Tk, Hq, H, D)
    if n < 0:
        raise ValueError(f"no workspace size for B={B}, T={T}, Tk={Tk}, Hq={Hq}, H={H}, D={D}")
    return n


def prompt_attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         out: torch.Tensor, lse: torch.Tensor, cu_seqlens: torch.Tensor,
                         sm_scale: float, cu_seqlens_k: torch.Tensor | None = None,
                         dq: torch.Tensor | None = None, dk: torch.Tensor | None = None,
                         dv: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """Gradients of ``prompt_attention``: dout [T, Hq, D] (strided as q may be) is that of its
    output, ``out`` and ``lse`` are what it returned, the other arguments its inputs.  Returns
    ``(dq, dk, dv)`` of q's type, allocated unless given (views of a fused gradient included).
    Gradients are written, not added to; rows behind the last sequence are left as they were in
    given ones, zeros otherwise.  Equal calls give equal bits.  ``workspace`` (optional): a uint8
    GPU tensor of at least ``bwd_workspace_bytes(...)`` bytes, which calls that may overlap do not
    share.  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(q) if workspace is None else (None, None)
    if mod is not None:
        r = mod.prompt_bwd(q, k, v, cu_seqlens, cu_seqlens_k, sm_scale, dout, out, lse, dq, dk, dv,
                           fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_prompt_attention_bwd_launch")
        # An argument the binding leaves to the checks below.
    B, T, Tk, Hq, H, D = _check(q, k, v, cu_seqlens, cu_seqlens_k)
    dev = q.device
    if out.dtype != q.dtype or tuple(out.shape) != (T, Hq, D) or not out.is_contiguous() \
            or out.device != dev:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of shape {(T, Hq, D)} on {dev}")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (Hq, T) or not lse.is_contiguous() \
            or lse.device != dev:
        raise ValueError(f"lse must be a contiguous float32 tensor of shape {(Hq, T)} on {dev}")
    fill = (FILL_DQ if dq is None else 0) | (FILL_DK if dk is None else 0) | (FILL_DV if dv is None else 0)
    shapes = ((T, Hq, D), (Tk, H, D), (Tk, H, D))
    dq, dk, dv = (torch.empty(s, dtype=q.dtype, device=dev) if t is None else t
                  for t, s in zip((dq, dk, dv), shapes))
    strides = []
    for name, t, shape in (("dout", dout, shapes[0]), ("q", q, shapes[0]), ("k", k, shapes[1]),
                           ("v", v, shapes[1]), ("dq", dq, shapes[0]), ("dk", dk, shapes[1]),
                           ("dv", dv, shapes[1])):
        strides += _heads(t, name, shape, q.dtype, dev)
    need = bwd_workspace_bytes(B, T, Tk, Hq, H, D)
    if workspace is not None:
        check_workspace(workspace, need, dev)
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if T > 0 or Tk > 0:
        lib = _lib.load()
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream(dev).cuda_stream
            st = lib.fagq_prompt_attention_bwd_launch(
                _ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(cu_seqlens),
                _ptr(cu_seqlens_k), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(workspace) if need else None,
                workspace.numel() * workspace.element_size() if need else 0,
                (ctypes.c_int64 * 14)(*strides), B, T, Tk, Hq, H, D, float(sm_scale),
                _DTYPES[q.dtype], fill, ctypes.c_void_p(stream))
        _lib.check(st, "fagq_prompt_attention_bwd_launch")
    return dq, dk, dv
