"""The index tensors of a step, made on the GPU from the lengths of its requests.

``batch_tables`` gives what the attention side's calls of a step take: positions for
``qk_norm_rope``, slots for ``kv_cache_write``, cumulative lengths for ``prompt_attention`` and
``kv_cache_read``, lengths and page table for ``paged_attention`` and ``paged_tree_attention``.
The kernel is libfagq.so's ``fagq_batch_tables_launch`` (include/fagq_cache.h); there is no
fallback.

No counterpart in the reference repository, whose page tables are made outside of it
(src/task02_dsa_topk_page_table_transform.py:1666-1726 takes one).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv_cache import MAX_PAGE, MIN_PAGE
from .qk_rope import index_code


def _ptr(t: torch.Tensor | None):
    return None if t is None or t.numel() == 0 else ctypes.c_void_p(t.data_ptr())


def batch_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                 page_table: torch.Tensor, page_size: int, num_tokens: int,
                 free_start: torch.Tensor | None = None):
    """A step of B requests: request b has ``context_lens[b]`` tokens in the cache, on the first
    pages of its row of page_table (int32 [B, width]), and ``new_lens[b]`` new ones (both int32 or
    both int64 [B]), packed request by request in ``num_tokens`` rows.  The new pages that they
    need are taken from free_pages (int32 [F]) from entry ``free_start`` (int32 [1], default 0) on,
    and written into page_table.

    Returns ``(cu_seqlens, cu_seqlens_k, kv_lens, positions, slots, free_end)``: where each
    request's rows begin (int32 [B + 1]); the running sums of kv_lens, context and new tokens
    (int32 [B + 1], [B]); each row's position in its request (int32) and slot in the cache (int64,
    ``page * page_size + offset``), both -1 in rows behind the last; and free_start plus the pages
    taken (int32 [1]), which the next step starts from.

    Nothing is read on the host.  New tokens past ``num_tokens`` are no part of the step.  Where
    free_pages runs out, ``free_end`` is larger than F, and the missing entries and slots are -1,
    as are slots past the table's width.  page_table's other entries are left as they were: a call
    with the same lengths gives the same results again.  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(page_table)
    if mod is not None:
        r = mod.tables(context_lens, new_lens, free_pages, page_table, page_size, num_tokens, free_start,
                       fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_batch_tables_launch")
        # An argument the binding leaves to the checks below.
    dev = page_table.device
    if dev.type != "cuda":
        raise ValueError("page_table must be a GPU (HIP) tensor; this operator has no CPU path")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or not page_table.is_contiguous():
        raise ValueError(f"page_table must be a contiguous int32 [B, width] tensor on {dev}")
    B, width = (int(s) for s in page_table.shape)
    idx = index_code(context_lens, "context_lens")
    for name, t in (("context_lens", context_lens), ("new_lens", new_lens)):
        if t.device != dev or t.dtype != context_lens.dtype or tuple(t.shape) != (B,) \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {context_lens.dtype} tensor of shape "
                             f"({B},) on {dev}")
    if free_pages.device != dev or free_pages.dtype != torch.int32 or free_pages.dim() != 1 \
            or not free_pages.is_contiguous():
        raise ValueError(f"free_pages must be a contiguous int32 [F] tensor on {dev}")
    if free_start is not None and (free_start.device != dev or free_start.dtype != torch.int32
                                   or tuple(free_start.shape) != (1,)):
        raise ValueError(f"free_start must be an int32 tensor of shape (1,) on {dev}")
    page_size, num_tokens = int(page_size), int(num_tokens)
    if page_size < MIN_PAGE or page_size > MAX_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page size must be a power of two of {MIN_PAGE} to {MAX_PAGE}, got {page_size}")
    if num_tokens < 0:
        raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
    i32 = dict(dtype=torch.int32, device=dev)
    cu, cu_k = torch.empty(B + 1, **i32), torch.empty(B + 1, **i32)
    lens, positions, end = torch.empty(B, **i32), torch.empty(num_tokens, **i32), torch.empty(1, **i32)
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.fagq_batch_tables_launch(
            _ptr(context_lens), _ptr(new_lens), _ptr(free_pages), _ptr(free_start),
            _ptr(page_table), _ptr(cu), _ptr(cu_k), _ptr(lens), _ptr(positions), _ptr(slots),
            _ptr(end), B, num_tokens, free_pages.shape[0], page_size, width, idx,
            ctypes.c_void_p(stream))
    _lib.check(st, "fagq_batch_tables_launch")
    return cu, cu_k, lens, positions, slots, end
