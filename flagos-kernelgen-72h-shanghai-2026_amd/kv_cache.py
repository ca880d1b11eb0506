"""A quantised paged key/value cache: written as it is quantised, read back, and attended over.

Layout (contiguous tensors, ``empty_kv_cache`` allocates them):

    codes   [num_pages, H, page_size, D]      float8_e4m3fn or int8
    scales  [num_pages, H, D / G, page_size]  float32 or uint8 (UE8M0)

A value is ``code * scale``, one scale for each group of G values of a token's head row, in the
formats of ``fused_add_rmsnorm_group_quant``.  ``kv_cache_write`` quantises keys and values into
slots (page * page_size + offset), ``kv_cache_read`` gathers the pages of a ragged batch, and
``paged_attention`` and, for drafted trees, ``paged_tree_attention`` attend over them.  The kernels
are libfagq.so's (include/fagq_cache.h); there is no fallback.

No counterpart in the reference repository; the page tables are those that
``dsa_topk_page_table_transform`` reads
(src/task02_dsa_topk_page_table_transform.py:1666-1726).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mla_bwd import check_workspace
from .qk_rope import _heads, index_code

_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
_CODES = {torch.float8_e4m3fn: _lib.Q_FP8_E4M3FN, torch.int8: _lib.Q_INT8}
_SCALES = {torch.float32: _lib.SCALE_F32, torch.uint8: _lib.SCALE_UE8M0}
GROUPS = (64, 128, 256)
MIN_PAGE, MAX_PAGE, MAX_D = 16, 65536, 1024
ATTENTION_DIMS = (64, 128, 256)


def _ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def empty_kv_cache(num_pages: int, heads: int, page_size: int, head_dim: int,
                   group_size: int | None = None, dtype: torch.dtype = torch.float8_e4m3fn,
                   scale_ue8m0: bool = False, device="cuda"):
    """(codes, scales) of one cache, uninitialised; group_size defaults to the head dim."""
    G = head_dim if group_size is None else group_size
    if G not in GROUPS or head_dim % G:
        raise ValueError(f"group size must be one of {GROUPS} and divide {head_dim}, got {G}")
    if dtype not in _CODES:
        raise TypeError(f"a cache's codes are float8_e4m3fn or int8, got {dtype}")
    codes = torch.empty(num_pages, heads, page_size, head_dim, dtype=dtype, device=device)
    scales = torch.empty(num_pages, heads, head_dim // G, page_size, device=device,
                         dtype=torch.uint8 if scale_ue8m0 else torch.float32)
    return codes, scales


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    """Checks a cache's tensors; returns (pages, H, page size, D, G, code format, scale format)."""
    if k_cache.dim() != 4 or k_scale.dim() != 4:
        raise ValueError("k_cache must be [pages, H, page_size, D] and k_scale "
                         f"[pages, H, D / G, page_size], got {tuple(k_cache.shape)} and "
                         f"{tuple(k_scale.shape)}")
    if k_cache.dtype not in _CODES:
        raise TypeError(f"k_cache must be float8_e4m3fn or int8, got {k_cache.dtype}")
    if k_scale.dtype not in _SCALES:
        raise TypeError(f"k_scale must be float32 or uint8 (ue8m0), got {k_scale.dtype}")
    dev = k_cache.device
    if dev.type != "cuda":
        raise ValueError("the cache must be on a GPU (HIP); these operators have no CPU path")
    P, H, page, D = (int(s) for s in k_cache.shape)
    groups = int(k_scale.shape[2])
    if groups < 1 or D % groups or D // groups not in GROUPS:
        raise ValueError(f"k_scale must hold a scale for each group of {GROUPS} of {D} values, "
                         f"got {groups} for a row")
    if page < MIN_PAGE or page > MAX_PAGE or page & (page - 1):
        raise ValueError(f"page size must be a power of two of {MIN_PAGE} to {MAX_PAGE}, got {page}")
    if D > MAX_D:
        raise ValueError(f"head dim must be at most {MAX_D}, got {D}")
    if (v_cache is None) != (v_scale is None):
        raise ValueError("v_cache and v_scale go together")
    for name, t, shape, dt in (("k_cache", k_cache, (P, H, page, D), k_cache.dtype),
                               ("v_cache", v_cache, (P, H, page, D), k_cache.dtype),
                               ("k_scale", k_scale, (P, H, groups, page), k_scale.dtype),
                               ("v_scale", v_scale, (P, H, groups, page), k_scale.dtype)):
        if t is None:
            continue
        if t.device != dev or t.dtype != dt or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dt} tensor of shape {shape} on {dev}")
    return P, H, page, D, D // groups, _CODES[k_cache.dtype], _SCALES[k_scale.dtype]


def kv_cache_write(k: torch.Tensor, v: torch.Tensor | None, slots: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor | None, k_scale: torch.Tensor,
                   v_scale: torch.Tensor | None) -> None:
    """Quantises k and v [T, H, D] (bfloat16, float16 or float32, contiguous rows at any 16-byte
    aligned token and head strides) into the slots [T] (int32 or int64) of the cache.  A token
    whose slot is negative or past the cache is left out; no two tokens may name one slot.
    Values are finite (others spoil their own group, no other).  A cache of latents passes None
    for v, v_cache and v_scale.  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(k_cache)
    if mod is not None:
        st = mod.cache_write(k, v, slots, k_cache, v_cache, k_scale, v_scale, fast_stream)
        if st == 0:
            return
        if st != _lib.FAST_ARG_ERROR:
            _lib.check(st, "fagq_kv_cache_write_launch")
        # An argument the binding leaves to the checks below.
    P, H, page, D, G, qf, sf = _check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    if (v is None) != (v_cache is None):
        raise ValueError("v, v_cache and v_scale go together")
    if k.dim() != 3:
        raise ValueError(f"k must be [T, H, D], got {tuple(k.shape)}")
    if k.dtype not in _DTYPES:
        raise TypeError(f"k must be bfloat16, float16 or float32, got {k.dtype}")
    T = int(k.shape[0])
    strides = _heads(k, "k", (T, H, D), k.dtype, dev)
    strides += [0, 0] if v is None else _heads(v, "v", (T, H, D), k.dtype, dev)
    idx = index_code(slots, "slots")
    if slots.device != dev or tuple(slots.shape) != (T,) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous tensor of shape ({T},) on {dev}")
    if T == 0 or P == 0:            # empty tensors have no address to pass
        return
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.fagq_kv_cache_write_launch(
            _ptr(k), _ptr(v), _ptr(slots), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale),
            _ptr(v_scale), (ctypes.c_int64 * 4)(*strides), T, H, D, G, P, page, _DTYPES[k.dtype],
            qf, sf, idx, ctypes.c_void_p(stream))
    _lib.check(st, "fagq_kv_cache_write_launch")


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor | None, k_scale: torch.Tensor,
                  v_scale: torch.Tensor | None, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
                  k_out: torch.Tensor, v_out: torch.Tensor | None):
    """Gathers B sequences from their pages: page_table int32 [B, width], cu_seqlens int32
    [B + 1] ascending from 0 (token j of sequence b goes to row cu_seqlens[b] + j); k_out, v_out
    [rows, H, D] contiguous, bfloat16, float16 or float32.  Tokens without a page (an entry
    outside the cache, such as -1) become zeros; rows behind cu_seqlens[B] are left as they
    were.  Returns ``(k_out, v_out)``.  Asynchronous on the current stream."""
    mod, fast_stream = _lib.fast_module(k_cache)
    if mod is not None:
        st = mod.cache_read(k_cache, v_cache, k_scale, v_scale, page_table, cu_seqlens, k_out, v_out,
                            fast_stream)
        if st == 0:
            return k_out, v_out
        if st != _lib.FAST_ARG_ERROR:
            _lib.check(st, "fagq_kv_cache_read_launch")
        # An argument the binding leaves to the checks below.
    P, H, page, D, G, qf, sf = _check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    if (v_out is None) != (v_cache is None):
        raise ValueError("v_out, v_cache and v_scale go together")
    if k_out.dtype not in _DTYPES:
        raise TypeError(f"k_out must be bfloat16, float16 or float32, got {k_out.dtype}")
    rows = int(k_out.shape[0]) if k_out.dim() else 0
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None and (t.device != dev or t.dtype != k_out.dtype
                              or tuple(t.shape) != (rows, H, D) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {k_out.dtype} tensor of shape "
                             f"({rows}, {H}, {D}) on {dev}")
    B, width = _check_table(page_table, dev)
    if cu_seqlens.device != dev or cu_seqlens.dtype != torch.int32 or \
            tuple(cu_seqlens.shape) != (B + 1,) or not cu_seqlens.is_contiguous():
        raise ValueError(f"cu_seqlens must be a contiguous int32 tensor of shape ({B + 1},) on {dev}")
    if B == 0 or rows == 0 or H == 0:
        return k_out, v_out
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.fagq_kv_cache_read_launch(
            _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(page_table),
            _ptr(cu_seqlens), _ptr(k_out), _ptr(v_out), B, rows, H, D, G, P, page, width,
            _DTYPES[k_out.dtype], qf, sf, ctypes.c_void_p(stream))
    _lib.check(st, "fagq_kv_cache_read_launch")
    return k_out, v_out


def _check_table(page_table: torch.Tensor, dev: torch.device) -> tuple[int, int]:
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != dev \
            or not page_table.is_contiguous():
        raise ValueError(f"page_table must be a contiguous int32 [B, width] tensor on {dev}")
    return int(page_table.shape[0]), int(page_table.shape[1])


def attention_workspace_bytes(B: int, S: int, Hq: int, H: int, D: int, prefix_len: int,
                              max_kv_len: int) -> int:
    """Workspace bytes of a ``paged_attention`` of exactly these sizes, where max_kv_len is the
    smaller of its argument and the page table's capacity.  Not monotone: a smaller batch or bound
    is cut into more parts and may need more, so a workspace that serves several calls is as large
    as the largest of theirs."""
    n = _lib.load().fagq_paged_attention_workspace_bytes(B, S, Hq, H, D, prefix_len, max_kv_len)
    if n < 0:
        raise ValueError(f"no workspace size for B={B}, S={S}, Hq={Hq}, H={H}, D={D}, "
                         f"prefix_len={prefix_len}, max_kv_len={max_kv_len}")
    return n


def tree_attention_workspace_bytes(B: int, S: int, Hq: int, H: int, D: int, prefix_len: int,
                                   max_kv_len: int) -> int:
    """The same for a ``paged_tree_attention``."""
    n = _lib.load().fagq_paged_tree_attention_workspace_bytes(B, S, Hq, H, D, prefix_len, max_kv_len)
    if n < 0:
        raise ValueError(f"no workspace size for B={B}, S={S}, Hq={Hq}, H={H}, D={D}, "
                         f"prefix_len={prefix_len}, max_kv_len={max_kv_len}")
    return n


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, sm_scale: float,
                    prefix_pages: torch.Tensor | None = None, prefix_len: int = 0,
                    max_kv_len: int | None = None, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the newest S tokens of each of B sequences over the cache.

    q: bfloat16 or float16 [B, S, Hq, D] with contiguous rows at 16-byte aligned strides; D is
    64, 128 or 256, Hq a multiple of the cache's H, and the cache has one scale for each token
    and head.  page_table: int32 [B, width]; kv_lens [B] (int32 or int64) counts the tokens on
    a sequence's own pages, its newest S among them, so that token s sees the first
    ``kv_lens[b] - S + s + 1``.  Before those, every token sees the ``prefix_len`` tokens of
    ``prefix_pages`` (int32, at least ``ceil(prefix_len / page_size)``), which the batch shares
    and which is computed once for all of it.  A query that sees nothing gets zeros; tokens
    without a page (an entry outside the cache, such as -1) are left out.

    ``max_kv_len`` (default: the table's capacity) bounds kv_lens; longer ones are cut to it.  The
    split of the work and whether codes are read past the caches go by it and not by kv_lens: give
    a close one where the table is wide (up to 2.4 times as fast).  ``workspace`` (optional): a
    uint8 GPU tensor of at least ``attention_workspace_bytes(...)`` bytes for these sizes (a
    smaller call may need more), which calls that may overlap do not share.  Codes and scales of
    the tokens that are seen are finite, value scales 0 to 2^64.  Returns ``out`` [B, S, Hq, D]
    (contiguous, allocated unless given), asynchronously on the current stream."""
    mod, fast_stream = _lib.fast_module(k_cache) if workspace is None else (None, None)
    if mod is not None:
        r = mod.attention(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, sm_scale,
                          prefix_pages, prefix_len, max_kv_len, out, fast_stream)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_paged_attention_launch")
        # An argument the binding leaves to the checks below.
    return _attention(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, None, sm_scale,
                      prefix_pages, prefix_len, max_kv_len, out, workspace)


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
                         kv_lens: torch.Tensor, tree_mask: torch.Tensor, sm_scale: float,
                         prefix_pages: torch.Tensor | None = None, prefix_len: int = 0,
                         max_kv_len: int | None = None, out: torch.Tensor | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the S drafted tokens of each of B sequences over the cache: ``paged_attention``
    for a tree of drafts.  The newest S of a sequence's ``kv_lens[b]`` tokens are its drafts.  Query
    s sees the shared prefix, all tokens before the drafts, and the drafts t with
    ``tree_mask[b, s, t]`` (bool or uint8, [B, S, S], or [S, S] for all sequences; contiguous):
    itself only if the mask says so.  Where a sequence has fewer than S tokens, its first drafts do
    not exist.  Any mask will do; a query that sees nothing gets zeros, and the slots of drafts that no
    row of the mask names (a padded tree's) may hold anything.

    S is at most 4096.  The other arguments, and what is returned, as in ``paged_attention``;
    ``workspace`` has ``tree_attention_workspace_bytes(...)`` bytes.  Asynchronous on the current
    stream."""
    if not isinstance(tree_mask, torch.Tensor):
        raise TypeError(f"tree_mask must be a tensor, got {type(tree_mask).__name__}")
    mod, fast_stream = _lib.fast_module(k_cache) if workspace is None else (None, None)
    if mod is not None:
        r = mod.tree_attention(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, sm_scale,
                               prefix_pages, prefix_len, max_kv_len, out, fast_stream, tree_mask)
        if type(r) is not int:
            return r
        if r != _lib.FAST_ARG_ERROR:
            _lib.check(r, "fagq_paged_tree_attention_launch")
        # An argument the binding leaves to the checks below.
    return _attention(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, tree_mask, sm_scale,
                      prefix_pages, prefix_len, max_kv_len, out, workspace)


def _attention(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, tree_mask, sm_scale,
               prefix_pages, prefix_len, max_kv_len, out, workspace):
    """Either attention from its checks on; tree_mask: None without a tree."""
    P, H, page, D, G, qf, sf = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if v_cache is None:
        name = "paged_attention" if tree_mask is None else "paged_tree_attention"
        raise ValueError(f"{name} needs a cache of keys and values")
    dev = k_cache.device
    if q.dim() != 4 or q.shape[3] != D:
        raise ValueError(f"q must be [B, S, Hq, {D}], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    B, S, Hq = (int(s) for s in q.shape[:3])
    if D not in ATTENTION_DIMS or G != D:
        raise ValueError(f"attention takes one scale for each token and head and a head dim of "
                         f"{ATTENTION_DIMS}, got {D // G} for {D}")
    if H < 1 or Hq < 1 or Hq % H:
        raise ValueError(f"{Hq} query heads do not share {H} cache heads evenly")
    if q.device != dev or q.stride(3) != 1:
        raise ValueError(f"q must be on {dev} with contiguous rows, strides {q.stride()}")
    tb, width = _check_table(page_table, dev)
    idx = index_code(kv_lens, "kv_lens")
    if tb != B:
        raise ValueError(f"page_table must have {B} rows, got {tb}")
    if kv_lens.device != dev or tuple(kv_lens.shape) != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be a contiguous tensor of shape ({B},) on {dev}")
    if tree_mask is not None and (
            tree_mask.device != dev or tree_mask.dtype not in (torch.bool, torch.uint8)
            or tuple(tree_mask.shape) not in ((B, S, S), (S, S)) or not tree_mask.is_contiguous()):
        raise ValueError(f"tree_mask must be a contiguous bool or uint8 tensor of shape ({B}, {S}, {S}) "
                         f"or ({S}, {S}) on {dev}")
    prefix_len = int(prefix_len)
    if prefix_len < 0:
        raise ValueError(f"prefix_len must not be negative, got {prefix_len}")
    if prefix_len:
        need = -(-prefix_len // page)
        if prefix_pages is None or prefix_pages.device != dev or prefix_pages.dim() != 1 \
                or prefix_pages.dtype != torch.int32 or not prefix_pages.is_contiguous() \
                or prefix_pages.shape[0] < need:
            raise ValueError(f"prefix_pages must be a contiguous int32 tensor of at least {need} "
                             f"pages on {dev}")
    room = width * page
    most = room if max_kv_len is None else min(int(max_kv_len), room)
    if most < 0:
        raise ValueError(f"max_kv_len must not be negative, got {max_kv_len}")
    if out is None:
        out = torch.empty(B, S, Hq, D, dtype=q.dtype, device=dev)
    elif out.dtype != q.dtype or tuple(out.shape) != (B, S, Hq, D) or not out.is_contiguous() \
            or out.device != dev:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of shape {(B, S, Hq, D)} on {dev}")
    if B == 0 or S == 0:
        return out
    if P == 0:
        return out.zero_()
    size = attention_workspace_bytes if tree_mask is None else tree_attention_workspace_bytes
    need = size(B, S, Hq, H, D, prefix_len, most)
    if workspace is not None:
        check_workspace(workspace, need, dev)
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    strides = [q.stride(i) if q.shape[i] > 1 else 0 for i in range(3)]
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        head = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                _ptr(page_table) if width else None, _ptr(kv_lens),
                _ptr(prefix_pages) if prefix_len else None)
        rest = (_ptr(out), _ptr(workspace) if need else None,
                workspace.numel() * workspace.element_size() if need else 0,
                (ctypes.c_int64 * 3)(*strides), B, S, Hq, H, D, P, page, width, prefix_len, most,
                float(sm_scale), _DTYPES[q.dtype], qf, sf, idx, ctypes.c_void_p(stream))
        if tree_mask is None:
            name, st = "fagq_paged_attention_launch", lib.fagq_paged_attention_launch(*head, *rest)
        else:
            name = "fagq_paged_tree_attention_launch"
            st = lib.fagq_paged_tree_attention_launch(*head, _ptr(tree_mask),
                                                      int(tree_mask.dim() == 2), *rest)
    _lib.check(st, name)
    return out
