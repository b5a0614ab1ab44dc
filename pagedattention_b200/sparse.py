"""Page-sparse decode: attend to the pages of a context that a query's bound
ranks highest.

The reference attends to every page (src/kernel_triton.py:8-117) and has no
counterpart.  ``update_page_bounds`` keeps, for every page of a cache of any
kind, the elementwise minimum and maximum of its keys as tokens are appended;
``select_pages`` scores the pages of every (sequence, kv head) with them and
returns the block tables and lengths of those to attend to, which any decode
entry point takes; ``paged_attention_sparse`` selects and attends in one call.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .int4_cache import _check_offsets, _length_strides
from .kernel_b200 import (_DTYPES, _append_status_word, _as_int32, _check_device,
                          _current_stream_handle, _keep_workspace, _paged_args, _raise_for)


def _check_bounds(page_bounds, block_table, num_seqs, num_kv_heads, head_size, dtype):
    """Checks of the bounds and their table; returns (table, page count, page
    mul, page add, max_blocks, table strides)."""
    if page_bounds.dtype != dtype:
        raise TypeError(f"page_bounds must have the keys' dtype {dtype}, got {page_bounds.dtype}")
    if not page_bounds.is_contiguous():
        raise ValueError("page_bounds must be contiguous")
    if tuple(page_bounds.shape[-2:]) != (2, head_size):
        raise ValueError("page_bounds must end in (2, head_size)")
    bt = _as_int32(block_table, "block_table")
    if page_bounds.dim() == 4:
        if page_bounds.shape[1] != num_kv_heads:
            raise ValueError(f"page_bounds has {page_bounds.shape[1]} kv heads, not {num_kv_heads}")
        num_pages, mul, add = page_bounds.shape[0] * num_kv_heads, num_kv_heads, 1
    elif page_bounds.dim() == 3:
        if bt.dim() != 3:
            raise ValueError("3-D (per-head page) bounds need a block table "
                             "(num_seqs, num_kv_heads, max_blocks)")
        num_pages, mul, add = page_bounds.shape[0], 1, 0
    else:
        raise ValueError("page_bounds must be (num_blocks, num_kv_heads, 2, head_size) or "
                         "(num_pages, 2, head_size)")
    if bt.dim() == 3 and tuple(bt.shape[:2]) == (num_seqs, num_kv_heads):
        strides, maxb = bt.stride(), bt.shape[2]
    elif bt.dim() == 2 and bt.shape[0] == num_seqs:
        strides, maxb = (bt.stride(0), 0, bt.stride(1)), bt.shape[1]
    else:
        raise ValueError("block table must be (num_seqs, max_blocks) or "
                         "(num_seqs, num_kv_heads, max_blocks)")
    return bt, num_pages, mul, add, maxb, strides


def update_page_bounds(page_bounds, k_new, cache_seqlens, block_table, block_size, cu_new=None):
    """Bounds of the pages that new tokens go to, in place.

    page_bounds: (num_blocks, num_kv_heads, 2, head_size) for a pool of either
    layout or (num_pages, 2, head_size) for per-head pages, of the keys' dtype:
    minimum and maximum.  k_new, cu_new as for ``kv_append_int4``;
    cache_seqlens: the lengths BEFORE the tokens (call this before the append
    that advances them), not changed here.  A page whose first row is new starts
    afresh, any other is widened.  Tokens without a place are left out and set a
    bit read by ``kv_append_status``.
    """
    if k_new.dim() != 3:
        raise ValueError("k_new must be (num_tokens, num_kv_heads, head_size)")
    if k_new.dtype not in _DTYPES:
        raise TypeError(f"k_new must be bfloat16 or float16, got {k_new.dtype}")
    if k_new.stride(2) != 1:
        raise ValueError("k_new must be contiguous in head_size")
    N, Hkv, D = k_new.shape
    lens = _as_int32(cache_seqlens, "cache_seqlens")
    B = lens.shape[0]
    cu = _check_offsets(cu_new, B, "cu_new")
    if cu is None and N != B:
        raise ValueError(f"{N} tokens for {B} sequences need cu_new")
    bt, num_pages, mul, add, maxb, bts = _check_bounds(page_bounds, block_table, B, Hkv, D,
                                                       k_new.dtype)
    lsb, lsh = _length_strides(lens, B, Hkv, "cache_seqlens")
    device = _check_device(*([page_bounds, k_new, lens, bt] + ([] if cu is None else [cu])))
    a = _lib.PageBoundsArgs()
    a.page_bounds, a.k_rows = page_bounds.data_ptr(), k_new.data_ptr()
    a.seqlens, a.block_table = lens.data_ptr(), bt.data_ptr()
    a.cu_tokens = None if cu is None else cu.data_ptr()
    a.status = _append_status_word(device).data_ptr()
    a.dtype, a.num_seqs, a.num_kv_heads = _DTYPES[k_new.dtype], B, Hkv
    a.head_size, a.block_size, a.max_blocks = D, block_size, maxb
    a.num_pages, a.num_tokens = num_pages, N
    a.row_stride_t, a.row_stride_h = k_new.stride(0), k_new.stride(1)
    a.seqlens_stride_b, a.seqlens_stride_h = lsb, lsh
    a.bt_stride_b, a.bt_stride_h, a.bt_stride_i = bts
    a.bounds_page_mul, a.bounds_page_add = mul, add
    lib = _lib.load()
    with torch.cuda.device(device):
        rc = lib.pab200_update_page_bounds(ctypes.byref(a), _current_stream_handle(device))
    _raise_for(lib, rc, "pab200_update_page_bounds")


def _select_args(query, page_bounds, block_tables, context_lens, block_size, num_selected, num_sink,
                 num_recent, num_kv_heads):
    if query.dim() != 3:
        raise ValueError("query must be (num_seqs, num_q_heads, head_size)")
    if query.dtype not in _DTYPES:
        raise TypeError(f"query must be bfloat16 or float16, got {query.dtype}")
    if query.stride(2) != 1:
        raise ValueError("query must be contiguous in head_size")
    if num_sink < 0 or num_recent < 1 or num_sink + num_recent > num_selected:
        raise ValueError("need num_sink >= 0, num_recent >= 1 and "
                         "num_sink + num_recent <= num_selected")
    B, Hq, D = query.shape
    if B < 1 or Hq % num_kv_heads != 0:
        raise ValueError(f"num_q_heads {Hq} is not a multiple of num_kv_heads {num_kv_heads}, "
                         "or there is no sequence")
    bt, num_pages, mul, add, maxb, bts = _check_bounds(page_bounds, block_tables, B, num_kv_heads, D,
                                                       query.dtype)
    lens = _as_int32(context_lens, "context_lens")
    lsb, lsh = _length_strides(lens, B, num_kv_heads, "context_lens")
    device = _check_device(query, page_bounds, bt, lens)
    tables = torch.empty((B, num_kv_heads, num_selected), dtype=torch.int32, device=device)
    out_lens = torch.empty((B, num_kv_heads), dtype=torch.int32, device=device)
    a = _lib.SelectArgs()
    a.q, a.page_bounds = query.data_ptr(), page_bounds.data_ptr()
    a.seqlens, a.block_table = lens.data_ptr(), bt.data_ptr()
    a.tables, a.selected_lens = tables.data_ptr(), out_lens.data_ptr()
    a.status = _append_status_word(device).data_ptr()
    a.dtype, a.num_seqs, a.num_q_heads, a.num_kv_heads = _DTYPES[query.dtype], B, Hq, num_kv_heads
    a.head_size, a.block_size, a.max_blocks = D, block_size, maxb
    a.num_selected, a.num_sink, a.num_recent = num_selected, num_sink, num_recent
    a.num_pages = num_pages
    a.q_stride_b, a.q_stride_h = query.stride(0), query.stride(1)
    a.seqlens_stride_b, a.seqlens_stride_h = lsb, lsh
    a.bt_stride_b, a.bt_stride_h, a.bt_stride_i = bts
    a.bounds_page_mul, a.bounds_page_add = mul, add
    return a, device, tables, out_lens, (bt, lens)


def select_pages(query, page_bounds, block_tables, context_lens, block_size, num_selected,
                 num_sink=1, num_recent=1):
    """The pages of every (sequence, kv head) that ``query`` attends to.

    Returns (tables, lens): int32 block tables (num_seqs, num_kv_heads,
    num_selected), the entries of ``block_tables`` for the kept pages in
    ascending page order and -1 behind them, and int32 lens (num_seqs,
    num_kv_heads), their tokens.  Both go to ``paged_attention``,
    ``paged_attention_states`` or ``paged_attention_int4`` as they are.

    A context of at most ``num_selected`` pages keeps them all.  Otherwise its
    first ``num_sink`` and last ``num_recent`` (>= 1) pages are kept, and of the
    others those with the highest score: the sum over the kv head's query group
    and the head elements of max(q * min, q * max), which no token of the page
    exceeds.  Scores are summed in 64 bits and rounded to fp32; ties go to the
    earlier page, a NaN score ranks first.  query: (num_seqs, num_q_heads,
    head_size); page_bounds as kept by ``update_page_bounds``; block_tables,
    context_lens as for ``paged_attention``.
    """
    heads = page_bounds.shape[1] if page_bounds.dim() == 4 else block_tables.shape[1]
    a, device, tables, lens, keep = _select_args(query, page_bounds, block_tables, context_lens,
                                                 block_size, num_selected, num_sink, num_recent,
                                                 heads)
    lib = _lib.load()
    with torch.cuda.device(device):
        need = lib.pab200_select_pages_workspace_size(ctypes.byref(a))
        if need == 0:
            raise ValueError(f"pab200_select_pages: {lib.pab200_last_error().decode()}")
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        rc = lib.pab200_select_pages(ctypes.byref(a), ws.data_ptr(), need,
                                     _current_stream_handle(device))
    _raise_for(lib, rc, "pab200_select_pages")
    del keep
    return tables, lens


def paged_attention_sparse(out, query, key_cache, value_cache, page_bounds, block_tables,
                           context_lens, scale, block_size, num_selected, num_sink=1, num_recent=1,
                           kv_layout="HND", num_splits=0):
    """In-place paged decode over the pages ``select_pages`` keeps: writes
    ``out`` and returns the (tables, lens) it attended to.

    Arguments as for ``paged_attention`` (16-bit caches of either layout) and
    ``select_pages``.
    """
    args, device, keep = _paged_args(query, key_cache, value_cache, block_tables, context_lens,
                                     scale, block_size, kv_layout, num_splits)
    if out.shape != query.shape or out.dtype != query.dtype or out.device != device:
        raise ValueError("out must match query in shape, dtype and device")
    if out.stride(2) != 1:
        raise ValueError("out must be contiguous in head_size")
    if num_splits < 0:
        raise ValueError("num_splits must be >= 0")
    args.out = out.data_ptr()
    args.out_stride_b, args.out_stride_h = out.stride(0), out.stride(1)
    sel, dev, tables, lens, kept = _select_args(query, page_bounds, block_tables, context_lens,
                                                block_size, num_selected, num_sink, num_recent,
                                                args.num_kv_heads)
    if dev != device:
        raise ValueError(f"page_bounds must be on {device}")
    lib = _lib.load()
    with torch.cuda.device(device):
        need = lib.pab200_decode_sparse_workspace_size(ctypes.byref(args), ctypes.byref(sel))
        if need == 0:
            raise ValueError(f"pab200_decode_sparse: {lib.pab200_last_error().decode()}")
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        stream = _current_stream_handle(device)
        rc = lib.pab200_decode_sparse(ctypes.byref(args), ctypes.byref(sel), ws.data_ptr(), need,
                                      stream)
    _raise_for(lib, rc, "pab200_decode_sparse")
    _keep_workspace(device, ws, stream)
    del keep, kept
    return tables, lens
