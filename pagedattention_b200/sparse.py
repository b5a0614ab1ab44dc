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

import torch

from . import _lib
from .int4 import _append_status_ptr, _check_offsets, _check_table, _length_strides
from .kernel_b200 import (_DTYPES, _as_int32, _call_with_workspace, _check_device,
                          _keep_workspace, _on_device, _paged_args, _raise_for, _take_events)


def _check_bounds(page_bounds, block_table, num_seqs, num_kv_heads, head_size, dtype):
    """Checks of the bounds and their table; returns (table, page count, page
    mul, page add, max_blocks, table strides)."""
    if page_bounds.dtype != dtype:
        raise TypeError(f"page_bounds must have the keys' dtype {dtype}, got {page_bounds.dtype}")
    if not page_bounds.is_contiguous():
        raise ValueError("page_bounds must be contiguous")
    shape = page_bounds.shape
    if len(shape) < 2 or shape[-2] != 2 or shape[-1] != head_size:
        raise ValueError("page_bounds must end in (2, head_size)")
    if len(shape) == 4:
        if shape[1] != num_kv_heads:
            raise ValueError(f"page_bounds has {shape[1]} kv heads, not {num_kv_heads}")
        num_pages, mul, add = shape[0] * num_kv_heads, num_kv_heads, 1
    elif len(shape) == 3:
        if block_table.dim() != 3:
            raise ValueError("3-D (per-head page) bounds need a block table "
                             "(num_seqs, num_kv_heads, max_blocks)")
        num_pages, mul, add = shape[0], 1, 0
    else:
        raise ValueError("page_bounds must be (num_blocks, num_kv_heads, 2, head_size) or "
                         "(num_pages, 2, head_size)")
    bt, maxb, strides = _check_table(block_table, num_seqs, num_kv_heads)
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
    shape, st = k_new.shape, k_new.stride()
    if len(shape) != 3:
        raise ValueError("k_new must be (num_tokens, num_kv_heads, head_size)")
    code = _DTYPES.get(k_new.dtype)
    if code is None:
        raise TypeError(f"k_new must be bfloat16 or float16, got {k_new.dtype}")
    if st[2] != 1:
        raise ValueError("k_new must be contiguous in head_size")
    N, Hkv, D = shape
    lens = _as_int32(cache_seqlens, "cache_seqlens")
    B = lens.shape[0]
    cu = _check_offsets(cu_new, B, "cu_new")
    bt, num_pages, mul, add, maxb, bts = _check_bounds(page_bounds, block_table, B, Hkv, D,
                                                       k_new.dtype)
    lsb, lsh = _length_strides(lens, B, Hkv, "cache_seqlens")
    if cu is None:
        if N != B:
            raise ValueError(f"{N} tokens for {B} sequences need cu_new")
        device = _check_device(page_bounds, k_new, lens, bt)
    else:
        device = _check_device(page_bounds, k_new, lens, bt, cu)
    a = _lib.PageBoundsArgs(
        page_bounds.data_ptr(), k_new.data_ptr(), lens.data_ptr(), bt.data_ptr(),
        None if cu is None else cu.data_ptr(), _append_status_ptr(device), code, B, Hkv, D,
        block_size, maxb, num_pages, N, st[0], st[1], lsb, lsh, *bts, mul, add)
    lib = _lib.load()
    rc = _on_device(device, lib.pab200_update_page_bounds, a)
    if rc:
        _raise_for(lib, rc, "pab200_update_page_bounds")


def _select_args(query, page_bounds, block_tables, context_lens, block_size, num_selected, num_sink,
                 num_recent, num_kv_heads):
    shape, qst = query.shape, query.stride()
    if len(shape) != 3:
        raise ValueError("query must be (num_seqs, num_q_heads, head_size)")
    code = _DTYPES.get(query.dtype)
    if code is None:
        raise TypeError(f"query must be bfloat16 or float16, got {query.dtype}")
    if qst[2] != 1:
        raise ValueError("query must be contiguous in head_size")
    if num_sink < 0 or num_recent < 1 or num_sink + num_recent > num_selected:
        raise ValueError("need num_sink >= 0, num_recent >= 1 and "
                         "num_sink + num_recent <= num_selected")
    B, Hq, D = shape
    if Hq % num_kv_heads != 0:
        raise ValueError(f"num_q_heads {Hq} is not a multiple of num_kv_heads {num_kv_heads}")
    bt, num_pages, mul, add, maxb, bts = _check_bounds(page_bounds, block_tables, B, num_kv_heads, D,
                                                       query.dtype)
    lens = _as_int32(context_lens, "context_lens")
    lsb, lsh = _length_strides(lens, B, num_kv_heads, "context_lens")
    device = _check_device(query, page_bounds, bt, lens)
    tables = torch.empty((B, num_kv_heads, num_selected), dtype=torch.int32, device=device)
    out_lens = torch.empty((B, num_kv_heads), dtype=torch.int32, device=device)
    a = _lib.SelectArgs(
        query.data_ptr(), page_bounds.data_ptr(), lens.data_ptr(), bt.data_ptr(), tables.data_ptr(),
        out_lens.data_ptr(), _append_status_ptr(device), code, B, Hq, num_kv_heads, D, block_size,
        maxb, num_selected, num_sink, num_recent, num_pages, qst[0], qst[1], lsb, lsh, *bts, mul, add)
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
    exceeds.  Scores are those of a sum in 64 bits, rounded to fp32; ties go to the
    earlier page, a NaN score (a NaN in the query or the bounds, 0 times an
    infinite bound) ranks first, an invalid page id last (it, and a
    length out of range, set bits read by ``kv_append_status``).  At most 65,535
    (sequence, kv head) pairs.  query: (num_seqs, num_q_heads,
    head_size); page_bounds as kept by ``update_page_bounds``; block_tables,
    context_lens as for ``paged_attention``.
    """
    heads = page_bounds.shape[1] if page_bounds.dim() == 4 else block_tables.shape[1]
    a, device, tables, lens, keep = _select_args(query, page_bounds, block_tables, context_lens,
                                                 block_size, num_selected, num_sink, num_recent,
                                                 heads)
    if a.num_seqs:
        _on_device(device, _run_select, a, device)
    del keep
    return tables, lens


def _run_select(a, device, stream):
    _call_with_workspace(_lib.load(), "pab200_select_pages", device,
                         (a.num_seqs, a.num_kv_heads, a.max_blocks), (a,), stream)


def paged_attention_sparse(out, query, key_cache, value_cache, page_bounds, block_tables,
                           context_lens, scale, block_size, num_selected, num_sink=1, num_recent=1,
                           kv_layout="HND", num_splits=0):
    """In-place paged decode over the pages ``select_pages`` keeps: writes
    ``out`` and returns the (tables, lens) it attended to.

    Arguments as for ``paged_attention`` (16-bit caches of either layout) and
    ``select_pages``, whose ranking takes ``scale`` for positive; ``out`` must not
    overlap ``query``.
    """
    args, device, keep = _paged_args(query, key_cache, value_cache, block_tables, context_lens,
                                     scale, block_size, kv_layout, num_splits)
    if out.shape != query.shape or out.dtype != query.dtype or out.device != device:
        raise ValueError("out must match query in shape, dtype and device")
    if out.stride(2) != 1:
        raise ValueError("out must be contiguous in head_size")
    if out.data_ptr() == query.data_ptr() and query.numel():
        raise ValueError("out must not be query: queries are read until the call ends")
    if num_splits < 0:
        raise ValueError("num_splits must be >= 0")
    args.out = out.data_ptr()
    args.out_stride_b, args.out_stride_h = out.stride(0), out.stride(1)
    sel, dev, tables, lens, kept = _select_args(query, page_bounds, block_tables, context_lens,
                                                block_size, num_selected, num_sink, num_recent,
                                                args.num_kv_heads)
    if dev != device:
        raise ValueError(f"page_bounds must be on {device}")
    if args.num_seqs:
        _on_device(device, _run_sparse, args, sel, device)
    del keep, kept
    return tables, lens


def _run_sparse(args, sel, device, stream):
    _take_events(args)
    ws = _call_with_workspace(
        _lib.load(), "pab200_decode_sparse", device,
        (args.dtype, args.num_seqs, args.num_q_heads, args.num_kv_heads, args.head_size,
         args.block_size, args.num_splits, sel.max_blocks, sel.num_selected), (args, sel), stream)
    _keep_workspace(device, ws, stream)
