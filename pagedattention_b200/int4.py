"""4-bit page caches: append, read-back and decode attention.

The reference's caches hold 16-bit rows (src/common.py:1-14) and it has no
counterpart.  A 4-bit cache is a uint8 tensor of pages, one per (sequence, kv
head)'s block of ``block_size`` tokens, ``int4_page_bytes(head_size,
block_size)`` bytes each: a pool (num_blocks, num_kv_heads, page_bytes) with
block tables (num_seqs, max_blocks), or pages (num_pages, page_bytes) with
per-head block tables (num_seqs, num_kv_heads, max_blocks).  ``int4_cache``
allocates a pool.

Rows are quantised in groups of 64 elements: minimum lo and scale s = T((max -
lo) / 15) in the rows' 16-bit type T, codes rint((x - lo) / s) in 0..15.  A
group stands for lo + s * code; a group with a NaN or an infinity for NaN.  A
page takes 9/32 of the bytes of its 16-bit rows.
"""
from __future__ import annotations

import torch

from . import _lib
from .kernel_b200 import (_DTYPES, _append_status_word, _as_int32, _call_with_workspace,
                          _check_device, _keep_workspace, _on_device, _raise_for, _take_events)

_HEAD_SIZES = (64, 128, 256)
_BLOCK_SIZES = (8, 16, 32, 64)


def _append_status_ptr(device) -> int:
    return _append_status_word(device).data_ptr()


def int4_page_bytes(head_size: int, block_size: int) -> int:
    """Bytes of one page of a 4-bit cache (block_size * head_size * 9 / 16)."""
    if head_size not in _HEAD_SIZES or block_size not in _BLOCK_SIZES:
        raise ValueError(f"head_size must be one of {_HEAD_SIZES} and block_size one of "
                         f"{_BLOCK_SIZES}, got {head_size} and {block_size}")
    return block_size * head_size * 9 // 16


def int4_cache(num_blocks, num_kv_heads, block_size, head_size, device="cuda"):
    """Two zeroed 4-bit pools (num_blocks, num_kv_heads, page_bytes): keys and
    values."""
    shape = (num_blocks, num_kv_heads, int4_page_bytes(head_size, block_size))
    return tuple(torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))


def _check_table(block_table, num_seqs, num_kv_heads):
    """The block table as int32, its max_blocks and strides (b, h, i)."""
    bt = _as_int32(block_table, "block_table")
    shape, st = bt.shape, bt.stride()
    if len(shape) == 2 and shape[0] == num_seqs:
        return bt, shape[1], (st[0], 0, st[1])
    if len(shape) == 3 and shape[0] == num_seqs and shape[1] == num_kv_heads:
        return bt, shape[2], st
    raise ValueError("block table must be (num_seqs, max_blocks) or "
                     "(num_seqs, num_kv_heads, max_blocks)")


def _check_caches(key_cache, value_cache, block_table, head_size, block_size, num_seqs,
                  num_kv_heads):
    """Checks of the caches and their table; returns (table, page count, kv
    heads, bt_page_mul, bt_page_add, max_blocks, table strides)."""
    if key_cache.dtype != torch.uint8 or value_cache.dtype != torch.uint8:
        raise TypeError("4-bit caches must be uint8 tensors")
    shape = key_cache.shape
    if shape != value_cache.shape:
        raise ValueError("key_cache and value_cache shapes differ")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("key_cache and value_cache must be contiguous")
    if shape[-1] != int4_page_bytes(head_size, block_size):
        raise ValueError(f"pages of {shape[-1]} bytes, head_size {head_size} and "
                         f"block_size {block_size} need {int4_page_bytes(head_size, block_size)}")
    if len(shape) == 3:
        heads = shape[1]
        num_pages, mul, add = shape[0] * heads, heads, 1
    elif len(shape) == 2:
        if block_table.dim() != 3:
            raise ValueError("a 2-D (per-head page) cache needs a block table "
                             "(num_seqs, num_kv_heads, max_blocks)")
        num_pages, heads, mul, add = shape[0], block_table.shape[1], 1, 0
    else:
        raise ValueError(f"unsupported 4-bit cache rank {len(shape)}")
    if num_kv_heads is not None and heads != num_kv_heads:
        raise ValueError(f"cache has {heads} kv heads, the rows {num_kv_heads}")
    bt, maxb, strides = _check_table(block_table, num_seqs, heads)
    return bt, num_pages, heads, mul, add, maxb, strides


def _length_strides(lens, num_seqs, heads, name):
    shape = lens.shape
    if len(shape) == 1 and shape[0] == num_seqs:
        return lens.stride(0), 0
    if len(shape) == 2 and shape[0] == num_seqs and shape[1] == heads:
        return lens.stride()
    raise ValueError(f"{name} must be (num_seqs,) or (num_seqs, num_kv_heads)")


def _check_offsets(cu, num_seqs, name):
    """Token offsets: an int32 tensor (num_seqs + 1,), or None."""
    if cu is None:
        return None
    if cu.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if cu.dim() != 1 or cu.shape[0] != num_seqs + 1 or not cu.is_contiguous():
        raise ValueError(f"{name} must be a contiguous (num_seqs + 1,) tensor")
    return cu


def _rows_args(key_cache, value_cache, k, v, lens, block_table, cu, block_size, what):
    """The arguments append and read-back share."""
    shape, st = k.shape, k.stride()
    if len(shape) != 3 or shape != v.shape:
        raise ValueError(f"{what} must be (num_tokens, num_kv_heads, head_size)")
    code = _DTYPES.get(k.dtype)
    if code is None or v.dtype != k.dtype:
        raise TypeError(f"{what} must share one dtype, bfloat16 or float16")
    N, Hkv, D = shape
    vst = v.stride()
    # the stride of a dimension of one element means nothing
    st_t, st_h = (st[0] if N > 1 else 0), (st[1] if Hkv > 1 else 0)
    if (st[2] != 1 or vst[2] != 1 or (N > 1 and vst[0] != st_t) or (Hkv > 1 and vst[1] != st_h)):
        raise ValueError(f"{what} must share strides, contiguous in head_size")
    B = lens.shape[0]
    bt, num_pages, _, mul, add, maxb, bts = _check_caches(key_cache, value_cache, block_table, D,
                                                          block_size, B, Hkv)
    lsb, lsh = _length_strides(lens, B, Hkv, "cache_seqlens")
    if cu is None:
        if N != B:
            raise ValueError(f"{N} tokens for {B} sequences need token offsets")
        device = _check_device(key_cache, value_cache, k, v, lens, bt)
    else:
        device = _check_device(key_cache, value_cache, k, v, lens, bt, cu)
    args = _lib.Int4RowsArgs(
        key_cache.data_ptr(), value_cache.data_ptr(), k.data_ptr(), v.data_ptr(), lens.data_ptr(),
        bt.data_ptr(), None if cu is None else cu.data_ptr(), _append_status_ptr(device), code, B, Hkv,
        D, block_size, maxb, num_pages, N, st_t, st_h, lsb, lsh, *bts, mul, add)
    return args, device, bt


def kv_append_int4(key_cache, value_cache, k_new, v_new, cache_seqlens, block_table, block_size,
                   cu_new=None, increment=True):
    """Quantise new tokens into a 4-bit cache, in place.

    The 4-bit form of ``kv_append``, for one token per sequence or for ragged
    runs of them (prompts).  k_new, v_new: (num_tokens, num_kv_heads,
    head_size), bfloat16 or float16.  ``cu_new``: int32 (num_seqs + 1,), ascending
    in 0 .. num_tokens, tokens cu_new[s] .. cu_new[s+1] - 1 belong to sequence s
    (one whose offsets are out of order or range is left out); None: one token per
    sequence.  cache_seqlens: int32 (num_seqs,) or (num_seqs, num_kv_heads), the
    lengths L before the call; token j goes to position L + j and, with
    ``increment``, L grows in place by the tokens written (sequences may not share
    one length).  Tokens from the
    first one without a page slot or with an invalid page id are not counted,
    and a bit read by ``kv_append_status`` is set.
    """
    if cache_seqlens.dtype != torch.int32:
        raise TypeError("cache_seqlens must be int32 (it is updated in place)")
    cu = _check_offsets(cu_new, cache_seqlens.shape[0], "cu_new")
    a, device, keep = _rows_args(key_cache, value_cache, k_new, v_new, cache_seqlens, block_table,
                                 cu, block_size, "k_new and v_new")
    lib = _lib.load()
    rc = _on_device(device, lib.pab200_kv_append_int4, a, 1 if increment else 0)
    if rc:
        _raise_for(lib, rc, "pab200_kv_append_int4")
    del keep


def kv_read_int4(key_cache, value_cache, block_table, cache_seqlens, block_size, head_size, dtype,
                 starts=None, cu_out=None, num_tokens=None, out=None):
    """Read tokens of a 4-bit cache back as 16-bit rows.

    Returns (k, v), each (num_tokens, num_kv_heads, head_size) of ``dtype``, the
    type the tokens were appended in.  Rows cu_out[s] .. cu_out[s+1] - 1 are
    positions starts[s], starts[s] + 1, ... of sequence s (``starts`` None: from
    0); ``cu_out`` int32 (num_seqs + 1,), ascending in 0 .. ``num_tokens``, the
    rows in all (rows of a sequence whose offsets are not are not written), or
    None: one row per sequence.  Positions at or past cache_seqlens and pages
    with an invalid id read as zeros, and so do rows of no sequence.  ``out``: a
    (k, v) pair to fill; its rows of no sequence are left as they were.
    """
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    lens = _as_int32(cache_seqlens, "cache_seqlens")
    B = lens.shape[0]
    cu = _check_offsets(cu_out, B, "cu_out")
    fresh = out is None
    if fresh:
        if cu is not None and num_tokens is None:
            raise ValueError("cu_out needs num_tokens (or out)")
        n = B if cu is None else int(num_tokens)
        heads = key_cache.shape[1] if key_cache.dim() == 3 else block_table.shape[1]
        k, v = torch.empty((2, n, heads, head_size), dtype=dtype,
                           device=key_cache.device).unbind(0)
    else:
        k, v = out
    if k.dtype != dtype or k.dim() != 3 or k.shape[2] != head_size:
        raise ValueError("out must be a pair of (num_tokens, num_kv_heads, head_size) of dtype")
    if starts is not None:
        starts = _as_int32(starts, "starts")
        if starts.dim() != 1 or starts.shape[0] != B:
            raise ValueError("starts must be (num_seqs,)")
        _check_device(key_cache, starts)
        first, step = starts.data_ptr(), starts.stride(0)
    else:
        first, step = None, 0
    a, device, keep = _rows_args(key_cache, value_cache, k, v, lens, block_table, cu, block_size,
                                 "out")
    lib = _lib.load()
    rc = _on_device(device, lib.pab200_kv_read_int4, a, first, step, 1 if fresh else 0)
    if rc:
        _raise_for(lib, rc, "pab200_kv_read_int4")
    del keep
    return k, v


def paged_attention_int4(out, query, key_cache, value_cache, block_tables, context_lens, scale,
                         block_size, num_splits=0):
    """In-place paged decode over 4-bit caches: ``paged_attention`` with the
    caches of ``kv_append_int4``, appended in query's dtype.

    out, query: (num_seqs, num_q_heads, head_size); block_tables (num_seqs,
    max_blocks) or, per kv head, (num_seqs, num_kv_heads, max_blocks);
    context_lens (num_seqs,) or (num_seqs, num_kv_heads).  Query groups as for
    ``paged_attention``.  ``out`` must not overlap ``query``.  An invalid page id
    reads as rows of zeros and sets a bit read by ``read_status``.
    """
    shape, qst, ost = query.shape, query.stride(), out.stride()
    if len(shape) != 3:
        raise ValueError("query must be (num_seqs, num_q_heads, head_size)")
    code = _DTYPES.get(query.dtype)
    if code is None:
        raise TypeError(f"query must be bfloat16 or float16, got {query.dtype}")
    if qst[2] != 1:
        raise ValueError("query must be contiguous in head_size")
    if out.shape != shape or out.dtype != query.dtype:
        raise ValueError("out must match query in shape and dtype")
    if ost[2] != 1:
        raise ValueError("out must be contiguous in head_size")
    if out.data_ptr() == query.data_ptr() and query.numel():
        raise ValueError("out must not be query: queries are read until the call ends")
    if num_splits < 0:
        raise ValueError("num_splits must be >= 0")
    B, Hq, D = shape
    bt, num_pages, Hkv, mul, add, maxb, bts = _check_caches(key_cache, value_cache, block_tables, D,
                                                            block_size, B, None)
    if Hq % Hkv != 0:
        raise ValueError(f"num_q_heads {Hq} is not a multiple of num_kv_heads {Hkv}")
    lens = _as_int32(context_lens, "context_lens")
    lsb, lsh = _length_strides(lens, B, Hkv, "context_lens")
    device = _check_device(query, out, key_cache, value_cache, bt, lens)
    if B == 0:
        return
    args = _lib.DecodeArgs(
        out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        lens.data_ptr(), bt.data_ptr(), code, _lib.LAYOUT_PAGES, B, Hq, Hkv, D, block_size, maxb,
        num_pages, qst[0], qst[1], ost[0], ost[1], lsb, lsh, *bts, mul, add, float(scale),
        int(num_splits))
    _on_device(device, _run_int4, args, device)


def _run_int4(args, device, stream):
    _take_events(args)
    ws = _call_with_workspace(
        _lib.load(), "pab200_decode_int4", device,
        (args.dtype, args.num_seqs, args.num_q_heads, args.num_kv_heads, args.head_size,
         args.block_size, args.max_blocks, args.num_splits), (args,), stream)
    _keep_workspace(device, ws, stream)
