"""4-bit and page-sparse operators without a GPU: struct layouts, host-side
refusals of the C ABI and of the Python entry points, and the oracle's format."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import pagedattention_b200 as pa
from oracle import pages as op
from pagedattention_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("struct,mirror", [("pab200_int4_rows_args", _lib.Int4RowsArgs),
                                           ("pab200_page_bounds_args", _lib.PageBoundsArgs),
                                           ("pab200_select_args", _lib.SelectArgs)])
def test_struct_layouts_match_c(tmp_path, struct, mirror):
    fields = [f for f, _ in mirror._fields_]
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "pab200.h"', 'int main(void){',
           f'printf("size %zu\\n", sizeof({struct}));']
    src += [f'printf("{f} %zu\\n", offsetof({struct}, {f}));' for f in fields]
    c = tmp_path / "layout.c"
    c.write_text("\n".join(src + ['return 0;}']))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(c), "-o", str(exe)],
                   check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(mirror)
    for f in fields:
        assert int(out[f]) == getattr(mirror, f).offset, f


def test_page_bytes():
    lib = _lib.load()
    for D in (64, 128, 256):
        for bs in (8, 16, 32, 64):
            want = op.page_bytes(D, bs)
            assert pa.int4_page_bytes(D, bs) == lib.pab200_int4_page_bytes(D, bs) == want
            assert want % 16 == 0 and want * 32 == bs * D * 2 * 9
    assert lib.pab200_int4_page_bytes(96, 16) == 0 and lib.pab200_int4_page_bytes(64, 12) == 0
    with pytest.raises(ValueError):
        pa.int4_page_bytes(128, 4)
    k, v = pa.int4_cache(3, 2, 8, 64, device="cpu")
    assert k.shape == v.shape == (3, 2, 288) and k.dtype == torch.uint8 and not k.any()


@pytest.mark.parametrize("value", [False, True])
@pytest.mark.parametrize("D,bs", [(64, 8), (128, 16), (256, 64)])
def test_format_places_are_a_permutation(D, bs, value):
    """Every nibble of the code area belongs to exactly one (row, element)."""
    seen = {op.code_place(D, r, d, value) for r in range(bs) for d in range(D)}
    assert seen == {(b, s) for b in range(bs * D // 2) for s in (0, 4)}


def test_oracle_round_trip_is_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    for dt in (torch.bfloat16, torch.float16):
        x = torch.randn((16, 128), generator=g).to(dt)
        c, s, lo = op.quantise(x)
        for value in (False, True):
            page = np.zeros(op.page_bytes(128, 16), np.uint8)
            for r in range(16):
                op.put_row(page, 16, r, c[r], s[r], lo[r], value)
            got = torch.from_numpy(op.get_rows(page[None], 128, 16, dt, value)[0])
            # half a step, and what the rounding of s (half a unit) moves code 15 by
            sd = s.double().repeat_interleave(64, -1)
            tol = sd * (0.5 + 15 * torch.finfo(dt).eps / 2)
            assert ((got - x.double()).abs() <= tol).all()


# ------------------------------------------------------------ C ABI refusals

def _rows():
    a = _lib.Int4RowsArgs()
    a.k_cache = a.v_cache = a.k_rows = a.v_rows = a.seqlens = a.block_table = 4096
    a.dtype, a.num_seqs, a.num_kv_heads, a.head_size = _lib.DTYPE_BF16, 2, 2, 128
    a.block_size, a.max_blocks, a.num_pages, a.num_tokens = 16, 4, 16, 2
    a.row_stride_t, a.row_stride_h = 256, 128
    a.seqlens_stride_b, a.bt_stride_b, a.bt_stride_i, a.bt_page_mul = 1, 4, 1, 1
    return a


@pytest.mark.parametrize("field,value,code", [
    ("dtype", 2, _lib.ERR_UNSUPPORTED), ("head_size", 96, _lib.ERR_UNSUPPORTED),
    ("block_size", 4, _lib.ERR_UNSUPPORTED), ("num_kv_heads", 0, _lib.ERR_INVALID_ARGUMENT),
    ("num_tokens", 3, _lib.ERR_INVALID_ARGUMENT), ("num_tokens", -1, _lib.ERR_INVALID_ARGUMENT),
    ("max_blocks", -1, _lib.ERR_INVALID_ARGUMENT), ("max_blocks", 1 << 28, _lib.ERR_UNSUPPORTED),
    ("k_rows", 0, _lib.ERR_INVALID_ARGUMENT), ("seqlens", 0, _lib.ERR_INVALID_ARGUMENT),
    ("block_table", 0, _lib.ERR_INVALID_ARGUMENT), ("v_cache", 4104, _lib.ERR_ALIGNMENT),
    ("k_rows", 4097, _lib.ERR_ALIGNMENT)])
def test_rows_refusals(field, value, code):
    lib = _lib.load()
    a = _rows()
    setattr(a, field, value)
    assert lib.pab200_kv_append_int4(ctypes.byref(a), 1, None) == code
    assert lib.pab200_kv_read_int4(ctypes.byref(a), None, 0, 0, None) == code
    assert lib.pab200_last_error() != b""


def test_append_refuses_a_length_of_many_sequences():
    """An expanded length would be advanced once per sequence, in any order."""
    lib = _lib.load()
    a = _rows()
    a.seqlens_stride_b = 0
    assert lib.pab200_kv_append_int4(ctypes.byref(a), 1, None) == _lib.ERR_INVALID_ARGUMENT
    assert b"share a length" in lib.pab200_last_error()


def test_rows_edge_calls():
    lib = _lib.load()
    assert lib.pab200_kv_append_int4(None, 1, None) == _lib.ERR_INVALID_ARGUMENT
    a = _rows()
    a.num_seqs = a.num_tokens = 0
    assert lib.pab200_kv_append_int4(ctypes.byref(a), 1, None) == _lib.OK     # nothing to do
    assert lib.pab200_kv_read_int4(ctypes.byref(a), None, 0, 0, None) == _lib.OK
    a = _rows()
    a.row_stride_t = 260                                                     # reads back in 16 bytes
    assert lib.pab200_kv_read_int4(ctypes.byref(a), None, 0, 0, None) == _lib.ERR_ALIGNMENT


def _decode():
    a = _lib.DecodeArgs()
    a.out = a.q = a.k_cache = a.v_cache = a.seqlens = a.block_table = 4096
    a.dtype, a.layout = _lib.DTYPE_BF16, _lib.LAYOUT_PAGES
    a.num_seqs, a.num_q_heads, a.num_kv_heads = 2, 8, 2
    a.head_size, a.block_size, a.max_blocks, a.num_pages = 128, 16, 4, 16
    a.q_stride_b, a.q_stride_h, a.out_stride_b, a.out_stride_h = 1024, 128, 1024, 128
    a.seqlens_stride_b, a.seqlens_stride_h = 2, 1
    a.bt_stride_b, a.bt_stride_h, a.bt_stride_i, a.bt_page_mul = 8, 4, 1, 1
    a.softmax_scale = 0.1
    return a


@pytest.mark.parametrize("field,value,code", [
    ("layout", _lib.LAYOUT_NHD, _lib.ERR_UNSUPPORTED), ("head_size", 96, _lib.ERR_UNSUPPORTED),
    ("num_q_heads", 128, _lib.ERR_UNSUPPORTED), ("num_q_heads", 7, _lib.ERR_INVALID_ARGUMENT),
    ("k_cache", 4104, _lib.ERR_ALIGNMENT), ("out", 0, _lib.ERR_INVALID_ARGUMENT),
    ("num_seqs", 0, _lib.ERR_INVALID_ARGUMENT)])
def test_decode_int4_refusals(field, value, code):
    lib = _lib.load()
    a = _decode()
    setattr(a, field, value)
    assert lib.pab200_decode_int4_workspace_size(ctypes.byref(a)) == 0
    assert lib.pab200_decode_int4(ctypes.byref(a), 1 << 20, 1 << 30, None) == code


def _select():
    a = _lib.SelectArgs()
    a.q = a.page_bounds = a.seqlens = a.block_table = a.tables = a.selected_lens = 4096
    a.dtype, a.num_seqs, a.num_q_heads, a.num_kv_heads = _lib.DTYPE_BF16, 2, 8, 2
    a.head_size, a.block_size, a.max_blocks, a.num_pages = 128, 16, 64, 256
    a.num_selected, a.num_sink, a.num_recent = 8, 1, 1
    a.q_stride_b, a.q_stride_h, a.seqlens_stride_b = 1024, 128, 1
    a.bt_stride_b, a.bt_stride_i, a.bounds_page_mul, a.bounds_page_add = 64, 1, 2, 1
    return a


@pytest.mark.parametrize("field,value,code", [
    ("dtype", 2, _lib.ERR_UNSUPPORTED), ("head_size", 80, _lib.ERR_UNSUPPORTED),
    ("block_size", 128, _lib.ERR_UNSUPPORTED), ("num_recent", 0, _lib.ERR_INVALID_ARGUMENT),
    ("num_sink", -1, _lib.ERR_INVALID_ARGUMENT), ("num_sink", 8, _lib.ERR_INVALID_ARGUMENT),
    ("num_selected", 1, _lib.ERR_INVALID_ARGUMENT), ("num_q_heads", 7, _lib.ERR_INVALID_ARGUMENT),
    ("tables", 0, _lib.ERR_INVALID_ARGUMENT), ("page_bounds", 4104, _lib.ERR_ALIGNMENT),
    ("max_blocks", 1 << 28, _lib.ERR_UNSUPPORTED)])
def test_select_refusals(field, value, code):
    lib = _lib.load()
    a = _select()
    setattr(a, field, value)
    assert lib.pab200_select_pages_workspace_size(ctypes.byref(a)) == 0
    assert lib.pab200_select_pages(ctypes.byref(a), 1 << 20, 1 << 30, None) == code
    d = _decode()
    d.max_blocks, d.num_pages = 64, 256
    assert lib.pab200_decode_sparse(ctypes.byref(d), ctypes.byref(a), 1 << 20, 1 << 30, None) == code


def test_select_workspace_and_sparse_agreement():
    lib = _lib.load()
    a, d = _select(), _decode()
    assert lib.pab200_select_pages(ctypes.byref(a), None, 0, None) == _lib.ERR_WORKSPACE
    d.num_seqs = 3                                                # not the selection's
    assert lib.pab200_decode_sparse(ctypes.byref(d), ctypes.byref(a), 1 << 20, 1 << 30, None) == \
        _lib.ERR_INVALID_ARGUMENT
    assert lib.pab200_decode_sparse(None, ctypes.byref(a), 1 << 20, 1 << 30, None) == \
        _lib.ERR_INVALID_ARGUMENT


def _bounds():
    a = _lib.PageBoundsArgs()
    a.page_bounds = a.k_rows = a.seqlens = a.block_table = 4096
    a.dtype, a.num_seqs, a.num_kv_heads, a.head_size = _lib.DTYPE_F16, 2, 2, 64
    a.block_size, a.max_blocks, a.num_pages, a.num_tokens = 16, 4, 16, 2
    a.row_stride_t, a.row_stride_h, a.seqlens_stride_b = 128, 64, 1
    a.bt_stride_b, a.bt_stride_i, a.bounds_page_mul, a.bounds_page_add = 4, 1, 2, 1
    return a


@pytest.mark.parametrize("field,value,code", [
    ("dtype", 2, _lib.ERR_UNSUPPORTED), ("head_size", 32, _lib.ERR_UNSUPPORTED),
    ("block_size", 1, _lib.ERR_UNSUPPORTED), ("num_tokens", 5, _lib.ERR_INVALID_ARGUMENT),
    ("k_rows", 0, _lib.ERR_INVALID_ARGUMENT), ("page_bounds", 0, _lib.ERR_INVALID_ARGUMENT),
    ("page_bounds", 4100, _lib.ERR_ALIGNMENT), ("num_kv_heads", 0, _lib.ERR_INVALID_ARGUMENT)])
def test_bounds_refusals(field, value, code):
    lib = _lib.load()
    a = _bounds()
    setattr(a, field, value)
    assert lib.pab200_update_page_bounds(ctypes.byref(a), None) == code


# --------------------------------------------------------- Python refusals

def _tensors(B=2, Hkv=2, D=128, bs=16, maxb=4, dtype=torch.bfloat16):
    k, v = pa.int4_cache(16, Hkv, bs, D, device="cpu")
    rows = torch.zeros((B, Hkv, D), dtype=dtype)
    lens = torch.zeros(B, dtype=torch.int32)
    bt = torch.zeros((B, maxb), dtype=torch.int32)
    return k, v, rows, lens, bt


def test_append_refusals():
    k, v, x, lens, bt = _tensors()
    for bad, err in [
            (dict(k_cache=k.to(torch.int8)), TypeError), (dict(k_cache=k[:8]), ValueError),
            (dict(k_new=x.float(), v_new=x.float()), TypeError), (dict(k_new=x[:, :1]), ValueError),
            (dict(lens=lens.long()), TypeError), (dict(lens=lens[:1]), ValueError),
            (dict(bt=bt[:1]), ValueError), (dict(bs=8), ValueError), (dict(bs=12), ValueError),
            (dict(cu=torch.zeros(2, dtype=torch.int32)), ValueError),
            (dict(cu=torch.zeros(3, dtype=torch.int64)), TypeError),
            (dict(k_new=torch.zeros((3, 2, 128), dtype=torch.bfloat16),
                  v_new=torch.zeros((3, 2, 128), dtype=torch.bfloat16)), ValueError),
            (dict(k_cache=k.transpose(0, 1), v_cache=v.transpose(0, 1)), ValueError),
            (dict(), ValueError)]:                      # all is well, but nothing is on a GPU
        a = dict(k_cache=k, v_cache=v, k_new=x, v_new=x, lens=lens, bt=bt, bs=16, cu=None) | bad
        with pytest.raises(err):
            pa.kv_append_int4(a["k_cache"], a["v_cache"], a["k_new"], a["v_new"], a["lens"],
                              a["bt"], a["bs"], cu_new=a["cu"])


def test_read_refusals():
    k, v, x, lens, bt = _tensors()
    cu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        pa.kv_read_int4(k, v, bt, lens, 16, 128, torch.float32)
    with pytest.raises(ValueError):
        pa.kv_read_int4(k, v, bt, lens, 16, 128, torch.bfloat16, cu_out=cu)     # no num_tokens
    with pytest.raises(ValueError):
        pa.kv_read_int4(k, v, bt, lens, 16, 128, torch.bfloat16, starts=lens[:1])
    with pytest.raises(ValueError):
        pa.kv_read_int4(k, v, bt, lens, 16, 128, torch.bfloat16, out=(x[..., :64], x[..., :64]))


def test_attention_int4_refusals():
    k, v, x, lens, bt = _tensors()
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    o = q.clone()
    for bad, err in [
            (dict(q=q.float(), out=q.float()), TypeError), (dict(q=q[0]), ValueError),
            (dict(out=q), ValueError),                 # in place
            (dict(out=q.half()), ValueError), (dict(out=q[:1]), ValueError),
            (dict(q=q[:, :7], out=q[:, :7]), ValueError), (dict(lens=lens[:1]), ValueError),
            (dict(bt=bt[0]), ValueError), (dict(bs=32), ValueError), (dict(n=-1), ValueError),
            (dict(k=k.view(torch.int8)), TypeError), (dict(k=k.view(32, -1)), ValueError),
            (dict(q=q[:, :, ::2], out=q[:, :, ::2]), ValueError), (dict(), ValueError)]:
        a = dict(out=o, q=q, k=k, v=v, bt=bt, lens=lens, bs=16, n=0) | bad
        with pytest.raises(err):
            pa.paged_attention_int4(a["out"], a["q"], a["k"], a["v"], a["bt"], a["lens"], 0.1,
                                    a["bs"], num_splits=a["n"])


def test_bounds_and_select_python_refusals():
    _, _, x, lens, bt = _tensors()
    bounds = torch.zeros((16, 2, 2, 128), dtype=torch.bfloat16)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    for b, err in [(bounds.half(), TypeError), (bounds[:, :1], ValueError),
                   (bounds[..., :64], ValueError), (bounds[0, 0], ValueError),
                   (bounds.view(32, 2, 128), ValueError), (bounds, ValueError)]:
        with pytest.raises(err):
            pa.update_page_bounds(b, x, lens, bt, 16)
    for kw in (dict(num_selected=1), dict(num_selected=4, num_recent=0),
               dict(num_selected=4, num_sink=4), dict(num_selected=4, num_sink=-1),
               dict(num_selected=4)):
        with pytest.raises(ValueError):
            pa.select_pages(q, bounds, bt, lens, 16, **kw)
    pool = torch.zeros((16, 2, 16, 128), dtype=torch.bfloat16)
    for kw in (dict(num_selected=1), dict(num_selected=4, kv_layout="NHD"),
               dict(num_selected=4, num_splits=-1), dict(num_selected=4)):
        with pytest.raises(ValueError):
            pa.paged_attention_sparse(q, q, pool, pool, bounds, bt, lens, 0.1, 16, **kw)
    with pytest.raises(ValueError):
        pa.paged_attention_sparse(q[:1], q, pool, pool, bounds, bt, lens, 0.1, 16, 4)
