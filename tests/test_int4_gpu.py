"""4-bit page cache on a GPU: append and read-back bit for bit against the
64-bit restatement, decode attention within derived bounds, and the places
where they can go wrong."""
import math

import numpy as np
import pytest
import torch

import pagedattention_b200 as pa
from oracle import pages as op
from pagedattention_b200 import _lib

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tables(lens, bs, pool_extra=3, per_head=0, seed=0, maxb=None):
    """Random block tables (CPU) covering lens (B,) or (B, Hkv); -1 where unused."""
    g = torch.Generator().manual_seed(seed)
    need = (lens.long() + bs - 1) // bs
    pool = int(need.sum()) + pool_extra
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    width = maxb or max(int(need.max()) + 1, 1)
    bt = torch.full(tuple(lens.shape) + (width,), -1, dtype=torch.int32)
    at = 0
    flat, nf = bt.view(-1, width), need.reshape(-1)
    for i in range(nf.numel()):
        flat[i, :nf[i]] = perm[at:at + nf[i]]
        at += int(nf[i])
    return bt, pool


def random_pages(P, D, bs, dt, g, value, scale=1.0):
    """Pages of quantised random rows, uint8 [P, bytes] (CPU), by the oracle."""
    x = (torch.randn((P, bs, D), generator=g) * scale).to(dt)
    c, s, lo = op.quantise(x)
    out = np.zeros((P, op.page_bytes(D, bs)), np.uint8)
    for r in range(bs):
        at, sh = op._places(D, r, value)
        for i in range(D):
            out[:, at[i]] |= (c[:, r, i].numpy().astype(np.uint8) << np.uint8(sh[i]))
    sl = torch.stack((s, lo), -1).contiguous().view(torch.uint8).numpy().reshape(P, -1)
    out[:, bs * D // 2:] = sl
    return out


# ------------------------------------------------------------------ append

def expect_append(kc, vc, k, v, lens, bt, bs, cu, per_head_pages):
    """The oracle's append on CPU copies: caches (numpy) changed in place, new lens."""
    N, Hkv, D = k.shape
    B = lens.shape[0]
    per_len = lens.dim() == 2
    after = lens.clone()
    cap = bt.shape[-1]
    P = kc.shape[0] if per_head_pages else kc.shape[0] * Hkv
    kf, vf = kc.reshape(-1, kc.shape[-1]), vc.reshape(-1, vc.shape[-1])
    quant = [op.quantise(k), op.quantise(v)]
    for s in range(B):
        a, b = (s, s + 1) if cu is None else (int(cu[s]), int(cu[s + 1]))
        grown = []
        for h in range(Hkv):
            L = int(lens[s, h] if per_len else lens[s])
            got, ok = 0, L >= 0
            for j in range(b - a):
                if L < 0:
                    break
                i = (L + j) // bs
                pid = -1
                if i < cap:
                    e = int(bt[s, h, i] if bt.dim() == 3 else bt[s, i])
                    pid = e if per_head_pages else e * Hkv + h
                    if e < 0 and not per_head_pages:
                        pid = e * Hkv + h
                if pid < 0 or pid >= P:
                    ok = False
                    continue
                r = (L + j) % bs
                for page, (c, sc, lo), value in ((kf[pid], quant[0], False), (vf[pid], quant[1], True)):
                    op.put_row(page, bs, r, c[a + j, h], sc[a + j, h], lo[a + j, h], value)
                if ok:
                    got += 1
            grown.append(got)
            if per_len:
                after[s, h] += got
        if not per_len:
            after[s] += min(grown)
    return after


def same_pages(got, want, D, bs):
    """Byte equality, with any NaN standing for any NaN in the scale area."""
    g, w = torch.from_numpy(got.reshape(-1, got.shape[-1])), torch.from_numpy(
        want.reshape(-1, want.shape[-1]))
    assert torch.equal(g[:, :bs * D // 2], w[:, :bs * D // 2])
    return g[:, bs * D // 2:].contiguous(), w[:, bs * D // 2:].contiguous()


APPEND = [  # dtype, D, bs, Hkv, lens before, new tokens (None: one each), pages per head, lens per head
    (BF, 128, 16, 8, [0, 15, 16, 100], None, False, False),
    (HF, 64, 8, 1, [0, 7, 3, 61], [1, 20, 0, 33], False, False),
    (BF, 256, 32, 2, [5, 0], [70, 1], False, True),
    (HF, 128, 64, 3, [63, 1, 0], [2, 200, 65], True, True),
    (BF, 64, 16, 5, [0], [513], True, False),
    (HF, 256, 8, 1, [0, 9], [0, 17], False, False),
]


@pytest.mark.parametrize("dt,D,bs,Hkv,lens,new,per_head,per_len", APPEND)
@pytest.mark.parametrize("rows", ["plain", "strided", "odd"])
def test_append_bytes(cuda_device, dt, D, bs, Hkv, lens, new, per_head, per_len, rows):
    g = torch.Generator().manual_seed(len(lens) + D)
    lens = torch.tensor(lens, dtype=torch.int32)
    B = lens.numel()
    n = torch.ones(B, dtype=torch.int32) if new is None else torch.tensor(new, dtype=torch.int32)
    total = lens + n
    if per_head:
        bt, pool = tables(total[:, None].expand(B, Hkv).contiguous(), bs)
        shape = (pool, op.page_bytes(D, bs))
    else:
        bt, pool = tables(total, bs)
        shape = (pool, Hkv, op.page_bytes(D, bs))
    ll = lens[:, None].expand(B, Hkv).contiguous() if per_len else lens
    N = int(n.sum())
    cu = None
    if new is not None:
        cu = torch.zeros(B + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(n, 0)
        N += 3                                    # rows behind the last sequence
    if rows == "plain":
        k, v = (torch.randn((N, Hkv, D), generator=g).to(dt) for _ in range(2))
        kd, vd = k.to(cuda_device), v.to(cuda_device)
    else:
        # a fused projection's rows; "odd": at an offset no 16-byte load may use
        off, width = (Hkv * D, 3 * Hkv * D) if rows == "strided" else (1, 2 * Hkv * D + 3)
        fused = torch.randn((N, width), generator=g).to(dt)
        fd = fused.to(cuda_device)
        k, v = (fused[:, o:o + Hkv * D].unflatten(1, (Hkv, D)) for o in (off, off + Hkv * D))
        kd, vd = (fd[:, o:o + Hkv * D].unflatten(1, (Hkv, D)) for o in (off, off + Hkv * D))
    kc, vc = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2))
    kcd, vcd, ld, btd = kc.to(cuda_device), vc.to(cuda_device), ll.to(cuda_device), bt.to(cuda_device)
    cud = None if cu is None else cu.to(cuda_device)
    pa.kv_append_status()
    pa.kv_append_int4(kcd, vcd, kd, vd, ld, btd, bs, cu_new=cud)
    assert pa.kv_append_status() == 0
    wk, wv = kc.numpy(), vc.numpy()
    after = expect_append(wk, wv, k, v, ll, bt, bs, cu, per_head)
    assert torch.equal(ld.cpu(), after)
    assert np.array_equal(kcd.cpu().numpy(), wk)   # every byte, the untouched ones too
    assert np.array_equal(vcd.cpu().numpy(), wv)
    # read back what was appended: lo + s c, one rounding
    out_shape = (N, Hkv, D)
    out = tuple(torch.full(out_shape, 7.0, dtype=dt, device=cuda_device) for _ in range(2))
    k2, v2 = pa.kv_read_int4(kcd, vcd, btd, ld, bs, D, dt, starts=lens.to(cuda_device), cu_out=cud,
                             out=out)
    M = int(n.sum())
    for got, src in ((k2, k), (v2, v)):
        c, s, lo = op.quantise(src)
        want = (lo.double()[..., None] + s.double()[..., None] * c.unflatten(-1, (-1, 64)).double())
        want = want.flatten(-2).to(torch.float64)
        g64 = got.cpu().double()[:M]
        assert ((g64 - want[:M]).abs() <= half_step(dt) * want[:M].abs()
                + 2.0 ** -23 * want[:M].abs() + torch.finfo(dt).smallest_normal * half_step(dt)).all()
        assert (got[M:] == 7.0).all()


def test_append_and_read_one_row_of_any_stride(cuda_device):
    """Strides of dimensions of one element mean nothing: neither their agreement
    nor their alignment is asked for."""
    dt, D, bs = BF, 64, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn((2, 1, 1, D), generator=g).to(dt)
    xd = x.to(cuda_device)
    k, v = xd[0].as_strided((1, 1, D), (D, D, 1)), xd[1].as_strided((1, 1, D), (7, 3, 1))
    kc, vc = pa.int4_cache(1, 1, bs, D, device=cuda_device)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    bt = torch.zeros((1, 1), dtype=torch.int32, device=cuda_device)
    pa.kv_append_int4(kc, vc, k, v, lens, bt, bs)
    out = torch.full((2, D), 7.0, dtype=dt, device=cuda_device)
    start = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    k2, v2 = pa.kv_read_int4(kc, vc, bt, lens, bs, D, dt, starts=start,
                             out=(out[0].as_strided((1, 1, D), (1, 5, 1)),
                                  out[1].as_strided((1, 1, D), (2, 3, 1))))
    for got, src in ((k2, x[0]), (v2, x[1])):
        c, s, lo = op.quantise(src)
        want = (lo.double()[..., None] + s.double()[..., None] * c.unflatten(-1, (-1, 64)).double())
        want = want.flatten(-2)
        # the one rounding of lo + s c
        assert ((got.cpu().double() - want).abs() <= half_step(dt) * want.abs()).all()


def test_append_places_that_do_not_exist(cuda_device):
    """A full table, bad page ids and a negative length: nothing else is
    touched, lengths stop before the first token without a place."""
    dt, D, bs, Hkv = BF, 64, 8, 2
    lens = torch.tensor([30, 4, -2, 0], dtype=torch.int32)
    new = [5, 20, 3, 9]
    cu = torch.tensor([0, 5, 25, 28, 37], dtype=torch.int32)
    bt = torch.tensor([[0, 1, 2, 3], [4, 99, 5, 6], [7, 8, 9, 10], [11, -1, 12, 13]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((sum(new), Hkv, D), generator=g).to(dt) for _ in range(2))
    kc, vc = (torch.randint(0, 256, (14, Hkv, op.page_bytes(D, bs)), generator=g, dtype=torch.uint8)
              for _ in range(2))
    kcd, vcd, ld = kc.to(cuda_device), vc.to(cuda_device), lens.to(cuda_device)
    pa.kv_append_status()
    pa.kv_append_int4(kcd, vcd, k.to(cuda_device), v.to(cuda_device), ld, bt.to(cuda_device), bs,
                      cu_new=cu.to(cuda_device))
    assert pa.kv_append_status() == (_lib.STATUS_APPEND_FULL | _lib.STATUS_BAD_PAGE_ID
                                     | _lib.STATUS_NEG_SEQLEN)
    wk, wv = kc.numpy(), vc.numpy()
    after = expect_append(wk, wv, k, v, lens, bt, bs, cu, False)
    assert after.tolist() == [32, 8, -2, 8]
    assert torch.equal(ld.cpu(), after)
    assert np.array_equal(kcd.cpu().numpy(), wk) and np.array_equal(vcd.cpu().numpy(), wv)


@pytest.mark.parametrize("dt", [BF, HF])
def test_append_values_at_the_edges(cuda_device, dt):
    """Constant groups, tiny and huge ranges, exact ties, NaN and infinities."""
    D, bs, Hkv = 128, 8, 1
    big = torch.finfo(dt).max
    rows = torch.zeros((12, Hkv, D), dtype=torch.float32)
    rows[1] = 3.25
    rows[2, 0] = torch.arange(D) % 16                      # codes exactly
    rows[3, 0] = torch.arange(D) % 31 * 0.5                # ties
    rows[4, 0] = torch.randn(D) * torch.finfo(dt).smallest_normal * 4
    rows[5, 0, :64] = torch.linspace(-1, 1, 64) * big * (0.25 if dt == BF else 1.0)
    rows[6, 0, 3] = float("nan")
    rows[7, 0, 70] = float("inf")
    rows[8, 0, 0] = -float("inf")
    rows[9, 0, :] = -0.0
    rows[10, 0] = torch.randn(D) * 1e-3 + 100
    rows[11, 0, 5] = 1.0
    k = rows.to(dt)
    v = (rows.flip(0)).to(dt)
    cu = torch.tensor([0, 12], dtype=torch.int32)
    lens = torch.zeros(1, dtype=torch.int32)
    bt = torch.tensor([[1, 0]], dtype=torch.int32)
    kc, vc = (torch.zeros((2, Hkv, op.page_bytes(D, bs)), dtype=torch.uint8) for _ in range(2))
    kcd, vcd, ld = kc.to(cuda_device), vc.to(cuda_device), lens.to(cuda_device)
    pa.kv_append_int4(kcd, vcd, k.to(cuda_device), v.to(cuda_device), ld, bt.to(cuda_device), bs,
                      cu_new=cu.to(cuda_device))
    wk, wv = kc.numpy(), vc.numpy()
    expect_append(wk, wv, k, v, lens, bt, bs, cu, False)
    for got, want in ((kcd, wk), (vcd, wv)):
        a, b = same_pages(got.cpu().numpy(), want, D, bs)
        x, y = a.view(dt).float(), b.view(dt).float()
        # the minimum of +0 and -0 may carry either sign
        assert torch.equal(torch.nan_to_num(x, nan=12345.0), torch.nan_to_num(y, nan=12345.0))
    k2, _ = pa.kv_read_int4(kcd, vcd, bt.to(cuda_device), ld, bs, D, dt, cu_out=cu.to(cuda_device),
                            num_tokens=12)
    nan = torch.isnan(k2.cpu().float()).view(12, 2, 64).all(-1)
    assert nan.nonzero().tolist() == [[6, 0], [7, 1], [8, 0]]
    assert torch.isfinite(k2.cpu().float().view(12, 2, 64)[~nan]).all()
    assert torch.equal(k2.cpu()[:3].float(), rows[:3])     # held exactly


def test_read_ranges(cuda_device):
    """Starts in the middle, past the end, before 0; bad pages read as zeros."""
    dt, D, bs, Hkv = HF, 128, 16, 2
    g = torch.Generator().manual_seed(3)
    lens = torch.tensor([40, 0, 20], dtype=torch.int32)
    bt = torch.tensor([[0, 77, 1], [-1, -1, -1], [2, 3, -1]], dtype=torch.int32)
    kp = random_pages(4 * Hkv, D, bs, dt, g, False)
    vp = random_pages(4 * Hkv, D, bs, dt, g, True)
    starts, cu = torch.tensor([10, 0, -3], dtype=torch.int32), torch.tensor([0, 34, 36, 60], dtype=torch.int32)
    kcd, vcd = (torch.from_numpy(p).view(4, Hkv, -1).to(cuda_device) for p in (kp, vp))
    pa.kv_append_status()
    k, v = pa.kv_read_int4(kcd, vcd, bt.to(cuda_device), lens.to(cuda_device), bs, D, dt,
                           starts=starts.to(cuda_device), cu_out=cu.to(cuda_device), num_tokens=62)
    assert pa.kv_append_status() == _lib.STATUS_BAD_PAGE_ID
    for got, pages, value in ((k, kp, False), (v, vp, True)):
        vals = op.get_rows(pages, D, bs, dt, value)
        want = torch.zeros((62, Hkv, D), dtype=torch.float64)
        for s in range(3):
            for j in range(int(cu[s + 1] - cu[s])):
                pos = int(starts[s]) + j
                if 0 <= pos < int(lens[s]):
                    e = int(bt[s, pos // bs])
                    for h in range(Hkv if 0 <= e < 4 else 0):
                        want[int(cu[s]) + j, h] = torch.from_numpy(vals[e * Hkv + h, pos % bs])
        err = (got.cpu().double() - want).abs()
        assert (err <= (half_step(dt) + 2.0 ** -23) * want.abs() + 1e-8).all()


@pytest.mark.parametrize("cu,N", [([5, 12, 12, 20], 40), ([0, 0, 0, 0], 9), ([9, 9, 9, 9], 9),
                                  ([3, 4, 70, 71], 71)])
def test_read_rows_of_no_sequence(cuda_device, cu, N):
    """Fresh outputs are zero before the first sequence's rows and behind the last's."""
    dt, D, bs, Hkv = BF, 64, 8, 3
    g = torch.Generator().manual_seed(4)
    lens = torch.tensor([70, 70, 70], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    kp = random_pages(pool * Hkv, D, bs, dt, g, False)
    vp = random_pages(pool * Hkv, D, bs, dt, g, True)
    kcd, vcd = (torch.from_numpy(p).view(pool, Hkv, -1).to(cuda_device) for p in (kp, vp))
    torch.full((2, N, Hkv, D), 7.0, dtype=dt, device=cuda_device)  # freed: the memory is not zero
    k, v = pa.kv_read_int4(kcd, vcd, bt.to(cuda_device), lens.to(cuda_device), bs, D, dt,
                           cu_out=torch.tensor(cu, dtype=torch.int32, device=cuda_device), num_tokens=N)
    for got, pages, value in ((k, kp, False), (v, vp, True)):
        vals = op.get_rows(pages, D, bs, dt, value)
        want = torch.zeros((N, Hkv, D), dtype=torch.float64)
        for s in range(3):
            for j in range(cu[s + 1] - cu[s]):
                for h in range(Hkv):
                    want[cu[s] + j, h] = torch.from_numpy(vals[int(bt[s, j // bs]) * Hkv + h, j % bs])
        err = (got.cpu().double() - want).abs()
        assert (err <= (half_step(dt) + 2.0 ** -23) * want.abs() + 1e-8).all()


@pytest.mark.parametrize("N,first", [(1, 0), (9, 0), (70, 3), (70, 70)])
@pytest.mark.parametrize("bs", [8, 16])
def test_read_of_an_empty_batch(cuda_device, N, first, bs):
    """Without sequences every row is a row of no sequence."""
    dt, D, Hkv = BF, 64, 3
    kc, vc = pa.int4_cache(2, Hkv, bs, D, device=cuda_device)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    bt = torch.zeros((0, 4), dtype=torch.int32, device=cuda_device)
    cu = torch.full((1,), first, dtype=torch.int32, device=cuda_device)
    x = torch.full((2, N, Hkv, D), 7.0, dtype=dt, device=cuda_device)
    del x                                          # freed: the memory is not zero
    k, v = pa.kv_read_int4(kc, vc, bt, lens, bs, D, dt, cu_out=cu, num_tokens=N)
    assert k.shape == v.shape == (N, Hkv, D) and not k.any() and not v.any()
    out = tuple(torch.full((N, Hkv, D), 7.0, dtype=dt, device=cuda_device) for _ in range(2))
    pa.kv_read_int4(kc, vc, bt, lens, bs, D, dt, cu_out=cu, out=out)
    assert (out[0] == 7.0).all() and (out[1] == 7.0).all()


@pytest.mark.parametrize("length,start", [(-2 ** 31, 16), (-1, 0), (0, 2 ** 31 - 8), (24, 2 ** 31 - 8)])
def test_read_lengths_and_starts_at_the_ends_of_int32(cuda_device, length, start):
    """Positions past every length read as zeros, however far."""
    dt, D, bs, Hkv = HF, 64, 8, 1
    g = torch.Generator().manual_seed(5)
    kc, vc = (torch.from_numpy(random_pages(4, D, bs, dt, g, val)).view(4, 1, -1).to(cuda_device)
              for val in (False, True))
    bt = torch.arange(4, dtype=torch.int32, device=cuda_device)[None]

    def mk(*x):
        return torch.tensor(x, dtype=torch.int32, device=cuda_device)

    k, v = pa.kv_read_int4(kc, vc, bt, mk(length), bs, D, dt, starts=mk(start), cu_out=mk(0, 24),
                           num_tokens=24)
    assert not k.any() and not v.any()


# --------------------------------------------------------------- attention

def check_attention(got, q, kp, vp, bt, lens, scale, bs, Hkv, dt, per_head_pages=False):
    """Against 64 bits.  Error: the output's rounding; each probability times
    its scale is rounded to T once, and multiplies s (c - 8), at most 8 s; the
    scores' fp32 sums move every probability by 2^-18 of itself and more with
    the score's size (128 roundings of 2^-24 of sums below |q| |k| sum)."""
    B, Hq, D = q.shape
    G = Hq // Hkv
    kv, vv = op.get_rows(kp, D, bs, dt, False), op.get_rows(vp, D, bs, dt, True)
    vs = torch.from_numpy(np.ascontiguousarray(vp[:, bs * D // 2:])).view(dt).double()
    vs = torch.nan_to_num(vs.view(-1, bs, D // 64, 2)[..., 0]).numpy()
    for s in range(B):
        for h in range(Hkv):
            L = int(lens[s, h] if lens.dim() == 2 else lens[s])
            n = (L + bs - 1) // bs
            ks, vals, smax = [], [], 0.0
            for i in range(n):
                e = int(bt[s, h, i] if bt.dim() == 3 else bt[s, i])
                pid = e if per_head_pages else e * Hkv + h
                take = min(bs, L - i * bs)
                if pid < 0 or pid >= kp.shape[0]:
                    ks.append(np.zeros((take, D)))
                    vals.append(np.zeros((take, D)))
                    continue
                ks.append(kv[pid, :take])
                vals.append(vv[pid, :take])
                smax = max(smax, vs[pid, :take].max())
            k = np.concatenate(ks) if ks else np.zeros((0, D))
            v = np.concatenate(vals) if vals else np.zeros((0, D))
            qq = q[s, h * G:(h + 1) * G].double().cpu().numpy()
            want = op.attention(qq, k, v, scale)
            have = got[s, h * G:(h + 1) * G].double().cpu().numpy()
            if L == 0:
                assert (have == 0).all()
                continue
            size = np.abs(qq) @ np.abs(k).T.max(1) * scale if L else 0
            u = half_step(dt)
            tol = u * np.abs(want) + u * 8 * smax \
                + (2.0 ** -18 + 128 * 2.0 ** -24 * 2 * size[:, None]) * np.abs(v).max() \
                + torch.finfo(dt).smallest_normal * u
            bad = np.abs(have - want) > tol
            assert not bad.any(), (s, h, L, np.abs(have - want).max(), tol.min())


ATTEND = [  # dtype, D, G, Hkv, bs, lens
    (BF, 128, 4, 2, 16, [1, 0, 333, 16, 17, 1000]),
    (HF, 128, 1, 4, 16, [5, 130, 64]),
    (BF, 64, 8, 1, 8, [2000, 1, 7, 9]),
    (HF, 64, 32, 1, 8, [777, 64, 65]),
    (BF, 64, 12, 2, 64, [129, 3]),
    (HF, 128, 16, 1, 32, [95, 513]),
    (BF, 128, 32, 1, 16, [400, 31]),
    (HF, 128, 17, 2, 64, [100, 65]),
    (BF, 256, 8, 1, 16, [200, 33, 0]),
    (HF, 256, 2, 3, 64, [65, 640]),
    (BF, 256, 5, 1, 8, [99]),
    (HF, 64, 3, 2, 32, [33, 1500]),
]


@pytest.mark.parametrize("dt,D,G,Hkv,bs,lens", ATTEND)
def test_attention_matches_64_bits(cuda_device, dt, D, G, Hkv, bs, lens):
    g = torch.Generator().manual_seed(D + G)
    lens = torch.tensor(lens, dtype=torch.int32)
    B = lens.numel()
    bt, pool = tables(lens, bs)
    kp = random_pages(pool * Hkv, D, bs, dt, g, False, 2.0)
    vp = random_pages(pool * Hkv, D, bs, dt, g, True)
    # rows past a sequence's end and unused pages: every bit set (NaN scales)
    used = np.zeros((pool * Hkv, bs), bool)
    for s in range(B):
        for i in range((int(lens[s]) + bs - 1) // bs):
            used[int(bt[s, i]) * Hkv:(int(bt[s, i]) + 1) * Hkv, :min(bs, int(lens[s]) - i * bs)] = True
    for p in (kp, vp):
        sl = p[:, bs * D // 2:].reshape(pool * Hkv, bs, -1)
        sl[~used] = 255
        p[:, bs * D // 2:] = sl.reshape(pool * Hkv, -1)
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    scale = 1 / math.sqrt(D)
    args = [torch.from_numpy(p).view(pool, Hkv, -1).to(cuda_device) for p in (kp, vp)]
    args += [bt.to(cuda_device), lens.to(cuda_device)]
    out = torch.full_like(q, 9.0).to(cuda_device)
    pa.paged_attention_int4(out, q.to(cuda_device), *args, scale, bs)
    assert pa.read_status() == 0
    check_attention(out, q, kp, vp, bt, lens, scale, bs, Hkv, dt)
    # the split asked for, strided query and output, lengths and tables per head
    big = torch.zeros((B, G * Hkv + 1, 2 * D), dtype=dt, device=cuda_device)
    qs = big[:, 1:, D:]
    qs.copy_(q)
    outs = torch.full((G * Hkv, B, D), 3.0, dtype=dt, device=cuda_device).transpose(0, 1)
    lh = lens[:, None].expand(B, Hkv)
    bh = bt[:, None].expand(B, Hkv, -1)
    pa.paged_attention_int4(outs, qs, args[0], args[1], bh.to(cuda_device), lh.to(cuda_device),
                            scale, bs, num_splits=3)
    check_attention(outs, q, kp, vp, bt, lens, scale, bs, Hkv, dt)
    again = torch.empty_like(out)
    pa.paged_attention_int4(again, q.to(cuda_device), *args, scale, bs)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dt,D,G,Hkv,bs,lens", ATTEND)
@pytest.mark.parametrize("splits", [0, 1, 4])
def test_attention_is_finite(cuda_device, dt, D, G, Hkv, bs, lens, splits):
    """No NaN or infinity comes out of finite rows (a comparison with a bound
    would let a NaN pass)."""
    g = torch.Generator().manual_seed(D + G + splits)
    lens = torch.tensor(lens, dtype=torch.int32)
    bt, pool = tables(lens, bs)
    kp, vp = (random_pages(pool * Hkv, D, bs, dt, g, value) for value in (False, True))
    q = torch.randn((lens.numel(), G * Hkv, D), generator=g).to(dt).to(cuda_device)
    out = torch.full_like(q, float("nan"))
    pa.paged_attention_int4(out, q, *(torch.from_numpy(p).view(pool, Hkv, -1).to(cuda_device) for p in (kp, vp)),
                            bt.to(cuda_device), lens.to(cuda_device), 0.1, bs, num_splits=splits)
    assert torch.isfinite(out).all()


# Binary exponents of the values' standard deviation, page by page.
UP = list(range(-96, 100, 4))
SCALES = [(BF, [UP, UP[::-1], [-118] * 40, [117] * 12, [0, 60, -20, 30, -60, 100] * 6]),
          (HF, [list(range(-6, 11)) * 2, list(range(10, -7, -1)) * 2, [-7] * 40, [12] * 40])]


@pytest.mark.parametrize("dt,exps", SCALES)
@pytest.mark.parametrize("D,G,bs", [(64, 8, 8), (128, 4, 16), (128, 20, 8)])
def test_attention_values_of_many_scales(cuda_device, dt, exps, D, G, bs):
    """Values whose size jumps from page to page, tiny and huge ones."""
    g = torch.Generator().manual_seed(9)
    lens = torch.tensor([len(e) * bs - 3 for e in exps], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    mul = torch.ones((pool, 1, 1))
    for s, es in enumerate(exps):
        for i, e in enumerate(es):
            mul[int(bt[s, i])] = 2.0 ** e
    kp = random_pages(pool, D, bs, dt, g, False)
    vp = random_pages(pool, D, bs, dt, g, True, mul)
    q = (torch.randn((len(exps), G, D), generator=g) * 0.5).to(dt)
    out = torch.empty_like(q).to(cuda_device)
    for splits in (0, 2):
        pa.paged_attention_int4(out, q.to(cuda_device),
                                *(torch.from_numpy(p).view(pool, 1, -1).to(cuda_device)
                                  for p in (kp, vp)), bt.to(cuda_device), lens.to(cuda_device),
                                0.1, bs, num_splits=splits)
        check_attention(out, q, kp, vp, bt, lens, 0.1, bs, 1, dt)


def flat_values(D, L, bs, dt, g, size, sink):
    """Keys and values of one head: a first token with a score of `sink` and values
    of 0, and L - 1 like tokens with scores of 0 and values of one size, whose codes
    lie at the top but for one element of each group."""
    base = torch.randn(D, generator=g)
    k = torch.zeros((L, D))
    k[0] = base * sink / (base @ base)
    v = torch.full((L, D), size) * (1 - 0.02 * torch.rand(D, generator=g))
    v[:, ::64] = 0.0
    v[0] = 0.0
    return base, k.to(dt), v.to(dt)


def pages_of(x, bs, dt, value):
    L, D = x.shape
    n = (L + bs - 1) // bs
    pad = torch.zeros((n * bs, D), dtype=dt)
    pad[:L] = x
    c, s, lo = op.quantise(pad.view(n, bs, D))
    out = np.zeros((n, op.page_bytes(D, bs)), np.uint8)
    for p in range(n):
        for r in range(bs):
            op.put_row(out[p], bs, r, c[p, r], s[p, r], lo[p, r], value)
    return out


@pytest.mark.parametrize("D,G,bs,sink", [(64, 1, 8, 8.0), (128, 4, 16, 10.0), (64, 32, 8, 10.0),
                                         (256, 2, 16, 12.0)])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.02, 0.005])
def test_attention_small_values_beside_a_dominating_token(cuda_device, D, G, bs, sink, size):
    """fp16 values whose probability x scale lies far below fp16's normal numbers."""
    dt, L = HF, 1025
    g = torch.Generator().manual_seed(D + G)
    base, k, v = flat_values(D, L, bs, dt, g, size, sink)
    q = base.expand(1, G, D).to(dt)
    kp, vp = pages_of(k, bs, dt, False), pages_of(v, bs, dt, True)
    n = kp.shape[0]
    bt = torch.arange(n, dtype=torch.int32)[None]
    out = torch.empty_like(q).to(cuda_device)
    for splits in (0, 2):
        pa.paged_attention_int4(out, q.to(cuda_device),
                                *(torch.from_numpy(p).view(n, 1, -1).to(cuda_device) for p in (kp, vp)),
                                bt.to(cuda_device), torch.tensor([L], dtype=torch.int32, device=cuda_device),
                                1.0, bs, num_splits=splits)
        kv, vv = (op.get_rows(p, D, bs, dt, val).reshape(-1, D)[:L] for p, val in ((kp, False), (vp, True)))
        sc = torch.from_numpy(np.ascontiguousarray(vp[:, bs * D // 2:])).view(dt).double()
        sc = sc.view(-1, D // 64, 2)[:L, :, 0].repeat_interleave(64, -1).numpy()   # scales
        qq = q[0].double().numpy()
        w = np.exp(qq @ kv.T - (qq @ kv.T).max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        want, u = w @ vv, half_step(dt)
        size_ = (np.abs(qq) @ np.abs(kv).T).max(1)[:, None]
        # The output's rounding; each probability x scale rounded once, times codes
        # of at most 8; below fp16's normal numbers, that is 2^24 under the largest
        # scale, 2^-35 of that scale per token; the scores' sums as in
        # check_attention, against the mean size of the values.
        tol = u * np.abs(want) + torch.finfo(dt).smallest_normal * u + u * 8 * (w @ sc) \
            + L * 8 * 2.0 ** -35 * sc.max() + 2 * (2.0 ** -18 + 256 * 2.0 ** -24 * size_) * (w @ np.abs(vv))
        err = np.abs(out[0].double().cpu().numpy() - want)
        assert (err <= tol).all()


@pytest.mark.parametrize("D,G", [(64, 8), (128, 4), (128, 20), (256, 2)])
@pytest.mark.parametrize("e,same", [(60, False), (108, False), (118, False), (124, False), (126, True)])
def test_attention_queries_near_the_largest(cuda_device, D, G, e, same):
    """bf16 queries up to the type's largest; `same`: sums of a group's elements pass it."""
    dt, bs, L = BF, 16, 333
    g = torch.Generator().manual_seed(e + G)
    lens = torch.tensor([L, 1], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    kp = random_pages(pool, D, bs, dt, g, False, 2.0 ** -60)
    vp = random_pages(pool, D, bs, dt, g, True)
    q = torch.rand((2, G, D), generator=g) + 0.5 if same else torch.randn((2, G, D), generator=g)
    q[:, 0] *= 2.0 ** -4                           # heads of other sizes beside the largest
    q = (q * 2.0 ** e).clamp(-torch.finfo(dt).max, torch.finfo(dt).max).to(dt)
    scale = 2.0 ** (60 - e) / math.sqrt(D)
    out = torch.empty_like(q).to(cuda_device)
    pa.paged_attention_int4(out, q.to(cuda_device),
                            *(torch.from_numpy(p).view(pool, 1, -1).to(cuda_device) for p in (kp, vp)),
                            bt.to(cuda_device), lens.to(cuda_device), scale, bs)
    assert torch.isfinite(out).all()
    check_attention(out, q, kp, vp, bt, lens, scale, bs, 1, dt)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D,G,bs", [(64, 8, 8), (128, 4, 16), (128, 20, 64), (256, 2, 16)])
def test_attention_nan_in_a_group_or_a_query(cuda_device, dt, D, G, bs):
    """A NaN group of values makes its 64 elements NaN, one of keys or a NaN in a
    query the heads that read it; everything else stays what it is."""
    g = torch.Generator().manual_seed(D)
    lens = torch.tensor([200, 200, 200, 77], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    kp = random_pages(pool, D, bs, dt, g, False)
    vp = random_pages(pool, D, bs, dt, g, True)
    q = torch.randn((4, G, D), generator=g).to(dt)

    def run(kp, vp, q):
        out = torch.empty_like(q).to(cuda_device)
        pa.paged_attention_int4(out, q.to(cuda_device),
                                *(torch.from_numpy(p).view(pool, 1, -1).to(cuda_device) for p in (kp, vp)),
                                bt.to(cuda_device), lens.to(cuda_device), 0.1, bs)
        return out.cpu()

    clean, clean_q = run(kp, vp, q), q
    clean_kp, clean_vp = kp, vp
    assert torch.isfinite(clean).all()
    bad = torch.zeros(clean.shape, dtype=torch.bool)
    nan = torch.full((1, D), float("nan")).to(dt)
    kp, vp, q = kp.copy(), vp.copy(), q.clone()
    at = bs * D // 2 + 5 * (D // 64) * 4           # pairs of row 5
    vp[int(bt[0, 1]), at:at + 4] = nan.view(torch.uint8).numpy()[0, :4]
    bad[0, :, :64] = True
    kp[int(bt[1, 0]), at + (D // 64 - 1) * 4:at + (D // 64) * 4] = nan.view(torch.uint8).numpy()[0, :4]
    bad[1] = True
    q[2, G - 1, 9] = float("nan")
    bad[2, G - 1] = True
    q[3, 0, 3] = float("inf")
    bad[3, 0] = True
    got = run(kp, vp, q)
    assert torch.isnan(got[bad]).all()
    assert torch.isfinite(got[~bad]).all()
    # not bit for bit: a head whose scores are infinite makes its warp take new
    # reference points, which moves the roundings of the warp's other heads
    check_attention(torch.where(bad, clean, got), clean_q, clean_kp, clean_vp, bt, lens, 0.1, bs, 1, dt)


@pytest.mark.parametrize("dt,D,G,bs", [(BF, 128, 2, 16), (BF, 64, 32, 8), (BF, 256, 4, 64),
                                       (HF, 128, 2, 16)])
def test_attention_long_range_of_one_cta(cuda_device, dt, D, G, bs):
    """20,001 tokens over two CTAs: hundreds of stages of one head per CTA."""
    g = torch.Generator().manual_seed(10)
    L, pages = 20001, 48
    bt = torch.randint(0, pages, (1, (L + bs - 1) // bs), generator=g, dtype=torch.int32)
    kp = random_pages(pages, D, bs, dt, g, False)
    vp = random_pages(pages, D, bs, dt, g, True)
    q = torch.randn((1, G, D), generator=g).to(dt)
    out = torch.empty_like(q).to(cuda_device)
    lens = torch.tensor([L], dtype=torch.int32)
    pa.paged_attention_int4(out, q.to(cuda_device), *(torch.from_numpy(p).view(pages, 1, -1).to(cuda_device)
                                                      for p in (kp, vp)),
                            bt.to(cuda_device), lens.to(cuda_device), 0.05, bs, num_splits=2)
    check_attention(out, q, kp, vp, bt, lens, 0.05, bs, 1, dt)


@pytest.mark.parametrize("dt", [BF, HF])
def test_attention_many_heads(cuda_device, dt):
    """1,200 (sequence, kv head) pairs, many of them empty or of one token."""
    D, G, Hkv, bs, B = 64, 2, 4, 8, 300
    g = torch.Generator().manual_seed(11)
    lens = torch.randint(0, 60, (B, Hkv), generator=g, dtype=torch.int32)
    lens[::7] = 0
    lens[::11] = 1
    bt, pool = tables(lens, bs)
    kp = random_pages(pool, D, bs, dt, g, False)
    vp = random_pages(pool, D, bs, dt, g, True)
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    out = torch.full_like(q, 5.0).to(cuda_device)
    pa.paged_attention_int4(out, q.to(cuda_device), torch.from_numpy(kp).to(cuda_device),
                            torch.from_numpy(vp).to(cuda_device), bt.to(cuda_device),
                            lens.to(cuda_device), 0.125, bs)
    assert pa.read_status() == 0
    check_attention(out, q, kp, vp, bt, lens, 0.125, bs, Hkv, dt, per_head_pages=True)


@pytest.mark.parametrize("dt", [BF, HF])
def test_states_of_two_ranges(cuda_device, dt):
    """The C entry's state outputs: attention and log-sum-exp of a range; two
    ranges of a context merge to the whole."""
    D, G, Hkv, bs, B, scale = 128, 4, 2, 16, 3, 0.08
    g = torch.Generator().manual_seed(14)
    lens = torch.tensor([3000, 0, 40], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    kp = random_pages(pool * Hkv, D, bs, dt, g, False)
    vp = random_pages(pool * Hkv, D, bs, dt, g, True)
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    qd = q.to(cuda_device)
    kc, vc = (torch.from_numpy(p).view(pool, Hkv, -1).to(cuda_device) for p in (kp, vp))
    lib = _lib.load()
    cut = 32                                     # pages of the first range
    parts = [(bt[:, :cut].contiguous(), lens.clamp(max=cut * bs)),
             (bt[:, cut:].contiguous(), (lens - cut * bs).clamp(min=0))]
    rows, states = B * G * Hkv, []
    for table, ln in parts:
        td, ld = table.to(cuda_device), ln.to(cuda_device)
        o = torch.full((rows, D), 9.0, device=cuda_device)
        lse = torch.full((rows,), 9.0, device=cuda_device)
        a = _lib.DecodeArgs(
            None, qd.data_ptr(), kc.data_ptr(), vc.data_ptr(), ld.data_ptr(), td.data_ptr(),
            0 if dt == BF else 1, _lib.LAYOUT_PAGES, B, G * Hkv, Hkv, D, bs, table.shape[1],
            pool * Hkv, G * Hkv * D, D, 0, 0, 1, 0, table.shape[1], 0, 1, Hkv, 1, scale, 0)
        a.state_o, a.state_lse = o.data_ptr(), lse.data_ptr()
        need = lib.pab200_decode_int4_workspace_size(a)
        ws = torch.empty(need, dtype=torch.uint8, device=cuda_device)
        st = torch.cuda.current_stream().cuda_stream
        assert lib.pab200_decode_int4(a, ws.data_ptr(), need, st) == 0
        states.append((o.view(B, G * Hkv, D), lse.view(B, G * Hkv)))
        torch.cuda.synchronize()
        check_attention(states[-1][0], q, kp, vp, table, ln, scale, bs, Hkv, dt)
        kv = op.get_rows(kp, D, bs, dt, False)
        for s in range(B):
            for h in range(G * Hkv):
                n = int(ln[s])
                got = float(states[-1][1][s, h])
                if n == 0:
                    assert got == -math.inf
                    continue
                k = np.concatenate([kv[int(e) * Hkv + h // G] for e in table[s, :(n + bs - 1) // bs]])[:n]
                sc = k @ q[s, h].double().numpy() * scale
                want = sc.max() + math.log(np.exp(sc - sc.max()).sum())
                # scores: as in check_attention; the sum and its logarithm: 2^-18
                size = np.abs(q[s, h].double().numpy()) @ np.abs(k).max(0) * scale
                assert abs(got - want) <= 128 * 2.0 ** -24 * 2 * size + 2.0 ** -18 * (1 + abs(want))
    out = pa.merge_states(torch.stack([o for o, _ in states]), torch.stack([l for _, l in states]),
                          out_dtype=dt)
    check_attention(out.view_as(q), q, kp, vp, bt, lens, scale, bs, Hkv, dt)


def test_attention_per_head_pages_and_bad_ids(cuda_device):
    """Reference page layout with lengths per head; pages out of range read as zeros."""
    dt, D, G, Hkv, bs = BF, 128, 4, 3, 16
    g = torch.Generator().manual_seed(5)
    lens = torch.tensor([[50, 0, 300], [16, 700, 1]], dtype=torch.int32)
    bt, pool = tables(lens, bs)
    bt[0, 2, 3], bt[1, 1, 0], bt[1, 1, 40] = 10 ** 6, -5, -1
    kp = random_pages(pool, D, bs, dt, g, False)
    vp = random_pages(pool, D, bs, dt, g, True)
    q = torch.randn((2, G * Hkv, D), generator=g).to(dt)
    out = torch.empty_like(q).to(cuda_device)
    pa.paged_attention_int4(out, q.to(cuda_device), torch.from_numpy(kp).to(cuda_device),
                            torch.from_numpy(vp).to(cuda_device), bt.to(cuda_device),
                            lens.to(cuda_device), 0.09, bs)
    assert pa.read_status() == _lib.STATUS_BAD_PAGE_ID
    check_attention(out, q, kp, vp, bt, lens, 0.09, bs, Hkv, dt, per_head_pages=True)


def test_attention_long_context_is_split(cuda_device):
    """One sequence of 40,001 tokens over every warp; lengths past the table are clamped."""
    dt, D, G, Hkv, bs = HF, 128, 2, 1, 16
    g = torch.Generator().manual_seed(6)
    L = 40001
    n = (L + bs - 1) // bs
    pages = 64                                   # pages repeat: a table may name one twice
    kp = random_pages(pages, D, bs, dt, g, False)
    vp = random_pages(pages, D, bs, dt, g, True)
    bt = torch.randint(0, pages, (1, n), generator=g, dtype=torch.int32)
    q = torch.randn((1, G, D), generator=g).to(dt)
    out = torch.empty_like(q).to(cuda_device)
    args = [torch.from_numpy(p).view(pages, 1, -1).to(cuda_device) for p in (kp, vp)]
    pa.paged_attention_int4(out, q.to(cuda_device), *args, bt.to(cuda_device),
                            torch.tensor([L], dtype=torch.int32, device=cuda_device), 0.1, bs)
    check_attention(out, q, kp, vp, bt, torch.tensor([L]), 0.1, bs, Hkv, dt)
    pa.paged_attention_int4(out, q.to(cuda_device), *args, bt.to(cuda_device),
                            torch.tensor([n * bs + 999], dtype=torch.int32, device=cuda_device), 0.1, bs)
    assert pa.read_status() == _lib.STATUS_SEQLEN_CLAMP
    check_attention(out, q, kp, vp, bt, torch.tensor([n * bs]), 0.1, bs, Hkv, dt)


def test_attention_offsets_past_32_bits(cuda_device):
    """Pages beyond 4 GiB of the cache."""
    dt, D, G, Hkv, bs = BF, 128, 4, 1, 64
    g = torch.Generator().manual_seed(7)
    pool = (5 << 30) // op.page_bytes(D, bs)
    ids = torch.tensor([[pool - 1, 3, pool - 2, pool // 2]], dtype=torch.int32)
    kp = random_pages(4, D, bs, dt, g, False)
    vp = random_pages(4, D, bs, dt, g, True)
    kc, vc = (torch.empty((pool, 1, op.page_bytes(D, bs)), dtype=torch.uint8, device=cuda_device)
              for _ in range(2))
    kc[ids[0].long().to(cuda_device), 0] = torch.from_numpy(kp).to(cuda_device)
    vc[ids[0].long().to(cuda_device), 0] = torch.from_numpy(vp).to(cuda_device)
    q = torch.randn((1, G, D), generator=g).to(dt)
    out = torch.empty_like(q).to(cuda_device)
    lens = torch.tensor([250], dtype=torch.int32)
    pa.paged_attention_int4(out, q.to(cuda_device), kc, vc, ids.to(cuda_device), lens.to(cuda_device),
                            0.1, bs)
    check_attention(out, q, kp, vp, torch.tensor([[0, 1, 2, 3]]), lens, 0.1, bs, Hkv, dt)
    # and an append there
    x = torch.randn((1, 1, D), generator=g).to(dt)
    pa.kv_append_int4(kc, vc, x.to(cuda_device), x.to(cuda_device), lens.to(cuda_device),
                      ids.to(cuda_device), bs)
    c, s, lo = op.quantise(x)
    op.put_row(kp[3], bs, 250 % bs, c[0, 0], s[0, 0], lo[0, 0], False)
    assert np.array_equal(kc[pool // 2, 0].cpu().numpy(), kp[3])


def test_two_streams_and_graph(cuda_device):
    """Calls on two streams at once, and a captured append + attention step
    replayed while its inputs change."""
    dt, D, G, Hkv, bs, B = BF, 128, 4, 2, 16, 3
    g = torch.Generator().manual_seed(8)
    lens = torch.tensor([100, 31, 0], dtype=torch.int32)
    bt, pool = tables(lens + 40, bs)
    kp = random_pages(pool * Hkv, D, bs, dt, g, False)
    vp = random_pages(pool * Hkv, D, bs, dt, g, True)
    q = torch.randn((2, B, G * Hkv, D), generator=g).to(dt)
    kc, vc = (torch.from_numpy(p).view(pool, Hkv, -1).to(cuda_device) for p in (kp, vp))
    btd, ld, qd = bt.to(cuda_device), lens.to(cuda_device), q.to(cuda_device)
    outs = [torch.empty_like(qd[0]) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                pa.paged_attention_int4(outs[i], qd[i], kc, vc, btd, ld, 0.1, bs)
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(outs[i], q[i], kp, vp, bt, lens, 0.1, bs, Hkv, dt)
    x = torch.zeros((B, Hkv, D), dtype=dt, device=cuda_device)
    out, qs = torch.empty_like(qd[0]), qd[0].clone()

    def step():
        pa.kv_append_int4(kc, vc, x, x, ld, btd, bs)
        pa.paged_attention_int4(out, qs, kc, vc, btd, ld, 0.1, bs)

    with torch.cuda.stream(streams[0]):
        step()                                     # warm-up: writes one token of zeros
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    zero = torch.zeros((B, Hkv, D), dtype=dt)
    cur = lens.clone()
    views = kp.reshape(pool, Hkv, -1), vp.reshape(pool, Hkv, -1)
    cur = expect_append(*views, zero, zero, cur, bt, bs, None, False)
    for i in range(3):
        xn = torch.randn((B, Hkv, D), generator=g).to(dt)
        x.copy_(xn)
        qs.copy_(q[i % 2])
        graph.replay()
        torch.cuda.synchronize()
        cur = expect_append(*views, xn, xn, cur, bt, bs, None, False)
        assert torch.equal(ld.cpu(), cur)
        check_attention(out, q[i % 2], kp, vp, bt, cur, 0.1, bs, Hkv, dt)
