"""Key bounds, page selection and page-sparse decode on a GPU: bounds and
selected pages exactly, attention against the dense call over the same pages."""
import math

import numpy as np
import pytest
import torch

import pagedattention_b200 as pa
from oracle import pages as op
from pagedattention_b200 import _lib, kernel_b200
from tests.test_int4_gpu import check_attention, half_step, tables

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def expect_bounds(bounds, k, lens, bt, bs, cu, per_head):
    """Restatement on CPU copies, in place.  bounds (P, 2, D) by page id."""
    Hkv = k.shape[1]
    for s in range(lens.shape[0]):
        a, b = (s, s + 1) if cu is None else (int(cu[s]), int(cu[s + 1]))
        for h in range(Hkv):
            L = int(lens[s, h] if lens.dim() == 2 else lens[s])
            for j in range(b - a):
                i = (L + j) // bs
                if L < 0 or i >= bt.shape[-1]:
                    continue
                e = int(bt[s, h, i] if bt.dim() == 3 else bt[s, i])
                pid = e if per_head else e * Hkv + h
                if pid < 0 or pid >= bounds.shape[0]:
                    continue
                x = k[a + j, h]
                if (L + j) % bs == 0:
                    bounds[pid, 0] = bounds[pid, 1] = x
                else:
                    bounds[pid, 0] = torch.minimum(bounds[pid, 0], x)
                    bounds[pid, 1] = torch.maximum(bounds[pid, 1], x)


@pytest.mark.parametrize("dt,D,bs,Hkv,lens,new,per_head", [
    (BF, 128, 16, 8, [0, 15, 16, 100], None, False),
    (HF, 64, 8, 1, [0, 7, 3, 61], [1, 20, 0, 33], False),
    (BF, 256, 32, 2, [5, 0], [70, 1], True),
    (HF, 128, 64, 3, [63, 1, 0, 64], [2, 200, 65, 64], False),
    (BF, 64, 16, 5, [0], [513], True),
])
@pytest.mark.parametrize("off", [0, 1])
def test_bounds_exact(cuda_device, dt, D, bs, Hkv, lens, new, per_head, off):
    g = torch.Generator().manual_seed(D)
    lens = torch.tensor(lens, dtype=torch.int32)
    B = lens.numel()
    n = torch.ones(B, dtype=torch.int32) if new is None else torch.tensor(new, dtype=torch.int32)
    cu = None
    if new is not None:
        cu = torch.zeros(B + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(n, 0)
    total = lens + n
    bt, pool = tables(total[:, None].expand(B, Hkv).contiguous() if per_head else total, bs)
    P = pool if per_head else pool * Hkv
    N = int(n.sum()) + (0 if cu is None else 2)
    flat = torch.randn((N, Hkv * D + 8), generator=g).to(dt)
    k = flat[:, off:off + Hkv * D].unflatten(1, (Hkv, D))
    kd = flat.to(cuda_device)[:, off:off + Hkv * D].unflatten(1, (Hkv, D))
    k[0, 0, 3] = kd[0, 0, 3] = float("nan")
    bounds = torch.randn((P, 2, D), generator=g).to(dt)
    bd = bounds.to(cuda_device).view((P, 2, D) if per_head else (pool, Hkv, 2, D))
    ld = lens.to(cuda_device)
    pa.kv_append_status()
    pa.update_page_bounds(bd, kd, ld, bt.to(cuda_device), bs,
                          cu_new=None if cu is None else cu.to(cuda_device))
    assert pa.kv_append_status() == 0
    expect_bounds(bounds, k, lens, bt, bs, cu, per_head)
    assert torch.equal(torch.nan_to_num(bd.cpu().view(P, 2, D), nan=99.0),
                       torch.nan_to_num(bounds, nan=99.0))
    assert torch.equal(ld.cpu(), lens)


def test_bounds_places_that_do_not_exist(cuda_device):
    dt, D, bs, Hkv = BF, 64, 8, 2
    lens = torch.tensor([30, 4, -2, 0], dtype=torch.int32)
    cu = torch.tensor([0, 5, 25, 28, 37], dtype=torch.int32)
    bt = torch.tensor([[0, 1, 2, 3], [4, 99, 5, 6], [7, 8, 9, 10], [11, -1, 12, 13]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    k = torch.randn((37, Hkv, D), generator=g).to(dt)
    bounds = torch.randn((28, 2, D), generator=g).to(dt)
    bd = bounds.to(cuda_device).view(14, Hkv, 2, D)
    pa.kv_append_status()
    pa.update_page_bounds(bd, k.to(cuda_device), lens.to(cuda_device), bt.to(cuda_device), bs,
                          cu_new=cu.to(cuda_device))
    assert pa.kv_append_status() == (_lib.STATUS_APPEND_FULL | _lib.STATUS_BAD_PAGE_ID
                                     | _lib.STATUS_NEG_SEQLEN)
    expect_bounds(bounds, k, lens, bt, bs, cu, False)
    assert torch.equal(bd.cpu().view(28, 2, D), bounds)


# --------------------------------------------------------------- selection

def expect_select(q, bounds, bt, lens, bs, keep, sink, recent, Hkv, per_head):
    B, Hq, _ = q.shape
    G = Hq // Hkv
    tabs = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    out = torch.zeros((B, Hkv), dtype=torch.int32)
    cap = bt.shape[-1] * bs
    for s in range(B):
        for h in range(Hkv):
            L = int(lens[s, h] if lens.dim() == 2 else lens[s])
            L = min(max(L, 0), cap)
            n = (L + bs - 1) // bs
            row = bt[s, h] if bt.dim() == 3 else bt[s]
            ids = [int(e) if per_head else int(e) * Hkv + h for e in row[:n]]
            b, bad = np.zeros((n, 2, q.shape[2])), set()
            for i, pid in enumerate(ids):
                if 0 <= pid < bounds.shape[0]:
                    b[i] = bounds[pid].double().numpy()
                else:
                    bad.add(i)
            got = op.select(q[s, h * G:(h + 1) * G].double().numpy(), b, n, keep, sink, recent, bad)
            tabs[s, h, :len(got)] = row[torch.tensor(got, dtype=torch.long)]
            out[s, h] = (len(got) - 1) * bs + L - (n - 1) * bs if n else 0
    return tabs, out


SELECT = [  # dtype, D, G, Hkv, bs, lens, keep, sink, recent
    (BF, 128, 4, 2, 16, [1000, 0, 1, 333, 128, 129], 8, 1, 1),
    (HF, 64, 8, 1, 8, [5000, 63, 64, 65], 8, 0, 1),
    (BF, 256, 2, 3, 32, [700, 2000], 5, 2, 2),
    (HF, 128, 1, 2, 64, [4097, 260], 4, 3, 1),       # nothing left to choose
    (BF, 64, 32, 1, 8, [9000], 300, 1, 4),
    (HF, 128, 3, 5, 16, [17, 600], 1, 0, 1),         # only the last page
    (BF, 128, 8, 1, 8, [20000], 1030, 1, 1),
]


@pytest.mark.parametrize("dt,D,G,Hkv,bs,lens,keep,sink,recent", SELECT)
@pytest.mark.parametrize("per_head", [False, True])
def test_select_exact(cuda_device, dt, D, G, Hkv, bs, lens, keep, sink, recent, per_head):
    g = torch.Generator().manual_seed(keep + D)
    lens = torch.tensor(lens, dtype=torch.int32)
    B = lens.numel()
    ll = lens[:, None].expand(B, Hkv).contiguous() if per_head else lens
    bt, pool = tables(ll, bs)
    P = pool if per_head else pool * Hkv
    x = torch.randn((P, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    bd = bounds.to(cuda_device).view((P, 2, D) if per_head else (pool, Hkv, 2, D))
    pa.kv_append_status()
    tabs, out = pa.select_pages(q.to(cuda_device), bd, bt.to(cuda_device), ll.to(cuda_device), bs, keep,
                                num_sink=sink, num_recent=recent)
    assert pa.kv_append_status() == 0
    want, wl = expect_select(q, bounds, bt, ll, bs, keep, sink, recent, Hkv, per_head)
    assert torch.equal(out.cpu(), wl)
    assert torch.equal(tabs.cpu(), want)


def test_select_ties_nan_and_bad_pages(cuda_device):
    """Equal scores go to the lower page, NaN ranks first, bad ids last; -0 is +0."""
    dt, D, G, Hkv, bs = BF, 64, 2, 1, 8
    n, keep = 400, 50
    bounds = torch.zeros((n, 2, D), dtype=dt)
    bounds[::2, 1, 0] = 1.0                          # two scores in all
    bounds[1::4, 0, 1], bounds[1::4, 1, 1] = -0.0, -0.0
    bounds[100] = float("nan")
    bounds[301] = float("nan")
    bounds[200:203, 1, 0] = 5.0
    q = torch.zeros((1, G, D), dtype=dt)
    q[:, :, 0] = 1.0
    bt = torch.arange(n, dtype=torch.int32)[None].clone()
    bt[0, 7], bt[0, 11] = -3, 10 ** 6
    lens = torch.tensor([n * bs - 3], dtype=torch.int32)
    for keep in (50, 4, 380, 399):
        pa.kv_append_status()
        tabs, out = pa.select_pages(q.to(cuda_device), bounds.to(cuda_device).view(n, 1, 2, D),
                                    bt.to(cuda_device), lens.to(cuda_device), bs, keep)
        assert pa.kv_append_status() == _lib.STATUS_BAD_PAGE_ID
        want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, Hkv, False)
        assert torch.equal(out.cpu(), wl) and torch.equal(tabs.cpu(), want)


def select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, Hkv):
    """The C entry's tables and lengths, with words before and behind them that
    no unit may touch."""
    B, Hq, D = q.shape
    lib = _lib.load()
    qd, bd, btd, ld = (x.to(cuda_device) for x in (q, bounds, bt, lens))
    units, guard = B * Hkv, 4096
    tabs = torch.full((units * keep + 2 * guard,), 77, dtype=torch.int32, device=cuda_device)
    out = torch.full((units + 2 * guard,), 77, dtype=torch.int32, device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    a = _lib.SelectArgs(
        qd.data_ptr(), bd.data_ptr(), ld.data_ptr(), btd.data_ptr(), tabs[guard:].data_ptr(),
        out[guard:].data_ptr(), status.data_ptr(), 0 if q.dtype == BF else 1, B, Hq, Hkv, D, bs,
        bt.shape[1], keep, 1, 1, bounds.shape[0], Hq * D, D, 1, 0, bt.shape[1], 0, 1, Hkv, 1)
    need = lib.pab200_select_pages_workspace_size(a)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    assert lib.pab200_select_pages(a, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    tabs, out = tabs.cpu(), out.cpu()
    for x in (tabs, out):
        assert (x[:guard] == 77).all() and (x[-guard:] == 77).all()
    return tabs[guard:-guard].view(B, Hkv, keep), out[guard:-guard].view(B, Hkv), int(status[0])


@pytest.mark.parametrize("n,nans,keep", [
    (300, 100, 32),        # more NaN pages than places
    (300, 299, 32), (700, 500, 64),
    (2500, 1000, 256),     # 1,024 threads: more open pages than are compared directly
    (2500, 2, 4), (700, 65, 64),
])
def test_select_many_nan_pages(cuda_device, n, nans, keep):
    """NaN pages beyond the free places: the earlier ones are kept, and neither the
    recent pages nor another unit's table nor anything behind the last is written."""
    dt, D, G, Hkv, bs, B = BF, 64, 2, 2, 8, 3
    g = torch.Generator().manual_seed(n + nans)
    pool = B * n
    x = torch.randn((pool * Hkv, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    bt = torch.randperm(pool, generator=g).to(torch.int32).view(B, n)
    for s in range(B - 1):                        # the last sequence has none
        for h in range(Hkv):
            at = torch.randperm(n, generator=g)[:nans]
            bounds[bt[s, at].long() * Hkv + h, :, 3] = float("nan")
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    lens = torch.full((B,), n * bs - 1, dtype=torch.int32)
    tabs, out, status = select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, Hkv)
    want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, Hkv, False)
    assert status == 0 and torch.equal(out, wl) and torch.equal(tabs, want)


@pytest.mark.parametrize("n,keep", [(300, 32), (2500, 256)])
def test_select_nan_query_and_a_bad_page(cuda_device, n, keep):
    """A NaN in the query makes every page NaN but the one whose id is out of range."""
    dt, D, G, Hkv, bs, B = HF, 64, 2, 1, 8, 2
    g = torch.Generator().manual_seed(n)
    x = torch.randn((B * n, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    bt = torch.randperm(B * n, generator=g).to(torch.int32).view(B, n)
    bt[0, 5] = -1
    q = torch.randn((B, G, D), generator=g).to(dt)
    q[0, 1, 7] = float("nan")
    lens = torch.full((B,), n * bs, dtype=torch.int32)
    tabs, out, status = select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, Hkv)
    want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, Hkv, False)
    assert status == _lib.STATUS_BAD_PAGE_ID and torch.equal(out, wl) and torch.equal(tabs, want)


@pytest.mark.parametrize("threads", [256, 1024])
def test_select_nan_pages_after_large_terms(cuda_device, threads):
    """Scores that only 64 bits tell apart (large terms that cancel), read before
    NaN pages and those before small ones: the NaNs hide none of the sizes."""
    dt, D, G, bs = BF, 64, 1, 8
    g = torch.Generator().manual_seed(threads)
    n, keep = 3 * threads + 2, threads + threads // 2 + 2
    rows = torch.zeros((n, D))
    first = rows[1:1 + threads]
    first[:, 0], first[:, 63] = 4096.0, -4096.0
    first[:, 1:63] = torch.randint(-64, 65, (threads, 62), generator=g) * 2.0 ** -18
    rows[1 + threads:1 + 2 * threads] = float("nan")
    rows[1 + 2 * threads:-1, 0] = -1.0
    bounds = rows[:, None].expand(n, 2, D).to(dt).contiguous()
    q = torch.ones((1, G, D), dtype=dt)
    bt = torch.arange(n, dtype=torch.int32)[None].contiguous()
    lens = torch.tensor([n * bs], dtype=torch.int32)
    tabs, out, _ = select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, 1)
    want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, 1, False)
    assert torch.equal(out, wl) and torch.equal(tabs, want)


@pytest.mark.parametrize("dt,n,keep,spread", [
    (BF, 3000, 700, 0.0),      # all alike but one page in seven: only the order decides
    (HF, 5000, 1200, 2.0 ** -22), (BF, 9000, 40, 2.0 ** -20), (HF, 600, 300, 2.0 ** -24)])
def test_select_scores_next_to_the_border(cuda_device, dt, n, keep, spread):
    """Scores that an fp32 sum cannot tell apart: a common large part, and
    differences of a few fp32 units, across hundreds of pages."""
    D, G, bs = 128, 4, 8
    g = torch.Generator().manual_seed(n)
    q = torch.randn((1, G, D), generator=g).to(dt)
    q[:, :, 1] = spread
    base = torch.randn((1, 2, D), generator=g).abs() + 0.5
    bounds = base.expand(n, 2, D).clone()
    bounds[:, 0] = -bounds[:, 0]
    bounds = bounds.to(dt)
    # element 1 moves the score by spread * its value
    bounds[:, :, 1] = torch.randint(0, 40, (n, 1), generator=g).to(dt)
    if spread == 0.0:
        bounds[::7, 1, 2] += 1.0
    bt = torch.randperm(n, generator=g).to(torch.int32)[None]
    lens = torch.tensor([n * bs], dtype=torch.int32)
    tabs, out = pa.select_pages(q.to(cuda_device), bounds.to(cuda_device).view(n, 1, 2, D),
                                bt.to(cuda_device), lens.to(cuda_device), bs, keep)
    want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, 1, False)
    assert torch.equal(out.cpu(), wl) and torch.equal(tabs.cpu(), want)


def test_select_infinite_bounds(cuda_device):
    """A page with infinite bounds leaves its unit to the 64-bit scores."""
    dt, D, bs, n = HF, 64, 8, 2500
    g = torch.Generator().manual_seed(4)
    x = torch.randn((n, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    bounds[77, 1, 5] = float("inf")
    bounds[1234, 0, 5] = -float("inf")
    q = torch.randn((1, 3, D), generator=g).to(dt)
    q[0, :, 5] = torch.tensor([1.0, -1.0, 2.0])    # no 0 * inf in either form of the sum
    bt = torch.randperm(n, generator=g).to(torch.int32)[None]
    lens = torch.tensor([n * bs - 1], dtype=torch.int32)
    tabs, out = pa.select_pages(q.to(cuda_device), bounds.to(cuda_device).view(n, 1, 2, D),
                                bt.to(cuda_device), lens.to(cuda_device), bs, 200)
    want, wl = expect_select(q, bounds, bt, lens, bs, 200, 1, 1, 1, False)
    assert torch.equal(out.cpu(), wl) and torch.equal(tabs.cpu(), want)


@pytest.mark.parametrize("n", [300, 2500])
@pytest.mark.parametrize("dt", [BF, HF])
def test_select_infinite_bounds_by_definition(cuda_device, dt, n):
    """max(q min, q max) of an infinite bound: the finite product where the infinite
    one is the smaller, NaN only where the query is 0."""
    D, bs, G, keep = 64, 8, 3, 40
    g = torch.Generator().manual_seed(n)
    x = torch.randn((n, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    inf = float("inf")
    q = torch.randn((4, G, D), generator=g).to(dt)
    q[:, :, 5], q[:, :, 6] = q[:, :, 5].abs() + 0.1, -q[:, :, 6].abs() - 0.1
    q[1, 1, 5] = 0.0                              # 0 * inf
    q[2, :, 5] = torch.tensor([inf, 1.0, 2.0])    # an infinite query
    q[3, 1, 9] = -0.0
    for i in range(20, 40):
        bounds[i, 0, 5] = -inf
        bounds[i + 50, 1, 6] = inf
    bounds[100, 1, 5] = inf                       # ranks first
    bounds[101, 0, 6] = -inf
    bounds[102, :, 5] = -inf                      # ranks last
    bounds[103, 0, 9] = -inf
    bounds[104, 1, 9] = 0.0
    bt = torch.randperm(n, generator=g).to(torch.int32)[None].expand(4, n).contiguous()
    lens = torch.full((4,), n * bs - 1, dtype=torch.int32)
    tabs, out, _ = select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, 1)
    with np.errstate(invalid="ignore"):          # 0 * inf, inf - inf
        want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, 1, False)
    for s in range(4):
        assert torch.equal(out[s], wl[s]) and torch.equal(tabs[s], want[s]), s


@pytest.mark.parametrize("width", [2000, 9000])
def test_select_wide_tables(cuda_device, width):
    """Tables far wider than the contexts; what lies behind a context is not read."""
    dt, D, G, Hkv, bs, keep = BF, 128, 2, 2, 16, 20
    g = torch.Generator().manual_seed(width)
    lens = torch.tensor([3000, 0, 5000, 17], dtype=torch.int32)
    bt, pool = tables(lens, bs, maxb=width)
    x = torch.randn((pool * Hkv, 2, D), generator=g).to(dt)
    bounds = torch.stack((x.amin(1), x.amax(1)), 1)
    q = torch.randn((4, G * Hkv, D), generator=g).to(dt)
    tabs, out, status = select_within_guards(cuda_device, q, bounds, bt, lens, bs, keep, Hkv)
    want, wl = expect_select(q, bounds, bt, lens, bs, keep, 1, 1, Hkv, False)
    assert status == 0 and torch.equal(out, wl) and torch.equal(tabs, want)


def test_select_lengths_out_of_range(cuda_device):
    dt, D, bs = HF, 64, 8
    g = torch.Generator().manual_seed(0)
    bounds = torch.randn((20, 2, D), generator=g).to(dt).sort(1).values
    q = torch.randn((2, 2, D), generator=g).to(dt)
    bt = torch.arange(20, dtype=torch.int32).view(2, 10)
    lens = torch.tensor([-1, 10 ** 6], dtype=torch.int32)
    pa.kv_append_status()
    tabs, out = pa.select_pages(q.to(cuda_device), bounds.view(20, 1, 2, D).to(cuda_device),
                                bt.to(cuda_device), lens.to(cuda_device), bs, 4)
    assert pa.kv_append_status() == _lib.STATUS_NEG_SEQLEN | _lib.STATUS_SEQLEN_CLAMP
    want, wl = expect_select(q, bounds, bt, lens, bs, 4, 1, 1, 1, False)
    assert torch.equal(out.cpu(), wl) and torch.equal(tabs.cpu(), want)


# --------------------------------------------------------- sparse attention

@pytest.mark.parametrize("dt,D,G,Hkv,bs,lens,keep,layout", [
    (BF, 128, 4, 2, 16, [1000, 0, 1, 333, 128, 129], 8, "HND"),
    (HF, 64, 8, 1, 8, [3000, 63], 16, "HND"),
    (HF, 128, 8, 2, 32, [1500, 40], 7, "NHD"),
    (BF, 256, 2, 1, 64, [3000], 3, "NHD"),
    (BF, 128, 32, 1, 16, [900], 12, "HND"),
])
def test_sparse_attention(cuda_device, dt, D, G, Hkv, bs, lens, keep, layout):
    g = torch.Generator().manual_seed(D + G)
    lens = torch.tensor(lens, dtype=torch.int32)
    B = lens.numel()
    bt, pool = tables(lens, bs)
    k = torch.randn((pool, Hkv, bs, D), generator=g).to(dt)
    v = torch.randn((pool, Hkv, bs, D), generator=g).to(dt)
    bounds = torch.stack((k.amin(2), k.amax(2)), 2).contiguous()
    q = torch.randn((B, G * Hkv, D), generator=g).to(dt)
    scale = 1 / math.sqrt(D)

    def lay(x):
        return (x if layout == "HND" else x.transpose(1, 2)).contiguous().to(cuda_device)

    kd, vd, qd, bd = lay(k), lay(v), q.to(cuda_device), bounds.to(cuda_device)
    btd, ld = bt.to(cuda_device), lens.to(cuda_device)
    out = torch.full_like(qd, 9.0)
    tabs, sl = pa.paged_attention_sparse(out, qd, kd, vd, bd, btd, ld, scale, bs, keep,
                                         kv_layout=layout)
    want, wl = expect_select(q, bounds.view(-1, 2, D), bt, lens, bs, keep, 1, 1, Hkv, False)
    assert torch.equal(tabs.cpu(), want) and torch.equal(sl.cpu(), wl)
    t2, s2 = pa.select_pages(qd, bd, btd, ld, bs, keep)
    assert torch.equal(t2, tabs) and torch.equal(s2, sl)
    # in 64 bits over the selected pages: the probabilities' rounding to T
    # (half a step of each, against values up to max |v|) and the output's
    for s in range(B):
        for h in range(Hkv):
            L = int(wl[s, h])
            ids = want[s, h, :(L + bs - 1) // bs].long()
            kk, vv = (x[ids, h].reshape(-1, D)[:L].double().numpy() for x in (k, v))
            qq = q[s, h * G:(h + 1) * G].double().numpy()
            ref = op.attention(qq, kk, vv, scale)
            have = out[s, h * G:(h + 1) * G].double().cpu().numpy()
            if L == 0:
                assert (have == 0).all()
                continue
            size = (np.abs(qq) @ np.abs(kk).T).max(1)[:, None] * scale
            tol = half_step(dt) * (np.abs(ref) + np.abs(vv).max()) + \
                (2.0 ** -18 + 128 * 2.0 ** -24 * 2 * size) * np.abs(vv).max()
            assert (np.abs(have - ref) <= tol).all(), (s, h)
    # keeping every page is the dense call
    full = torch.empty_like(out)
    pa.paged_attention(full, qd, kd, vd, btd, ld, scale, bs, kv_layout=layout)
    n = max(int((lens.max() + bs - 1) // bs), 2)
    pa.paged_attention_sparse(out, qd, kd, vd, bd, btd, ld, scale, bs, n, kv_layout=layout)
    tol = 2 * half_step(dt) * (full.float().abs() + v.float().abs().max()) + 1e-3
    assert ((out.float() - full.float()).abs() <= tol).all()


def test_empty_batch(cuda_device):
    """No sequences: empty results, like the other calls of a step."""
    dt, D, Hkv, bs = BF, 64, 2, 8
    q = torch.zeros((0, 4, D), dtype=dt, device=cuda_device)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    bt = torch.zeros((0, 5), dtype=torch.int32, device=cuda_device)
    pool = torch.zeros((3, Hkv, bs, D), dtype=dt, device=cuda_device)
    bounds = torch.zeros((3, Hkv, 2, D), dtype=dt, device=cuda_device)
    for tabs, sl in (pa.select_pages(q, bounds, bt, lens, bs, 4),
                     pa.paged_attention_sparse(q.clone(), q, pool, pool, bounds, bt, lens, 0.1, bs, 4)):
        assert tabs.shape == (0, Hkv, 4) and sl.shape == (0, Hkv)
        assert tabs.dtype == sl.dtype == torch.int32
    kc, vc = pa.int4_cache(3, Hkv, bs, D, device=cuda_device)
    x = torch.zeros((0, Hkv, D), dtype=dt, device=cuda_device)
    pa.update_page_bounds(bounds, x, lens, bt, bs)
    pa.kv_append_int4(kc, vc, x, x, lens, bt, bs)
    pa.paged_attention_int4(q.clone(), q, kc, vc, bt, lens, 0.1, bs)


@pytest.mark.parametrize("int4", [False, True])
def test_kernel_events_of_the_new_decode_calls(cuda_device, int4):
    """Events set around the decode kernel of every decode call are recorded by
    the 4-bit and the page-sparse calls too."""
    dt, D, Hkv, bs = BF, 64, 2, 8
    q = torch.zeros((2, 4, D), dtype=dt, device=cuda_device)
    lens = torch.full((2,), 300, dtype=torch.int32, device=cuda_device)
    bt = torch.zeros((2, 40), dtype=torch.int32, device=cuda_device)
    pool = torch.zeros((3, Hkv, bs, D), dtype=dt, device=cuda_device)
    bounds = torch.zeros((3, Hkv, 2, D), dtype=dt, device=cuda_device)
    kc, vc = pa.int4_cache(3, Hkv, bs, D, device=cuda_device)
    before, after, mark = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    for e in (before, after, mark):
        e.record()
    with kernel_b200.kernel_events(before, after):
        if int4:
            pa.paged_attention_int4(q.clone(), q, kc, vc, bt, lens, 0.1, bs)
        else:
            pa.paged_attention_sparse(q.clone(), q, pool, pool, bounds, bt, lens, 0.1, bs, 4)
    torch.cuda.synchronize()
    assert mark.elapsed_time(before) > 0 and before.elapsed_time(after) > 0


def test_sparse_attention_on_the_tcgen05_kernel(cuda_device, monkeypatch):
    """The opt-in decode kernel takes a selection's tables too."""
    monkeypatch.setenv("PAB200_TC", "1")
    # freed: workspaces that come from here are not zero
    torch.full((64 << 20,), 0x7f, dtype=torch.uint8, device=cuda_device)
    test_sparse_attention(cuda_device, BF, 64, 32, 1, 16, [900, 0, 40, 333], 12, "HND")


def test_captured_ragged_and_sparse_calls(cuda_device):
    """A chunk of a prompt (bounds, append, read-back) and a page-sparse decode in
    two graphs, replayed in turn on two streams while their inputs change."""
    dt, D, G, Hkv, bs, B, keep = HF, 64, 8, 2, 8, 3, 5
    g = torch.Generator().manual_seed(12)
    lens = torch.tensor([3, 0, 40], dtype=torch.int32)
    new = torch.tensor([20, 1, 9], dtype=torch.int32)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(new, 0)
    bt, pool = tables(lens + new, bs)
    N = int(new.sum())
    kc, vc = pa.int4_cache(pool, Hkv, bs, D, device=cuda_device)
    bounds = torch.zeros((pool, Hkv, 2, D), dtype=dt, device=cuda_device)
    kp = torch.randn((pool, Hkv, bs, D), generator=g).to(dt).to(cuda_device)
    vp = torch.randn((pool, Hkv, bs, D), generator=g).to(dt).to(cuda_device)
    kb = torch.stack((kp.amin(2), kp.amax(2)), 2).contiguous()
    x = torch.zeros((2, N, Hkv, D), dtype=dt, device=cuda_device)
    q = torch.zeros((B, G * Hkv, D), dtype=dt, device=cuda_device)
    out = torch.empty_like(q)
    l0, l1 = lens.to(cuda_device), lens.to(cuda_device)
    tot = (lens + new).to(cuda_device)
    btd, cud = bt.to(cuda_device), cu.to(cuda_device)
    res = {}

    def chunk():
        l1.copy_(l0)
        pa.update_page_bounds(bounds, x[0], l1, btd, bs, cu_new=cud)
        pa.kv_append_int4(kc, vc, x[0], x[1], l1, btd, bs, cu_new=cud)
        res["k"], res["v"] = pa.kv_read_int4(kc, vc, btd, l1, bs, D, dt, starts=l0, cu_out=cud,
                                             num_tokens=N)

    def attend():
        res["t"], res["l"] = pa.paged_attention_sparse(out, q, kp, vp, kb, btd, tot, 0.1, bs, keep)

    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for fn, st in zip((chunk, attend), streams):
        with torch.cuda.stream(st):
            fn()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            fn()
        graphs.append(gr)
    for _ in range(3):
        xn = torch.randn((2, N, Hkv, D), generator=g).to(dt)
        qn = torch.randn((B, G * Hkv, D), generator=g).to(dt)
        x.copy_(xn)
        q.copy_(qn)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(l1.cpu(), lens + new)
        for i, name in enumerate(("k", "v")):
            c, s, lo = op.quantise(xn[i])
            want = lo.double()[..., None] + s.double()[..., None] * c.unflatten(-1, (-1, 64)).double()
            err = (res[name].cpu().double() - want.flatten(-2)).abs()
            assert (err <= half_step(dt) * want.flatten(-2).abs() + 2.0 ** -25).all()
        b = torch.zeros((pool * Hkv, 2, D), dtype=dt)
        expect_bounds(b, xn[0], lens, bt, bs, cu, False)
        fresh = [int(bt[s, i]) for s in range(B)
                 for i in range((int(lens[s]) + bs - 1) // bs, (int(lens[s] + new[s]) + bs - 1) // bs)]
        assert torch.equal(bounds.cpu()[fresh], b.view(pool, Hkv, 2, D)[fresh])
        want, wl = expect_select(qn, kb.cpu().view(-1, 2, D), bt, lens + new, bs, keep, 1, 1, Hkv, False)
        assert torch.equal(res["t"].cpu(), want) and torch.equal(res["l"].cpu(), wl)
        full = torch.empty_like(out)
        pa.paged_attention(full, q, kp, vp, res["t"], res["l"], 0.1, bs)
        # the same tables through the dense call: other splits of the same sums
        tol = 2 * half_step(dt) * (full.float().abs() + vp.float().abs().max()) + 1e-3
        assert ((out.float() - full.float()).abs() <= tol).all()


def test_selections_used_by_the_next_call(cuda_device):
    """Tables and lengths of a selection, read by a decode call that follows it at
    once in a graph, are this replay's, not the last one's."""
    dt, D, G, Hkv, bs, B, keep = BF, 128, 4, 4, 16, 8, 16
    g = torch.Generator().manual_seed(13)
    lens = torch.tensor([900, 16, 0, 333, 1000, 50, 700, 257], dtype=torch.int32)
    bt, pool = tables(torch.full((B,), 1000, dtype=torch.int32), bs)
    k, v = (torch.randn((pool, Hkv, bs, D), generator=g).to(dt).to(cuda_device) for _ in range(2))
    bounds = torch.stack((k.amin(2), k.amax(2)), 2).contiguous()
    q, ld, btd = torch.zeros((B, G * Hkv, D), dtype=dt, device=cuda_device), lens.to(cuda_device), bt.to(cuda_device)
    out1, out2, out3 = (torch.empty_like(q) for _ in range(3))
    res = {}

    def step():
        res["a"] = pa.select_pages(q, bounds, btd, ld, bs, keep)
        pa.paged_attention(out1, q, k, v, *res["a"], 0.1, bs)
        res["b"] = pa.paged_attention_sparse(out2, q, k, v, bounds, btd, ld, 0.1, bs, keep)
        pa.paged_attention(out3, q, k, v, *res["b"], 0.1, bs)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        qn = torch.randn((B, G * Hkv, D), generator=g).to(dt)
        q.copy_(qn)
        lens = lens.roll(1)
        ld.copy_(lens)
        graph.replay()
        torch.cuda.synchronize()
        want, wl = expect_select(qn, bounds.cpu().view(-1, 2, D), bt, lens, bs, keep, 1, 1, Hkv, False)
        for t, n in res.values():
            assert torch.equal(t.cpu(), want) and torch.equal(n.cpu(), wl)
        full = torch.empty_like(q)
        pa.paged_attention(full, q, k, v, want.to(cuda_device), wl.to(cuda_device), 0.1, bs)
        assert torch.equal(out1, full) and torch.equal(out3, full)


def test_serving_steps_together(cuda_device):
    """Prompts and steps: bounds, 4-bit append, selection and 4-bit attention
    over the selection, eager and then replayed from a graph."""
    dt, D, G, Hkv, bs, B, keep = BF, 128, 4, 2, 16, 3, 6
    g = torch.Generator().manual_seed(11)
    prompt = torch.tensor([150, 17, 401], dtype=torch.int32)
    bt, pool = tables(prompt + 40, bs)
    btd = bt.to(cuda_device)
    kc, vc = pa.int4_cache(pool, Hkv, bs, D, device=cuda_device)
    bounds = torch.zeros((pool, Hkv, 2, D), dtype=dt, device=cuda_device)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda_device)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(prompt, 0)
    N = int(cu[-1])
    rows = torch.randn((2, N, Hkv, D), generator=g).to(dt)
    cud = cu.to(cuda_device)
    kd, vd = rows.to(cuda_device)
    pa.update_page_bounds(bounds, kd, lens, btd, bs, cu_new=cud)
    pa.kv_append_int4(kc, vc, kd, vd, lens, btd, bs, cu_new=cud)
    keys = [[rows[0, int(cu[s]) + j] for j in range(int(prompt[s]))] for s in range(B)]
    x = torch.zeros((2, B, Hkv, D), dtype=dt, device=cuda_device)
    q = torch.zeros((B, G * Hkv, D), dtype=dt, device=cuda_device)
    out = torch.empty_like(q)
    res = {}

    def step():
        pa.update_page_bounds(bounds, x[0], lens, btd, bs)
        pa.kv_append_int4(kc, vc, x[0], x[1], lens, btd, bs)
        res["t"], res["l"] = pa.select_pages(q, bounds, btd, lens, bs, keep)
        pa.paged_attention_int4(out, q, kc, vc, res["t"], res["l"], 0.09, bs)

    def fill():
        xn = torch.randn((2, B, Hkv, D), generator=g).to(dt)
        qn = torch.randn((B, G * Hkv, D), generator=g).to(dt)
        x.copy_(xn)
        q.copy_(qn)
        for s in range(B):
            keys[s].append(xn[0, s])
        return qn

    def check(qn):
        torch.cuda.synchronize()
        n = torch.tensor([len(k) for k in keys], dtype=torch.int32)
        assert torch.equal(lens.cpu(), n)
        b = torch.zeros((pool, Hkv, 2, D), dtype=dt)
        for s in range(B):
            kk = torch.stack(keys[s])
            for i in range((len(keys[s]) + bs - 1) // bs):
                part = kk[i * bs:(i + 1) * bs]
                b[int(bt[s, i])] = torch.stack((part.amin(0), part.amax(0)), 1)
        used = torch.cat([bt[s, :(int(n[s]) + bs - 1) // bs] for s in range(B)]).long()
        assert torch.equal(bounds.cpu()[used], b[used])
        want, wl = expect_select(qn, b.view(-1, 2, D), bt, n, bs, keep, 1, 1, Hkv, False)
        assert torch.equal(res["t"].cpu(), want) and torch.equal(res["l"].cpu(), wl)
        check_attention(out, qn, kc.cpu().numpy().reshape(pool * Hkv, -1),
                        vc.cpu().numpy().reshape(pool * Hkv, -1), want, wl, 0.09, bs, Hkv, dt)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(18):                        # over a page's end
            qn = fill()
            step()
        check(qn)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        qn = fill()
        graph.replay()
        check(qn)


def test_append_status_word_is_not_a_graphs(cuda_device):
    """A first call inside a capture: the bits outlive the graph's replays."""
    dt, D, bs = BF, 64, 8
    bounds = torch.zeros((2, 1, 2, D), dtype=dt, device=cuda_device)
    k = torch.zeros((1, 1, D), dtype=dt, device=cuda_device)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    good = torch.zeros((1, 1), dtype=torch.int32, device=cuda_device)
    bad = good - 5
    pa.update_page_bounds(bounds, k, lens, good, bs)
    pa.kv_append_status()
    torch.cuda.synchronize()
    old = dict(kernel_b200._append_status)
    kernel_b200._append_status.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pa.update_page_bounds(bounds, k, lens, good, bs)
        assert pa.kv_append_status(reset=False) == 0
        pa.update_page_bounds(bounds, k, lens, bad, bs)
        graph.replay()
        assert pa.kv_append_status() == _lib.STATUS_BAD_PAGE_ID
    finally:
        kernel_b200._append_status.update(old)
