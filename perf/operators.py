"""Measured cases of the operators around a compressed or sparsely read page
cache: the 4-bit append and read-back, decode attention over the 4-bit cache,
the key bounds of pages, and decode attention over the pages they select.

``run`` computes a case with elementary torch operations (``own`` false), or
through this package's entry points (``own`` true).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 64                              # head elements per (scale, minimum) pair
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]      # element of a code word held by nibble n


# ----------------------------------------------------------------- cases

def _case(name, op, dtype, seqs, q_heads, kv_heads, head, block, lens, new=(1, 1), select=0,
          layout="HND", k_scale=1.0):
    return {"name": name, "op": op, "dtype": dtype, "seqs": seqs, "q_heads": q_heads,
            "kv_heads": kv_heads, "head": head, "block": block, "len_lo": lens[0],
            "len_hi": lens[1], "new_lo": new[0], "new_hi": new[1], "select": select,
            "layout": layout, "k_scale": k_scale}


def listed():
    return [
        # a batch of ragged prompts enters an empty 4-bit cache (8 kv heads of 128)
        _case("append_prompts", "append", "bf16", 12, 32, 8, 128, 16, (0, 0), (700, 4099)),
        # one decode step of a large batch: latency
        _case("append_step", "append", "bf16", 64, 32, 8, 128, 16, (0, 4096)),
        # chunks of a prompt behind tokens that are there, one kv head, small pages, fp16
        _case("append_chunks_mqa", "append", "f16", 37, 32, 1, 64, 8, (0, 500), (1, 513)),
        # decode over the 4-bit cache: the grouped-query batch of the default benchmark
        _case("attend_gqa", "attend", "bf16", 64, 32, 8, 128, 16, (4096, 4096)),
        # few long contexts: work split over a long axis
        _case("attend_long", "attend", "bf16", 4, 32, 8, 128, 16, (32768, 131072)),
        # one kv head for 32 query heads, small pages, fp16, large keys
        _case("attend_mqa", "attend", "f16", 128, 32, 1, 64, 8, (512, 8192), k_scale=4.0),
        # a small multi-head batch: latency
        _case("attend_small", "attend", "f16", 8, 32, 32, 128, 16, (0, 1024)),
        # bounds of prompts' keys
        _case("bounds_prompts", "bounds", "bf16", 12, 32, 8, 128, 16, (0, 0), (700, 4099)),
        # bounds in a decode step
        _case("bounds_step", "bounds", "f16", 64, 32, 8, 128, 16, (0, 4096)),
        # few long contexts read through 256 pages each
        _case("sparse_long", "sparse", "bf16", 4, 32, 8, 128, 16, (32768, 131072), select=256),
        # a batch of mixed contexts, larger pages and groups, token-major pool
        _case("sparse_mixed", "sparse", "f16", 48, 64, 8, 128, 32, (64, 16384), select=64,
              layout="NHD"),
        # one user: latency
        _case("sparse_single", "sparse", "bf16", 1, 32, 8, 128, 16, (8000, 8000), select=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "bounds", "sparse"])
    dtype = rng.choice(["bf16", "f16"])
    head = rng.choice([64, 128, 128, 256])
    block = rng.choice([8, 16, 32, 64])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    group = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 12, 16, 32)
                        if g * head <= 2048 or (g <= 32 and head <= 128)])
    row = kv * head
    new, lens, select, layout = (1, 1), (0, 0), 0, "HND"
    if op in ("append", "bounds"):
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, 8192) if rng.random() < 0.7 else 1
        hi = max(1, min(hi, 26000 * 1024 // (row * seqs)))
        new = (rng.randint(1, hi), hi)
        lens = (0, rng.choice([0, 0, 600, 4096]))
        lens = (0, min(lens[1], max(1, 64 * 4096 * 1024 // (row * seqs))))
    elif op == "attend":
        seqs = _log(rng, 1, 256)
        room = int(240e6 / (row * seqs) / max(1, group / 4))
        hi = min(_log(rng, 1, 131072), max(1, room))
        lens = (rng.randint(0, hi), hi)
    else:
        seqs = min(_log(rng, 1, 64), max(1, int(18e6 / (row * block) / max(1, group / 8))))
        hi = min(_log(rng, 256, 131072), max(64, int(240e6 / (row * seqs))))
        lens = (rng.randint(0, hi), hi)
        room = int(80e6 / (row * seqs * block) / max(1, group / 8))
        select = max(4, min(_log(rng, 4, 300), room))
        layout = rng.choice(["HND", "NHD"])
    c = _case("", op, dtype, seqs, group * kv, kv, head, block, lens, new, select, layout,
              rng.choice([1.0, 1.0, 4.0]))
    del c["name"]
    return c


# ----------------------------------------------------- the page format

def _page_bytes(head, block):
    return block * (head // 2) + block * (head // GROUP) * 4


def _quantise(x):
    """x (..., D) -> codes uint8 (..., D), scale and minimum (..., D / 64) of x's type."""
    f = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = f.amin(-1), f.amax(-1)
    s = ((hi - lo) / 15).to(x.dtype)
    sf = s.float().unsqueeze(-1)
    c = torch.where(sf > 0, torch.round((f - lo.unsqueeze(-1)) / sf), 0.0).clamp_(0, 15)
    return c.to(torch.uint8).flatten(-2), s, lo.to(x.dtype)


def _words(codes):
    """(..., 8) codes -> (..., 4) bytes of the code word."""
    n = codes[..., NIBBLES]
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _key_words(codes):
    """(N, D) -> (N, D / 2) bytes: chunk c of 4 holds elements 16 c .. 16 c + 15 of every group."""
    n, d = codes.shape
    w = _words(codes.view(n, d // GROUP, 4, 2, 8))           # group, chunk, word, byte
    return w.permute(0, 2, 1, 3, 4).reshape(n, d // 2)


def _value_words(codes):
    """(N, D) -> (N, 8, D / 64, 4) bytes: octet, group, byte."""
    n, d = codes.shape
    return _words(codes.view(n, d // GROUP, 8, 8)).permute(0, 2, 1, 3)


def _value_view(pages, head, block):
    """The value codes of pages (P, bytes) as (P, tile, octet, pair, parity, group, byte)."""
    return pages[:, :block * head // 2].unflatten(1, (block // 8, 8, 4, 2, head // GROUP, 4))


def _scales(pages, head, block, dtype):
    """(P, bs, D / 64, 2) scale and minimum, a view of the pages."""
    return pages[:, block * head // 2:].view(dtype).unflatten(1, (block, head // GROUP, 2))


def _unwords(b):
    """(..., 4) bytes -> (..., 8) codes."""
    n = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    out = torch.empty_like(n)
    out[..., NIBBLES] = n
    return out


def _rows(pages, head, block, dtype, value, wide=torch.float32):
    """Every row of pages (P, bytes) as the values it stands for, (P, bs, D)."""
    p, g = pages.shape[0], head // GROUP
    if value:
        c = _unwords(_value_view(pages, head, block))        # P tile octet pair parity group 8
        c = c.permute(0, 1, 3, 4, 5, 2, 6).reshape(p, block, g, GROUP)
    else:
        c = _unwords(pages[:, :block * head // 2].unflatten(1, (block, 4, g, 2, 4)))
        c = c.permute(0, 1, 3, 2, 4, 5).reshape(p, block, g, GROUP)
    sl = _scales(pages, head, block, dtype).to(wide)
    return (c.to(wide) * sl[..., :1] + sl[..., 1:]).flatten(-2)


# --------------------------------------------------------------- inputs

def _lengths(case):
    """Lengths before the call and new tokens of every sequence, on the host:
    the case's own, so that its outputs have one shape whatever the seed."""
    g = torch.Generator().manual_seed(1000003 * case["len_hi"] + 1009 * case["new_hi"] + case["seqs"])
    lens = torch.randint(case["len_lo"], case["len_hi"] + 1, (case["seqs"],), generator=g)
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (case["seqs"],), generator=g)
    return lens, new


def _tables(case, total, seed):
    """(B, max_blocks) int32 ids, slices of one random permutation of the pool."""
    bs = case["block"]
    need = (total + bs - 1) // bs
    pool = max(int(need.sum()) + 3, 4)
    g = torch.Generator().manual_seed(seed + 1)
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    width = max(int(need.max()), 1)
    bt = torch.zeros((case["seqs"], width), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need.tolist()):
        bt[s, :n] = perm[at:at + n]
        at += n
    return bt, pool


def _randn(shape, dtype, g, scale=1.0, chunk=1 << 27):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), chunk):
        n = min(chunk, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda") * scale
    return out


def _random_pages(case, pool, g, value):
    """Pages of a filled cache: quantised N(0, 1) rows in the page format."""
    head, bs, dtype = case["head"], case["block"], DTYPES[case["dtype"]]
    pages = torch.empty((pool * case["kv_heads"], _page_bytes(head, bs)), dtype=torch.uint8,
                        device="cuda")
    step = max(1, (1 << 25) // (bs * head))
    for i in range(0, pages.shape[0], step):
        part = pages[i:i + step]
        n = part.shape[0]
        x = torch.randn((n * bs, head), generator=g, device="cuda")
        c, s, lo = _quantise((x if value else x * case["k_scale"]).to(dtype))
        if value:
            w = _value_words(c).unflatten(0, (n, bs // 8, 4, 2))   # P tile pair parity octet ..
            part[:, :bs * head // 2] = w.permute(0, 1, 4, 2, 3, 5, 6).reshape(n, -1)
        else:
            part[:, :bs * head // 2] = _key_words(c).view(n, -1)
        sl = torch.stack((s, lo), -1)
        part[:, bs * head // 2:] = sl.view(torch.uint8).reshape(n, -1)
    return pages.view(pool, case["kv_heads"], -1)


def prepare(case, seed):
    dtype, head, bs, hkv = DTYPES[case["dtype"]], case["head"], case["block"], case["kv_heads"]
    lens, new = _lengths(case)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    st = {"case": case, "scale": 1.0 / math.sqrt(head)}
    if case["op"] in ("append", "bounds"):
        bt, pool = _tables(case, lens + new, seed)
        n = int(new.sum())
        st["k"] = _randn((n, hkv, head), dtype, g, case["k_scale"])
        cu = torch.zeros(case["seqs"] + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(new, 0)
        # one token per sequence is the call without offsets
        st["cu"] = None if case["new_hi"] == 1 else cu.cuda()
        st["cu_host"] = cu.tolist()
        if case["op"] == "append":
            st["v"] = _randn((n, hkv, head), dtype, g)
            # random bytes: what recycled pages hold
            for name in ("key_cache", "value_cache"):
                st[name] = torch.randint(0, 256, (pool, hkv, _page_bytes(head, bs)),
                                         dtype=torch.uint8, generator=g, device="cuda")
        else:
            x = _randn((2, pool, hkv, head), dtype, g)
            st["bounds"] = torch.stack((x.amin(0), x.amax(0)), 2).contiguous()
    else:
        bt, pool = _tables(case, lens, seed)
        st["q"] = _randn((case["seqs"], case["q_heads"], head), dtype, g)
        st["out"] = torch.empty_like(st["q"])
        if case["op"] == "attend":
            st["key_cache"] = _random_pages(case, pool, g, False)
            st["value_cache"] = _random_pages(case, pool, g, True)
        else:
            hnd = case["layout"] == "HND"
            shape = (pool, hkv, bs, head) if hnd else (pool, bs, hkv, head)
            st["key_cache"] = _randn(shape, dtype, g, case["k_scale"])
            st["value_cache"] = _randn(shape, dtype, g)
            # the bounds such a program keeps; rows past a sequence's end are not in them
            k = st["key_cache"] if hnd else st["key_cache"].transpose(1, 2)
            st["bounds"] = torch.stack((k.amin(2), k.amax(2)), 2).contiguous()
            for s, n in enumerate(lens.tolist()):
                if n % bs:
                    last = k[int(bt[s, n // bs]), :, :n % bs]
                    st["bounds"][int(bt[s, n // bs])] = torch.stack((last.amin(1), last.amax(1)), 1)
    st["bt"], st["lens"], st["lens_host"] = bt.cuda(), lens.to(torch.int32).cuda(), lens.tolist()
    return st


# ---------------------------------------------------------- plain forms

def _places(st):
    """Page and row of every new token, on the device."""
    c = st["case"]
    n = st["k"].shape[0]
    i = torch.arange(n, device="cuda")
    if st["cu"] is None:
        s, pos = i, st["lens"].long()
    else:
        s = torch.searchsorted(st["cu"][1:].contiguous(), i.to(torch.int32), right=True)
        pos = st["lens"].long()[s] + i - st["cu"].long()[s]
    return st["bt"].long()[s, pos // c["block"]], pos % c["block"], s, pos


def _plain_append(st):
    c = st["case"]
    head, bs, hkv, dtype = c["head"], c["block"], c["kv_heads"], DTYPES[c["dtype"]]
    block, row, _, _ = _places(st)
    n = block.numel()
    page = (block[:, None] * hkv + torch.arange(hkv, device="cuda")).view(-1)
    row = row[:, None].expand(n, hkv).reshape(-1)
    out = []
    for x, cache, value in ((st["k"], st["key_cache"], False), (st["v"], st["value_cache"], True)):
        pages = cache.view(-1, cache.shape[-1])
        codes, s, lo = _quantise(x.reshape(n * hkv, head))
        if value:
            view = _value_view(pages, head, bs)
            view[page, row // 8, :, row % 8 // 2, row % 2] = _value_words(codes)
        else:
            pages[:, :bs * head // 2].unflatten(1, (bs, head // 2))[page, row] = _key_words(codes)
        _scales(pages, head, bs, dtype)[page, row] = torch.stack((s, lo), -1)
        # what the cache now holds for these tokens
        sl = _scales(pages, head, bs, dtype)[page, row].float()
        if value:
            cc = _unwords(view[page, row // 8, :, row % 8 // 2, row % 2]).permute(0, 2, 1, 3)
        else:
            b = pages[:, :bs * head // 2].unflatten(1, (bs, head // 2))[page, row]
            cc = _unwords(b.view(-1, 4, head // GROUP, 2, 4)).permute(0, 2, 1, 3, 4)
        cc = cc.reshape(n * hkv, head // GROUP, GROUP).float()
        out.append((cc * sl[..., :1] + sl[..., 1:]).to(dtype).view(n, hkv, head))
    return out[0], out[1], _lens_after(st)


def _lens_after(st):
    if st["cu"] is None:
        return st["lens"] + 1
    return st["lens"] + (st["cu"][1:] - st["cu"][:-1])


def _softmax_out(q, k, v, scale, wide):
    """q (Hq, D), k and v (Hkv, L, D) -> (Hq, D) in ``wide``."""
    hkv = k.shape[0]
    qg = q.to(wide).view(hkv, -1, q.shape[-1])
    sc = torch.matmul(qg, k.to(wide).transpose(1, 2)) * scale
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    return (torch.matmul(p, v.to(wide)) / p.sum(-1, keepdim=True)).reshape(q.shape)


def _plain_attend(st, wide=torch.float32):
    c = st["case"]
    head, bs, hkv, dtype = c["head"], c["block"], c["kv_heads"], DTYPES[c["dtype"]]
    out = torch.zeros(st["q"].shape, dtype=wide, device="cuda")
    for s, n in enumerate(st["lens_host"]):
        if n == 0:
            continue
        ids = st["bt"][s, :(n + bs - 1) // bs].long()
        kv = []
        for cache, value in ((st["key_cache"], False), (st["value_cache"], True)):
            pages = cache[ids].view(-1, cache.shape[-1])
            r = _rows(pages, head, bs, dtype, value, wide).view(-1, hkv, bs, head)
            kv.append(r.transpose(0, 1).reshape(hkv, -1, head)[:, :n])
        out[s] = _softmax_out(st["q"][s], kv[0], kv[1], st["scale"], wide)
    return out


def _plain_bounds(st):
    bounds, k = st["bounds"], st["k"]
    pool = bounds.shape[0]
    block, row, _, _ = _places(st)
    # a page whose row 0 is new starts afresh, the others go on (row `pool` takes the rest)
    fresh = torch.where(row == 0, block, pool)
    idx = block[:, None, None].expand(k.shape)
    for i, (start, how) in enumerate(((float("inf"), "amin"), (-float("inf"), "amax"))):
        b = torch.cat((bounds[:, :, i], bounds[:1, :, i])).float()
        b[fresh] = start
        bounds[:, :, i] = b.scatter_reduce_(0, idx, k.float(), how)[:pool].to(k.dtype)
    return bounds


def _plain_sparse(st):
    """Selection in 64 bits (scores next to the border), attention in 32."""
    c = st["case"]
    bs, hkv, keep, hnd = c["block"], c["kv_heads"], c["select"], c["layout"] == "HND"
    out = torch.zeros(st["q"].shape, dtype=torch.float32, device="cuda")
    tables = torch.full((c["seqs"], hkv, keep), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros((c["seqs"], hkv), dtype=torch.int32, device="cuda")
    heads = torch.arange(hkv, device="cuda")[:, None]
    for s, n in enumerate(st["lens_host"]):
        if n == 0:
            continue
        pages = (n + bs - 1) // bs
        ids = st["bt"][s, :pages].long()
        if pages <= keep:
            sel = torch.arange(pages, device="cuda").expand(hkv, pages)
        else:
            qg = st["q"][s].double().view(hkv, -1, c["head"])
            up, dn = qg.clamp(min=0).sum(1), qg.clamp(max=0).sum(1)
            b = st["bounds"][ids]
            u = torch.matmul(b[:, :, 1].double().transpose(0, 1), up[:, :, None])[..., 0]
            u = u + torch.matmul(b[:, :, 0].double().transpose(0, 1), dn[:, :, None])[..., 0]
            u = u.float()
            u[:, 0] = u[:, pages - 1] = float("inf")     # the first and the last page
            sel = torch.sort(u, dim=1, descending=True, stable=True).indices[:, :keep]
            sel = sel.sort(dim=1).values
        m = sel.shape[1]
        tables[s, :, :m] = ids[sel].to(torch.int32)
        got = (m - 1) * bs + n - (pages - 1) * bs
        lens[s] = got
        at = (ids[sel], heads) if hnd else (ids[sel], slice(None), heads)
        k = st["key_cache"][at].reshape(hkv, m * bs, -1)[:, :got]
        v = st["value_cache"][at].reshape(hkv, m * bs, -1)[:, :got]
        out[s] = _softmax_out(st["q"][s], k, v, st["scale"], torch.float32)
    return out.to(st["q"].dtype), tables, lens


# ------------------------------------------------------------------ run

def run(st):
    c = st["case"]
    if not own:
        if c["op"] == "append":
            return _plain_append(st)
        if c["op"] == "attend":
            return _plain_attend(st).to(st["q"].dtype)
        if c["op"] == "bounds":
            return _plain_bounds(st)
        return _plain_sparse(st)
    import pagedattention_b200 as pa
    if c["op"] == "append":
        lens = st["lens"].clone()       # the call advances it
        pa.kv_append_int4(st["key_cache"], st["value_cache"], st["k"], st["v"], lens, st["bt"],
                          c["block"], cu_new=st["cu"])
        k, v = pa.kv_read_int4(st["key_cache"], st["value_cache"], st["bt"], lens, c["block"],
                               c["head"], DTYPES[c["dtype"]], starts=st["lens"], cu_out=st["cu"],
                               num_tokens=st["k"].shape[0])
        return k, v, lens
    if c["op"] == "attend":
        pa.paged_attention_int4(st["out"], st["q"], st["key_cache"], st["value_cache"], st["bt"],
                                st["lens"], st["scale"], c["block"])
        return st["out"]
    if c["op"] == "bounds":
        bounds = st["bounds"]
        pa.update_page_bounds(bounds, st["k"], st["lens"], st["bt"], c["block"], cu_new=st["cu"])
        return bounds
    tables, lens = pa.paged_attention_sparse(
        st["out"], st["q"], st["key_cache"], st["value_cache"], st["bounds"], st["bt"], st["lens"],
        st["scale"], c["block"], c["select"], kv_layout=c["layout"])
    return st["out"], tables, lens


# ----------------------------------------------------------------- work

def work(case):
    row, bs = case["kv_heads"] * case["head"], case["block"]
    lens, new = _lengths(case)
    n, total = int(new.sum()), int(lens.sum())
    if case["op"] == "append":
        # rows in, codes with their scales out, the values they stand for out
        return {"bytes": int(2 * n * row * (2 + 9 / 16 + 2)), "flops": 2 * n * row * 8}
    q = case["seqs"] * case["q_heads"] * case["head"]
    if case["op"] == "attend":
        return {"bytes": int(2 * total * row * 9 / 16 + 4 * q),
                "flops": 4 * total * case["q_heads"] * case["head"]}
    if case["op"] == "bounds":
        touched = int(((lens + new + bs - 1) // bs - lens // bs).sum())
        old = int((lens % bs > 0).sum())        # pages that go on: their bounds are read
        return {"bytes": 2 * n * row + 4 * (touched + old) * row, "flops": 2 * n * row}
    pages = (lens + bs - 1) // bs
    scored = int(pages[pages > case["select"]].sum())
    kept = int(torch.where(pages > case["select"], case["select"] * bs, lens).sum())
    return {"bytes": 4 * scored * row + 4 * kept * row + 4 * q,
            "flops": 4 * scored * row + 4 * kept * case["q_heads"] * case["head"]}


# ---------------------------------------------------------------- exact

def exact(case, seed):
    """The operators' definitions in 64 bits, token by token or page by page."""
    st = prepare(case, seed)
    f64 = torch.float64
    head, bs, hkv, dtype = case["head"], case["block"], case["kv_heads"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        out = []
        for x in (st["k"], st["v"]):
            y = torch.empty(x.shape, dtype=f64, device="cuda")
            for g in range(head // GROUP):
                part = x[..., g * GROUP:(g + 1) * GROUP].to(f64)
                low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
                step = ((high - low) / 15).to(dtype).to(f64)    # held in the rows' type
                code = torch.round((part - low) / torch.where(step > 0, step, torch.ones_like(step)))
                code = torch.where(step > 0, code, torch.zeros_like(code)).clamp(0, 15)
                y[..., g * GROUP:(g + 1) * GROUP] = low + step * code
            out.append(y)
        new = torch.tensor(st["cu_host"], device="cuda").diff().to(torch.int32)
        return out[0], out[1], st["lens"] + new
    if case["op"] == "bounds":
        want = st["bounds"].to(f64)
        cu = st["cu_host"]
        for s, n in enumerate(st["lens_host"]):
            at = cu[s]
            while at < cu[s + 1]:
                pos = n + at - cu[s]
                take = min(bs - pos % bs, cu[s + 1] - at)
                rows = st["k"][at:at + take].to(f64)
                b = want[st["bt"][s, pos // bs].long()]
                low, high = rows.min(0).values, rows.max(0).values
                if pos % bs:
                    low, high = torch.minimum(low, b[:, 0]), torch.maximum(high, b[:, 1])
                want[st["bt"][s, pos // bs].long()] = torch.stack((low, high), 1)
                at += take
        return want
    if case["op"] == "attend":
        out = torch.zeros(st["q"].shape, dtype=f64, device="cuda")
        g = head // GROUP
        # byte offset and shift of element d of row r of a page
        d = torch.arange(head, device="cuda")
        r = torch.arange(bs, device="cuda")[:, None]
        grp, e = d // GROUP, d % GROUP
        nib = e % 8 // 2 + 4 * (e % 2)
        shift = nib % 2 * 4
        key_at = r * (head // 2) + e // 16 * (head // 8) + grp * 8 + e % 16 // 8 * 4 + nib // 2
        word = ((e // 8 * 4 + r % 8 // 2) * 2 + r % 2) * g + grp
        value_at = r // 8 * (4 * head) + word * 4 + nib // 2
        for s, n in enumerate(st["lens_host"]):
            if n == 0:
                continue
            ids = st["bt"][s, :(n + bs - 1) // bs].long()
            for h in range(hkv):
                kv = []
                for cache, at in (("key_cache", key_at), ("value_cache", value_at)):
                    pages = st[cache][ids, h]
                    code = (pages[:, at] >> shift.to(torch.uint8)) & 15
                    sl = pages[:, bs * head // 2:].contiguous().view(dtype).view(-1, bs, g, 2)
                    sl = sl.to(f64).repeat_interleave(GROUP, 2)
                    kv.append((sl[..., 1] + sl[..., 0] * code).view(-1, head)[:n])
                mine = slice(h * (case["q_heads"] // hkv), (h + 1) * (case["q_heads"] // hkv))
                w = torch.softmax(st["q"][s, mine].to(f64) @ kv[0].T * st["scale"], -1)
                out[s, mine] = w @ kv[1]
        return out
    grp = case["q_heads"] // hkv
    keep = case["select"]
    out = torch.zeros(st["q"].shape, dtype=f64, device="cuda")
    tables = torch.full((case["seqs"], hkv, keep), -1, dtype=torch.int32)
    lens = torch.zeros((case["seqs"], hkv), dtype=torch.int32)
    for s, n in enumerate(st["lens_host"]):
        count = (n + bs - 1) // bs
        ids = st["bt"][s, :count].long()
        for h in range(hkv if n else 0):
            q = st["q"][s, h * grp:(h + 1) * grp].to(f64)
            chosen = list(range(count))
            if count > keep:
                b = st["bounds"][ids, h].to(f64)
                u = torch.zeros(count, dtype=f64, device="cuda")
                for i in range(grp):
                    u += torch.maximum(b[:, 0] * q[i], b[:, 1] * q[i]).sum(1)
                u = u.float().tolist()
                order = sorted(range(1, count - 1), key=lambda p: (-u[p], p))
                chosen = sorted([0, count - 1] + order[:keep - 2])
            pick = ids[torch.tensor(chosen, device="cuda")]
            tables[s, h, :len(chosen)] = pick.to(torch.int32).cpu()
            got = (len(chosen) - 1) * bs + n - (count - 1) * bs
            lens[s, h] = got
            if case["layout"] == "HND":
                k, v = st["key_cache"][pick, h], st["value_cache"][pick, h]
            else:
                k, v = st["key_cache"][pick, :, h], st["value_cache"][pick, :, h]
            k, v = k.reshape(-1, head)[:got].to(f64), v.reshape(-1, head)[:got].to(f64)
            out[s, h * grp:(h + 1) * grp] = torch.softmax(q @ k.T * st["scale"], -1) @ v
    return out, tables.cuda(), lens.cuda()


if __name__ == "__main__":
    for c in listed():
        print(c["name"], work(c))
    print(draw(random.Random(0)))
