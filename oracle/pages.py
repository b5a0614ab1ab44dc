"""64-bit restatement of the 4-bit page format and the page-sparse selection
(test infrastructure only: plain loops and numpy, no kernels).

The reference (src/kernel_eager.py:29-56) attends to every page of a 16-bit
cache; these are the operators' definitions, written token by token.
"""
from __future__ import annotations

import numpy as np
import torch

GROUP = 64


def page_bytes(D, bs):
    return bs * D // 2 + bs * (D // GROUP) * 4


def quantise(x: torch.Tensor):
    """x (..., D) 16-bit -> codes (..., D) int64, scale and minimum (..., D/64) of x's type."""
    g = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    rng = hi - lo
    s = (rng.float() / 15).to(x.dtype)
    ok = torch.isfinite(rng) & torch.isfinite(rng.float())
    nan = torch.tensor(float("nan"), dtype=x.dtype)
    s, lo = torch.where(ok, s, nan), torch.where(ok, lo.to(x.dtype), nan)
    sd = s.double()[..., None]
    c = torch.where(sd > 0, torch.round((g - lo.double()[..., None]) / sd), 0.0).clamp(0, 15)
    c = torch.where(ok[..., None], c, 0.0)
    return c.long().flatten(-2), s, lo


def _nibble(i):
    return i // 2 + 4 * (i % 2)


def code_place(D, r, d, value):
    """(byte, shift) of element d of row r in a page."""
    g, e = divmod(d, GROUP)
    o, i = divmod(e, 8)
    if value:
        word = ((o * 4 + (r % 8) // 2) * 2 + r % 2) * (D // GROUP) + g
        at = (r // 8) * 4 * D + word * 4
    else:
        at = r * (D // 2) + (o // 2) * (D // 8) + g * 8 + (o % 2) * 4
    return at + _nibble(i) // 2, 4 * (_nibble(i) % 2)


def _places(D, r, value):
    p = [code_place(D, r, d, value) for d in range(D)]
    return np.array([x[0] for x in p]), np.array([x[1] for x in p])


def put_row(page: np.ndarray, bs, r, codes, scale, lo, value):
    """Writes one row into a page (uint8 [page_bytes])."""
    D = codes.shape[-1]
    at, sh = _places(D, r, value)
    c = codes.numpy().astype(np.uint8)
    for b in np.unique(at):
        page[b] = 0
    np.bitwise_or.at(page, at, c << sh.astype(np.uint8))
    pair = torch.stack((scale, lo), -1).contiguous().view(torch.uint8).numpy().reshape(-1)
    o = bs * D // 2 + r * (D // GROUP) * 4
    page[o:o + pair.size] = pair


def get_rows(pages: np.ndarray, D, bs, dtype, value):
    """pages uint8 [P, page_bytes] -> the values they stand for, float64 [P, bs, D]."""
    P = pages.shape[0]
    out = np.empty((P, bs, D))
    raw = np.ascontiguousarray(pages[:, bs * D // 2:])
    sl = torch.from_numpy(raw).view(dtype).double().numpy().reshape(P, bs, D // GROUP, 2)
    for r in range(bs):
        at, sh = _places(D, r, value)
        c = (pages[:, at] >> sh.astype(np.uint8)) & 15
        s = np.repeat(sl[:, r, :, 0], GROUP, 1)
        lo = np.repeat(sl[:, r, :, 1], GROUP, 1)
        out[:, r] = lo + s * c
    return out


def attention(q, k, v, scale):
    """q (G, D), k and v (L, D), float64 -> (G, D); zeros for L = 0."""
    if k.shape[0] == 0:
        return np.zeros_like(q)
    s = q @ k.T * scale
    p = np.exp(s - s.max(1, keepdims=True))
    return p @ v / p.sum(1, keepdims=True)


def page_score(q, lo, hi):
    """Sum over heads and elements of max(q * lo, q * hi), rounded to fp32.
    q (G, D), lo and hi (D,), float64."""
    return np.float32(np.maximum(q * lo, q * hi).sum())


def select(q, bounds, n, keep, sink, recent, bad=()):
    """Indices of the kept pages of n, ascending.  bounds (n, 2, D) float64;
    pages in ``bad`` (ids out of range) have no bounds and rank last."""
    if n <= keep:
        return list(range(n))
    mid = list(range(sink, n - recent))
    u = {p: -np.inf if p in bad else page_score(q, bounds[p, 0], bounds[p, 1]) for p in mid}

    def order(p):
        return (0, 0.0, p) if np.isnan(u[p]) else (1, -float(u[p]), p)

    best = sorted(mid, key=order)[:keep - sink - recent]
    return sorted(list(range(sink)) + best + list(range(n - recent, n)))
