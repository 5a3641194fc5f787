"""The 8-bit paged cache on CPU tensors: :class:`kitty.kernels.Cache8`'s calls
in torch code, with the rules of include/kitty_hip.h (kitty_cache8_*).
Codes and scales are bit-identical to the HIP kernels'."""
from __future__ import annotations

import math
from collections import Counter
from typing import List, Optional, Tuple

import torch

E4M3 = torch.float8_e4m3fn


def scale_for(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two s >= 2^-64 with amax <= 448 s (float32)."""
    m, e = torch.frexp(amax)            # 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).masked_fill(amax == 0, -64).clamp(min=-64)
    return (e + 127 << 23).view(torch.float32)


def _page_ids(table: torch.Tensor, number: torch.Tensor, num_pages: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(page ids, whether they exist) of page numbers (B, n); ids 0 where they do not."""
    W = table.shape[1]
    ok = (number >= 0) & (number < W)
    if W == 0:
        return torch.zeros_like(number), ok
    ids = table.long().gather(1, number.clamp(0, W - 1))
    ok = ok & (ids >= 0) & (ids < num_pages)
    return torch.where(ok, ids, torch.zeros_like(ids)), ok


def write(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
          table: torch.Tensor, start: torch.Tensor, lens: Optional[torch.Tensor]) -> None:
    B, H, T, D = k.shape
    G = key.shape[2]
    start = start.long()
    n = torch.full_like(start, T) if lens is None else lens.long().clamp(0, T)
    n = torch.where(start < 0, torch.zeros_like(n), n)
    first = start.clamp(min=0)
    off, slots = first % G, (T + G - 2) // G + 1
    row = torch.arange(slots * G)
    new = ((row >= off[:, None]) & (row < (off + n)[:, None])).view(B, slots, G)
    ids, ok = _page_ids(table, first[:, None] // G + torch.arange(slots), key.shape[0])
    touched = new.any(-1) & ok
    pid, new = ids[touched], new[touched]
    old = (row < off[:, None]).view(B, slots, G)[touched]
    src = (row - off[:, None]).clamp(0, T - 1)[:, None, :, None].expand(B, H, slots * G, D)
    for i, (x, pool) in enumerate(((k, key), (v, value))):
        x = x.float().gather(2, src).view(B, H, slots, G, D).transpose(1, 2)[touched]
        x = torch.where(new[:, None, :, None], x, torch.zeros_like(x))
        finite = x.isfinite()
        s = scale_for(torch.where(finite, x, torch.zeros_like(x)).abs().amax((2, 3)))
        was = scale[pid, :, i]
        s = torch.where(old.any(-1)[:, None], torch.fmax(s, was), s)
        codes = torch.where(finite, x / s[..., None, None], torch.full_like(x, math.nan)).to(E4M3).view(torch.uint8)
        codes = torch.where(finite, codes, torch.full_like(codes, 0x7F))
        held = pool.view(torch.uint8)[pid]
        again = (held.view(E4M3).float() * (was / s)[..., None, None]).to(E4M3).view(torch.uint8)
        again = torch.where((s != was)[..., None, None], again, held)
        held = torch.where(old[:, None, :, None], again, held)
        pool.view(torch.uint8)[pid] = torch.where(new[:, None, :, None], codes, held)
        scale[pid, :, i] = s


def read(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
         start: Optional[torch.Tensor], out: Tuple[torch.Tensor, torch.Tensor]) -> None:
    B, H, T, D = out[0].shape
    G = key.shape[2]
    first = torch.zeros_like(lens).long() if start is None else start.long()
    pos = first[:, None] + torch.arange(T)
    ids, ok = _page_ids(table, torch.div(pos, G, rounding_mode="floor"), key.shape[0])
    here = pos < lens.long()[:, None]
    for i, pool in enumerate((key, value)):
        x = torch.zeros(B, T, H, D)
        if key.shape[0]:
            x = pool.view(torch.uint8)[ids, :, pos % G].view(E4M3).float() * scale[ids][..., i, None]
        x = torch.where(ok[..., None, None], x, torch.full_like(x, math.nan))
        out[i].copy_(torch.where(here[..., None, None], x, torch.zeros_like(x)).transpose(1, 2))


def _tokens(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, table: torch.Tensor, n: int):
    """Codes (H, n, D) and scales (H, 1, n) of keys and values of the n tokens that a
    table row names, apart, as in the kernels: their products may pass fp32's range."""
    P, H, G, D = key.shape
    ids, ok = _page_ids(table[None], torch.arange(-(-n // G))[None], P)
    codes, scales = [], []
    for i, pool in enumerate((key, value)):
        x, f = torch.zeros(ids.shape[1], H, G, D), torch.ones(ids.shape[1], H)
        if P:
            x, f = pool.view(torch.uint8)[ids[0]].view(E4M3).float(), torch.where(ok[0][:, None], scale[ids[0], :, i], f)
        x = torch.where(ok[0][:, None, None, None], x, torch.full_like(x, math.nan))
        codes.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
        scales.append(f.t().repeat_interleave(G, 1)[:, None, :n])
    return codes, scales


def _rows(q: torch.Tensor, codes, scales, causal: bool, sm_scale: float):
    """Attention of q (Hq, t, D) over tokens as _tokens has them, the queries their last:
    (out, log-sum-exp, softmax weights (H, gq, t, n), 0 where a row does not see a token)."""
    Hq, t, D = q.shape
    H, n, _ = codes[0].shape
    gq = Hq // H
    sees = torch.ones(t, n, dtype=torch.bool)
    if causal:
        sees = torch.arange(n) <= torch.arange(n - t, n)[:, None]
    s = (q.reshape(H, gq * t, D) @ codes[0].transpose(1, 2) * (scales[0] * sm_scale)).view(H, gq, t, n)
    s = s.masked_fill(~sees, -math.inf)
    l = torch.logsumexp(s, -1)
    none = ~sees.any(-1)                                   # rows that see nothing
    w = torch.exp(s - torch.where(none, torch.zeros_like(l), l)[..., None])
    gone = codes[1].isnan()                                # masked NaN values stay out of the product
    o = (w.view(H, gq * t, n) * scales[1]) @ codes[1].masked_fill(gone, 0.0)
    met = (sees.float().repeat(gq, 1) @ gone.float()) > 0
    o = o.masked_fill(met, math.nan).view(H, gq, t, D).masked_fill(none[:, None], 0.0)
    w = w.masked_fill((l == math.inf)[..., None], math.nan)     # inf / inf, as the kernels have every weight of such a row
    return o.reshape(Hq, t, D), l.masked_fill(none, -math.inf).reshape(Hq, t), w.masked_fill(~sees, 0.0)


def attend(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, q: torch.Tensor, table: torch.Tensor,
           lens: torch.Tensor, q_lens: Optional[torch.Tensor], causal: bool, sm_scale: float, out: torch.Tensor,
           lse: torch.Tensor, weights: Optional[torch.Tensor] = None) -> None:
    B, Hq, T, D = q.shape
    G = key.shape[2]
    q = q.float()       # a copy: out may be q
    out.zero_()
    lse.fill_(-math.inf)
    rows = [T] * B if q_lens is None else q_lens.tolist()
    for b, (n, t) in enumerate(zip(lens.tolist(), rows)):
        if n < 0 or n > table.shape[1] * G or not 0 <= t <= T:
            out[b] = math.nan
            lse[b] = math.nan
            continue
        if n == 0 or t == 0:
            continue
        o, l, w = _rows(q[b, :, :t], *_tokens(key, value, scale, table[b], n), causal, sm_scale)
        out[b, :, :t] = o.to(out.dtype)
        lse[b, :, :t] = l
        if weights is not None:
            n = min(n, weights.shape[2])
            weights[b, :, :n] += w[..., :n].sum((1, 2))


def attend_shared(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, q: torch.Tensor, prefix_table: torch.Tensor,
                  prefix_lens: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, q_lens: Optional[torch.Tensor],
                  causal: bool, sm_scale: float, out: torch.Tensor, lse: torch.Tensor) -> None:
    B, Hq, T, D = q.shape
    G, each = key.shape[2], B // prefix_table.shape[0]
    q = q.float()       # a copy: out may be q
    out.zero_()
    lse.fill_(-math.inf)
    rows = [T] * B if q_lens is None else q_lens.tolist()
    prefix = prefix_lens.tolist()
    for b, (n, t) in enumerate(zip(lens.tolist(), rows)):
        f = b // each
        before = prefix[f]
        if n < 0 or n > table.shape[1] * G or not 0 <= t <= T or before < 0 or before > prefix_table.shape[1] * G:
            out[b] = math.nan
            lse[b] = math.nan
            continue
        if n + before == 0 or t == 0:
            continue
        parts = _tokens(key, value, scale, prefix_table[f], before), _tokens(key, value, scale, table[b], n)
        codes = [torch.cat([p[0][i] for p in parts], 1) for i in range(2)]
        scales = [torch.cat([p[1][i] for p in parts], 2) for i in range(2)]
        o, l, _ = _rows(q[b, :, :t], codes, scales, causal, sm_scale)
        out[b, :, :t] = o.to(out.dtype)
        lse[b, :, :t] = l


def _named(row: torch.Tensor, pages: int, num_pages: int) -> List[int]:
    """Ids of the first `pages` pages that a table's row names, without those outside the pool."""
    return [p for p in row[:max(pages, 0)].tolist() if 0 <= p < num_pages]


def evict(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
          weights: torch.Tensor, keep: int, first: int, last: int, into: Optional[torch.Tensor], out_lens: torch.Tensor,
          kept: torch.Tensor, out_weights: torch.Tensor) -> None:
    P, H, G, D = key.shape
    N, K = weights.shape[2], kept.shape[2]
    heads = torch.arange(H)[:, None]
    kept.fill_(-1)
    out_weights.zero_()
    lens = [n if 0 <= n <= min(table.shape[1] * G, N) else -1 for n in lens.tolist()]
    # pages that each sequence needs and writes, and how often the call names each: written ones once
    if into is None:
        needed = [_named(table[b], -(-min(n, keep) // G), P) for b, n in enumerate(lens)]
        written = [pages if n > keep else [] for pages, n in zip(needed, lens)]
        count = Counter(p for pages in needed for p in pages)
    else:
        written = [_named(into[b], -(-min(n, keep) // G), P) for b, n in enumerate(lens)]
        count = Counter(p for b, n in enumerate(lens) for p in _named(table[b], -(-n // G), P) + written[b])
    moves = []          # all that moves is read before any of it is written
    for b, n in enumerate(lens):
        if n < 0 or any(count[p] > 1 for p in written[b]):
            out_lens[b] = -1
            continue
        m = out_lens[b] = min(n, keep)
        at = torch.arange(n).expand(H, n)
        if n > m:
            between = weights[b, :, first:n - last].sort(dim=-1, descending=True, stable=True).indices[:, :m - first - last]
            at = torch.cat([at[:, :first], first + between.sort(-1).values, at[:, n - last:]], 1)
        kept[b, :, :m] = at
        out_weights[b, :, :m] = weights[b].gather(1, at)
        if m == 0 or P == 0 or (into is None and m == n):     # in place only what is cut is written
            continue
        ids, ok = _page_ids(table[b:b + 1].expand(H, -1), at // G, P)
        new, there = _page_ids((table if into is None else into)[b:b + 1], torch.arange(-(-m // G))[None], P)
        moved = []
        for i, pool in enumerate((key, value)):
            was = torch.where(ok, scale[ids, heads, i], torch.full(ids.shape, -1.0))
            codes = torch.where(ok[..., None], pool.view(torch.uint8)[ids, heads, at % G], torch.tensor(0x7F, dtype=torch.uint8))
            moved.append((was, codes))
        moves.append((new[0].tolist(), there[0].tolist(), moved))
    for new, there, moved in moves:
        for page, (p, there_) in enumerate(zip(new, there)):
            if not there_:
                continue
            for i, pool in enumerate((key, value)):
                was, codes = (x[:, page * G:(page + 1) * G] for x in moved[i])
                top = was.amax(1, keepdim=True)
                top = torch.where(top < 0, torch.ones_like(top), top)
                again = (codes.contiguous().view(E4M3).float() * (was / top)[..., None]).to(E4M3).view(torch.uint8)
                pool.view(torch.uint8)[p, :, :codes.shape[1]] = torch.where(((was == top) | (was < 0))[..., None], codes, again)
                scale[p, :, i] = top[:, 0]
