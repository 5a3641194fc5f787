"""The 8-bit paged cache on CPU tensors: :class:`kitty.kernels.Cache8`'s three
calls in torch code, with the rules of include/kitty_hip.h (kitty_cache8_*).
Codes and scales are bit-identical to the HIP kernels'."""
from __future__ import annotations

import math
from typing import Optional, Tuple

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


def attend(key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor, q: torch.Tensor, table: torch.Tensor,
           lens: torch.Tensor, q_lens: Optional[torch.Tensor], causal: bool, sm_scale: float, out: torch.Tensor,
           lse: torch.Tensor) -> None:
    B, Hq, T, D = q.shape
    P, H, G = key.shape[:3]
    gq = Hq // H
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
        ids, ok = _page_ids(table[b:b + 1], torch.arange(-(-n // G))[None], P)
        # codes and scales apart, as in the kernels: their products may pass fp32's range
        kv, factors = [], []
        for i, pool in enumerate((key, value)):
            x, f = torch.zeros(ids.shape[1], H, G, D), torch.ones(ids.shape[1], H)
            if P:
                x, f = pool.view(torch.uint8)[ids[0]].view(E4M3).float(), torch.where(ok[0][:, None], scale[ids[0], :, i], f)
            x = torch.where(ok[0][:, None, None, None], x, torch.full_like(x, math.nan))
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
            factors.append(f.t().repeat_interleave(G, 1)[:, None, :n])       # (H, 1, n)
        sees = torch.ones(t, n, dtype=torch.bool)
        if causal:
            sees = torch.arange(n) <= torch.arange(n - t, n)[:, None]
        s = (q[b, :, :t].reshape(H, gq * t, D) @ kv[0].transpose(1, 2) * (factors[0] * sm_scale)).view(H, gq, t, n)
        s = s.masked_fill(~sees, -math.inf)
        l = torch.logsumexp(s, -1)
        none = ~sees.any(-1)                                   # rows that see nothing
        w = torch.exp(s - torch.where(none, torch.zeros_like(l), l)[..., None])
        gone = kv[1].isnan()                                   # masked NaN values stay out of the product
        o = (w.view(H, gq * t, n) * factors[1]) @ kv[1].masked_fill(gone, 0.0)
        met = (sees.float().repeat(gq, 1) @ gone.float()) > 0
        o = o.masked_fill(met, math.nan).view(H, gq, t, D).masked_fill(none[:, None], 0.0)
        out[b, :, :t] = o.reshape(Hq, t, D).to(out.dtype)
        lse[b, :, :t] = l.masked_fill(none, -math.inf).reshape(Hq, t)
