"""attend_shared of more rows than its workspace takes at once: calls that run in pieces of
prefixes, of sequences and of KV heads."""
import ctypes

import pytest
import torch

from test_cache8 import F16, filled

GIB = 1 << 30


def size(F, B, Hq, H, T, D, G=64, Wp=256, W=64):
    from kitty import _hip
    c = _hip.Cache8(4096, 8192, 16384, H * G * D, G * D, D, H * G * D, G * D, D, 2 * H, 2, 4, H, D, G)
    a = _hip.Cache8SharedArgs()
    a.prefixes, a.batch, a.num_q_heads, a.tokens, a.prefix_pages, a.table_pages, a.sm_scale = F, B, Hq, T, Wp, W, 1.0
    got = ctypes.c_size_t(0)
    assert _hip.load().kitty_cache8_shared_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(got)) == _hip.KITTY_OK
    return got.value


def test_workspaces_stay_within_a_gibibyte():
    """Many queries, many sequences of one prefix and of many, one long sequence; the bound of one sequence and head."""
    for F, B, Hq, H, T, D in ((1, 16, 32, 8, 2048, 128), (1, 64, 32, 8, 2048, 128), (64, 64, 32, 8, 2048, 128), (3, 51, 64, 8, 3001, 64),
                              (1, 8192, 32, 32, 1, 128), (4, 8192, 128, 128, 1, 128), (1, 5000, 16, 1, 70, 256), (1, 1, 64, 8, 33000, 128),
                              (700, 2100, 96, 8, 40, 192), (1, 1, 64, 64, 200000, 64)):
        got = size(F, B, Hq, H, T, D)
        assert 0.3 * GIB < got <= GIB, (F, B, Hq, H, T, D, got)
    assert GIB < size(1, 1, 16, 1, 100000, 256) <= 2 * (16 * 100000 + 128) * (256 * 4 + 8 + 8) + 80 * 2 ** 20


def exact(cache, q, ptable, plens, table, lens, end, causal):
    """Some queries of some sequences in float64: out, its tolerance, log-sum-exp and its own; a sequence's own tokens
    stand behind its prefix's, and the queries end with its token `end`."""
    B, Hq, T, D = q.shape
    H, G = cache.num_kv_heads, cache.page_tokens
    ids = torch.cat([ptable, table], 1).long()
    kv = []
    for i, pool in enumerate((cache.key, cache.value)):
        x = pool.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * cache.scale[ids][..., i, None, None].double()
        kv.append(x.transpose(1, 2).flatten(2, 3))                      # (B, H, tokens, D)
    L, n = ptable.shape[1] * G, kv[0].shape[2]
    j, t = torch.arange(n, device=q.device), torch.arange(T, device=q.device)
    place = torch.where(j < L, j, j - L + plens[:, None])               # of each token in its sequence
    held = torch.where(j < L, j < plens[:, None], j - L < lens[:, None])
    sees = held[:, None].expand(B, T, n)
    if causal:
        sees = sees & (place[:, None] <= (plens + end - T)[:, None, None] + t[:, None])
    rows = q.double().view(B, H, Hq // H * T, D)
    s = (rows @ kv[0].transpose(2, 3)).view(B, H, -1, T, n) * D ** -0.5
    s = s.masked_fill(~sees[:, None, None], -float("inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.nan_to_num(torch.exp(s - lse[..., None])).view(B, H, -1, n)
    out, spread = p @ kv[1], p @ kv[1].abs()
    mag = (rows.abs() @ kv[0].abs().transpose(2, 3)).amax(-1, keepdim=True) * D ** -0.5
    w = 2 * ((D + 6) * 2.0 ** -24 * mag + 2.0 ** -20 + n * 2.0 ** -24) + 2.0 ** -16      # cache8_ref.tolerance's, fp16
    tol = 2.0 ** -11 * out.abs() + w * spread + 2.0 ** -24
    room = (D + 8) * 2.0 ** -24 * mag.view(lse.shape) + 2.0 ** -21 * (1 + torch.nan_to_num(lse, neginf=0.0).abs()) + n * 2.0 ** -24
    return out.view(q.shape), tol.view(q.shape), lse.view(B, Hq, T), room.view(B, Hq, T)


# (prefixes, sequences of each, query heads, KV heads, queries, head size, causal, sequences at a time in float64):
# pieces of two prefixes and one, of three and two sequences, of KV heads, of many short sequences
@pytest.mark.gpu
@pytest.mark.parametrize("F,each,Hq,H,T,D,causal,step", [(3, 1, 32, 8, 13000, 128, False, 1), (1, 5, 16, 4, 13500, 128, True, 1),
                                                         (1, 1, 24, 6, 46000, 128, False, 1), (1, 1, 9, 3, 240000, 64, True, 1),
                                                         (4, 1100, 32, 32, 1, 128, True, 275), (2, 2, 40, 5, 10000, 80, True, 1)])
def test_pieces_match_float64(dev, F, each, Hq, H, T, D, causal, step):
    gen = torch.Generator().manual_seed(F + T)
    B, G = F * each, 16
    DP = 64 if D <= 64 else 128
    in_one = 2 * B * Hq * T * 4 * DP if T > 1 else B * H * 16 * 4 * DP
    assert in_one > GIB >= size(F, B, Hq, H, T, D, G, 5, 3)
    cache = filled(gen, 5 * F + 200, H, D, G, dev)
    cache.scale.mul_(0.25)
    ptable = torch.randperm(5 * F, generator=gen).view(F, 5).int().to(dev)
    table = (5 * F + torch.stack([torch.randperm(200, generator=gen)[:3] for _ in range(B)])).int().to(dev)   # read alone: shared
    plens = torch.randint(1, 81, (F,), generator=gen).int().to(dev)
    lens = torch.randint(0, 49, (B,), generator=gen).int().to(dev)
    q = torch.randn(B, Hq, T, D, generator=torch.Generator(dev).manual_seed(1), device=dev, dtype=F16)
    out, lse = cache.attend_shared(q, ptable, plens, table, lens, causal=causal, return_lse=True)
    worst = 0.0
    part = max(1, min(T, (1 << 28) // (step * Hq * 128 * 8)))            # queries at a time, the last of them where causal
    for b in range(0, B, step):
        rows = slice(b, b + step)
        f = torch.arange(b, b + step, device=dev) // each
        starts = range(0, T, part)
        if causal and T > 1:
            starts = sorted({max(0, T - part), 0, max(0, T // 2 - part)})
        for t in starts:
            some = q[rows, :, t:t + part]
            end = lens[rows] - (T - t - some.shape[2])
            want, tol, wlse, room = exact(cache, some, ptable[f], plens[f], table[rows], lens[rows], end, causal)
            assert ((out[rows, :, t:t + part].double() - want).abs() <= tol).all(), (b, t)
            got = lse[rows, :, t:t + part].double()
            assert ((got == wlse) | ((got - wlse).abs() <= room)).all(), (b, t)
            worst = max(worst, float(want.abs().max()))
    assert worst > 0
