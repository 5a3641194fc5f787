"""Attention over the 8-bit cache that weighs its tokens (Cache8.attend_weighed) against
float64, on the CPU path and on the GPU, and its refusals."""
import ctypes
import math

import numpy as np
import pytest
import torch

from cache8_plan import widened
from cache8_ref import Ref, numpy, tolerance
from test_cache8 import BF16, DEVICES, F16, filled, i32, tables


def want_weights(cache, q, table, lens, q_lens, causal, sm_scale, weights):
    """(weights after the call, how far they may be off) in float64.

    A row's p = exp(score - lse) is off by that factor's exponent's error: the score's, D products and sums
    and 6 factors of 2^-24 of the largest sum of |q k| each, in the attention and again here; the
    log-sum-exp's own, 2^-21 (1 + |lse|) and the sum's n 2^-24; 4 roundings on the way to the exponent, of
    numbers up to |score| + |lse|; exp2 2^-22.  Adding R rows takes R roundings of the sum, adding it to
    the weight one more of the result."""
    ref = Ref(cache)
    B, Hq, T, D = q.shape
    sm = D ** -0.5 if sm_scale is None else sm_scale
    gq, N = Hq // ref.H, weights.shape[2]
    out, off = weights.copy(), np.zeros_like(weights)
    for b in range(B):
        n, t = int(lens[b]), T if q_lens is None else int(q_lens[b])
        if n < 0 or n > table.shape[1] * ref.G or not 0 <= t <= T:
            continue
        keys = ref.tokens(table, b, 0, n)[0]
        for h in range(Hq):
            for i in range(t):
                e = n - t + i + 1 if causal else n
                if e <= 0:
                    continue
                with np.errstate(invalid="ignore"):
                    s = keys[h // gq, :e] @ q[b, h, i] * sm
                    top = s.max()
                    lse = top + np.log(np.exp(s - top).sum())
                    p = np.exp(s - lse)
                    mag = np.max(np.abs(keys[h // gq, :e]) @ np.abs(q[b, h, i]) * sm)
                    rel = (2 * (D + 6) * 2.0 ** -24 * mag + 2.0 ** -21 * (1 + abs(lse)) + n * 2.0 ** -24
                           + 4 * 2.0 ** -24 * (mag + abs(lse)) + 2.0 ** -22)
                e = min(e, N)
                out[b, h // gq, :e] += p[:e]
                off[b, h // gq, :e] += p[:e] * (rel + (gq * t + 1) * 2.0 ** -24)
    return out, off + np.abs(out) * 2.0 ** -24


def check_weighed(cache, q, table, lens, N=None, q_lens=None, causal=True, sm_scale=None, weights=None, infinite=False, **kw):
    """Output and log-sum-exp as check_attend has them of attend, and the weights; infinite: of rows
    with infinite scores the log-sum-exp (-inf of no finite one, and +inf or NaN) is not looked at."""
    dev = cache.device
    gen = torch.Generator().manual_seed(len(lens))
    if weights is None:
        weights = torch.rand(q.shape[0], cache.num_kv_heads, max(max(lens), 0) if N is None else N, generator=gen).to(dev)
    before = numpy(weights)
    args = table, i32(lens, dev)
    more = dict(q_lens=None if q_lens is None else i32(q_lens, dev), causal=causal, sm_scale=sm_scale, return_lse=True, **kw)
    out, lse = cache.attend_weighed(q.to(dev), *args, weights, **more)
    want, off = want_weights(cache, numpy(q), table.cpu().numpy(), lens, q_lens, causal, sm_scale, before)
    got = numpy(weights)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > off
    assert not bad.any(), (float(np.nanmax(np.abs(got - want) - off)), np.argwhere(bad)[:4])
    assert (got[want == before] == before[want == before]).all()             # what no row sees stays as it is
    ref, rlse, spread, mag, small = Ref(cache).attend(numpy(q), table.cpu().numpy(), lens, q_lens, causal, sm_scale)
    n, D = max(max(lens), 1), q.shape[3]
    tol = tolerance(q.dtype, ref, spread, mag, small, q.shape[1] // cache.num_kv_heads * q.shape[2], D, n)
    out, lse = numpy(out), numpy(lse)
    np.testing.assert_array_equal(np.isnan(out), np.isnan(ref))
    assert not (np.abs(out - ref) > tol).any()
    if not infinite:
        np.testing.assert_array_equal(np.isnan(lse), np.isnan(rlse))
    seen = np.isfinite(rlse)
    assert (lse[np.isneginf(rlse)] == -np.inf).all()
    room = (D + 8) * 2.0 ** -24 * mag[seen] + 2.0 ** -21 * (1 + np.abs(rlse[seen])) + n * 2.0 ** -24
    assert (np.abs(lse[seen] - rlse[seen]) <= room).all()
    return weights


SHAPES = [
    # one query: lengths around the tiles, groups around the row blocks, every page and head size
    (1, 1, 1, 1, 16, 16, [1]), (1, 4, 1, 1, 64, 16, [31]), (2, 8, 8, 1, 128, 128, [32, 33]), (1, 7, 1, 1, 128, 32, [129]),
    (3, 16, 2, 1, 128, 64, [0, 127, 700]), (1, 20, 1, 1, 80, 16, [257]), (2, 3, 3, 1, 256, 256, [5, 511]),
    (4, 34, 2, 1, 64, 32, [1, 0, 64, 300]), (1, 2, 2, 1, 192, 128, [1025]), (70, 2, 1, 1, 32, 16, list(range(70))),
    # a few queries, more queries than tokens
    (2, 4, 1, 3, 128, 16, [2, 50]), (1, 8, 2, 4, 128, 128, [300]), (3, 4, 2, 8, 64, 32, [8, 100, 9]), (2, 6, 2, 9, 256, 16, [3, 90]),
    # chunks: heads that begin and end inside a block of rows, tokens that later queries alone see
    (1, 4, 2, 40, 128, 64, [40]), (2, 8, 2, 33, 64, 16, [33, 200]), (1, 3, 1, 130, 128, 128, [131]), (1, 4, 4, 70, 80, 32, [500]),
    (2, 2, 1, 65, 256, 128, [64, 300]), (1, 4, 1, 100, 48, 16, [170]),
    # rows in several parts, whose sums are added
    (1, 4, 1, 150, 64, 16, [200]), (1, 3, 1, 200, 112, 32, [333]), (2, 2, 1, 300, 256, 16, [300, 31])]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,H,T,D,G,lens", SHAPES)
def test_matches_float64(dev, dtype, causal, B, Hq, H, T, D, G, lens):
    gen = torch.Generator().manual_seed(B * 100 + Hq * 10 + T + D)
    W = max(1, (max(lens) + G - 1) // G)
    cache = filled(gen, B * W + 1, H, D, G, dev)
    cache.scale[::3] *= 1.61                     # not only powers of two
    q = torch.randn(B, Hq, T, D, generator=gen).to(dtype)
    table = tables(gen, B, W, B * W + 1, dev)
    check_weighed(cache, q, table, lens, causal=causal)
    # a table that could hold far more, weights of more tokens and of fewer than there are
    wide = widened(table, 8192 // G)
    check_weighed(cache, q, wide, lens, causal=causal, N=max(lens) + 77)
    check_weighed(cache, q, wide, lens, causal=causal, N=max(lens) // 2, max_tokens=1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,q_lens", [(1, [1, 0, 1, 1]), (5, [5, 1, 0, 3]), (60, [1, 60, 33, 0])])
def test_padded(dev, dtype, causal, T, q_lens):
    """Padded query rows, sequences without tokens or queries, more queries than tokens."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 40, 2, 64, 16, dev)
    q = torch.randn(4, 6, T, 64, generator=gen).to(dtype)
    q[:, :, T // 2:] *= math.nan if T == 60 else 1.0          # padding may hold anything
    table = tables(gen, 4, 9, 40, dev)
    if T == 60:
        q_lens = [min(n, 30) for n in q_lens]
    check_weighed(cache, q, table, [130, 40, 7, 0], q_lens=q_lens, causal=causal)
    check_weighed(cache, q, table, [130, 40, 7, 0], q_lens=q_lens, causal=causal, N=9 * 16)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("Hq,T", [(4, 1), (2, 6), (4, 50), (4, 80)])
def test_masked_and_missing_places(dev, Hq, T):
    """NaN codes and wild page ids behind the last token, NaN keys of later tokens, NaN
    values, a missing page: the weights of what rows with a NaN softmax see are NaN, no others."""
    gen = torch.Generator().manual_seed(T)
    D, G, n = 128, 16, 150
    cache = filled(gen, 24, 2, D, G, dev)
    table = 1 + tables(gen, 1, 12, 23, dev)
    table[0, 10:12] = torch.tensor([1 << 30, -5], dtype=torch.int32)
    last = int(table[0, 9])
    for pool in (cache.key, cache.value):        # rows 6 .. of the page that ends inside a tile
        pool.view(torch.uint8)[last, :, n % G:] = 0xFF
    q = torch.randn(1, Hq, T, D, generator=gen).half()
    check_weighed(cache, q, table, [n])
    cache.value.view(torch.uint8)[last, 0, 1, 7] = 0x7F                      # values are not in the softmax
    check_weighed(cache, q, table, [n])
    if T > 1:
        cache.key.view(torch.uint8)[last, 1, n % G - 2, 3] = 0x7F            # a token that the first queries do not see
        check_weighed(cache, q, table, [n])
    table[0, 9] = 24                             # outside the pool: rows that see tokens 144 .. are NaN
    check_weighed(cache, q, table, [n])
    cache.scale[0] = math.nan                    # page 0's scales stand for no missing page
    check_weighed(cache, q, table, [n], causal=False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,wide", [(1, 0), (1, 500), (5, 0), (40, 500), (100, 0)])
def test_infinite_queries(dev, T, wide):
    """Infinite scores: the weights of what a row of NaN weights sees are NaN, a score of -inf
    beside finite ones weighs nothing."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 12, 2, 64, 16, dev)
    cache.key.view(torch.uint8)[..., 7] = 0x38                               # 1.0
    cache.key.view(torch.uint8)[..., 9] = 0x00
    table = torch.cat([tables(gen, 1, 12, 12, dev), torch.zeros(1, wide, dtype=torch.int32, device=dev)], 1)
    cache.key.view(torch.uint8)[int(table[0, 2]), 1, 5, 9] = 0xB8            # -1.0 in one token
    q = torch.randn(1, 4, T, 64, generator=gen).half()
    q[..., 9] = 1.0
    q[0, 2, T // 2, 9] = 60000.0                                             # far below all others
    check_weighed(cache, q, table, [180], N=192)
    for row, value in (((0, 1, 0, 7), math.inf), ((0, 1, 0, 7), -math.inf)):
        x = q.clone()
        x[row] = value
        w = check_weighed(cache, x, table, [180], N=192, infinite=True)
        assert w[0, 0, :180 - T + 1].isnan().all() and w[0, 0, 180:].isfinite().all() and w[0, 1].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,T,cut", [(128, 1, 0), (64, 1, 5000), (8, 13, 0), (40, 3, 16369)])
def test_scores_in_bursts(dev, Hq, T, cut):
    """Runs of more steps than a wave keeps scores of: several bursts, of whole pairs and of parts; weights
    that end inside a burst."""
    gen = torch.Generator().manual_seed(Hq)
    B, H, D, G, W = 12, 8, 16, 256, 64
    cache = filled(gen, 1 + B * W, H, D, G, dev)
    table = (1 + torch.randperm(B * W, generator=gen)).view(B, W).int().to(dev)
    lens = [16384, 16383, 1, 9000, 16370, 12345, 16384, 40, 16129, 16384, 15000, 16384]
    q = torch.randn(B, Hq, T, D, generator=gen).half()
    check_weighed(cache, q, table, lens, N=cut or 16384)


@pytest.mark.gpu
def test_scores_beyond_a_gibibyte(dev):
    """Weights for so many tokens that the scores of 16 rows are not kept: a second pass over the keys instead."""
    gen = torch.Generator().manual_seed(3)
    cache = filled(gen, 4, 1, 64, 256, dev)
    q = torch.randn(1, 16, 1, 64, generator=gen).half()
    for columns in (1 << 16, (1 << 16) + 1):
        table = widened(tables(torch.Generator().manual_seed(9), 1, 4, 4, dev), columns)
        weights = torch.zeros(1, 1, columns * 256, device=dev)
        check_weighed(cache, q, table, [700], weights=weights, max_tokens=700)
        assert (weights[..., 700:] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [1, 4, 20, 48])
def test_broken_lengths(dev, T):
    """Sequences whose lengths break the rules change no weight."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 60, 1, 64, 16, dev)
    q = torch.randn(5, 2, T, 64, generator=gen).half()
    table = tables(gen, 5, 4, 60, dev)
    check_weighed(cache, q, table, [32, 65, -1, 20, 1 << 30], N=64)
    check_weighed(cache, q, table, [64, 30, 1, 20, 0], N=64, q_lens=[T, T + 1, 0, -1, 1])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("Hq,T", [(4, 1), (2, 6), (4, 50)])
def test_layouts(dev, Hq, T):
    """Queries, outputs and weights in other memory orders, unaligned, negated, q and out in
    one memory; pools of other strides."""
    gen = torch.Generator().manual_seed(T)
    D, B, H = 64, 3, 2
    cache = filled(gen, 31, H, D, 16, dev)
    table = tables(gen, B, 10, 31, dev)
    q = torch.randn(B, Hq, T, D, generator=gen).half()
    lens = [150, 3, 97]
    weights = torch.rand(B, H, 160, generator=gen).to(dev)
    held = weights.clone()
    check_weighed(cache, q, table, lens, weights=weights)
    q, n = q.to(dev), i32(lens, dev)
    want = cache.attend(q, table, n)

    def same(x, cache=cache, w=None, **kw):
        w = held.clone() if w is None else w.copy_(held)
        got = cache.attend_weighed(x, table, n, w, **kw)
        assert torch.equal(got, want) and torch.equal(w, weights)
        return got

    same(q)
    same(q.transpose(1, 2).contiguous().transpose(1, 2))
    odd = torch.zeros(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)
    same(odd.copy_(q))
    same(q.transpose(2, 3).contiguous().transpose(2, 3))                     # channels not contiguous
    same(torch._neg_view(-q))
    for out in (torch.empty(B, T, Hq, D, dtype=F16, device=dev).transpose(1, 2), torch.zeros_like(odd), q.clone(),
                torch._neg_view(torch.zeros_like(q))):
        assert same(q, out=out) is out and torch.equal(out, want)
    x = q.clone()
    assert same(x, out=x) is x and torch.equal(x, want)
    long = torch.zeros(B + 1, Hq, T, D, dtype=F16, device=dev)               # rows of out over other rows of q
    long[:B] = q
    w = held.clone()
    assert torch.equal(cache.attend_weighed(long[:B], table, n, w, out=long[1:]), want) and torch.equal(w, weights)
    same(q, w=torch.zeros(H, B, 161, device=dev)[:, :, 1:].transpose(0, 1))
    from kitty.kernels import Cache8
    turned = [t.view(torch.uint8).permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3) for t in (cache.key, cache.value)]
    same(q, cache=Cache8(*(t.view(torch.float8_e4m3fn) for t in turned), cache.scale.transpose(0, 1).contiguous().transpose(0, 1)))
    assert cache.attend_weighed(q[:0], table[:0], n[:0], held[:0]).shape == (0, Hq, T, D)
    assert cache.attend_weighed(q[:, :, :0], table, n, held).shape == (B, Hq, 0, D)
    assert torch.equal(cache.attend_weighed(q, table, n, held[..., :0]), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_weights_and_gradients(dev):
    gen = torch.Generator().manual_seed(9)
    cache = filled(gen, 9, 2, 64, 16, dev)
    table, lens = tables(gen, 2, 4, 9, dev), i32([60, 5], dev)
    q = torch.randn(2, 4, 3, 64, generator=gen).half().to(dev)
    w = torch.zeros(2, 2, 64, device=dev)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend_weighed(q.clone().requires_grad_(), table, lens, w)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend_weighed(q, table, lens, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend_weighed(q, table, lens, w, out=torch.zeros_like(q).requires_grad_())
    for _ in range(2):
        x = torch.ones(w.shape, device=dev, requires_grad=True)
        y = (x * w).sum()                       # saves w
        cache.attend_weighed(q, table, lens, w)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda x: cache.attend_weighed(x, table, lens, w), (q,), check_trace=False)


def test_refusals():
    gen = torch.Generator().manual_seed(3)
    cache = filled(gen, 9, 2, 64, 16, "cpu")
    table, lens = tables(gen, 2, 4, 9, "cpu"), i32([60, 5], "cpu")
    q, w = torch.randn(2, 4, 1, 64, generator=gen).half(), torch.zeros(2, 2, 64)
    cache.attend_weighed(q, table, lens, w)
    for bad in (w.double(), w[:1], w[:, :1], w[0], w.half(), w.transpose(1, 2), torch.zeros(2, 64, 2).transpose(1, 2),
                torch._neg_view(w), w[:, :1].expand(2, 2, 64), w[:1].expand(2, 2, 64)):
        with pytest.raises(ValueError):
            cache.attend_weighed(q, table, lens, bad)
    for kw in (dict(q_lens=lens[:1]), dict(sm_scale=0.0), dict(sm_scale=math.nan), dict(out=q.float()), dict(max_tokens=-1)):
        with pytest.raises(ValueError):
            cache.attend_weighed(q, table, lens, w, **kw)
    for args in ((q.float(), table, lens), (q[:, :3], table, lens), (q, table.long(), lens), (q, table, lens.long()), (q, table[:1], lens)):
        with pytest.raises(ValueError):
            cache.attend_weighed(*args, w)
    with pytest.raises(RuntimeError):
        cache.attend_weighed(q, table, lens, w.to("meta"))


def test_abi_refusals():
    from kitty import _hip
    L = _hip.load()
    c = _hip.Cache8(4096, 8192, 16384, 1024, 1024, 64, 1024, 1024, 64, 4, 2, 4, 1, 64, 16)

    def call(fn=L.kitty_cache8_weighed_attention, w=(4096, 64, 64, 64), last=None, **kw):
        a, x = _hip.Cache8AttentionArgs(), _hip.Cache8Weights(*w)
        a.q = a.out = a.block_table = a.lens = a.workspace = 4096
        a.batch, a.num_q_heads, a.tokens, a.table_pages, a.sm_scale, a.workspace_bytes = 2, 2, 1, 4, 1.0, 1 << 40
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(c), ctypes.byref(a), ctypes.byref(x), last)

    assert L.kitty_cache8_weighed_attention(ctypes.byref(c), None, None, None) == _hip.KITTY_E_INVALID
    a = _hip.Cache8AttentionArgs()
    assert L.kitty_cache8_weighed_attention(ctypes.byref(c), ctypes.byref(a), None, None) == _hip.KITTY_E_INVALID
    for w in ((None, 64, 64, 64), (4096, 64, 64, -1), (4097, 64, 64, 64)):
        assert call(w=w) == _hip.KITTY_E_INVALID, w
    for kw in (dict(batch=-1), dict(tokens=-1), dict(num_q_heads=0), dict(dtype=2), dict(sm_scale=0.0), dict(q=None),
               dict(out=None), dict(lens=None), dict(block_table=None), dict(q=4098), dict(out=4104), dict(q_s_tok=4),
               dict(workspace=None), dict(workspace=4100), dict(workspace_bytes=15)):
        assert call(**kw) == _hip.KITTY_E_INVALID, kw
    for kw in (dict(table_pages=1 << 27), dict(tokens=1 << 26), dict(batch=1 << 26)):
        assert call(**kw) == _hip.KITTY_E_UNSUPPORTED, kw
    assert call(batch=0) == _hip.KITTY_OK and call(tokens=0) == _hip.KITTY_OK
    size, plain = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert call(L.kitty_cache8_weighed_attention_workspace_size, last=ctypes.byref(size)) == _hip.KITTY_OK
    assert call(lambda c, a, w, s: L.kitty_cache8_attention_workspace_size(c, a, s), last=ctypes.byref(plain)) == _hip.KITTY_OK
    assert size.value >= plain.value + 2 * 2 * 4
    assert call(workspace_bytes=size.value - 1) == _hip.KITTY_E_INVALID
    assert call(L.kitty_cache8_weighed_attention_workspace_size) == _hip.KITTY_E_INVALID


def test_packed_arguments_are_the_structures():
    from kitty import _hip
    from kitty.kernels import cache8
    fields = [n for n, _ in _hip.Cache8Weights._fields_]
    a = _hip.Cache8Weights.from_buffer_copy(cache8._WEIGHTS.pack(1, 2, 3, 4).ljust(ctypes.sizeof(_hip.Cache8Weights), b"\0"))
    assert [getattr(a, n) for n in fields] == [1, 2, 3, 4]
