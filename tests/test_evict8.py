"""Eviction from the 8-bit cache by weight (Cache8.evict) against its definition, token
by token, on the CPU path and on the GPU, and its refusals."""
import ctypes
import math

import numpy as np
import pytest
import torch

from cache8_ref import NAN, VALUES, Ref, encode
from test_cache8 import DEVICES, filled, i32, same_pools, tables


def order(w):
    """Positions from the heaviest on, the earlier of equals first, NaN above all."""
    return sorted(range(len(w)), key=lambda i: (0 if np.isnan(w[i]) else 1, 0.0 if np.isnan(w[i]) else -w[i], i))


def evict_ref(ref, table, lens, weights, keep, first, last, into):
    """The pools of `ref` after the call; lengths, positions and weights."""
    B, H, N = weights.shape
    out_lens = np.zeros(B, np.int32)
    kept = np.full((B, H, min(keep, N)), -1, np.int32)
    out = np.zeros((B, H, N), np.float32)
    old = [p.copy() for p in ref.pools], ref.scale.astype(np.float32)
    for b in range(B):
        n = int(lens[b])
        if n < 0 or n > table.shape[1] * ref.G or n > N:
            out_lens[b] = -1
            continue
        m = out_lens[b] = min(n, keep)
        for h in range(H):
            at = list(range(n))
            if n > keep:
                mid = [first + i for i in order(weights[b, h, first:n - last])[:keep - first - last]]
                at = sorted(at[:first] + mid + at[n - last:])
            assert len(at) == m
            kept[b, h, :m], out[b, h, :m] = at, weights[b, h, at]
            for number in range(-(-m // ref.G)):
                p = ref.page(into, b, number)
                if p < 0:
                    continue
                src = at[number * ref.G:(number + 1) * ref.G]
                ids = [ref.page(table, b, i // ref.G) for i in src]
                for st in range(2):
                    there = [old[1][j, h, st] for j in ids if j >= 0]
                    top = max(there) if there else np.float32(1)
                    for r, (i, j) in enumerate(zip(src, ids)):
                        if j < 0:
                            ref.pools[st][p, h, r] = NAN
                            continue
                        codes, was = old[0][st][j, h, i % ref.G], old[1][j, h, st]
                        if was != top:      # the quotient and the product in fp32, then e4m3
                            codes = encode((VALUES[codes].astype(np.float32) * (was / top)).astype(np.float64))
                        ref.pools[st][p, h, r] = codes
                    ref.scale[p, h, st] = top
    return out_lens, kept, out


def check_evict(cache, table, lens, weights, keep, first=0, last=0, into=None):
    dev = cache.device
    ref = Ref(cache)
    before = weights.clone()
    got = cache.evict(table, i32(lens, dev), weights, keep, first=first, last=last, into=into)
    want = evict_ref(ref, table.cpu().numpy(), lens, weights.cpu().numpy(), keep, first, last, (table if into is None else into).cpu().numpy())
    for g, w in zip(got, want):
        assert tuple(g.shape) == w.shape
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    same_pools(cache, ref)
    np.testing.assert_array_equal(weights.cpu().numpy(), before.cpu().numpy())
    return got


def heavy(gen, *shape):
    """Weights over orders of magnitude, with zeros and equals among them."""
    w = (torch.randn(shape, generator=gen) * 2).exp()
    w[torch.rand(shape, generator=gen) < 0.2] = 0.0
    return torch.where(torch.rand(shape, generator=gen) < 0.2, w.round(), w)


# (sequences, KV heads, head size, page, lengths, keep, first, last)
SHAPES = [
    (1, 1, 16, 16, [1], 1, 0, 0), (1, 1, 16, 16, [2], 1, 0, 0), (2, 2, 64, 16, [40, 17], 16, 1, 4), (1, 8, 128, 128, [300], 200, 4, 64),
    (3, 2, 80, 32, [0, 100, 500], 77, 3, 0), (1, 3, 128, 64, [700], 699, 0, 0), (2, 1, 256, 256, [511, 256], 256, 10, 10),
    (1, 2, 48, 16, [333], 64, 32, 32), (1, 1, 64, 32, [1030], 1, 0, 1), (2, 2, 32, 16, [1024, 1025], 1000, 0, 0),
    (1, 1, 16, 16, [5000], 2100, 1024, 1000), (1, 1, 16, 256, [2100], 2048, 0, 9), (2, 1, 112, 32, [1300, 1171], 1170, 7, 0), (2, 1, 48, 64, [2700, 10], 2049, 7, 0), (4, 1, 192, 64, [64, 65, 0, 128], 64, 0, 63), (1, 2, 144, 128, [90], 0, 0, 0), (70, 1, 16, 16, list(range(70)), 33, 2, 5)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,H,D,G,lens,keep,first,last", SHAPES)
def test_matches_the_definition(dev, B, H, D, G, lens, keep, first, last):
    gen = torch.Generator().manual_seed(B * 100 + keep + D)
    W = max(1, -(-max(lens) // G))
    K = max(1, -(-min(keep, max(lens)) // G))
    P = B * (W + K) + 2
    for place in (False, True):
        cache = filled(gen, P, H, D, G, dev)
        if place:
            cache.scale[::3] *= 1.61             # not only powers of two
        ids = torch.randperm(P, generator=gen).to(torch.int32)
        table, into = ids[:B * W].view(B, W).to(dev), ids[B * W:B * (W + K)].view(B, K).to(dev)
        w = heavy(gen, B, H, W * G).to(dev)
        check_evict(cache, table, lens, w, keep, first, last, None if place else into)
    # weights of no more tokens than there are, of far more, and more to keep than either
    cache = filled(gen, P, H, D, G, dev)
    check_evict(cache, table, lens, w[..., :max(lens)], keep, first, last)
    lens = [min(n, keep) for n in lens]
    check_evict(cache, table, lens, torch.cat([w, w, w], 2), keep // 2, min(first, keep // 4), min(last, keep // 4))
    check_evict(cache, table, [n // 2 for n in lens], w, 1 << 29, first, last, into if max(lens) <= K * G and W <= K else None)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["zeros", "equal", "signs", "nan", "bits", "inf", "one byte"])
@pytest.mark.parametrize("n", [40, 1500])
def test_weights_of_every_kind(dev, kind, n):
    """Equal weights, both zeros, negative ones, NaN of either sign, infinities, subnormals,
    weights that differ in their last or first bits alone: the earlier of equals stays."""
    gen = torch.Generator().manual_seed(n)
    G, W = 64, -(-n // 64)
    cache = filled(gen, 2 * W, 2, 16, G, dev)
    w = heavy(gen, 1, 2, n)
    if kind == "zeros":
        w = torch.where(torch.rand(w.shape, generator=gen) < 0.5, 0.0, -0.0)
    elif kind == "equal":
        w = torch.full_like(w, 0.7)
    elif kind == "signs":
        w = torch.randn(w.shape, generator=gen).round(decimals=1)
    elif kind == "nan":
        w[..., ::3] = math.nan
        w[..., ::6] = -math.nan
    elif kind == "inf":
        w[..., ::3], w[..., 1::7] = math.inf, -math.inf
    elif kind == "bits":
        w = (0x3F800000 + torch.randint(0, 9, w.shape, generator=gen, dtype=torch.int32)).view(torch.float32)
        w[..., :n // 3] = torch.randint(0, 5, (n // 3,), generator=gen, dtype=torch.int32).view(torch.float32)   # subnormal
    else:
        w = torch.randint(0, 256, w.shape, generator=gen, dtype=torch.int32).bitwise_left_shift(8).view(torch.float32)
    for keep in (n // 2, n - 1, 7, n // 3 + 1, 2):
        check_evict(cache, tables(gen, 1, W, 2 * W, dev), [n], w.to(dev), keep, 1, 1)


@pytest.mark.parametrize("dev", DEVICES)
def test_codes_rounded_again(dev):
    """Scales far apart: codes that become subnormal or zero, NaN codes, tokens of the largest
    scale that move unchanged; a page whose light tokens alone had the large scale gets a smaller one."""
    gen = torch.Generator().manual_seed(4)
    G, W = 16, 8
    cache = filled(gen, 3 * W, 2, 64, G, dev)
    cache.scale.copy_(2.0 ** torch.randint(-20, 1, cache.scale.shape, generator=gen).float().to(dev))
    cache.value.view(torch.uint8)[::2, :, 3, 5] = 0xFF
    table = tables(gen, 1, W, 3 * W, dev)
    w = torch.arange(128.0).repeat(1, 2, 1)
    w[0, 1] = w[0, 1].flip(0)
    check_evict(cache, table, [128], w.to(dev), 50, 0, 3)
    cache.scale[int(table[0, 0])] = 2.0 ** 10
    w[0, :, :16] = -1.0
    lens, kept, _ = check_evict(cache, table, [50], w.to(dev), 20, 0, 0)
    assert int(kept.min()) == -1 or int(kept.min()) >= 16
    assert (cache.scale[int(table[0, 0])] <= 1.0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_pages_that_are_not_there_and_broken_lengths(dev):
    """Tokens without a page move as NaN and set no scale, tokens whose new page is not there
    are dropped; lengths that break the rules come back as -1 and leave everything as it was."""
    gen = torch.Generator().manual_seed(6)
    G, W = 16, 6
    for place in (True, False):
        cache = filled(gen, 40, 2, 32, G, dev)
        table, into = tables(gen, 3, W, 18, dev), (18 + tables(gen, 3, 4, 22, dev)).to(torch.int32)
        table[0, 1], table[1, 3], table[2, 5], table[2, 1] = 40, -1, 1 << 30, -(1 << 31)
        table[1, 0] = table[1, 1] = 77
        if not place:
            into[0, 0], into[2, 1] = -7, 40
        w = heavy(gen, 3, 2, W * G).to(dev)
        check_evict(cache, table, [96, 90, 96], w, 60, 8, 8, None if place else into)
        check_evict(cache, table, [-1, 97, 1 << 30], w, 60, 8, 8, None if place else into)
        check_evict(cache, table, [96, 70, 0], w[..., :80], 60, 0, 0, None if place else into)


@pytest.mark.parametrize("dev", DEVICES)
def test_layouts(dev):
    """Weights, tables and pools of other strides, unaligned and negated weights, the table itself as `into`."""
    gen = torch.Generator().manual_seed(7)
    from kitty.kernels import Cache8
    B, H, D, G, W = 2, 3, 64, 16, 10
    first = filled(gen, 31, H, D, G, dev)
    table, w = tables(gen, B, W, 31, dev), heavy(gen, B, H, W * G).to(dev)
    wide = torch.full((B, W + 7), -1, dtype=torch.int32, device=dev)
    wide[:, :W] = table
    strange = torch.zeros(H, B, W * G + 1, device=dev)[:, :, 1:].transpose(0, 1)
    results = []
    for t, x, into, turn in ((table, w, None, False), (wide, w, None, False), (table, strange.copy_(w), table, False),
                             (wide[:, :W], torch._neg_view(-w), wide[:, :W], False), (table, w, None, True)):
        key, value, scale = first.key.clone(), first.value.clone(), first.scale.clone()
        if turn:
            key, value = (p.view(torch.uint8).permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3).view(torch.float8_e4m3fn) for p in (key, value))
            scale = scale.transpose(0, 1).contiguous().transpose(0, 1)
        cache = Cache8(key, value, scale)
        results.append((*cache.evict(t, i32([150, 33], dev), x, 70, 4, 16, into), key.view(torch.uint8).clone(), value.view(torch.uint8).clone(), scale.clone()))
    for r in results[1:]:
        for a, b in zip(r, results[0]):
            assert torch.equal(a, b)
    check_evict(first, table, [150, 33], w, 70, 4, 16)
    lens, kept, out = first.evict(table[:0], i32([], dev), w[:0], 70)
    assert lens.shape == (0,) and kept.shape == (0, H, 70) and out.shape == (0, H, W * G)
    lens, kept, out = first.evict(table, i32([0, 0], dev), w[..., :0], 70)
    assert lens.tolist() == [0, 0] and kept.shape == (B, H, 0) and out.shape == (B, H, 0)


@pytest.mark.parametrize("dev", DEVICES)
def test_weights_and_gradients(dev):
    gen = torch.Generator().manual_seed(9)
    cache = filled(gen, 9, 2, 64, 16, dev)
    table, lens, w = tables(gen, 2, 4, 9, dev), i32([60, 5], dev), torch.zeros(2, 2, 64, device=dev)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.evict(table, lens, w.clone().requires_grad_(), 30)
    with torch.no_grad():
        cache.evict(table, lens, w.clone().requires_grad_(), 30)
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda x: cache.evict(table, lens, x, 30)[2], (w,), check_trace=False)


def test_refusals():
    gen = torch.Generator().manual_seed(3)
    cache = filled(gen, 20, 2, 64, 16, "cpu")
    table, lens, w = tables(gen, 2, 4, 9, "cpu"), i32([60, 5], "cpu"), torch.zeros(2, 2, 64)
    cache.evict(table, lens, w, 30, 10, 20)
    for kw in (dict(keep=-1), dict(keep=1 << 31), dict(keep=30, first=-1), dict(keep=30, last=-1), dict(keep=30, first=20, last=11),
               dict(keep=30, into=table[:1]), dict(keep=30, into=table[:, :1]), dict(keep=30, into=table.long()),
               dict(keep=30, into=table[0])):
        with pytest.raises(ValueError):
            cache.evict(table, lens, w, **kw)
    for args in ((table, lens, w.double()), (table, lens, w[:1]), (table, lens, w[:, :1]), (table, lens, w.transpose(1, 2)), (table.long(), lens, w),
                 (table[0], lens, w), (table, lens.long(), w), (table, lens[:1], w)):
        with pytest.raises(ValueError):
            cache.evict(*args, 30)
    with pytest.raises(RuntimeError):
        cache.evict(table, lens, w.to("meta"), 30)


def test_abi_refusals():
    from kitty import _hip
    L = _hip.load()
    c = _hip.Cache8(4096, 8192, 16384, 1024, 1024, 64, 1024, 1024, 64, 4, 2, 4, 1, 64, 16)

    def call(fn=L.kitty_cache8_evict, last_arg=None, **kw):
        a = _hip.Cache8EvictArgs()
        a.weights = a.block_table = a.lens = a.out_lens = a.kept = a.out_weights = a.workspace = 4096
        a.batch, a.table_pages, a.weight_tokens, a.keep, a.first, a.last, a.workspace_bytes = 2, 4, 64, 30, 4, 4, 1 << 40
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(c), ctypes.byref(a), last_arg)

    assert L.kitty_cache8_evict(ctypes.byref(c), None, None) == _hip.KITTY_E_INVALID
    assert L.kitty_cache8_evict(None, None, None) == _hip.KITTY_E_INVALID
    for kw in (dict(batch=-1), dict(table_pages=-1), dict(into_pages=-1), dict(weight_tokens=-1), dict(keep=-1), dict(first=-1),
               dict(last=-1), dict(first=20, last=11), dict(weights=None), dict(block_table=None), dict(lens=None),
               dict(out_lens=None), dict(kept=None), dict(out_weights=None), dict(weights=4098), dict(out_weights=4097),
               dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=15)):
        assert call(**kw) == _hip.KITTY_E_INVALID, kw
    for kw in (dict(table_pages=1 << 27), dict(batch=1 << 26), dict(weight_tokens=(1 << 30) + 1)):
        assert call(**kw) == _hip.KITTY_E_UNSUPPORTED, kw
    assert call(batch=0) == _hip.KITTY_OK
    size = ctypes.c_size_t(7)
    assert call(L.kitty_cache8_evict_workspace_size, ctypes.byref(size)) == _hip.KITTY_OK and size.value == 2 * 2 * 30 * (64 + 4)
    assert call(workspace_bytes=size.value - 1) == _hip.KITTY_E_INVALID
    assert call(L.kitty_cache8_evict_workspace_size, ctypes.byref(size), into=4096) == _hip.KITTY_OK and size.value == 0
    assert call(L.kitty_cache8_evict_workspace_size) == _hip.KITTY_E_INVALID


def test_packed_arguments_are_the_structure():
    from kitty import _hip
    from kitty.kernels import cache8
    fields = [n for n, _ in _hip.Cache8EvictArgs._fields_]
    values = list(range(1, len(fields) + 1))
    a = _hip.Cache8EvictArgs.from_buffer_copy(cache8._EVICT.pack(*values))
    assert cache8._EVICT.size == ctypes.sizeof(a)
    assert [getattr(a, n) for n in fields] == values
