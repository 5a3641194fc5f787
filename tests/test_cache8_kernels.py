"""Attention over the 8-bit cache, kernel by kernel: each case names the kernel that
its sizes choose (on the CPU path the same numbers are asked of the torch code)."""
import numpy as np
import pytest
import torch

from cache8_plan import SPLIT, TILE, TILES, WHOLE, plan, planned, widened
from cache8_ref import Ref, numpy, tolerance
from test_cache8 import BF16, DEVICES, F16, check_attend, filled, tables


# every head size the tile kernel has an instance for and between them, in parts and in
# one; groups that begin and end inside a block of 128 rows, chunks longer than it
TILE_SHAPES = [
    (TILES, 1, 4, 1, 40, 128, 64, [700]), (TILES, 2, 3, 1, 43, 64, 16, [43, 300]), (TILES, 1, 4, 2, 70, 80, 32, [500]),
    (TILES, 1, 1, 1, 97, 96, 128, [400]), (TILES, 2, 5, 1, 27, 16, 16, [90, 27]), (TILES, 1, 2, 1, 65, 32, 256, [1]),
    (TILES, 1, 3, 1, 50, 192, 32, [200]), (TILES, 1, 2, 1, 66, 256, 16, [333]), (TILES, 2, 2, 2, 130, 128, 16, [0, 257]),
    (TILE, 29, 3, 3, 65, 64, 16, None), (TILE, 29, 3, 3, 65, 128, 32, None), (TILE, 29, 3, 3, 65, 80, 16, None), (TILE, 1, 6, 1, 7, 240, 64, [90])]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel,B,Hq,H,T,D,G,lens", TILE_SHAPES)
def test_tile_kernel_matches_float64(dev, dtype, causal, kernel, B, Hq, H, T, D, G, lens):
    gen = torch.Generator().manual_seed(B * 100 + Hq * 10 + T + D)
    if lens is None:
        lens = [(37 * b) % 131 if b % 5 == 0 else b % 3 for b in range(B)]
    W = max(1, (max(lens) + G - 1) // G)
    cache = filled(gen, B * W + 1, H, D, G, dev)
    cache.scale[::3] *= 1.61
    table = tables(gen, B, W, B * W + 1, dev)
    if kernel == TILES:
        table = widened(table, 4096 // G)
    q = torch.randn(B, Hq, T, D, generator=gen).to(dtype)
    assert planned(cache, q, table) == kernel
    check_attend(cache, q, table, lens, causal=causal)


# (kernel, sequences, query heads, KV heads, queries, head size): a batch whose other
# sequences make the sizes, and a first one that the test is about
PADDED = [(WHOLE, 2, 2, 2, 5, 64), (WHOLE, 2, 6, 1, 9, 128), (SPLIT, 2, 2, 1, 5, 64), (SPLIT, 2, 4, 2, 16, 128), (SPLIT, 2, 2, 1, 10, 256),
          (SPLIT, 130, 8, 1, 2, 64), (TILES, 2, 4, 2, 40, 64), (TILES, 2, 2, 1, 70, 96), (TILES, 2, 2, 1, 33, 256),
          (TILE, 87, 1, 1, 66, 64), (TILE, 87, 1, 1, 66, 128)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kernel,B,Hq,H,T,D", PADDED)
def test_padded_rows_are_zero_whatever_real_rows_see(dev, dtype, causal, kernel, B, Hq, H, T, D):
    """NaN keys, NaN values and a missing page in early tokens, which every real row of
    the block sees: NaN rows where the row is real, zeros and -inf behind q_lens."""
    gen = torch.Generator().manual_seed(B + T + D)
    G, n = 16, 150
    few = B > 2                                    # the others of a large batch hold a token or nothing
    cache = filled(gen, 2 * 10 + 2, H, D, G, dev)
    table = widened(tables(gen, 2, 10, 20, dev), 10 if kernel == TILE or kernel == WHOLE else 4096 // G)
    if few:
        table = torch.cat([table, table[1:].expand(B - 2, -1)])
    q = torch.randn(B, Hq, T, D, generator=gen).to(dtype)
    lens = [n, 140] + [b % 2 for b in range(B - 2)]
    q_lens = [max(T - 3, T // 2), T // 2] + [b % 3 % (T + 1) for b in range(B - 2)]
    assert planned(cache, q, table) == kernel

    def check():
        out = check_attend(cache, q, table, lens, q_lens=q_lens, causal=causal)
        for b in range(2):
            assert (out[b, :, q_lens[b]:] == 0).all()

    check()
    cache.value.view(torch.uint8)[int(table[0, 0]), 0, 3, 5] = 0x7F
    check()
    cache.key.view(torch.uint8)[int(table[1, 1]), H - 1, 7, D - 1] = 0xFF
    check()
    table[0, 1] = 22                               # outside the pool
    if few:
        table[2:, 0] = -1                          # of sequences whose one token no or one row sees
    check()


def test_plans_are_the_librarys():
    """The restated rule at both sides of its borders."""
    for args in ((1, 8, 8, 1, 128, 128, 8), (1, 8, 8, 1, 128, 128, 9), (1, 8, 8, 1, 64, 16, 128), (1, 8, 8, 1, 64, 16, 129),
                 (600, 32, 8, 1, 128, 16, 64), (1, 8, 8, 1, 192, 128, 1), (4, 16, 8, 32, 64, 16, 100), (5, 16, 8, 32, 64, 16, 100),
                 (1, 8, 1, 8, 128, 64, 999), (1, 8, 1, 9, 128, 64, 999), (1, 8, 1, 4, 256, 64, 999), (1, 11, 1, 3, 256, 64, 999),
                 (8, 32, 8, 2048, 128, 128, 300), (33, 32, 8, 2048, 128, 128, 300), (1, 1, 1, 1, 16, 16, 0)):
        plan(*args)
        plan(*args, max_tokens=100)
    assert plan(1, 8, 8, 1, 128, 128, 8) == WHOLE and plan(1, 8, 8, 1, 128, 128, 9) == SPLIT
    assert plan(1, 8, 8, 1, 128, 128, 9, max_tokens=1024) == WHOLE
    assert plan(1, 8, 1, 8, 128, 64, 999) == SPLIT and plan(1, 8, 1, 9, 128, 64, 999) == TILES


# (kernel, query heads, queries, head size) on one KV head
FAR = [(WHOLE, 4, 5, 64), (SPLIT, 4, 5, 64), (SPLIT, 8, 7, 128), (TILES, 4, 40, 64), (TILES, 2, 70, 128), (TILES, 2, 20, 256),
       (TILE, 2, 20, 192)]


def far_cache(gen, D, exponents, dev):
    """Pages of 16 tokens in order, the value scales 2^e; a page of 2^-64 is what a page of zeros leaves."""
    cache = filled(gen, len(exponents), 1, D, 16, dev)
    cache.scale[:, 0, 1] = torch.tensor([2.0 ** e for e in exponents], device=dev)
    for p, e in enumerate(exponents):
        if e == -64:
            cache.value.view(torch.uint8)[p] = 0
    table = torch.arange(len(exponents), dtype=torch.int32, device=dev)[None]
    return cache, table


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("exponents", [
    [-64, 90] * 5, [90] + [-64] * 9, [-64] * 9 + [90], [-8] * 6 + [-64, 100, -8, -8], [-100, 5] * 5, [100, -8] * 5,
    [-8] * 8 + [-100, 110], [3, -30, -8] * 3 + [4]])
@pytest.mark.parametrize("kernel,Hq,T,D", FAR)
def test_value_scales_far_apart(dev, kernel, Hq, T, D, exponents):
    """Pages of one sequence whose value scales lie up to 2^210 apart, as large values beside
    a page of zeros leave them: each page keeps its share of the softmax."""
    gen = torch.Generator().manual_seed(T + D)
    cache, table = far_cache(gen, D, exponents, dev)
    cache.scale[:, 0, 0] = 2.0 ** -8
    if kernel in (SPLIT, TILES):
        table = widened(table, 300)
    q = torch.randn(1, Hq, T, D, generator=gen).to(BF16)
    assert planned(cache, q, table) == kernel
    for causal in (True, False):
        check_attend(cache, q, table, [16 * len(exponents) - 3], causal=causal)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel,Hq,T,D", FAR)
def test_small_pages_beside_a_large_one(dev, kernel, Hq, T, D, dtype):
    """A page with one huge channel: in the others its codes are zeros, and what the small
    pages hold there keeps its bits, however much larger the weight times scale of that page."""
    gen = torch.Generator().manual_seed(T + D)
    for small, large in ((-20, 0), (-14, 6), (-100, -8)) if dtype == BF16 else ((-20, -5), (-100, -8)):
        cache, table = far_cache(gen, D, [small] * 4 + [large] + [small] * 5, dev)
        cache.value.view(torch.uint8)[4, :, :, 1:] = 0
        cache.scale[:, 0, 0] = 2.0 ** -9
        if kernel in (SPLIT, TILES):
            table = widened(table, 300)
        q = torch.randn(1, Hq, T, D, generator=gen).to(dtype)
        assert planned(cache, q, table) == kernel
        out = numpy(cache.attend(q.to(dev), table, torch.tensor([157], dtype=torch.int32, device=dev), causal=False))
        want, _, spread, mag, weak = Ref(cache).attend(numpy(q), table.cpu().numpy(), [157], causal=False)
        tol = tolerance(dtype, want, spread, mag, weak, 1, D, 157)          # of one row: weights of two terms
        if dtype == BF16 and kernel in (TILE, TILES):
            # the first 64 tokens are of small pages alone: one fp16 term, off by 2^-11 of a weight, and
            # by 2^-25 of the largest of them where that is more; weights here are within 2^6 of each other
            tol = tol + (2.0 ** -11 + 2.0 ** -25 * 2.0 ** 6) * spread
        assert (np.abs(out - want) <= tol).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scales", [[float("nan")] * 2, [0.0] * 2, [float("inf")] * 2, [1.0, float("nan")]])
@pytest.mark.parametrize("kernel,Hq,T,D", FAR)
def test_missing_page_takes_nothing_from_page_0(dev, kernel, Hq, T, D, dtype, scales):
    """Page 0 is nobody's and its scales are no numbers: a page id outside the pool reaches
    the rows that see its tokens and no other."""
    gen = torch.Generator().manual_seed(T + D)
    cache = filled(gen, 12, 1, D, 16, dev)
    table = torch.arange(1, 11, dtype=torch.int32, device=dev)[None]
    if kernel in (SPLIT, TILES):
        table = widened(table, 300)
    q = torch.randn(1, Hq, T, D, generator=gen).to(dtype)
    assert planned(cache, q, table) == kernel
    want = cache.attend(q.to(dev), table, torch.tensor([147], dtype=torch.int32, device=dev))
    table[0, 9] = 12
    cache.scale[0, 0] = torch.tensor(scales, device=dev)
    out = cache.attend(q.to(dev), table, torch.tensor([147], dtype=torch.int32, device=dev))
    assert out[:, :, -3:].isnan().all()                    # tokens 144 .. 146 are behind the table's last page
    assert torch.equal(out[:, :, :-3], want[:, :, :-3])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel,Hq,T,D", FAR)
def test_scores_that_underflow(dev, kernel, Hq, T, D, dtype):
    """Key scales and sm_scale whose product is below fp32's numbers: every visible token
    weighs the same, masked ones nothing."""
    gen = torch.Generator().manual_seed(T + D)
    cache, table = far_cache(gen, D, [-8] * 10, dev)
    cache.scale[:, 0, 0] = 2.0 ** -64
    if kernel in (SPLIT, TILES):
        table = widened(table, 300)
    q = torch.randn(1, Hq, T, D, generator=gen).to(dtype)
    assert planned(cache, q, table) == kernel
    check_attend(cache, q, table, [150], sm_scale=2.0 ** -90)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kernel,Hq,T,D", FAR)
def test_masked_values_beyond_fp32(dev, kernel, Hq, T, D):
    """A page written elsewhere whose codes times scale pass fp32's range, keys and values:
    rows that do not see its tokens keep their numbers."""
    gen = torch.Generator().manual_seed(T + D)
    cache, table = far_cache(gen, D, [-8] * 10, dev)
    cache.scale[:, 0, 0] = 2.0 ** -8
    if kernel in (SPLIT, TILES):
        table = widened(table, 300)
    q = torch.randn(1, Hq, T, D, generator=gen).to(BF16).to(dev)
    lens = torch.tensor([147], dtype=torch.int32, device=dev)
    want = numpy(cache.attend(q, table, lens))[:, :, :-3]
    cache.scale[9] = 2.0 ** 125
    got = numpy(cache.attend(q, table, lens))[:, :, :-3]          # tokens 144 .. 146 are the last page's
    assert np.isfinite(got).all()
    # both within half a step of the same sums, and with one fp16 term within 2^-11 of the values' size
    assert (np.abs(got - want) <= 2.0 ** -7 * np.abs(want) + 2.0 ** -10 * np.abs(want).max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tile_kernel_beyond_4_gib(dev, dtype):
    """Pages whose byte offsets pass 2^32 in either pool, chunks in tiles."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(4)
    P, H, D, G = 70000, 4, 128, 128            # 4.6 GB a pool
    near = filled(gen, 6, H, D, G, dev)
    key, value = (torch.zeros(P, H, G, D, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    cache = Cache8(key, value, torch.ones(P, H, 2, device=dev))
    pages = [P - 1, 3, P - 3, P - 2, 65537, 66000]
    for a, b in ((cache.key, near.key), (cache.value, near.value)):
        a.view(torch.uint8)[pages] = b.view(torch.uint8)
    cache.scale[pages] = near.scale
    table = widened(torch.tensor(pages, dtype=torch.int32, device=dev).view(2, 3), 40)
    at = widened(torch.arange(6, dtype=torch.int32, device=dev).view(2, 3), 40)
    q = torch.randn(2, 8, 100, D, generator=gen).to(dtype)
    assert planned(cache, q, table) == TILES
    lens = torch.tensor([300, 307], dtype=torch.int32, device=dev)
    assert torch.equal(cache.attend(q.to(dev), table, lens), near.attend(q.to(dev), at, lens))
    check_attend(near, q, at, [300, 307])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,D", [(80, 80), (90, 128), (30, 208)])
def test_tile_kernel_on_pools_in_other_orders(dev, dtype, T, D):
    """Pools with heads inside tokens, slices of larger ones: the same results."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(T)
    P, H, G = 20, 2, 32
    plain = filled(gen, P, H, D, G, dev)
    other = []
    for t in (plain.key, plain.value):
        big = torch.full((P + 1, G, H + 1, D + 16), 0xFF, dtype=torch.uint8, device=dev)
        view = big[1:, :, 1:, 16:].permute(0, 2, 1, 3)
        view.copy_(t.view(torch.uint8))
        other.append(view)
    scale = torch.full((P, H, 6), float("nan"), device=dev)[..., 2:4]
    scale.copy_(plain.scale)
    cache = Cache8(*other, scale)
    table = widened(tables(gen, 2, 9, P, dev), 300, -1)
    q = torch.randn(2, 6, T, D, generator=gen).to(dtype)
    assert planned(cache, q, table) == TILES
    lens = torch.tensor([250, 77], dtype=torch.int32, device=dev)
    assert torch.equal(cache.attend(q.to(dev), table, lens), plain.attend(q.to(dev), table, lens))
    check_attend(cache, q, table, [250, 77])


@pytest.mark.gpu
def test_tile_kernel_repeats_itself(dev):
    """Value scales near and far, in parts and in one: no order of arrival enters a result."""
    gen = torch.Generator().manual_seed(1)
    for far in (False, True):
        cache = filled(gen, 300, 4, 128, 64, dev)
        if far:
            cache.scale[::7, :, 1] = 2.0 ** 40
        table = tables(gen, 8, 32, 300, dev)
        lens = torch.tensor([2000, 1, 700, 64, 2048, 1999, 1024, 300], dtype=torch.int32, device=dev)
        for B, T, kernel in ((8, 130, TILES), (2, 500, TILES), (8, 2100, TILE)):
            q = torch.randn(B, 8, T, 128, generator=gen).bfloat16().to(dev)
            assert planned(cache, q, table) == kernel
            first = cache.attend(q, table[:B], lens[:B])
            for _ in range(4):
                assert torch.equal(cache.attend(q, table[:B], lens[:B]), first)
