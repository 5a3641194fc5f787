"""The 8-bit paged cache (kitty.kernels.Cache8): writing, reading back and
attention against float64, on the CPU path and on the GPU, and its refusals."""
import math

import numpy as np
import pytest
import torch

import kitty  # noqa: F401
from cache8_ref import NAN, VALUES, Ref, encode, numpy, scale_for, tolerance

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def filled(gen, P, H, D, G, dev, spread=3):
    """A cache whose every byte is set: random finite codes with power-of-two
    scales around 1 / 100; NaN codes nowhere."""
    from kitty.kernels import Cache8
    codes = [torch.randint(0, 256, (P, H, G, D), generator=gen, dtype=torch.uint8) for _ in range(2)]
    for c in codes:
        c[(c & 0x7F) == NAN] = 0x3A
    s = 2.0 ** torch.randint(-8 - spread, -7 + spread, (P, H, 2), generator=gen).float()
    return Cache8(*(c.to(dev).view(torch.float8_e4m3fn) for c in codes), s.to(dev))


def tables(gen, B, W, P, dev):
    return torch.randperm(P, generator=gen)[:B * W].view(B, W).to(torch.int32).to(dev)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def same_pools(cache, ref):
    for st, t in enumerate((cache.key, cache.value)):
        got, want = t.view(torch.uint8).cpu().numpy(), ref.pools[st]
        nan = (want & 0x7F) == NAN
        assert ((got & 0x7F) == NAN)[nan].all()
        assert (got[~nan] == want[~nan]).all(), int((got[~nan] != want[~nan]).sum())
    assert (cache.scale.cpu().numpy() == ref.scale).all()


def test_reference_rounds_as_torch_does():
    x = torch.randn(100000, generator=torch.Generator().manual_seed(1)).mul_(80).clamp_(-448, 448)
    x = torch.cat([x, x / 4096, torch.from_numpy(VALUES[:127].copy()).float()])
    assert (encode(x.double().numpy()) == x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()).all()
    assert [scale_for(m) for m in (0.0, 448.0, 449.0, 28.0)] == [2.0 ** -64, 1.0, 2.0, 2.0 ** -4]


# ------------------------------------------------------------------- writing

# one token, a page's last row and the next page's first, whole pages, chunks that
# begin and end inside pages, every page size; head sizes around the vector widths
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,H,T,D,G,start,dtype", [
    (1, 1, 1, 16, 16, [0], F16), (1, 8, 1, 128, 128, [77], F16), (3, 2, 1, 64, 32, [31, 32, 33], BF16),
    (2, 2, 2, 128, 16, [15, 16], F32), (2, 3, 16, 80, 16, [0, 16], BF16), (1, 2, 40, 256, 16, [5], F16),
    (2, 1, 129, 96, 64, [63, 1], F32), (1, 2, 300, 128, 128, [100], BF16), (2, 1, 520, 256, 256, [0, 255], F32),
    (5, 1, 33, 48, 32, [0, 1, 31, 95, 64], F16), (1, 1, 700, 144, 256, [3], F16)])
def test_write_matches_the_definition(dev, B, H, T, D, G, start, dtype):
    gen = torch.Generator().manual_seed(T * 7 + D)
    W = (max(start) + T + G - 1) // G
    cache = filled(gen, B * W + 2, H, D, G, dev)
    ref = Ref(cache)
    table = tables(gen, B, W, B * W + 2, dev)
    k, v = (torch.randn(B, H, T, D, generator=gen).to(dtype) for _ in range(2))
    k[..., 3] *= 50
    cache.write(k.to(dev), v.to(dev), table, i32(start, dev))
    ref.write(numpy(k), numpy(v), table.cpu().numpy(), start)
    same_pools(cache, ref)
    # and a larger token behind them: the scale of the last page rises, its codes round again
    big = (100 * torch.randn(B, H, 1, D, generator=gen)).to(dtype)
    ends = [s + T for s in start]
    ok = [b for b in range(B) if ends[b] < W * G]
    if ok:
        cache.write(big[ok].to(dev), big[ok].to(dev), table[ok], i32([ends[b] for b in ok], dev))
        ref.write(numpy(big[ok]), numpy(big[ok]), table[ok].cpu().numpy(), [ends[b] for b in ok])
        same_pools(cache, ref)


@pytest.mark.parametrize("dev", DEVICES)
def test_tokens_one_by_one(dev):
    """A page filled token by token of growing size, past its end; every state on the way."""
    gen = torch.Generator().manual_seed(5)
    B, H, D, G = 3, 2, 64, 16
    cache = filled(gen, 8, H, D, G, dev)
    ref = Ref(cache)
    table = tables(gen, B, 2, 8, dev)
    pos = [0, 3, 9]
    for step in range(18):
        x = torch.randn(2, B, H, 1, D, generator=gen) * 1.3 ** step
        cache.write(x[0].to(dev), x[1].to(dev), table, i32(pos, dev))
        ref.write(numpy(x[0]), numpy(x[1]), table.cpu().numpy(), pos)
        same_pools(cache, ref)
        pos = [p + 1 for p in pos]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_write_special_values(dev, dtype):
    """Zeros, the type's smallest and largest numbers, values at the border of a scale,
    NaN and infinities: finite rows keep the scale that the finite values need."""
    gen = torch.Generator().manual_seed(6)
    B, H, T, D, G = 7, 1, 5, 32, 16
    fi = torch.finfo(dtype)
    x = torch.randn(B, H, T, D, generator=gen)
    x[0] = 0.0
    x[1] = fi.smallest_normal * x[1].sign()
    x[2] = fi.max * x[2].sign()
    x[3, ..., 0] = 28.0                       # 448 / 16: the largest code
    x[4, 0, 2, 5], x[4, 0, 3, 1], x[4, 0, 0, 0] = math.nan, math.inf, -math.inf
    x[5] = math.nan
    x[6, ..., 1] = -0.0
    x = x.to(dtype)
    if dtype == F32:
        x[1, 0, 0, 0] = 1e-45                 # subnormal
    cache = filled(gen, B + 1, H, D, G, dev)
    ref = Ref(cache)
    table = tables(gen, B, 1, B + 1, dev)
    for start in ([0] * B, [4] * B):          # fresh, and behind tokens
        cache.write(x.to(dev), (-x).to(dev), table, i32(start, dev))
        ref.write(numpy(x), numpy(-x), table.cpu().numpy(), start)
        same_pools(cache, ref)


@pytest.mark.parametrize("dev", DEVICES)
def test_write_keeps_foreign_scales(dev):
    """Pages whose scales are no powers of two (written elsewhere): kept where the new
    token fits, the quotient rounded once; raised to the power of two it needs otherwise."""
    gen = torch.Generator().manual_seed(8)
    cache = filled(gen, 4, 2, 64, 16, dev)
    cache.scale.copy_((torch.rand(4, 2, 2, generator=gen) + 0.1).to(dev))
    table = tables(gen, 2, 2, 4, dev)
    ref = Ref(cache)
    x = torch.randn(2, 2, 1, 64, generator=gen) * 20
    x[1] *= 1000
    start = [7, 20]
    cache.write(x.to(dev), x.to(dev), table, i32(start, dev))
    # fp32 quotients: x / s rounded to fp32 first
    ref.write(numpy(x), numpy(x), table.cpu().numpy(), start)
    for st, t in enumerate((cache.key, cache.value)):
        got, want = t.view(torch.uint8).cpu().numpy(), ref.pools[st]
        # rounding to fp32 before e4m3 moves a value by at most 2^-24: another code only next to a tie
        assert (np.abs(VALUES[got] - VALUES[want]) <= 2.0 ** -3 * np.abs(VALUES[want]) + 2.0 ** -9).all()
        assert (got != want).mean() < 1e-3
    assert (cache.scale.cpu().numpy() == ref.scale).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_write_strided_padded_and_pages_that_are_not_there(dev):
    """Projections' views, rows of odd alignment, padded batches with empty sequences,
    pools in another order; tokens without a page are dropped and nothing else moves."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(9)
    B, H, T, D, G, W, P = 6, 2, 37, 48, 16, 4, 30
    base = filled(gen, P, H, D, G, "cpu")
    pools = [t.view(torch.uint8).permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3) for t in (base.key, base.value)]
    cache = Cache8(*pools, base.scale.to(dev))      # (P, G, H, D) in memory
    ref = Ref(cache)
    table = tables(gen, B, W, P, dev)
    table[1, 1], table[2, 0] = -1, P
    start, lens = [3, 0, 0, -1, 50, 20], [37, 37, 30, 10, 37, 0]   # the fifth runs past the table
    fused = torch.randn(B, T, 2 * H * D + 1, generator=gen).to(BF16).to(dev)
    k = fused[..., :H * D].unflatten(2, (H, D)).transpose(1, 2)
    v = fused[..., H * D + 1:].unflatten(2, (H, D)).transpose(1, 2)   # rows 2-byte aligned
    cache.write(k, v, table, i32(start, dev), i32(lens, dev))
    ref.write(numpy(k), numpy(v), table.cpu().numpy(), start, lens)
    same_pools(cache, ref)


# ------------------------------------------------------------------- reading

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,H,D,G,lens,tokens,start,dtype", [
    (1, 1, 16, 16, [1], 1, None, F16), (2, 2, 64, 16, [33, 0], 40, None, BF16), (3, 1, 128, 128, [1, 128, 300], 129, [0, 100, 250], F32),
    (1, 8, 128, 32, [500], 333, [77], F16), (2, 3, 80, 64, [70, 130], 65, [64, 70], BF16), (1, 2, 256, 256, [257], 300, [-2], F32)])
def test_read_back(dev, B, H, D, G, lens, tokens, start, dtype):
    gen = torch.Generator().manual_seed(tokens)
    W = max(1, (max(lens) + G - 1) // G)
    cache = filled(gen, B * W + 1, H, D, G, dev)
    cache.scale[0] *= 1.37
    table = tables(gen, B, W, B * W + 1, dev)
    got = cache.read(table, i32(lens, dev), tokens, start=None if start is None else i32(start, dev), dtype=dtype)
    want = torch.from_numpy(Ref(cache).read(table.cpu().numpy(), lens, tokens, start))
    # code * scale in fp32, then the type: at most half a step of each
    half = torch.finfo(dtype).eps / 2
    for g, w in zip(got, want):
        assert g.dtype == dtype and g.shape == w.shape
        g = g.double().cpu()
        assert (g.isnan() == w.isnan()).all()
        assert ((g - w).abs() <= (half + 2.0 ** -24) * w.abs() + torch.finfo(dtype).smallest_normal * half).nan_to_num(1).bool().logical_or(w.isnan()).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_read_into_tensors_and_missing_pages(dev):
    gen = torch.Generator().manual_seed(3)
    cache = filled(gen, 5, 2, 64, 16, dev)
    table = i32([[0, 5, 2], [3, -7, 1]], dev)
    out = [torch.full((2, 48, 2, 64), 9.0, device=dev).transpose(1, 2) for _ in range(2)]   # (B, T, H, D) in memory
    got = cache.read(table, i32([60, 20], dev), 48, out=tuple(out))
    assert got[0] is out[0] and got[1] is out[1]
    want = Ref(cache).read(table.cpu().numpy(), [60, 20], 48)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(numpy(g), w)


# ----------------------------------------------------------------- attention

def check_attend(cache, q, table, lens, q_lens=None, causal=True, sm_scale=None, **kw):
    dev = cache.device
    out, lse = cache.attend(q.to(dev), table, i32(lens, dev), q_lens=None if q_lens is None else i32(q_lens, dev),
                            causal=causal, sm_scale=sm_scale, return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape
    want, wlse, spread, mag, small = Ref(cache).attend(numpy(q), table.cpu().numpy(), lens, q_lens, causal, sm_scale)
    tol = tolerance(q.dtype, want, spread, mag, small, q.shape[1] // cache.num_kv_heads * q.shape[2], q.shape[3],
                    max(max(lens), 1))
    got, glse = numpy(out), numpy(lse)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > tol
    assert not bad.any(), (float(np.nanmax(np.abs(got - want) - tol)), np.argwhere(bad)[:4])
    np.testing.assert_array_equal(np.isnan(glse), np.isnan(wlse))
    seen = np.isfinite(wlse)
    assert (glse[np.isneginf(wlse)] == -np.inf).all()
    # lse: the scores' error, and fp32's of the logarithm and the sum
    room = (q.shape[3] + 8) * 2.0 ** -24 * mag[seen] + 2.0 ** -21 * (1 + np.abs(wlse[seen])) + max(lens) * 2.0 ** -24
    assert (np.abs(glse[seen] - wlse[seen]) <= room).all()
    return out


SHAPES = [
    # one query: lengths around the tiles, groups around the row blocks, every page and head size
    (1, 1, 1, 1, 16, 16, [1]), (1, 4, 1, 1, 64, 16, [31]), (2, 8, 8, 1, 128, 128, [32, 33]), (1, 7, 1, 1, 128, 32, [129]),
    (3, 16, 2, 1, 128, 64, [0, 127, 700]), (1, 20, 1, 1, 80, 16, [257]), (2, 3, 3, 1, 256, 256, [5, 511]),
    (4, 34, 2, 1, 64, 32, [1, 0, 64, 300]), (1, 2, 2, 1, 192, 128, [1025]), (70, 2, 1, 1, 32, 16, list(range(70))),
    # a few queries, as many rows as the blocks, more queries than tokens
    (2, 4, 1, 3, 128, 16, [2, 50]), (1, 8, 2, 4, 128, 128, [300]), (3, 4, 2, 8, 64, 32, [8, 100, 9]), (1, 10, 2, 5, 96, 64, [40]),
    (2, 6, 2, 9, 256, 16, [3, 90]),
    # chunks
    (1, 4, 2, 40, 128, 64, [40]), (2, 8, 2, 33, 64, 16, [33, 200]), (1, 3, 1, 130, 128, 128, [131]), (1, 4, 4, 70, 80, 32, [500]),
    (2, 2, 1, 65, 256, 128, [64, 300]), (1, 16, 1, 100, 128, 16, [170])]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,H,T,D,G,lens", SHAPES)
def test_attend_matches_float64(dev, dtype, causal, B, Hq, H, T, D, G, lens):
    gen = torch.Generator().manual_seed(B * 100 + Hq * 10 + T + D)
    W = max(1, (max(lens) + G - 1) // G)
    cache = filled(gen, B * W + 1, H, D, G, dev)
    cache.scale[::3] *= 1.61                     # not only powers of two
    q = torch.randn(B, Hq, T, D, generator=gen).to(dtype)
    check_attend(cache, q, tables(gen, B, W, B * W + 1, dev), lens, causal=causal)


# the same rows with a table that could hold far more (entries behind the last page are
# no ids): work shared by the lengths on the device instead of a workgroup a pair, more
# than 64 sequences, blocks of 16 to 64 rows, runs that end in the middle of a pair
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,H,T,D,G,lens", [
    (1, 4, 1, 1, 64, 16, [300]), (3, 16, 2, 1, 128, 64, [0, 127, 700]), (2, 3, 3, 1, 256, 256, [5, 511]),
    (70, 2, 1, 1, 32, 16, list(range(70))), (130, 1, 1, 1, 16, 16, [3 * (b % 7) for b in range(130)]), (2, 4, 2, 9, 128, 16, [9, 1000]),
    (1, 8, 2, 4, 128, 128, [300]), (2, 5, 1, 8, 96, 32, [400, 0]), (2, 4, 1, 15, 64, 16, [50, 333]), (2, 6, 2, 9, 256, 16, [3, 290]),
    (1, 2, 1, 40, 256, 64, [600]), (1, 16, 1, 4, 128, 64, [1500]), (1, 8, 1, 33, 64, 64, [1500]), (1, 1, 1, 1, 128, 16, [1]),
    (3, 4, 2, 1, 16, 256, [20000, 15001, 37]), (5, 1, 1, 3, 16, 256, [30000, 0, 40000, 129, 9000])])
def test_attend_shared_by_lengths(dev, dtype, causal, B, Hq, H, T, D, G, lens):
    gen = torch.Generator().manual_seed(B * 100 + Hq * 10 + T + D)
    W = (max(lens) + G - 1) // G
    cache = filled(gen, B * W + 1, H, D, G, dev)
    cache.scale[::3] *= 1.61
    wide = torch.full((B, max(8192 // G, W)), 1 << 30, dtype=torch.int32, device=dev)
    wide[:, :W] = tables(gen, B, W, B * W + 1, dev)
    q = torch.randn(B, Hq, T, D, generator=gen).to(dtype)
    check_attend(cache, q, wide, lens, causal=causal)
    check_attend(cache, q, wide, lens, causal=causal, max_tokens=1)      # a wrong hint changes no result


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,q_lens", [(1, [1, 0, 1, 1]), (5, [5, 1, 0, 3]), (60, [1, 60, 33, 0])])
def test_attend_padded(dev, dtype, causal, T, q_lens):
    """Padded query rows, sequences without tokens or queries, more queries than tokens."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 40, 2, 64, 16, dev)
    q = torch.randn(4, 6, T, 64, generator=gen).to(dtype)
    out = check_attend(cache, q, tables(gen, 4, 9, 40, dev), [130, 40, 7, 0], q_lens=q_lens, causal=causal)
    for b, n in enumerate(q_lens):
        assert (out[b, :, n:] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("wide", [0, 600])
@pytest.mark.parametrize("Hq,T", [(4, 1), (2, 6), (4, 50), (4, 80)])
def test_attend_masked_places_reach_no_row(dev, Hq, T, wide):
    """NaN codes and wild page ids behind the last token, NaN keys and values of later
    tokens, a missing page: only the rows that see them change."""
    gen = torch.Generator().manual_seed(T)
    D, G, n = 128, 16, 150
    cache = filled(gen, 24, 2, D, G, dev)
    table = torch.cat([tables(gen, 1, 12, 24, dev), torch.full((1, wide), -9, dtype=torch.int32, device=dev)], 1)
    table[0, 10:12] = torch.tensor([1 << 30, -5], dtype=torch.int32)
    last = int(table[0, 9])
    for pool in (cache.key, cache.value):        # rows 6 .. of the page that ends inside a tile
        pool.view(torch.uint8)[last, :, n % G:] = 0xFF
    q = torch.randn(1, Hq, T, D, generator=gen).half()
    check_attend(cache, q, table, [n])
    spare = [p for p in range(24) if p not in table[0].tolist()][0]
    if T > 1:
        cache.value.view(torch.uint8)[last, 0, n % G - 1, 7] = 0x7F      # the newest token's value
        cache.value.view(torch.uint8)[last, 1, n % G - 3, 100] = 0xFF
        cache.value.view(torch.uint8)[int(table[0, 8]), 1, 14, 100] = 0xFF
        check_attend(cache, q, table, [n])
        cache.key.view(torch.uint8)[last, 1, n % G - 2, 3] = 0x7F
        check_attend(cache, q, table, [n])
    cache.value.view(torch.uint8)[spare] = 0x30
    cache.key.view(torch.uint8)[spare] = 0x30
    table[0, 9] = spare
    check_attend(cache, q, table, [n])
    table[0, 9] = 24                             # outside the pool: rows that see tokens 144 .. are NaN
    check_attend(cache, q, table, [n])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("G", [16, 256])
@pytest.mark.parametrize("T", [1, 4, 20, 48, 300])
def test_attend_broken_lengths(dev, T, G):
    """Lengths that break the rules give NaN rows to their sequence alone."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 60, 1, 64, G, dev)
    q = torch.randn(5, 2, T, 64, generator=gen).half()
    table = tables(gen, 5, 2 if G == 16 else 10, 60, dev)
    most = table.shape[1] * G
    check_attend(cache, q, table, [32, most + 1, -1, 20, 1 << 30])
    check_attend(cache, q, table, [most, 30, 1, 20, 0], q_lens=[T, T + 1, 0, -1, 1])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [1, 20, 40, 100])
def test_attend_wide_scales(dev, T):
    """Value scales 2^-60 to 2^60 in one sequence, in bf16: weights keep the range of fp32."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 8, 1, 64, 16, dev)
    cache.scale[:, :, 1] = 2.0 ** (torch.arange(8, device=dev) * 17 - 60)[:, None].float()
    cache.scale[:, :, 0] *= 4.0                  # sharp rows: some page wins
    q = torch.randn(1, 4, T, 64, generator=gen).to(BF16)
    check_attend(cache, q, i32([[0, 1, 2, 3, 4, 5, 6, 7]], dev), [127])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,wide", [(1, 0), (1, 500), (5, 0), (40, 500), (100, 0)])
def test_attend_infinite_queries(dev, T, wide):
    """Infinite scores as the softmax has them: +inf (and inf - inf) make the row NaN, -inf
    weighs nothing, a row of nothing else is NaN; the other rows keep their numbers."""
    gen = torch.Generator().manual_seed(T)
    cache = filled(gen, 12, 1, 64, 16, dev)
    cache.key.view(torch.uint8)[..., 7] = 0x38                      # 1.0
    cache.key.view(torch.uint8)[..., 9].bitwise_or_(1).bitwise_and_(0x77)   # positive, not 0
    table = torch.cat([tables(gen, 1, 12, 12, dev), torch.zeros(1, wide, dtype=torch.int32, device=dev)], 1)
    q = torch.randn(1, 4, T, 64, generator=gen).half()
    clean, _, _, _, _ = Ref(cache).attend(numpy(q), table.cpu().numpy(), [180])
    q[0, 1, :, 7] = math.inf
    q[0, 2, :, 7] = -math.inf
    q[0, 3, 0, 9] = math.inf
    out, lse = cache.attend(q.to(dev), table, i32([180], dev), return_lse=True)
    assert out[0, 1].isnan().all() and out[0, 2].isnan().all() and out[0, 3, 0].isnan().all()
    assert (lse[0, 2] == -math.inf).all()
    keep = np.abs(numpy(out)[0, 0] - clean[0, 0]) <= 2.0 ** -10 * np.abs(clean[0, 0]) + 1e-3 * np.abs(clean).max()
    assert keep.all() and out[0, 3, 1:].isfinite().all()


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_layouts(dev):
    """Views of fused projections, outputs in (B, T, H, D) memory, shared pages, unaligned
    rows, single-entry dimensions of odd strides: the same numbers."""
    gen = torch.Generator().manual_seed(2)
    B, Hq, H, T, D = 2, 4, 2, 3, 64
    cache = filled(gen, 9, H, D, 32, dev)
    table = i32([[4, 1, 2], [4, 1, 8]], dev)     # a shared prefix
    lens = i32([70, 65], dev)
    x = torch.randn(B, T, Hq * D + 8, generator=gen).half().to(dev)
    q = x[..., :Hq * D].unflatten(2, (Hq, D)).transpose(1, 2)
    want = cache.attend(q.contiguous(), table, lens)
    check_attend(cache, q.cpu(), table, [70, 65])
    assert torch.equal(cache.attend(q, table, lens), want)
    out = torch.empty(B, T, Hq, D, dtype=F16, device=dev).transpose(1, 2)
    assert cache.attend(q, table, lens, out=out) is out and torch.equal(out, want)
    odd = torch.empty(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape).copy_(q)
    assert torch.equal(cache.attend(odd, table, lens), want)
    odd_out = torch.empty(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)
    cache.attend(q, table, lens, out=odd_out)
    assert torch.equal(odd_out, want)
    one = x[:1, :1, 3:3 + D].unsqueeze(1)        # (1, 1, 1, D), strides of the fused row
    wide = cache.attend(one.expand(1, Hq, 1, D), table[:1], lens[:1])
    assert torch.equal(wide, cache.attend(one.expand(1, Hq, 1, D).contiguous(), table[:1], lens[:1]))
    same = q.contiguous()
    assert cache.attend(same, table, lens, out=same) is same and torch.equal(same, want)
    neg = torch._neg_view(q)
    assert torch.equal(cache.attend(neg, table, lens), cache.attend((-q).contiguous(), table, lens))
    assert torch.equal(cache.attend(q, table, lens, max_tokens=70), want)


# --------------------------------------------------------- together, as used

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_request(dev, dtype):
    """Two prompts in chunks, then decode steps: written, attended at every step over what
    the cache then holds, read back at the end; against unquantised attention it stays near."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(1)
    B, Hq, H, D, G = 2, 8, 2, 64, 32
    cache = Cache8.empty(12, H, D, G, device=dev)
    ref = Ref(cache)
    table = tables(gen, B, 5, 12, dev)
    held, ks, vs = [0, 0], [], []
    for T, lens in ((50, [50, 37]), (20, [1, 20]), (1, None), (1, None), (1, None)):
        n = [T] * B if lens is None else lens
        q, k, v = (torch.randn(B, h, T, D, generator=gen).to(dtype) for h in (Hq, H, H))
        padded = None if lens is None else i32(lens, dev)
        cache.write(k.to(dev), v.to(dev), table, i32(held, dev), padded)
        ref.write(numpy(k), numpy(v), table.cpu().numpy(), held, lens)
        held = [a + b for a, b in zip(held, n)]
        same_pools(cache, ref)
        check_attend(cache, q, table, held, q_lens=n)
        ks.append([k[b, :, :n[b]] for b in range(B)])
        vs.append([v[b, :, :n[b]] for b in range(B)])
    back = cache.read(table, i32(held, dev), max(held), dtype=F32)
    for got, parts in zip(back, (ks, vs)):
        for b in range(B):
            x = torch.cat([p[b] for p in parts], 1).float()
            # e4m3: half a step 2^-4 of a value, twice where its page's scale rose, and 2^-10 of the scale
            s = 2.0 ** math.ceil(math.log2(float(x.abs().max()) / 448))
            err = (got[b, :, :held[b]].cpu() - x).abs()
            assert (err <= 2 * 2.0 ** -4 * x.abs() * 1.07 + 2 * 2.0 ** -10 * s).all()


# ------------------------------------------------------------------ refusals

def test_refusals():
    from kitty.kernels import Cache8
    E = torch.float8_e4m3fn
    pool = lambda *s, dt=E: torch.zeros(s, dtype=torch.uint8).view(dt)  # noqa: E731
    one = torch.ones(4, 2, 2)
    with pytest.raises(ValueError, match="float8"):
        Cache8(pool(4, 2, 16, 64).view(torch.int8), pool(4, 2, 16, 64), one)
    with pytest.raises(ValueError, match="alike"):
        Cache8(pool(4, 2, 16, 64), pool(4, 2, 32, 64), one)
    with pytest.raises(ValueError, match="tokens"):
        Cache8(pool(4, 2, 24, 64), pool(4, 2, 24, 64), one)
    with pytest.raises(ValueError, match="multiple of 16"):
        Cache8(pool(4, 2, 16, 72), pool(4, 2, 16, 72), one)
    with pytest.raises(NotImplementedError, match="256"):
        Cache8(pool(4, 2, 16, 512), pool(4, 2, 16, 512), one)
    with pytest.raises(ValueError, match="scale"):
        Cache8(pool(4, 2, 16, 64), pool(4, 2, 16, 64), one.half())
    with pytest.raises(ValueError, match="contiguous channels"):
        Cache8(pool(4, 2, 64, 16).transpose(2, 3), pool(4, 2, 64, 16).transpose(2, 3), one)
    c = Cache8.empty(4, 2, 64, 16, device="cpu")
    x, t, n = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 3, 64).half()
    for bad in (x[:, :1], x[..., :32], x[0]):
        with pytest.raises(ValueError):
            c.write(bad, bad, t, n)
    with pytest.raises(ValueError, match="value"):
        c.write(x, x.half(), t, n)
    with pytest.raises(ValueError, match="float16"):
        c.write(x.double(), x.double(), t, n)
    for table in (t.long(), t[0], t.expand(2, 2), torch.zeros(2, 1, dtype=torch.int32).t()[:, ::1].expand(2, 2)):
        with pytest.raises(ValueError, match="block_table"):
            c.write(x, x, table, n)
    for lens in (n.long(), n.expand(2), n[0]):
        with pytest.raises(ValueError, match="start"):
            c.write(x, x, t, lens)
        with pytest.raises(ValueError, match="lens"):
            c.attend(q, t, lens)
    with pytest.raises(ValueError, match="heads"):
        c.attend(q[:, :3], t, n)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        c.attend(q.float(), t, n)
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="sm_scale"):
            c.attend(q, t, n, sm_scale=s)
    with pytest.raises(ValueError, match="out"):
        c.attend(q, t, n, out=q.float())
    with pytest.raises(ValueError, match="share memory"):
        c.attend(q, t, n, out=q[:, :1].expand(1, 4, 3, 64))
    with pytest.raises(ValueError, match="share memory"):
        c.read(t, n, 3, out=(x, x[:, :, :1].expand(1, 2, 3, 64)))
    with pytest.raises(ValueError, match="out"):
        c.read(t, n, 3, out=(x, x.half()))
    with pytest.raises(ValueError, match="dtype"):
        c.read(t, n, 3, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no backward"):
        c.attend(q.requires_grad_(), t, n)
    with torch.no_grad():
        c.attend(q, t, n)
    with pytest.raises(RuntimeError, match="no backward"):
        c.write(x.clone().requires_grad_(), x, t, n)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda a: c.attend(a, t, n), (q.detach(),))
    assert c.attend(q.detach()[:, :, :0], t, n).shape == (1, 4, 0, 64)
    assert c.read(t, n, 0)[0].shape == (1, 2, 0, 64)
    empty = Cache8.empty(0, 2, 64, 16, device="cpu")
    assert empty.attend(q.detach(), t, n + 1).isnan().any()
    empty.write(x, x, t, n)


def test_abi_refusals():
    """The C entries refuse bad pools and calls before they touch a device."""
    import ctypes
    from kitty import _hip
    L = _hip.load()
    assert L.kitty_cache8_write(None, ctypes.byref(_hip.Cache8RowsArgs()), None) == _hip.KITTY_E_INVALID

    def cache(**kw):
        c = _hip.Cache8(4096, 8192, 16384, 4096, 1024, 64, 4096, 1024, 64, 4, 2, 4, 2, 64, 16)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def rc(fn, c, a):
        return getattr(L, fn)(ctypes.byref(c), ctypes.byref(a), None)

    rows = _hip.Cache8RowsArgs()
    assert rc("kitty_cache8_write", cache(), rows) == rc("kitty_cache8_read", cache(), rows) == _hip.KITTY_OK
    for bad, text in ((dict(head_dim=72), b"multiple of 16"), (dict(page_tokens=48), b"page_tokens"), (dict(key=4097), b"aligned"),
                      (dict(scale=16388), b"aligned"), (dict(value=0), b"NULL"), (dict(key_s_tok=8), b"multiples of 16"),
                      (dict(value_s_tok=48), b"at least head_dim"), (dict(scale_s_head=1), b"even"), (dict(num_kv_heads=0), b"positive")):
        for fn in ("kitty_cache8_write", "kitty_cache8_read"):
            assert rc(fn, cache(**bad), rows) == _hip.KITTY_E_INVALID and text in L.kitty_last_error(), bad
        assert rc("kitty_cache8_attention", cache(**bad), _hip.Cache8AttentionArgs()) == _hip.KITTY_E_INVALID
    assert rc("kitty_cache8_write", cache(head_dim=272), rows) == _hip.KITTY_E_UNSUPPORTED
    rows.batch = rows.tokens = 1
    for fn in ("kitty_cache8_write", "kitty_cache8_read"):
        assert rc(fn, cache(), rows) == _hip.KITTY_E_INVALID and b"NULL" in L.kitty_last_error()
        rows.dtype = 3
        assert rc(fn, cache(), rows) == _hip.KITTY_E_INVALID and b"dtype" in L.kitty_last_error()
        rows.dtype = 0
    rows.key, rows.value, rows.block_table, rows.start, rows.lens, rows.table_pages = 4096, 4104, 16, 16, 16, 1
    assert rc("kitty_cache8_read", cache(), rows) == _hip.KITTY_E_INVALID and b"16-byte" in L.kitty_last_error()
    rows.tokens = 1 << 30
    rows.value, rows.batch = 4096, 1 << 20
    assert rc("kitty_cache8_write", cache(), rows) == _hip.KITTY_E_UNSUPPORTED
    assert rc("kitty_cache8_read", cache(), rows) == _hip.KITTY_E_UNSUPPORTED
    a = _hip.Cache8AttentionArgs()
    a.num_q_heads, a.sm_scale = 3, 1.0
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_E_INVALID and b"multiple" in L.kitty_last_error()
    a.num_q_heads, a.sm_scale = 4, 0.0
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_E_INVALID and b"sm_scale" in L.kitty_last_error()
    a.sm_scale = 1.0
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_OK      # a batch of none
    a.batch, a.tokens, a.table_pages = 2, 1, 4000      # too long for the launch that needs no workspace
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_E_INVALID and b"NULL q" in L.kitty_last_error()
    a.q = a.out = a.block_table = a.lens = 4096
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_E_INVALID and b"workspace" in L.kitty_last_error()
    a.q_s_tok = 4
    assert rc("kitty_cache8_attention", cache(), a) == _hip.KITTY_E_INVALID and b"multiples of 8" in L.kitty_last_error()
    need = ctypes.c_size_t(0)
    assert L.kitty_cache8_attention_workspace_size(ctypes.byref(cache()), ctypes.byref(a), ctypes.byref(need)) == _hip.KITTY_OK
    assert need.value > 0
    a.table_pages = (1 << 26) + 1
    assert L.kitty_cache8_attention(ctypes.byref(cache()), ctypes.byref(a), None) == _hip.KITTY_E_UNSUPPORTED
    a.table_pages, a.tokens = 4000, 1 << 28
    assert L.kitty_cache8_attention_workspace_size(ctypes.byref(cache()), ctypes.byref(a), ctypes.byref(need)) == _hip.KITTY_E_UNSUPPORTED


def test_packed_arguments_are_the_structures():
    """The packed bytes of a call hold the fields of the C structures in their places."""
    import ctypes
    from kitty import _hip
    from kitty.kernels import cache8
    for packed, cls in ((cache8._ROWS, _hip.Cache8RowsArgs), (cache8._ATTENTION, _hip.Cache8AttentionArgs)):
        values = list(range(3, 3 + len(cls._fields_)))
        assert packed.size == ctypes.sizeof(cls)
        got = cls.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, f[0]) for f in cls._fields_] == values
