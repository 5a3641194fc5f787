"""Attention over the 8-bit cache for sequences that share prefixes
(Cache8.attend_shared) against float64, on the CPU path and on the GPU, and its refusals."""
import ctypes
import math

import numpy as np
import pytest
import torch

import shared8_ref
from cache8_ref import numpy, tolerance
from test_cache8 import BF16, DEVICES, F16, filled, i32


def check_shared(cache, q, ptable, plens, table, lens, q_lens=None, causal=True, sm_scale=None, infinite=False, **kw):
    """infinite: of rows with infinite scores the log-sum-exp (-inf of no finite one, and +inf or NaN) is not looked at."""
    dev, F = cache.device, len(plens)
    out, lse = cache.attend_shared(q.to(dev), ptable, i32(plens, dev), table, i32(lens, dev),
                                   q_lens=None if q_lens is None else i32(q_lens, dev), causal=causal, sm_scale=sm_scale,
                                   return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape
    want, wlse, spread, mag, small = shared8_ref.attend_shared(cache, numpy(q), ptable.cpu().numpy(), plens,
                                                               table.cpu().numpy(), lens, q_lens, causal, sm_scale)
    # joining parts multiplies by powers of two that exp2 gives, off by 2^-23 each, two a part at most: within
    # the 2^-20 that the tolerance has for exp2.  A prefix's rows are those of all its sequences.
    rows = q.shape[1] // cache.num_kv_heads * q.shape[2] * (q.shape[0] // F)
    n = max(max(plens), 0) + max(max(lens), 0)
    tol = tolerance(q.dtype, want, spread, mag, small, rows, q.shape[3], max(n, 1))
    got, glse = numpy(out), numpy(lse)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > tol
    assert not bad.any(), (float(np.nanmax(np.abs(got - want) - tol)), np.argwhere(bad)[:4])
    if not infinite:
        np.testing.assert_array_equal(np.isnan(glse), np.isnan(wlse))
    seen = np.isfinite(wlse)
    assert (glse[np.isneginf(wlse)] == -np.inf).all()
    room = (q.shape[3] + 8) * 2.0 ** -24 * mag[seen] + 2.0 ** -21 * (1 + np.abs(wlse[seen])) + n * 2.0 ** -24
    assert (np.abs(glse[seen] - wlse[seen]) <= room).all()
    return out


def pools(gen, F, B, Wp, W, H, D, G, dev, spare=1, wide=0):
    """A filled cache, tables of prefixes and sequences with pages of their own; page 0 is no one's.  wide: columns of
    the sequences' table that name no pages (its width says whether a call is one launch)."""
    P = F * Wp + B * W + spare
    cache = filled(gen, P, H, D, G, dev)
    cache.scale[::3] *= 1.61                     # not only powers of two
    ids = (1 + torch.randperm(P - 1, generator=gen)).to(torch.int32)
    own = torch.cat([ids[F * Wp:F * Wp + B * W].view(B, W), torch.full((B, wide), 1 << 30, dtype=torch.int32)], 1)
    return cache, ids[:F * Wp].view(F, Wp).to(dev), own.to(dev)


# prefixes and sequences: (prefixes, sequences of each, query heads, KV heads, queries, head size, page, prefix lengths, own lengths)
SHAPES = [
    # both in one launch of the row kernel: blocks of 16 to 64 rows, empty prefixes and sequences
    (1, 1, 1, 1, 1, 16, 16, [1], [0]), (1, 4, 8, 8, 1, 128, 128, [1000], [1, 40, 13, 0]), (2, 3, 4, 1, 1, 64, 16, [130, 0], [5, 0, 300, 1, 2, 0]),
    (3, 2, 4, 2, 3, 80, 32, [33, 64, 500], [3, 70, 2, 1, 40, 3]), (1, 11, 4, 1, 1, 128, 64, [777], [9 * b for b in range(11)]),
    (1, 16, 4, 1, 1, 128, 16, [300], [b % 3 for b in range(16)]), (1, 2, 16, 1, 1, 256, 32, [200], [0, 37]), (70, 1, 2, 1, 1, 32, 16, [(7 * f) % 90 for f in range(70)], [f % 40 for f in range(70)]),
    # more entries than workgroups: runs that hold several whole ones
    (200, 1, 16, 8, 1, 16, 16, [(5 * f) % 23 for f in range(200)], [f % 19 for f in range(200)]), (2, 150, 16, 8, 1, 16, 16, [70, 3], [(3 * b) % 40 for b in range(300)]),
    # the prefix in tiles, the sequences' own by rows
    (1, 17, 4, 1, 1, 128, 64, [700], [(31 * b) % 150 for b in range(17)]), (2, 40, 3, 1, 1, 64, 16, [150, 401], [b % 50 for b in range(80)]),
    (1, 9, 4, 1, 1, 256, 128, [600], [10] * 9), (1, 17, 4, 1, 1, 256, 128, [600], [10 + b for b in range(17)]), (1, 13, 5, 1, 3, 96, 32, [257], [3 + b for b in range(13)]), (3, 20, 4, 1, 1, 16, 256, [300, 0, 63], [b for b in range(60)]),
    (1, 3, 60, 1, 1, 128, 64, [1], [0, 0, 1]),
    # both in tiles
    (1, 2, 4, 2, 40, 64, 16, [300], [40, 55]), (2, 2, 3, 1, 43, 128, 32, [65, 500], [43, 43, 100, 50]), (1, 3, 2, 1, 33, 256, 16, [129], [33, 40, 200]),
    (1, 2, 4, 1, 100, 192, 64, [90], [100, 130])]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("F,each,Hq,H,T,D,G,plens,lens", SHAPES)
def test_matches_float64(dev, dtype, causal, F, each, Hq, H, T, D, G, plens, lens):
    gen = torch.Generator().manual_seed(F * 100 + each * 10 + T + D)
    Wp, W = (max(1, -(-max(n) // G)) for n in (plens, lens))
    cache, ptable, table = pools(gen, F, F * each, Wp, W, H, D, G, dev)
    q = torch.randn(F * each, Hq, T, D, generator=gen).to(dtype)
    check_shared(cache, q, ptable, plens, table, lens, causal=causal)
    # tables that could hold far more: never whole sequences in one launch
    wide = [torch.cat([t, torch.full((t.shape[0], 4096 // G), 1 << 30, dtype=torch.int32, device=dev)], 1) for t in (ptable, table)]
    check_shared(cache, q, wide[0], plens, wide[1], lens, causal=causal)


# (sequences of each, query heads, KV heads, queries, wide): whole sequences of 16 rows and of 32, rows, tiles and
# rows, tiles
WAYS = [(2, 4, 2, 6, 0), (5, 4, 2, 16, 0), (2, 4, 2, 6, 300), (5, 4, 2, 16, 300), (2, 4, 2, 70, 0)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("each,Hq,H,T,wide", WAYS)
def test_padded_rows_and_rows_in_the_prefix(dev, dtype, causal, each, Hq, H, T, wide):
    """Padded queries, sequences without queries or without tokens, queries that are tokens
    of the prefix themselves, and more of them than both hold."""
    gen = torch.Generator().manual_seed(T)
    cache, ptable, table = pools(gen, 3, 3 * each, 5, 9, H, 64, 16, dev, wide=wide)
    q = torch.randn(3 * each, Hq, T, 64, generator=gen).to(dtype)
    lens = [(0, 130, 2, T, 1, 140)[b % 6] for b in range(3 * each)]
    q_lens = [(T, 1, T // 2, 0, T, T - 1, 3)[b % 7] for b in range(3 * each)]
    for b, n in enumerate(q_lens):               # padding may hold anything
        q[b, :, n:] = (math.nan, math.inf, 0.0)[b % 3]
    out = check_shared(cache, q, ptable, [77, 3, 0], table, lens, q_lens=q_lens, causal=causal)
    for b, n in enumerate(q_lens):
        assert (out[b, :, n:] == 0).all()
    check_shared(cache, q.nan_to_num(0.5, 0.5), ptable, [80, 3, 1], table, lens, causal=causal)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("each,Hq,H,T,wide", WAYS)
def test_masked_and_missing_places(dev, dtype, each, Hq, H, T, wide):
    """NaN codes behind the last tokens, NaN keys and values that some rows see, missing
    pages of the prefix and of one sequence: they reach the rows that see them alone."""
    gen = torch.Generator().manual_seed(T + 1)
    B, G = 2 * each, 16
    cache, ptable, table = pools(gen, 2, B, 8, 9, H, 128, G, dev, wide=wide)
    q = torch.randn(B, Hq, T, 128, generator=gen).to(dtype)
    plens, lens = [100, 97], [(75, 0, 3, 130, 16, 1)[b % 6] for b in range(B)]
    q_lens = [(T, 2, T - 1)[b % 3] for b in range(B)]

    def check():
        check_shared(cache, q, ptable, plens, table, lens, q_lens=q_lens)
        check_shared(cache, q, ptable, plens, table, lens, q_lens=q_lens, causal=False)

    for pool in (cache.key, cache.value):
        pool = pool.view(torch.uint8)
        pool[int(ptable[0, 6]), :, 100 % G:] = 0x7F
        pool[int(ptable[1, 6]), :, 97 % G:] = 0xFF
        pool[int(ptable[1, 7])] = 0xFF
        for b in range(B):
            pool[int(table[b, lens[b] // G]), :, lens[b] % G:] = 0x7F
    check()
    cache.value.view(torch.uint8)[int(ptable[0, 6]), 0, 3, 9] = 0x7F        # the prefix's last token, which not every row sees
    cache.value.view(torch.uint8)[int(ptable[1, 0]), H - 1, 2, 127] = 0xFF  # one that all rows of real queries see
    check()
    cache.key.view(torch.uint8)[int(ptable[0, 6]), H - 1, 2, 0] = 0x7F
    check()
    ptable[1, 6] = -1                                                        # its last token has no page
    table[0, 1] = cache.num_pages
    check()
    cache.scale[0] = math.nan                                                # page 0's scales stand for no missing page
    check()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("each,Hq,H,T,wide", WAYS)
def test_broken_lengths(dev, each, Hq, H, T, wide):
    """Lengths that break the rules give NaN rows to their sequences alone: to all of a prefix, or to one."""
    gen = torch.Generator().manual_seed(T + 2)
    cache, ptable, table = pools(gen, 3, 3 * each, 3, 9, H, 64, 16, dev, wide=wide)
    q = torch.randn(3 * each, Hq, T, 64, generator=gen).half()
    lens = [100] * (3 * each)
    lens[1], lens[-1] = -1, (9 + wide) * 16 + 1
    check_shared(cache, q, ptable, [48, 49, 20], table, lens)
    check_shared(cache, q, ptable, [-1, 0, 1 << 30], table, lens)
    q_lens = [T] * (3 * each)
    q_lens[0], q_lens[-1] = T + 1, -1
    check_shared(cache, q, ptable, [40, 0, 20], table, lens, q_lens=q_lens)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("each,Hq,H,T,wide", WAYS)
def test_infinite_queries(dev, each, Hq, H, T, wide):
    """Infinite scores as the softmax has them, in the prefix's tokens and a sequence's own: NaN
    rows where one is +inf or none is finite, the others keep their numbers."""
    gen = torch.Generator().manual_seed(T + 5)
    B = 2 * each
    cache, ptable, table = pools(gen, 2, B, 6, 9, H, 64, 16, dev, wide=wide)
    cache.key.view(torch.uint8)[..., 7] = 0x38                               # 1.0
    cache.key.view(torch.uint8)[int(ptable[0, 1]), :, 3, 9] = 0x38           # and one token's -1.0 elsewhere
    cache.key.view(torch.uint8)[..., 9] = 0xB8
    cache.key.view(torch.uint8)[int(ptable[0, 1]), :, 3, 9] = 0x38
    q = torch.randn(B, Hq, T, 64, generator=gen).half()
    q[0, 0, :, 7] = math.inf                                                 # every score +inf
    q[1, 1, :, 7] = -math.inf                                                # every score -inf
    q[1, 0, 0, 9] = -math.inf                                                # all +inf but one
    q[0, 1, T // 2, 9] = math.inf                                            # one +inf in prefix 0, -inf elsewhere
    q[-1, 1, T // 2, 9] = math.inf                                           # -inf alone
    check_shared(cache, q, ptable, [90, 30], table, [T + b for b in range(B)], infinite=True)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("each,Hq,H,T,wide", WAYS)
def test_layouts(dev, each, Hq, H, T, wide):
    """Queries and outputs in other memory orders, unaligned, negated, one memory for both;
    pools of other strides; prefix and own pages the same; a scale of the program's own."""
    gen = torch.Generator().manual_seed(T + 3)
    D, B = 64, 2 * each
    cache, ptable, table = pools(gen, 2, B, 8, 9, H, D, 16, dev, wide=wide)
    q = torch.randn(B, Hq, T, D, generator=gen).half()
    lens = [T + b for b in range(B)]
    args = [ptable, i32([100, 128], dev), table, i32(lens, dev)]
    want = check_shared(cache, q, ptable, [100, 128], table, lens, sm_scale=0.2)
    q = q.to(dev)

    def same(x, **kw):
        got = cache.attend_shared(x, *args, sm_scale=0.2, **kw)
        assert torch.equal(got, want)
        return got

    same(q.transpose(1, 2).contiguous().transpose(1, 2))
    odd = torch.zeros(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)
    same(odd.copy_(q))
    same(q.transpose(2, 3).contiguous().transpose(2, 3))                     # channels not contiguous
    same(torch._neg_view(-q))
    for out in (torch.empty(B, T, Hq, D, dtype=F16, device=dev).transpose(1, 2), torch.zeros_like(odd), q.clone(),
                torch._neg_view(torch.zeros_like(q)), torch.zeros(q.numel() + 1, dtype=F16, device=dev)[1:].view(q.shape)):
        assert same(q, out=out) is out and torch.equal(out, want)
    x = q.clone()
    assert same(x, out=x) is x
    long = torch.zeros(B + 1, Hq, T, D, dtype=F16, device=dev)               # rows of out over other rows of q
    long[:B] = q
    assert torch.equal(cache.attend_shared(long[:B], *args, sm_scale=0.2, out=long[1:]), want)
    from kitty.kernels import Cache8
    turned = [t.view(torch.uint8).permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3) for t in (cache.key, cache.value)]
    other = Cache8(*(t.view(torch.float8_e4m3fn) for t in turned), cache.scale.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(other.attend_shared(q, *args, sm_scale=0.2), want)
    check_shared(cache, q.cpu(), ptable, [100, 128], ptable[:1].expand(B, -1), [min(T, 128)] * B)
    # one prefix of no pages at all, and a batch of none
    none = torch.zeros(1, 0, dtype=torch.int32, device=dev)
    check_shared(cache, q.cpu(), none, [0], table, lens)
    assert cache.attend_shared(q[:0], none, i32([0], dev), table[:0], i32([], dev)).shape == (0, Hq, T, D)
    assert cache.attend_shared(q[:, :, :0], *args).shape == (B, Hq, 0, D)


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_and_gradients(dev):
    gen = torch.Generator().manual_seed(9)
    cache, ptable, table = pools(gen, 1, 2, 4, 3, 2, 64, 16, dev)
    q = torch.randn(2, 4, 3, 64, generator=gen).half().to(dev)
    args = ptable, i32([60], dev), table, i32([5, 40], dev)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend_shared(q.clone().requires_grad_(), *args)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend_shared(q, *args, out=torch.zeros_like(q).requires_grad_())
    target = torch.zeros_like(q)
    for _ in range(2):
        x = torch.ones(q.shape, device=dev, requires_grad=True)
        y = (x * target).sum()
        cache.attend_shared(q, *args, out=target)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda x: cache.attend_shared(x, *args), (q,), check_trace=False)


def test_refusals():
    gen = torch.Generator().manual_seed(3)
    cache, ptable, table = pools(gen, 2, 4, 4, 3, 2, 64, 16, "cpu")
    q = torch.randn(4, 4, 1, 64, generator=gen).half()
    plens, lens = i32([60, 1], "cpu"), i32([5, 40, 1, 0], "cpu")
    cache.attend_shared(q, ptable, plens, table, lens)
    for bad in (lambda: cache.attend_shared(q[:3], ptable, plens, table[:3], lens[:3]),             # no multiple of two prefixes
                lambda: cache.attend_shared(q, ptable[:0], plens[:0], table, lens),
                lambda: cache.attend_shared(q, ptable[0], plens, table, lens),
                lambda: cache.attend_shared(q, ptable.long(), plens, table, lens),
                lambda: cache.attend_shared(q, ptable, plens.long(), table, lens),
                lambda: cache.attend_shared(q, ptable, plens[:1], table, lens),
                lambda: cache.attend_shared(q, ptable, plens, table, lens[:3]),
                lambda: cache.attend_shared(q, ptable, plens, table[:3], lens),
                lambda: cache.attend_shared(q, ptable, plens, table, lens, q_lens=lens[:2]),
                lambda: cache.attend_shared(q[:, :3], ptable, plens, table, lens),
                lambda: cache.attend_shared(q[..., :32], ptable, plens, table, lens),
                lambda: cache.attend_shared(q.float(), ptable, plens, table, lens),
                lambda: cache.attend_shared(q, ptable, plens, table, lens, sm_scale=0.0),
                lambda: cache.attend_shared(q, ptable, plens, table, lens, sm_scale=math.inf),
                lambda: cache.attend_shared(q, ptable, plens, table, lens, out=q.float()),
                lambda: cache.attend_shared(q, ptable, plens, table, lens, out=q[:, :1].expand(4, 4, 1, 64))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        cache.attend_shared(q.to("meta"), ptable, plens, table, lens)


def test_abi_refusals():
    """Each argument that the C entry cannot take is refused before anything is launched."""
    from kitty import _hip
    L = _hip.load()
    c = _hip.Cache8(4096, 8192, 16384, 1024, 1024, 64, 1024, 1024, 64, 4, 2, 4, 1, 64, 16)

    def call(fn=L.kitty_cache8_shared_attention, **kw):
        a = _hip.Cache8SharedArgs()
        a.q = a.out = a.prefix_table = a.prefix_lens = a.block_table = a.lens = a.workspace = 4096
        a.prefixes, a.batch, a.num_q_heads, a.tokens, a.prefix_pages, a.table_pages = 2, 4, 2, 1, 4, 400
        a.sm_scale, a.workspace_bytes = 1.0, 1 << 40
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(c), ctypes.byref(a), None)

    assert L.kitty_cache8_shared_attention(ctypes.byref(c), None, None) == _hip.KITTY_E_INVALID
    assert L.kitty_cache8_shared_attention(None, None, None) == _hip.KITTY_E_INVALID
    for kw in (dict(prefixes=0), dict(prefixes=-1), dict(prefixes=3), dict(batch=-1), dict(tokens=-1), dict(prefix_pages=-1),
               dict(table_pages=-1), dict(num_q_heads=0), dict(dtype=2),
               dict(sm_scale=0.0), dict(sm_scale=math.inf), dict(sm_scale=math.nan), dict(q=None), dict(out=None),
               dict(lens=None), dict(prefix_lens=None), dict(block_table=None), dict(prefix_table=None), dict(q=4098),
               dict(out=4104), dict(q_s_tok=4), dict(o_s_head=12), dict(workspace=None), dict(workspace=4100),
               dict(workspace_bytes=16)):
        assert call(**kw) == _hip.KITTY_E_INVALID, kw
    for kw in (dict(prefix_pages=1 << 27), dict(table_pages=1 << 27), dict(tokens=1 << 26), dict(batch=1 << 26)):
        assert call(**kw) == _hip.KITTY_E_UNSUPPORTED, kw
    assert call(batch=0) == _hip.KITTY_OK and call(tokens=0) == _hip.KITTY_OK
    size = ctypes.c_size_t(7)
    get = lambda cache, args, _: L.kitty_cache8_shared_attention_workspace_size(cache, args, ctypes.byref(size))  # noqa: E731
    assert call(get, batch=0) == _hip.KITTY_OK and size.value == 0
    assert call(get) == _hip.KITTY_OK and size.value > 0
    assert call(workspace_bytes=size.value - 1) == _hip.KITTY_E_INVALID
    assert call(get, table_pages=4) == _hip.KITTY_OK and size.value == 0       # one launch
    assert call(lambda cache, args, _: L.kitty_cache8_shared_attention_workspace_size(cache, args, None)) == _hip.KITTY_E_INVALID


def test_packed_arguments_are_the_structure():
    from kitty import _hip
    from kitty.kernels import cache8
    fields = [n for n, _ in _hip.Cache8SharedArgs._fields_]
    values = [float(i + 1) if n == "sm_scale" else i + 1 for i, n in enumerate(fields)]
    a = _hip.Cache8SharedArgs.from_buffer_copy(cache8._SHARED.pack(*values))
    assert cache8._SHARED.size == ctypes.sizeof(a)
    assert [getattr(a, n) for n in fields] == values
