"""The 8-bit paged cache in captured graphs, on several streams at once, in pools
beyond 4 GiB and in other memory orders."""
import numpy as np
import pytest
import torch

from cache8_ref import Ref, numpy, tolerance
from test_cache8 import filled, i32, tables

pytestmark = pytest.mark.gpu


def step(cache, q, k, v, table, start, lens, **kw):
    cache.write(k, v, table, start)
    return cache.attend(q, table, lens, **kw)


# a decode step of one launch, one whose work is shared by the lengths, a chunk in parts
@pytest.mark.parametrize("T,wide", [(1, 0), (1, 300), (3, 300), (70, 300)])
def test_captured_steps(dev, T, wide):
    """write, attend and read in a graph, replayed with other lengths, pages and tokens in
    the same tensors, other work and synchronisations between: every replay is the eager call."""
    gen = torch.Generator().manual_seed(T)
    B, Hq, H, D, G, W = 3, 4, 2, 128, 64, 6
    cache = filled(gen, 40, H, D, G, dev)
    twin = filled(torch.Generator().manual_seed(T), 40, H, D, G, dev)
    table = torch.zeros(B, W + wide, dtype=torch.int32, device=dev)
    start, lens = i32([0] * B, dev), i32([T] * B, dev)
    q, k, v = (torch.zeros(B, h, T, D, dtype=torch.float16, device=dev) for h in (Hq, H, H))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = step(cache, q, k, v, table, start, lens, return_lse=True)
        back = cache.read(table[:, :W], lens, 80, dtype=torch.bfloat16)
    for c, t in ((cache, twin),):       # what capture may have left
        for a, b in ((c.key, t.key), (c.value, t.value)):
            a.view(torch.uint8).copy_(b.view(torch.uint8))
        c.scale.copy_(t.scale)
    for i in range(4):
        table[:, :W] = tables(gen, B, W, 40, dev)
        start.copy_(torch.randint(0, 6 * G - T, (B,), generator=gen))
        lens.copy_(start + T)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        graph.replay()
        torch.randn(1 << 20, device=dev).sum().item()
        want, want_lse = step(twin, q, k, v, table, start, lens, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), i
        for a, b in zip(back, twin.read(table[:, :W], lens, 80, dtype=torch.bfloat16)):
            assert torch.equal(a, b), i
        for a, b in ((cache.key, twin.key), (cache.value, twin.value)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        assert torch.equal(cache.scale, twin.scale), i


def test_streams_and_graphs_at_once(dev):
    """Two captured graphs and two streams on one cache, overlapping: workspaces are each
    call's own, the results those of calls one after the other."""
    gen = torch.Generator().manual_seed(11)
    B, Hq, H, D, G = 4, 8, 2, 128, 32
    cache = filled(gen, 256, H, D, G, dev)
    table = torch.full((B, 400), -1, dtype=torch.int32, device=dev)
    table[:, :64] = tables(gen, B, 64, 256, dev)
    lens = [i32([2000, 37, 900, 1500], dev), i32([5, 2048, 0, 777], dev)]
    qs = [torch.randn(B, Hq, t, D, generator=gen).half().to(dev) for t in (1, 5)]
    want = [cache.attend(q, table, n) for q, n in zip(qs, lens)]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q, n, s in zip(qs, lens, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs.append(cache.attend(q, table, n))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.fill_(7)
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        eager = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[i] = cache.attend(qs[1 - i], table, lens[1 - i])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for i in range(2):
            assert torch.equal(outs[i], want[i]) and torch.equal(eager[i], want[1 - i])
    torch.cuda.synchronize()


def test_pools_beyond_4_gib(dev):
    """Pages whose byte offsets pass 2^32 in either pool, and scales past 2^16 pages."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(4)
    P, H, D, G = 70000, 4, 128, 128       # 4.6 GB a pool
    key, value = (torch.empty(P, H, G, D, dtype=torch.uint8, device=dev) for _ in range(2))
    cache = Cache8(key.view(torch.float8_e4m3fn), value.view(torch.float8_e4m3fn), torch.ones(P, H, 2, device=dev))
    table = i32([[P - 1, 3, P - 3], [P - 2, 65537, 66000]], dev)
    k, v = (torch.randn(2, H, 300, D, generator=gen).half() for _ in range(2))
    cache.write(k.to(dev), v.to(dev), table, i32([0, 7], dev))
    lens = [300, 307]
    q = torch.randn(2, 8, 4, D, generator=gen).half()
    small = Cache8.empty(6, H, D, G, device="cpu")
    near = i32([[0, 1, 2], [3, 4, 5]], "cpu")
    for i, p in enumerate(table.flatten().tolist()):       # the second sequence's first rows are the pool's own
        for a, b in ((cache.key, small.key), (cache.value, small.value)):
            codes = a.view(torch.uint8)[p].cpu()
            if p == P - 2:
                codes[:, :7] = 0x30
                a.view(torch.uint8)[p] = codes.to(dev)
            b.view(torch.uint8)[i] = codes
        small.scale[i] = cache.scale[p].cpu()
    ref = Ref(small)
    twin = Ref(Cache8.empty(6, H, D, G, device="cpu"))
    twin.write(numpy(k[:1]), numpy(v[:1]), near[:1].numpy(), [0])
    assert (twin.pools[0][:2] == ref.pools[0][:2]).all() and (twin.scale[:3] == ref.scale[:3]).all()
    got = cache.read(table, i32(lens, dev), 300, dtype=torch.float32)
    for g, w in zip(got, ref.read(near.numpy(), lens, 300)):
        np.testing.assert_array_equal(numpy(g), w)
    for t, extra in ((1, 0), (4, 0), (4, 60), (200, 0)):
        q = torch.randn(2, 8, t, D, generator=gen).half()
        wide = torch.cat([table, torch.zeros(2, extra, dtype=torch.int32, device=dev)], 1)
        want, _, spread, mag, sm = ref.attend(numpy(q), near.numpy(), lens)
        out = numpy(cache.attend(q.to(dev), wide, i32(lens, dev)))
        assert (np.abs(out - want) <= tolerance(q.dtype, want, spread, mag, sm, 2 * t, D, 307)).all()


@pytest.mark.parametrize("T,wide", [(1, 0), (1, 300), (6, 300), (80, 0)])
def test_pools_in_other_orders(dev, T, wide):
    """Pools with heads inside tokens and slices of larger ones: the same results."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(T)
    P, H, D, G = 20, 2, 80, 32
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
    table = torch.cat([tables(gen, 2, 9, P, dev), torch.full((2, wide), -1, dtype=torch.int32, device=dev)], 1)
    lens = i32([250, 77], dev)
    q, k, v = (torch.randn(2, h, T, D, generator=gen).bfloat16().to(dev) for h in (6, 2, 2))
    for c in (plain, cache):
        c.write(k, v, table, lens - T if T < 77 else i32([170, 0], dev))
    lens = i32([250, 80 if T == 80 else 77], dev)
    assert torch.equal(cache.attend(q, table, lens), plain.attend(q, table, lens))
    for a, b in zip(cache.read(table, lens, 200), plain.read(table, lens, 200)):
        assert torch.equal(a, b)
    for a, b in ((cache.key, plain.key), (cache.value, plain.value)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(cache.scale, plain.scale)


def test_repeated_calls_are_equal(dev):
    """No order of arrival enters a result."""
    gen = torch.Generator().manual_seed(1)
    cache = filled(gen, 300, 4, 128, 64, dev)
    table = tables(gen, 8, 32, 300, dev)
    lens = i32([2000, 1, 700, 64, 2048, 1999, 1024, 300], dev)
    for Hq, T in ((16, 1), (32, 5), (8, 130)):
        q = torch.randn(8, Hq, T, 128, generator=gen).bfloat16().to(dev)
        first = cache.attend(q, table, lens)
        for _ in range(5):
            assert torch.equal(cache.attend(q, table, lens), first)
