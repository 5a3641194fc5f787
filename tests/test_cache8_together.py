"""The 8-bit cache's shared prefixes, weighed attention and eviction as a program uses them
together, on the CPU path and on the GPU; captured, on several streams, on pools beyond
4 GiB and over long contexts on the GPU."""
import ctypes

import numpy as np
import pytest
import torch

import shared8_ref
from cache8_ref import Ref, numpy
from test_cache8 import BF16, DEVICES, F16, check_attend, filled, i32, tables
from test_evict8 import check_evict, evict_ref, heavy
from test_shared8 import check_shared, pools
from test_weighed8 import check_weighed


def _hip_lib():
    from kitty import _hip
    return _hip


def _hip_cache(H, D, G):
    return _hip_lib().Cache8(4096, 8192, 16384, H * G * D, G * D, D, H * G * D, G * D, D, 2 * H, 2, 4, H, D, G)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_samples_of_one_prompt(dev, dtype):
    """A prompt written once, three samples decoded behind it, each in pages of its own: every
    step's attention is that over the prompt and the sample in one."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(21)
    B, Hq, H, D, G = 3, 4, 2, 64, 16
    cache = Cache8.empty(20, H, D, G, device=dev)
    ptable, table = i32([[3, 17, 5, 9]], dev), i32([[0, 1], [10, 11], [19, 4]], dev)
    k, v = (torch.randn(2, 1, H, 50, D, generator=gen).to(dtype))
    cache.write(k.to(dev), v.to(dev), ptable, i32([0], dev))
    for step in range(18):                       # past the end of the first page
        k, v = (torch.randn(2, B, H, 1, D, generator=gen).to(dtype))
        cache.write(k.to(dev), v.to(dev), table, i32([step] * B, dev))
        q = torch.randn(B, Hq, 1, D, generator=gen).to(dtype)
        if step % 5 == 2:
            check_shared(cache, q, ptable, [50], table, [step + 1] * B)
    q = torch.randn(B, Hq, 4, D, generator=gen).to(dtype)      # the last four at once, as drafts are checked
    check_shared(cache, q, ptable, [50], table, [18, 18, 18], q_lens=[4, 2, 3])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_chat_within_a_budget(dev, dtype):
    """Prompts weighed by their last queries and cut down, then steps that weigh what they
    attend to and cut down again: pools, lengths, positions, weights and outputs as the
    definitions have them, evictions in place and into other pages in turn."""
    gen = torch.Generator().manual_seed(22)
    B, Hq, H, D, G, W, budget = 2, 6, 2, 64, 16, 10, 60
    cache = filled(gen, 45, H, D, G, dev)
    spare = [tables(gen, B, W, 22, dev), 22 + tables(gen, B, W, 22, dev)]
    table = spare[0]
    prompt = [130, 77]
    k, v = torch.randn(2, B, H, 130, D, generator=gen).to(dtype)
    cache.write(k.to(dev), v.to(dev), table, i32([0, 0], dev), i32(prompt, dev))
    weights = torch.zeros(B, H, W * G, device=dev)
    check_weighed(cache, torch.randn(B, Hq, 9, D, generator=gen).to(dtype), table, prompt, weights=weights)
    lens = prompt
    for turn in range(4):
        into = (spare[1 - turn // 2 % 2] if turn % 2 == 1 else None)
        got = check_evict(cache, table, lens, weights, budget, 2, 16, into)
        lens, weights = got[0].tolist(), got[2]
        assert lens == [min(n, budget) for n in lens] and float(weights[:, :, budget:].abs().max()) == 0.0
        table = table if into is None else into
        for step in range(7):
            k, v = torch.randn(2, B, H, 1, D, generator=gen).to(dtype)
            cache.write(k.to(dev), v.to(dev), table, i32(lens, dev))
            lens = [n + 1 for n in lens]
            check_weighed(cache, torch.randn(B, Hq, 1, D, generator=gen).to(dtype), table, lens, weights=weights)
    check_attend(cache, torch.randn(B, Hq, 2, D, generator=gen).to(dtype), table, lens)


# ------------------------------------------------------- graphs, streams, devices

def everything(cache, x, q, q2):
    """All three calls; evict in place and into other pages."""
    shared, lse = cache.attend_shared(q, x["ptable"], x["plens"], x["table"], x["lens"], q_lens=x["q_lens"], return_lse=True)
    weighed = cache.attend_weighed(q2, x["table"], x["lens"], x["weights"], q_lens=x["q_lens2"])
    moved = cache.evict(x["table"], x["lens"], x["weights"], 150, 4, 16, x["into"])
    cut = cache.evict(x["table"], x["lens"], x["weights"], 97, 3, 8)
    after = cache.attend(q2[:, :, :1], x["table"], cut[0])
    return [shared, lse, weighed, x["weights"], *moved, *cut, after]


def refill(x, gen, B, W, G, T, T2, P):
    order = torch.randperm(P, generator=gen).to(torch.int32)
    x["ptable"].copy_(order[:2 * W].view(2, W))
    x["table"].copy_(order[2 * W:2 * W + B * W].view(B, W))
    x["into"].copy_(order[2 * W + B * W:2 * W + 2 * B * W].view(B, W))
    x["plens"].copy_(torch.randint(0, W * G + 1, (2,), generator=gen))
    x["lens"].copy_(torch.randint(0, W * G + 1, (B,), generator=gen))
    x["q_lens"].copy_(torch.randint(0, T + 1, (B,), generator=gen))
    x["q_lens2"].copy_(torch.randint(0, T2 + 1, (B,), generator=gen))
    x["weights"].copy_(heavy(gen, *x["weights"].shape))


def tensors(dev, B, H, W, G):
    zeros = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(ptable=zeros(2, W), table=zeros(B, W), into=zeros(B, W), plens=zeros(2), lens=zeros(B), q_lens=zeros(B),
                q_lens2=zeros(B), weights=torch.zeros(B, H, W * G, device=dev))


def copy_pools(a, b):
    for x, y in ((a.key, b.key), (a.value, b.value)):
        x.view(torch.uint8).copy_(y.view(torch.uint8))
    a.scale.copy_(b.scale)


# queries of attend_shared and attend_weighed: each of the shared ways, weights from scores (whole contexts in
# one launch, split), from tiles in one part and several
@pytest.mark.gpu
@pytest.mark.parametrize("T,T2,Hq,W", [(1, 1, 4, 20), (40, 30, 4, 20), (8, 8, 4, 20), (3, 2, 4, 100), (5, 1, 16, 140), (12, 200, 4, 60), (1, 700, 2, 20)])
def test_captured(dev, T, T2, Hq, W):
    """In a graph, replayed with other lengths, pages, queries and weights in the same tensors,
    other work and synchronisations between: every replay is the eager call."""
    gen = torch.Generator().manual_seed(T + T2)
    B, H, D, G = 4, 2, 64, 16
    P = 2 * W + 2 * B * W + 1
    cache, twin, clean = (filled(torch.Generator().manual_seed(5), P, H, D, G, dev) for _ in range(3))
    x, y = tensors(dev, B, H, W, G), tensors(dev, B, H, W, G)
    q, q2 = (torch.zeros(B, Hq, t, D, dtype=F16, device=dev) for t in (T, T2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = everything(cache, x, q, q2)
    for i in range(4):
        refill(x, gen, B, W, G, T, T2, P)
        for t in (q, q2):
            t.copy_(torch.randn(t.shape, generator=gen))
        for k in x:
            y[k].copy_(x[k])
        copy_pools(cache, clean)
        copy_pools(twin, clean)
        graph.replay()
        torch.randn(1 << 20, device=dev).sum().item()
        for n, (a, b) in enumerate(zip(outs, everything(twin, y, q, q2))):
            assert torch.equal(a, b), (i, n)
        for a, b in ((cache.key, twin.key), (cache.value, twin.value)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        assert torch.equal(cache.scale, twin.scale), i


@pytest.mark.gpu
def test_streams_and_graphs_at_once(dev):
    """Two graphs and two streams that overlap, on caches of their own for what they write and
    one for what they read: workspaces are each call's own, results those of calls one after the other."""
    gen = torch.Generator().manual_seed(31)
    B, H, D, G, W = 4, 2, 64, 16, 60
    P = 2 * W + 2 * B * W + 1
    clean = filled(torch.Generator().manual_seed(6), P, H, D, G, dev)
    caches = [filled(torch.Generator().manual_seed(6), P, H, D, G, dev) for _ in range(4)]
    shapes = [(1, 1), (20, 150), (1, 1), (20, 150)]
    xs, qs = [tensors(dev, B, H, W, G) for _ in range(4)], []
    for x, (T, T2) in zip(xs, shapes):
        refill(x, gen, B, W, G, T, T2, P)
        qs.append([torch.randn(B, 8, t, D, generator=gen).half().to(dev) for t in (T, T2)])
    held = [x["weights"].clone() for x in xs]

    def reset():
        for c, x, w in zip(caches, xs, held):
            copy_pools(c, clean)
            x["weights"].copy_(w)

    want = []
    for c, x, q in zip(caches, xs, qs):
        want.append([t.clone() for t in everything(c, x, *q)])
    reset()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], [None] * 4
    for i in range(2):
        streams[0].wait_stream(torch.cuda.current_stream())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[0]):
            outs[i] = everything(caches[i], xs[i], *qs[i])
    for _ in range(6):
        reset()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                outs[2 + i] = everything(caches[2 + i], xs[2 + i], *qs[2 + i])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for got, w in zip(outs, want):
            for n, (a, b) in enumerate(zip(got, w)):
                assert torch.equal(a, b), n
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_repeated_calls_are_equal(dev):
    gen = torch.Generator().manual_seed(33)
    cache, ptable, table = pools(gen, 2, 8, 200, 60, 2, 128, 16, dev)
    args = ptable, i32([3100, 777], dev), table, i32([5, 900, 0, 333, 960, 1, 77, 500], dev)
    for T in (1, 6, 40, 90):
        q = torch.randn(8, 8, T, 128, generator=gen).half().to(dev)
        first = cache.attend_shared(q, *args)
        w = torch.zeros(8, 2, 960, device=dev)
        out = cache.attend_weighed(q, *args[2:], w)
        for _ in range(4):
            torch.randn(1 << 18, device=dev).sum()
            assert torch.equal(cache.attend_shared(q, *args), first)
            again = torch.zeros_like(w)
            assert torch.equal(cache.attend_weighed(q, *args[2:], again), out) and torch.equal(again, w)


@pytest.mark.gpu
def test_pools_beyond_4_gib(dev):
    """Pages whose byte offsets pass 2^32 in either pool, and scales past 2^16 pages, against
    the same pages at the front of a small one."""
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(4)
    P, H, D, G = 70000, 4, 128, 128       # 4.6 GB a pool
    key, value = (torch.zeros(P, H, G, D, dtype=torch.uint8, device=dev) for _ in range(2))
    cache = Cache8(key.view(torch.float8_e4m3fn), value.view(torch.float8_e4m3fn), torch.ones(P, H, 2, device=dev))
    far = [P - 1, 3, P - 3, P - 2, 65537, 66000, 69000, 1, 68001, 68000]
    small = filled(gen, len(far), H, D, G, dev)
    for a, b in ((cache.key, small.key), (cache.value, small.value), (cache.scale, small.scale)):
        a.view(torch.uint8)[far] = b.view(torch.uint8)
    at = lambda rows: i32([[far[i] for i in r] for r in rows], dev)  # noqa: E731
    prefix, own, into = [[0, 1, 2]], [[3, 4], [5, 6]], [[7], [9]]
    lens = i32([200, 256], dev)
    for T in (1, 9, 40):
        q = torch.randn(2, 8, T, D, generator=gen).half().to(dev)
        got = cache.attend_shared(q, at(prefix), i32([333], dev), at(own), lens)
        assert torch.equal(got, small.attend_shared(q, i32(prefix, dev), i32([333], dev), i32(own, dev), lens))
        w, v = torch.ones(2, 2, H, 256, device=dev)
        got = cache.attend_weighed(q, at(own), lens, w)
        assert torch.equal(got, small.attend_weighed(q, i32(own, dev), lens, v)) and torch.equal(w, v)
    for to in (into, None):
        got = cache.evict(at(own), lens, w, 120, 4, 16, None if to is None else at(to))
        want = small.evict(i32(own, dev), lens, w, 120, 4, 16, None if to is None else i32(to, dev))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in ((cache.key, small.key), (cache.value, small.value), (cache.scale, small.scale)):
            assert torch.equal(a.view(torch.uint8)[far], b.view(torch.uint8))


def exact64(cache, q, ids, n, causal=True):
    """float64 attention on the GPU over the n tokens of the pages `ids`, in one table: (out, softmax @ |v|,
    weights by KV head)."""
    H = cache.num_kv_heads
    kv = []
    for i, pool in enumerate((cache.key, cache.value)):
        x = pool.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * cache.scale[ids][..., i, None, None].double()
        kv.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
    Hq, T, D = q.shape
    s = (q.double().view(H, -1, D) @ kv[0].transpose(1, 2)).view(H, Hq // H, T, n) * D ** -0.5
    if causal:
        s = s.masked_fill(torch.arange(n, device=q.device) > torch.arange(n - T, n, device=q.device)[:, None], -float("inf"))
    p = torch.softmax(s, -1)
    flat = p.view(H, -1, n)
    return (flat @ kv[1]).view(Hq, T, D), (flat @ kv[1].abs()).view(Hq, T, D), p.sum((1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("T,per", [(1, 3), (3, 2), (40, 2)])
def test_long_contexts(dev, T, per):
    """A prefix of 150,000 tokens, and weights of as many; tolerances as cache8_ref's, with the weights' bound
    (mag, the sum of |q k|, is below 12 * 64 channels' root sums here: scores up to 40, 2 * 70 * 2^-24 * 400)."""
    gen = torch.Generator().manual_seed(T)
    n, Hq, H, D, G = 150000, 4, 2, 64, 64
    W = -(-n // G)
    cache = filled(gen, W + per * 2, H, D, G, dev)
    cache.scale.mul_(0.25)
    order = torch.randperm(W + per * 2, generator=gen).to(dev)
    ptable, table = order[:W].view(1, W).int(), order[W:].view(per, 2).int()
    q = torch.randn(per, Hq, T, D, generator=gen).half().to(dev)
    own = [64 + 13 * b for b in range(per)]
    out = cache.attend_shared(q, ptable, i32([W * G], dev), table, i32(own, dev))
    weights = torch.zeros(1, H, W * G, device=dev)
    out1 = cache.attend_weighed(q[:1], ptable, i32([n], dev), weights)
    mag = 0.0
    for b in range(per):
        ids = torch.cat([ptable[0], table[b]]).long()
        want, spread, _ = exact64(cache, q[b], ids, W * G + own[b])
        mag = max(mag, float((q[b].abs().double().sum(-1) * 448 * cache.scale[..., 0].max() * D ** -0.5).max()))
        tol = 2.0 ** -11 * want.abs() + (2 * (D + 6) * 2.0 ** -24 * mag + 2 * n * 2.0 ** -24 + 2.0 ** -15) * spread + 2.0 ** -24
        assert ((out[b].double() - want).abs() <= tol).all()
    want, spread, w = exact64(cache, q[0], ptable[0].long(), n)
    tol = 2.0 ** -11 * want.abs() + (2 * (D + 6) * 2.0 ** -24 * mag + 2 * n * 2.0 ** -24 + 2.0 ** -15) * spread + 2.0 ** -24
    assert ((out1[0].double() - want).abs() <= tol).all()
    rel = 2 * (D + 6) * 2.0 ** -24 * mag + n * 2.0 ** -24 + 2.0 ** -18 + Hq * T * 2.0 ** -24
    assert ((weights[0, :, :n].double() - w).abs() <= rel * w + 1e-30).all() and (weights[0, :, n:] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n,keep", [(9000, 4000), (33000, 17000), (40000, 39000), (70000, 1)])
def test_long_evictions(dev, n, keep):
    """As many weights as a lane holds in registers and more than that, against a sort."""
    gen = torch.Generator().manual_seed(n)
    G, W = 256, -(-n // 256)
    cache = filled(gen, W, 1, 16, G, dev)
    table, w = tables(gen, 1, W, W, dev), heavy(gen, 1, 1, W * G).to(dev)
    first, last = min(5, keep // 2), min(100, keep // 2)
    before, _ = cache.read(table, i32([n], dev), n, dtype=torch.float32)
    lens, kept, out = cache.evict(table, i32([n], dev), w, keep, first, last)
    x = w[0, 0, :n].cpu().numpy()
    order = np.argsort(-x[first:n - last], kind="stable")[:keep - first - last] + first
    want = np.sort(np.concatenate([np.arange(first), order, np.arange(n - last, n)]))
    assert lens.tolist() == [keep] and (kept[0, 0].cpu().numpy() == want).all()
    assert (out[0, 0, :keep].cpu().numpy() == x[want]).all() and float(out[0, 0, keep:].abs().max()) == 0.0
    got, _ = cache.read(table, lens, keep, dtype=torch.float32)
    moved = before[0, 0, torch.from_numpy(want).to(dev)]
    # a code rounds again only where its scale was smaller than its new page's: half a step of e4m3, or half of
    # its smallest subnormal 2^-9 at the largest scale
    assert ((got[0, 0] - moved).abs() <= 2.0 ** -4 * moved.abs() + 2.0 ** -10 * cache.scale[..., 0].max()).all()


# ----------------------------------------------------------------- which kernels

def shared_way(B, F, Hq, H, T, D, G, Wp, W, plan=256):
    """How attend_shared's rule (csrc/attend8_shared.hip, restated) takes a call; the library's workspace has to
    be that way's."""
    from kitty import _hip
    up = lambda n: -(-n // 16) * 16  # noqa: E731
    own, DP = Hq // H * T, 64 if D <= 64 else 128 if D <= 128 else 256
    prefix = own * (B // F)
    rows, both = own <= 32, prefix <= 64 and own <= 32
    whole = rows and D <= 128 and (Wp + W) * G * DP <= 1280 * 128 and B * H <= plan
    RT = 0 if not rows else 1 if (prefix if both else own) <= 16 else 2
    RM = 16 * RT if rows else 128
    nrb = -(-prefix // (RM if both else 128))
    items, own_items = F * H * nrb, B * H * (1 if rows else -(-own // 128))
    units = lambda n, cap, unit: n * (2 + -(-cap // unit))  # noqa: E731
    tile, mine = units(items, Wp * G, 64), units(own_items, W * G, 128 if rows else 64)
    if both:
        WG = min(plan * (2 if DP <= 128 else 1), units(items, Wp * G, 128) + mine)
    else:
        WG = max(min(plan * (2 if DP <= 128 else 1), tile + mine + 16) // 8 * 8, 16)
    area = lambda slots, rm, n: up(slots * rm * DP * 4) + up(slots * rm * 8) + up(n * 8)  # noqa: E731
    if both or not rows:
        size = area(2 * WG + items + own_items, RM if both else 128, items + own_items)
    else:
        size = area(2 * WG + items, 128, items) + area(2 * WG + own_items, RM, own_items)
    if not both:
        size += up((B * T + B + F) * 4)
    if whole:
        size = 0
    c = _hip.Cache8(4096, 8192, 16384, H * G * D, G * D, D, H * G * D, G * D, D, 2 * H, 2, 4, H, D, G)
    a = _hip.Cache8SharedArgs()
    a.prefixes, a.batch, a.num_q_heads, a.tokens, a.prefix_pages, a.table_pages, a.sm_scale = F, B, Hq, T, Wp, W, 1.0
    got = ctypes.c_size_t(0)
    L = _hip.load()
    assert L.kitty_cache8_shared_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(got)) == _hip.KITTY_OK
    assert got.value == size, (got.value, size)
    return "whole" if whole else "rows" if both else "tiles and rows" if rows else "tiles"


def test_every_way_is_tested():
    """The shapes of test_shared8 reach each way at every padded head size, and both sides of the rule's borders hold."""
    from test_shared8 import SHAPES, WAYS
    met = set()
    for F, each, Hq, H, T, D, G, plens, lens in SHAPES:
        W = [max(1, -(-max(n) // G)) for n in (plens, lens)]
        for wide in (0, 4096 // G):
            met.add((shared_way(F * each, F, Hq, H, T, D, G, W[0] + wide, W[1] + wide), 64 if D <= 64 else 128 if D <= 128 else 256))
    assert met == {(w, d) for w in ("whole", "rows", "tiles and rows", "tiles") for d in (64, 128, 256)} - {("whole", 256)}
    ways = ["whole", "whole", "rows", "tiles and rows", "tiles"]
    assert [shared_way(2 * e, 2, Hq, H, T, 64, 16, 8, 9 + wide) for e, Hq, H, T, wide in WAYS] == ways
    assert shared_way(16, 1, 4, 1, 1, 128, 16, 40, 41) == "rows" and shared_way(17, 1, 4, 1, 1, 128, 16, 40, 41) == "tiles and rows"
    assert shared_way(16, 1, 4, 1, 1, 128, 16, 40, 40) == "whole" and shared_way(1, 1, 32, 1, 1, 128, 16, 40, 40) == "whole"
    assert shared_way(1, 1, 33, 1, 1, 128, 16, 8, 8) == "tiles" and shared_way(1, 1, 32, 1, 1, 128, 16, 40, 41) == "rows"
    assert shared_way(600, 300, 4, 2, 2, 256, 16, 99, 99) == "rows" and shared_way(129, 1, 2, 2, 1, 64, 16, 8, 8) == "tiles and rows"


def test_a_sequence_and_its_prefix_are_limited_together():
    """Tables of 2^30 tokens between them pass, a page more is refused: places of rows are ints."""
    L = _hip_lib()
    c = _hip_cache(1, 16, 16)
    for pages, rc in (((1 << 26, 0), 0), ((1 << 25, 1 << 25), 0), ((0, 1 << 26), 0), ((1 << 25, (1 << 25) + 1), 2), ((1 << 26, 1), 2)):
        a = L.Cache8SharedArgs()
        a.prefixes = a.batch = a.num_q_heads = a.tokens = 1
        a.prefix_pages, a.table_pages, a.sm_scale = *pages, 1.0
        got = L.load().kitty_cache8_shared_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(ctypes.c_size_t(0)))
        assert got == (L.KITTY_E_UNSUPPORTED if rc else L.KITTY_OK), pages


def test_sums_of_parts_stay_within_a_gibibyte():
    """Many rows over a long table whose sequences are said to be short: parts, but not at any size."""
    L = _hip_lib()
    c = _hip_cache(8, 128, 128)
    sizes = []
    for plan, N in ((1, 1 << 30), (1, 1 << 20), (0, 1 << 30)):
        a = L.Cache8AttentionArgs()
        a.batch, a.num_q_heads, a.tokens, a.table_pages, a.sm_scale, a.plan_tokens = 1, 32, 8192, 1 << 17, 1.0, plan
        w = L.Cache8Weights(4096, 8 * N, N, N)
        size, plain = ctypes.c_size_t(0), ctypes.c_size_t(0)
        assert L.load().kitty_cache8_weighed_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(w), ctypes.byref(size)) == 0
        assert L.load().kitty_cache8_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(plain)) == 0
        sizes.append(size.value - plain.value)
    assert all(0 < s < 1.25 * 2 ** 30 for s in sizes) and sizes[1] > 2 ** 29, sizes


def test_merge_and_weights_are_one_grid():
    """Of more than half of a grid's pairs the scores are not kept: their launch would hold the merge as well."""
    L = _hip_lib()
    c = _hip_cache(1, 16, 16)
    kept = []
    for B in (0xffffffff // 512, 0xffffffff // 512 + 1):
        a = L.Cache8AttentionArgs()
        a.batch, a.num_q_heads, a.tokens, a.table_pages, a.sm_scale = B, 1, 1, 1, 1.0
        size = ctypes.c_size_t(0)
        w = L.Cache8Weights(4096, 16, 16, 16)
        assert L.load().kitty_cache8_weighed_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(w), ctypes.byref(size)) == 0
        kept.append(size.value > B * 16 * 4)
    assert kept == [True, False]


def test_references_agree():
    """shared8_ref on an aligned prefix is cache8_ref on the joined table; evict_ref's zeros and NaN are torch.sort's."""
    gen = torch.Generator().manual_seed(1)
    cache, ptable, table = pools(gen, 1, 2, 2, 2, 2, 16, 16, "cpu")
    q = numpy(torch.randn(2, 4, 3, 16, generator=gen))
    a = shared8_ref.attend_shared(cache, q, ptable.numpy(), [32], table.numpy(), [20, 5])
    b = Ref(cache).attend(q, np.concatenate([ptable.numpy().repeat(2, 0), table.numpy()], 1), [52, 37])
    for x, y in zip(a, b):
        np.testing.assert_allclose(x, y, rtol=1e-12, atol=0)
    w = torch.tensor([0.0, -0.0, float("nan"), 1.0, -1.0, float("inf"), -0.0]).expand(2, 2, 7)
    got = evict_ref(Ref(cache), table.numpy(), [7, 7], w.numpy(), 4, 0, 0, table.numpy())
    want = w[0, 0].sort(descending=True, stable=True).indices[:4].sort().values
    assert (got[1][0, 0] == want.numpy()).all()
