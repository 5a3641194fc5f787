"""Which pages an eviction from the 8-bit cache writes (Cache8.evict), on the CPU path and on the GPU."""
import math

import numpy as np
import pytest
import torch

from cache8_ref import Ref
from test_cache8 import DEVICES, filled, i32, same_pools, tables
from test_evict8 import evict_ref, heavy


def held(cache):
    """Copies of the pools, as bits."""
    return cache.key.view(torch.uint8).clone(), cache.value.view(torch.uint8).clone(), cache.scale.view(torch.int32).clone()


def same(cache, before, pages=slice(None)):
    for a, b in zip(held(cache), before):
        assert torch.equal(a[pages], b[pages])


@pytest.mark.parametrize("dev", DEVICES)
def test_sequences_within_the_budget_keep_their_pages(dev):
    """In place nothing is written for them: what a page holds stays as it is, a scale that stands for
    no number too, and two of them may share pages.  Sequences beside them are cut."""
    gen = torch.Generator().manual_seed(8)
    B, H, D, G, W = 4, 2, 64, 16, 6
    cache = filled(gen, 30, H, D, G, dev)
    table, w = tables(gen, B, W, 30, dev), heavy(gen, B, H, W * G).to(dev)
    table[3, :2] = table[0, :2]
    strange = table[0, :3].long()
    cache.scale[strange[0]], cache.scale[strange[1], 1], cache.scale[strange[2], :, 1] = math.nan, -3.0, math.inf
    before, lens = held(cache), [40, 96, 0, 32]
    out_lens, kept, out = cache.evict(table, i32(lens, dev), w, 40, 4, 8)
    assert out_lens.tolist() == [40, 40, 0, 32]
    for b in (0, 3):
        n = lens[b]
        assert (kept[b, :, :n].cpu() == torch.arange(n)).all() and (kept[b, :, n:] == -1).all()
        assert torch.equal(out[b, :, :n], w[b, :, :n]) and (out[b, :, n:] == 0).all()
    cut = set(table[1, :3].tolist())
    same(cache, before, [p for p in range(30) if p not in cut])
    moved = cache.read(table[1:2], i32([40], dev), 40, dtype=torch.float32)[0][0]
    for h in range(H):
        for i, at in enumerate(kept[1, h].tolist()):
            page, row = int(table[1, at // G]), at % G
            was = before[0][page, h, row].view(torch.float8_e4m3fn).float() * before[2][page, h, 0].view(torch.float32)
            top = cache.scale[int(table[1, i // G]), h, 0]
            assert ((moved[h, i] - was).abs() <= 2.0 ** -4 * was.abs() + 2.0 ** -10 * top).all()


def refused(table, lens, keep, into, N, G, P):
    """Sequences of which a page that they write is named once more, as one that another needs or writes."""
    B = len(lens)
    ok = [0 <= n <= min(N, table.shape[1] * G) for n in lens]
    used = [-(-n // G) if o else 0 for n, o in zip(lens, ok)]
    if into is None:          # all that moves is read before: pages that stay count
        used = [-(-min(n, keep) // G) if o else 0 for n, o in zip(lens, ok)]
        written = [-(-keep // G) if o and n > keep else 0 for n, o in zip(lens, ok)]
        read, rows = used, table
    else:
        written = [min(-(-min(n, keep) // G), into.shape[1]) if o else 0 for n, o in zip(lens, ok)]
        read, rows = written, into
    names = {}
    for b in range(B):
        for p in (rows[b, :read[b]].tolist() + ([] if into is None else table[b, :used[b]].tolist())):
            names[p] = names.get(p, 0) + 1
    return [any(0 <= p < P and names[p] > 1 for p in rows[b, :written[b]].tolist()) for b in range(B)]


def check_pages(cache, table, lens, weights, keep, first=0, last=0, into=None, want=None):
    """evict as the definition has it where sequences whose pages are named twice have a length that breaks the rules."""
    ref, B = Ref(cache), len(lens)
    no = refused(table.cpu(), lens, keep, None if into is None else into.cpu(), weights.shape[2], cache.page_tokens, cache.num_pages)
    assert want is None or no == want
    got = cache.evict(table, i32(lens, cache.device), weights, keep, first, last, into)
    left = [-1 if no[b] else lens[b] for b in range(B)]
    wanted = evict_ref(ref, table.cpu().numpy(), left, weights.cpu().numpy(), keep, first, last, (table if into is None else into).cpu().numpy())
    for g, w in zip(got, wanted):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    same_pools(cache, ref)
    return no


@pytest.mark.parametrize("dev", DEVICES)
def test_pages_of_the_call_are_not_written_over(dev):
    """`into` that names pages the call reads, by another tensor of the same numbers or one page of another
    sequence, or one page twice: those sequences come back as -1 and as they were."""
    gen = torch.Generator().manual_seed(11)
    B, H, D, G, W = 3, 2, 32, 16, 5
    cache = filled(gen, 40, H, D, G, dev)
    table, spare = tables(gen, B, W, 20, dev), (20 + tables(gen, B, 4, 20, dev)).to(torch.int32)
    w = heavy(gen, B, H, W * G).to(dev)
    args = [table, [80, 33, 70], w, 50, 3, 8]
    before = held(cache)
    for into in (table.clone(), table[:, :4].contiguous(), table.flip(0)):
        check_pages(cache, *args, into, want=[True] * 3)
        same(cache, before)
    check_pages(cache, *args, torch.cat([spare[:2], table[:1, :4]]), want=[False, False, True])
    for (b, i), p, want in (((0, 3), int(table[2, 0]), [True, False, False]), ((1, 2), int(table[1, 0]), [False, True, False]),
                            ((1, 0), int(spare[0, 1]), [True, True, False]), ((2, 1), int(spare[2, 3]), [False, False, True]),
                            # behind what is kept or held: no page of the call
                            ((1, 3), int(table[0, 0]), [False] * 3), ((0, 0), int(table[1, 3]), [False] * 3),
                            # ids outside the pool are no pages
                            ((0, 0), 40, [False] * 3)):
        into = spare.clone()
        into[b, i] = p
        check_pages(cache, *args, into, want=want)
    into = spare.clone()
    into[0, 0] = into[1, 0] = into[1, 1] = -1
    check_pages(cache, *args, into, want=[False] * 3)
    # sequences that read the same pages move each into its own
    table[1, :2], table[2, :3] = table[0, :2], table[0, :3]
    check_pages(cache, *args, spare, want=[False] * 3)
    # lengths that break the rules name no page
    check_pages(cache, table, [80, -1, 1 << 20], w, 50, 3, 8, torch.cat([spare[:1], spare[:1], table[:1, :4]]), want=[False] * 3)


@pytest.mark.parametrize("dev", DEVICES)
def test_shared_pages_are_not_cut_in_place(dev):
    """A page that a cut sequence would write and another one, or the same one elsewhere, names."""
    gen = torch.Generator().manual_seed(12)
    B, H, D, G, W = 4, 2, 32, 16, 5
    clean = tables(gen, B, W, 30, dev)
    w = heavy(gen, B, H, W * G).to(dev)

    def check(lens, want, *named):
        cache, table = filled(torch.Generator().manual_seed(13), 30, H, D, G, dev), clean.clone()
        for (b, i), (c, j) in named:
            table[b, i] = table[c, j]
        check_pages(cache, table, lens, w, 40, 2, 8, want=want)

    for kw in ([((1, 0), (0, 0))], [((1, 2), (0, 1))]):
        check([80, 80, 10, 66], [True, True, False, False], *kw)      # two cut ones share a page
        check([80, 40, 10, 66], [True, False, False, False], *kw)     # one within the budget holds it
    check([80, 40, 10, 66], [True, False, False, False], ((1, 1), (0, 2)))
    check([80, 80, 10, 66], [False] * 4, ((1, 4), (0, 0)))                       # read by one, written by the other
    check([80, 80, 10, 66], [False] * 4, ((1, 4), (0, 4)))                       # read by both
    check([80, 60, 10, 66], [False] * 4, ((1, 4), (0, 0)))                       # behind its tokens
    check([80, 80, 10, 66], [False, False, False, True], ((3, 2), (3, 0)))       # twice in one
    check([80, 80, 10, 66], [False] * 4, ((3, 4), (3, 0)))                       # and read once more
    check([80, 80, 10, 66], [False] * 4, ((0, 4), (3, 0)), ((1, 3), (2, 0)), ((2, 4), (1, 1)), ((3, 4), (0, 2)))
    check([80, -1, 10, 66], [False] * 4, ((1, 0), (0, 0)))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("seed", range(6))
def test_pages_drawn_at_random(dev, seed):
    """Tables and `into` of few enough pages that some sequences clash."""
    gen = torch.Generator().manual_seed(seed)
    G, H, D, W, B = (16, 32)[seed % 2], 1 + seed % 3, 16, 4, (3, 20, 40)[seed % 3]
    P = B * W * 6
    met = []
    for turn in range(6):
        cache = filled(gen, P, H, D, G, dev)
        table, into = (torch.randint(0, P, (B, W), generator=gen, dtype=torch.int32).to(dev) for _ in range(2))
        lens = torch.randint(-3, W * G + 1, (B,), generator=gen).tolist()
        met += check_pages(cache, table, lens, heavy(gen, B, H, W * G).to(dev), 2 * G + 5, 2, 3, into if turn % 2 else None)
    assert any(met) and not all(met)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("at", [None, (3, 5000), (4100, 4096), (4999, 0), (6, 9)])
@pytest.mark.parametrize("place", [False, True])
def test_many_pages(dev, at, place):
    """Sequences of more pages than are looked at together; a page named twice, far apart or near."""
    gen = torch.Generator().manual_seed(14)
    G, W, K = 16, 5300, 5100
    cache = filled(gen, W + K + 50, 1, 16, G, dev)
    ids = torch.randperm(W + K + 50, generator=gen).to(torch.int32)
    table, into = ids[:W].view(1, W).clone(), ids[W:W + K].view(1, K).clone()
    if at is not None:
        rows = table if place else into
        rows[0, at[0]] = rows[0, at[1]]
    table = torch.cat([table, ids[-50:].view(1, 50).repeat(1, 106)]).to(dev)         # the second reads pages many times over
    into = torch.cat([into, table[1:, :1].cpu().expand(1, K)]).to(dev)
    n, keep = W * G - 3, K * G - 5
    w = torch.rand(2, 1, W * G, generator=gen).to(dev)
    before = held(cache)
    lens, kept, out = cache.evict(table, i32([n, 0], dev), w, keep, 7, 9, None if place else into)
    assert lens.tolist() == [keep if at is None else -1, 0]
    if at is not None:
        same(cache, before)
        assert (kept == -1).all() and (out == 0).all()
    else:
        order = w[0, 0, 7:n - 9].cpu().sort(descending=True, stable=True).indices[:keep - 16] + 7
        want = torch.cat([torch.arange(7), order.sort().values, torch.arange(n - 9, n)])
        assert torch.equal(kept[0, 0].cpu().long(), want) and (kept[1] == -1).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,H,W,N", [(4100, 1, 1, 3), (2100, 2, 1, 3), (2048, 1, 1, 2), (1100, 1, 2, 20), (500, 1, 120, 1900), (1, 3, 4090, 65000)])
def test_many_sequences(dev, B, H, W, N):
    """Of few tokens and of many, whose written pages are more than fit one table, or than the weights' memory has
    room for; some of them clash."""
    gen = torch.Generator().manual_seed(16)
    G, D = 16, 16
    K = -(-N // G)
    P = B * (W + K) + 7
    cache = filled(gen, P, H, D, G, dev)
    ids = torch.randperm(P, generator=gen).to(torch.int32)
    table, into = ids[:B * W].view(B, W).clone(), ids[B * W:B * (W + K)].view(B, K).clone()
    lens = torch.randint(0, min(N, W * G) + 1, (B,), generator=gen)
    lens[::5] = min(N, W * G)
    for b in range(0, B, 701):                  # a page of another one, behind its group too
        into[b, 0] = table[(b + B // 2) % B, 0]
        table[(b + 3) % B, 0] = table[(b + 3 + B // 3) % B, 0]
    table, into, w = table.to(dev), into.to(dev), heavy(gen, B, H, N).to(dev)
    no = refused(table.cpu(), lens.tolist(), N, into.cpu(), N, G, P)
    before = held(cache)
    got = cache.evict(table, lens.int().to(dev), w, N, 0, 0, into)
    assert any(no) and got[0].tolist() == [-1 if x else n for x, n in zip(no, lens.tolist())]
    gone = torch.tensor(no)
    there = (torch.arange(N) < lens[:, None])[:, None] & ~gone[:, None, None]
    assert torch.equal(got[1].cpu(), torch.where(there, torch.arange(N, dtype=torch.int32), -1).expand(B, H, N))
    assert torch.equal(got[2].cpu(), torch.where(there, w.cpu(), 0.0))
    for b in range(0, B, 97):
        for i in range(-(-int(lens[b]) // G)):
            n = min(G, int(lens[b]) - i * G)
            a, c = int(table[b, i]), int(into[b, i])
            for x, y in zip(held(cache)[:2], before[:2]) if b % 4 == 0 and i < 2 else ():
                assert torch.equal(x[c, :, :n], y[c if no[b] else a, :, :n])
    keep = N // 2 + 1
    no = refused(table.cpu(), lens.tolist(), keep, None, N, G, P)
    got = cache.evict(table, lens.int().to(dev), w, keep)
    assert got[0].tolist() == [-1 if x else min(n, keep) for x, n in zip(no, lens.tolist())]


@pytest.mark.gpu
@pytest.mark.parametrize("B,W,keep", [(3, 6, 40), (50, 100, 1500)])
def test_refusals_in_a_graph(dev, B, W, keep):
    """Captured, replayed with tables that clash and tables that do not."""
    gen = torch.Generator().manual_seed(15)
    H, D, G, P = 2, 32, 16, 3 * B * W + 6
    cache, twin = (filled(torch.Generator().manual_seed(5), P, H, D, G, dev) for _ in range(2))
    w = heavy(gen, B, H, W * G).to(dev)
    table, into, lens = tables(gen, B, W, P, dev), tables(gen, B, W, P, dev), i32([0] * B, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = [*cache.evict(table, lens, w, keep, 2, 8, into), *cache.evict(table, lens, w, keep, 2, 8)]
    met = set()
    for i in range(8):
        pages = torch.randint(0, P, (2, B, W), generator=gen) if i % 4 == 1 else torch.randperm(P, generator=gen)[:2 * B * W].view(2, B, W)
        if i % 4 == 3:
            pages[1, 0, 0], pages[0, 1, 0] = pages[0, 1, 0], pages[0, 2, 0]
        table.copy_(pages[0])
        into.copy_(pages[1])
        lens.copy_(torch.randint(0, W * G + 1, (B,), generator=gen))
        graph.replay()
        torch.randn(1 << 18, device=dev).sum().item()
        want = [*twin.evict(table, lens, w, keep, 2, 8, into), *twin.evict(table, lens, w, keep, 2, 8)]
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        for a, b in zip(held(cache), held(twin)):
            assert torch.equal(a, b)
        met |= set((outs[0] == -1).tolist())
    assert met == {True, False}
