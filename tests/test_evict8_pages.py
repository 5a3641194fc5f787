"""Which pages an eviction from the 8-bit cache writes (Cache8.evict), on the CPU path and on the GPU."""
import math

import pytest
import torch

from test_cache8 import DEVICES, filled, i32, tables
from test_evict8 import heavy


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
