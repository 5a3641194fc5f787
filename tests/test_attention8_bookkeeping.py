"""Slots, pages and lengths of KittyCache8: what refused and reading calls leave."""
import numpy as np
import pytest
import torch

from test_attention8 import DEVICES, config


def state(cache):
    return (dict(cache._slot_of), sorted(cache._free_slots), [list(p) for p in cache._pages], cache.pages_free,
            cache._held.tolist(), cache.lens.tolist())


def tokens(B, T, H=2, D=64, dev="cpu", dtype=torch.float16):
    return torch.randn(B, H, T, D, generator=torch.Generator().manual_seed(B * 100 + T)).to(dev, dtype)


def test_refused_calls_leave_nothing_behind():
    from kitty import KittyCache8, KittyPagedAttention8
    cfg = config("cpu", max_seq_len=64, max_batch_size=3, pool_pages_override=7)
    cache = KittyCache8(cfg, 2)
    cache.push(0, tokens(1, 40), tokens(1, 40), [5])
    cache.push(1, tokens(1, 20), tokens(1, 20), [5])
    before = state(cache)
    x = tokens(2, 8)
    for layer, k, v, ids, error in (
            (0, x, x, [7, 7], "twice"), (0, tokens(4, 1), tokens(4, 1), [5, 6, 7, 8], "slots"),
            (0, tokens(2, 30), tokens(2, 30), [6, 5], "max_seq_len"), (0, tokens(2, 50), tokens(2, 50), [6, 7], "exhausted"),
            (0, x, x[:, :, :4], [5, 6], "value"), (0, x.double(), x.double(), [6, 5], "float16"), (0, x[:, :1], x[:, :1], [6, 7], "key"),
            (0, x.clone().requires_grad_(), x, [7, 6], "no backward"), (1, x, x, [5], "sequence ids")):
        with pytest.raises((ValueError, RuntimeError), match=error):
            cache.push(layer, k, v, ids)
        assert state(cache) == before, error
    mod = KittyPagedAttention8(cfg, 2, cache, 0)
    with pytest.raises(RuntimeError, match="exhausted"):
        mod(tokens(2, 50), tokens(2, 50), tokens(2, 50), seq_id=[6, 7])
    assert state(cache) == before
    for heads in (0, 3):
        with pytest.raises(ValueError, match="num_q_heads"):
            KittyPagedAttention8(cfg, heads, cache, 0)
    cache.push(0, tokens(2, 8), tokens(2, 8), [9, 8])      # the slots are free as before
    assert cache.tokens(9) == cache.tokens(8) == 8 and cache.tokens(5) == 40


@pytest.mark.parametrize("dev", DEVICES)
def test_reading_takes_no_slot(dev):
    """read and attend of sequences that hold nothing: zeros, and every slot stays free."""
    from kitty import KittyCache8
    cfg = config(dev, max_batch_size=2)
    cache = KittyCache8(cfg, 1)
    before = state(cache)
    assert cache.read(0, [1, 2, 3])[0].shape == (3, 2, 0, 64)
    assert (cache.attend(0, tokens(1, 3, 4, dev=dev), [1]) == 0).all() and state(cache) == before
    cache.push(0, tokens(1, 20, dev=dev), tokens(1, 20, dev=dev), [7])
    before = state(cache)
    q = tokens(4, 2, 4, dev=dev)
    for ids in ([1, 7, 2, 3], [7, 1, 2, 3]):
        out = cache.attend(0, q, ids)
        at = ids.index(7)
        assert torch.equal(out[at:at + 1], cache.attend(0, q[at:at + 1], [7]))
        assert (out[[i for i in range(4) if i != at]] == 0).all()
        k, v = cache.read(0, ids)
        want = cache.read(0, [7])
        for got, w in zip((k, v), want):
            assert torch.equal(got[at:at + 1], w) and (got[[i for i in range(4) if i != at]] == 0).all()
    with pytest.raises(ValueError, match="twice"):
        cache.read(0, [1, 1])
    assert state(cache) == before
    cache.push(0, tokens(1, 1, dev=dev), tokens(1, 1, dev=dev), [9])      # the slot that reading 1, 2 and 3 left
    np.testing.assert_array_equal(cache.lens[0].cpu().numpy()[:2], [20, 1])


def test_pages_of_a_layer():
    """Each layer has the pages that the slots' tables can name: not a pool sized for all
    layers together, and enough for every slot's max_seq_len whatever the sinks."""
    from kitty import KittyAttentionFactory, KittyCache8
    cfg = config("cpu", max_batch_size=2, num_layers=6)
    cfg.pool_pages_override = cfg.max_pages * cfg.num_layers
    bi = torch.full((6, 2, 64), cfg.sentinel, dtype=torch.uint8)
    bi[:, :, :cfg.d_boost] = torch.arange(cfg.d_boost, dtype=torch.uint8)
    cache = KittyAttentionFactory.from_config(cfg, bi, 4, eight_bit_layers=[0, 5])[2][0].cache
    assert [c.num_pages for c in cache.layers] == [32, 32] and cache.pages_free == 32      # 2 x 256 tokens
    for sinks in (4, 100):
        cfg = config("cpu", max_batch_size=2, max_seq_len=250, sink_size=sinks)
        cache = KittyCache8(cfg, 1)
        cache.push(0, tokens(2, 250), tokens(2, 250), [1, 2])
        assert cache.tokens(1) == cache.tokens(2) == 250
    small = KittyCache8(config("cpu", max_batch_size=2, pool_pages_override=3), 1)
    assert small.pages_free == small.layers[0].num_pages == 3


@pytest.mark.parametrize("dev", DEVICES)
def test_reset_of_a_mixed_model(dev):
    """pipeline.reset_sequence drops a sequence from the factory's 8-bit layers too: its id
    begins anew in every layer, and the other sequences stay."""
    from kitty import KittyAttentionFactory
    cfg = config(dev, max_batch_size=2, num_layers=2)
    cfg.pool_pages_override = cfg.max_pages * cfg.num_layers
    bi = torch.full((2, 2, 64), cfg.sentinel, dtype=torch.uint8)
    bi[:, :, :cfg.d_boost] = torch.arange(cfg.d_boost, dtype=torch.uint8)
    _, pipeline, mods = KittyAttentionFactory.from_config(cfg, bi, 4, eight_bit_layers=[1])
    cache = mods[1].cache

    def run(ids, T):
        x = [tokens(len(ids), T, h, dev=dev) for h in (4, 2, 2)]
        with torch.no_grad():
            return [m(*x, seq_id=ids) for m in mods]

    first = run([3, 8], 30)
    pipeline.reset_sequence(3)
    assert cache.tokens(3) == 0 and cache.tokens(8) == 30 and cache.pages_free == cache.layers[0].num_pages - 2
    cache.reset_sequence(3)                     # as programs that reset both do
    pipeline.reset_sequence(3)
    pipeline.reset_sequence(77)
    again = run([3], 30)
    assert cache.tokens(3) == 30
    x = [tokens(2, 30, h, dev=dev)[:1] for h in (4, 2, 2)]
    pipeline.reset_sequence(3)
    with torch.no_grad():
        assert torch.equal(mods[1](*x, seq_id=3), first[1][:1])
    assert again[1].shape == (1, 4, 30, 64)
