"""KittyPagedAttention8 and KittyCache8: layers in 8 bits next to the 2-bit ones,
against float64 attention over the same quantised tokens."""
import numpy as np
import pytest
import torch

from cache8_ref import Ref, numpy, tolerance

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def config(dev, **kw):
    from kitty import KittyConfig
    base = dict(num_layers=3, num_kv_heads=2, head_dim=64, sink_size=4, q_buffer_size=16, local_value_window=16,
                max_seq_len=256, max_batch_size=4, device=dev)
    return KittyConfig(**{**base, **kw})


def tolerance_of(q, want, spread, mag, small, H, n):
    return tolerance(q.dtype, want, spread, mag, small, q.shape[1] // H * q.shape[2], q.shape[3], n)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_sequences_of_two_layers(dev, dtype):
    """Prompts, chunks and steps of sequences in changing batches, in two layers: a
    run of slots, any other order, one sequence reset and its pages reused."""
    from kitty import KittyCache8, KittyPagedAttention8
    gen = torch.Generator().manual_seed(3)
    cfg = config(dev, dtype=dtype)
    cache = KittyCache8(cfg, 2)
    mods = [KittyPagedAttention8(cfg, 6, cache, i) for i in range(2)]
    refs = [Ref(c) for c in cache.layers]
    held = {}
    dt = torch.float16 if dtype == "float16" else torch.bfloat16
    for ids, T in (([7, 8], 20), ([9], 33), ([8, 7, 9], 1), ([7, 8, 9], 1), ([9, 7], 5), ("reset", 8), ([4, 8], 50), ([8, 4, 7], 1),
                   ([4], 40), ([4, 7, 8, 9], 2)):
        if ids == "reset":
            cache.reset_sequence(T)
            held.pop(T)
            continue
        for layer in range(2):
            q, k, v = (torch.randn(len(ids), h, T, 64, generator=gen).to(dt) for h in (6, 2, 2))
            out = mods[layer](q.to(dev), k.to(dev), v.to(dev), seq_id=ids)
            assert out.dtype == dt and out.shape == q.shape
            slots = [cache.slot(i) for i in ids]
            table = cache.block_table[slots].cpu().numpy()
            before = [held.get(i, 0) for i in ids]
            refs[layer].write(numpy(k), numpy(v), table, before)
            lens = [b + T for b in before]
            assert [cache.tokens(i, layer) for i in ids] == lens == cache.lens[layer, slots].tolist()
            want, _, spread, mag, small = refs[layer].attend(numpy(q), table, lens)
            assert (np.abs(numpy(out) - want) <= tolerance_of(q, want, spread, mag, small, 2, max(lens))).all()
        held.update({i: held.get(i, 0) + T for i in ids})
    used = sum(-(-n // 16) for n in held.values())
    assert cache.pages_free == cfg.pool_pages - used
    k, v = cache.read(1, [7, 4], dtype=torch.float32)
    want = refs[1].read(cache.block_table[[cache.slot(7), cache.slot(4)]].cpu().numpy(), [held[7], held[4]], max(held[7], held[4]))
    np.testing.assert_array_equal(numpy(k), want[0])      # code times a power of two: exact in fp32
    np.testing.assert_array_equal(numpy(v), want[1])


@pytest.mark.parametrize("dev", DEVICES)
def test_factory_mixes_layers(dev):
    """from_config with 8-bit layers: those modules take the same calls and stay nearer to
    unquantised attention than the 2-bit ones; without them nothing changes."""
    from kitty import KittyAttentionFactory, KittyPagedAttention, KittyPagedAttention8
    gen = torch.Generator().manual_seed(5)
    cfg = config(dev, max_batch_size=2)
    cfg.pool_pages_override = cfg.max_pages * cfg.num_layers
    bi = torch.full((3, 2, 64), cfg.sentinel, dtype=torch.uint8)
    bi[:, :, :cfg.d_boost] = torch.arange(cfg.d_boost, dtype=torch.uint8)
    plain = KittyAttentionFactory.from_config(cfg, bi, 4)[2]
    assert all(type(m) is KittyPagedAttention for m in plain)
    _, _, mods = KittyAttentionFactory.from_config(cfg, bi, 4, eight_bit_layers=[2, 0])
    assert [type(m) for m in mods] == [KittyPagedAttention8, KittyPagedAttention, KittyPagedAttention8]
    assert mods[0].cache is mods[2].cache and [mods[0].layer, mods[2].layer] == [0, 1]
    q, k, v = (torch.randn(2, h, 100, 64, generator=gen).half() for h in (4, 2, 2))
    errs = []
    with torch.no_grad():
        for m in mods:
            m(q[:, :, :-1].to(dev), k[:, :, :-1].to(dev), v[:, :, :-1].to(dev))
            got = m(q[:, :, -1:].to(dev), k[:, :, -1:].to(dev), v[:, :, -1:].to(dev))
            s = (q[:, :, -1:].double() @ k.double().repeat_interleave(2, 1).transpose(2, 3)) / 8
            want = torch.softmax(s, -1) @ v.double().repeat_interleave(2, 1)
            errs.append(float((got.double().cpu() - want).norm() / want.norm()))
    # e4m3 rounds a value by 2^-4 at most, keys and values together well below 2-bit codes' error
    assert errs[0] < 0.1 and errs[2] < 0.1 and errs[1] > 2 * errs[0]
    with pytest.raises(ValueError, match="eight_bit_layers"):
        KittyAttentionFactory.from_config(cfg, bi, 4, eight_bit_layers=[3])


def test_refusals_and_limits():
    from kitty import KittyCache8, KittyPagedAttention8
    cfg = config("cpu", max_seq_len=64, max_batch_size=2, pool_pages_override=5)
    cache = KittyCache8(cfg, 1)
    mod = KittyPagedAttention8(cfg, 2, cache, 0)
    x = lambda B, T, h=2: torch.zeros(B, h, T, 64).half()  # noqa: E731
    with pytest.raises(ValueError, match="sequence ids"):
        mod(x(2, 1), x(2, 1), x(2, 1), seq_id=[1])
    with pytest.raises(ValueError, match="twice"):
        mod(x(2, 1), x(2, 1), x(2, 1), seq_id=[1, 1])
    mod(x(1, 40), x(1, 40), x(1, 40), seq_id=1)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        mod(x(1, 25), x(1, 25), x(1, 25), seq_id=1)
    with pytest.raises(RuntimeError, match="exhausted"):
        mod(x(1, 33), x(1, 33), x(1, 33), seq_id=2)
    assert cache.tokens(1) == 40 and cache.tokens(2) == 0 and cache.pages_free == 2
    mod(x(1, 32), x(1, 32), x(1, 32), seq_id=2)
    with pytest.raises(RuntimeError, match="slots are in use"):
        mod(x(1, 1), x(1, 1), x(1, 1), seq_id=3)
    cache.reset_sequence(1)
    cache.reset_sequence(99)
    assert cache.pages_free == 3
    mod(x(1, 1), x(1, 1), x(1, 1), seq_id=3)
    assert mod(x(0, 1), x(0, 1), x(0, 1)).shape == (0, 2, 1, 64)
    assert cache.attend(0, x(0, 1), []).shape == (0, 2, 1, 64)
    assert [t.shape for t in cache.read(0, [])] == [(0, 2, 0, 64)] * 2
    assert mod(x(1, 1).float(), x(1, 1).float(), x(1, 1).float(), seq_id=3).dtype == torch.float32
    with pytest.raises(RuntimeError, match="no backward"):
        mod(x(1, 1).requires_grad_(), x(1, 1), x(1, 1), seq_id=3)
    with pytest.raises(ValueError):
        KittyCache8(config("cpu", q_buffer_size=12), 1)
