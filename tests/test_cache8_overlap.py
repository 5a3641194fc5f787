"""Outputs and weights of the 8-bit cache's calls whose rows share memory in part are refused,
rows that lie between each other are not."""
import pytest
import torch

from test_cache8 import DEVICES, F16, filled, i32, tables

# strides (sequence, head, query) of out (2, 4, 3, 64): rows of 64 in rows of 48, heads over the next
# sequence's first, queries over the next head's; strides of weights (2, 2, 64) likewise
OUT = [(1024, 256, 48), (640, 256, 64), (1024, 128, 64), (256, 64, 128), (64, 512, 64)]
WEIGHTS = [(64, 48), (96, 64), (32, 128), (0, 64), (64, 64)]


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_that_overlap_are_refused(dev):
    gen = torch.Generator().manual_seed(1)
    cache = filled(gen, 9, 2, 64, 16, dev)
    table, lens = tables(gen, 2, 4, 9, dev), i32([60, 5], dev)
    q, w = torch.randn(2, 4, 3, 64, generator=gen).half().to(dev), torch.zeros(2, 2, 64, device=dev)
    memory = torch.zeros(4096, dtype=F16, device=dev)
    for strides in OUT:
        out = memory.as_strided((2, 4, 3, 64), (*strides, 1))
        for call in (lambda: cache.attend(q, table, lens, out=out), lambda: cache.attend_weighed(q, table, lens, w, out=out),
                     lambda: cache.attend_shared(q, table, lens, table, lens, out=out)):
            with pytest.raises(ValueError, match="share memory"):
                call()
        pair = memory.as_strided((2, 2, 3, 64), (*strides, 1)), torch.zeros(2, 2, 3, 64, dtype=F16, device=dev)
        if strides != (640, 256, 64):      # with two heads those do not meet
            with pytest.raises(ValueError, match="share memory"):
                cache.read(table, lens, 3, out=pair)
    held = torch.zeros(4096, device=dev)
    for strides in WEIGHTS:
        with pytest.raises(ValueError, match="share memory"):
            cache.attend_weighed(q, table, lens, held.as_strided((2, 2, 64), (*strides, 1)))
    assert (memory == 0).all() and (held == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_between_each_other(dev):
    gen = torch.Generator().manual_seed(2)
    cache = filled(gen, 9, 2, 64, 16, dev)
    table, lens = tables(gen, 2, 4, 9, dev), i32([60, 5], dev)
    q = torch.randn(2, 4, 3, 64, generator=gen).half().to(dev)
    want = cache.attend(q, table, lens)
    # heads 128 apart, queries 576 (behind the heads), sequences 64: between the heads
    out = torch.zeros(4096, dtype=F16, device=dev).as_strided((2, 4, 3, 64), (64, 128, 576, 1))
    assert torch.equal(cache.attend(q, table, lens, out=out), want)
    w, v = torch.zeros(2, 2, 64, device=dev), torch.zeros(4096, device=dev).as_strided((2, 2, 64), (100, 200, 1))
    assert torch.equal(cache.attend_weighed(q, table, lens, w), cache.attend_weighed(q, table, lens, v, out=out))
    assert torch.equal(w, v)
