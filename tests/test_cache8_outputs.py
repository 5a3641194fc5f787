"""Tensors that a program gives read and attend of the 8-bit cache to write into."""
import pytest
import torch

from test_cache8 import DEVICES, F16, filled, i32, tables


def setup(dev, T=3, D=64):
    gen = torch.Generator().manual_seed(7)
    cache = filled(gen, 9, 2, D, 32, dev)
    q = torch.randn(2, 4, T, D, generator=gen).half().to(dev)
    return cache, tables(gen, 2, 4, 9, dev), i32([70, 65], dev), q


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_and_gradients(dev):
    """As torch's own in-place writes: a leaf that needs a gradient is refused, what a graph
    saved is found changed."""
    cache, table, lens, q = setup(dev)
    leaf = torch.zeros_like(q).requires_grad_()
    pair = [torch.zeros(2, 2, 8, 64, dtype=F16, device=dev) for _ in range(2)]
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend(q, table, lens, out=leaf)
    for at in (0, 1):
        out = list(pair)
        out[at] = out[at].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="gradient"):
            cache.read(table, lens, 8, out=tuple(out))
    with torch.no_grad():
        cache.attend(q, table, lens, out=leaf)
        assert torch.equal(leaf, cache.attend(q, table, lens))
    for write, target in ((lambda t: cache.attend(q, table, lens, out=t), torch.zeros_like(q)),
                          (lambda t: cache.read(table, lens, 8, out=(t, pair[1])), pair[0]),
                          (lambda t: cache.read(table, lens, 8, out=(pair[0], t)), pair[1])):
        for _ in range(2):                      # the first call of a signature and a later one
            x = torch.ones(target.shape, device=dev, requires_grad=True)
            y = (x * target).sum()              # saves target
            write(target)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_negated_outputs(dev):
    """A view whose elements are read negated gets the values, not their negatives."""
    cache, table, lens, q = setup(dev)
    want = cache.attend(q, table, lens)
    pair = cache.read(table, lens, 8)
    for _ in range(2):
        out = torch._neg_view(torch.zeros_like(q))
        assert cache.attend(q, table, lens, out=out) is out and torch.equal(out, want)
        outs = torch.zeros_like(pair[0]), torch._neg_view(torch.zeros_like(pair[1]))
        got = cache.read(table, lens, 8, out=outs)
        assert torch.equal(got[0], pair[0]) and torch.equal(got[1], pair[1])
