"""Tensors that a program gives read and attend of the 8-bit cache to write into."""
import pytest
import torch

from test_cache8 import BF16, DEVICES, F16, filled, i32, tables


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


# a call of one launch, one that is split, a chunk in tiles
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,wide", [(3, 0), (3, 300), (40, 300)])
def test_output_over_other_queries(dev, T, wide):
    """out in q's memory but in another place or order: the results of a tensor of its own."""
    cache, table, lens, q = setup(dev, T)
    table = torch.cat([table, torch.zeros(2, wide, dtype=torch.int32, device=dev)], 1)
    want = cache.attend(q, table, lens)
    n = q.numel()
    for _ in range(2):
        room = torch.zeros(n + 64 * T, dtype=F16, device=dev)
        for a, b in ((0, 64 * T), (64 * T, 0), (8, 0)):            # one head or a few channels apart
            room.zero_()
            src = room[a:a + n].view(q.shape).copy_(q)
            out = room[b:b + n].view(q.shape)
            cache.attend(src, table, lens, out=out)
            assert torch.equal(out, want)
        src = room[:n].view(q.shape).copy_(q)
        out = room[:n].view(2, T, 4, 64).transpose(1, 2)           # the same memory as (B, T, H, D)
        cache.attend(src, table, lens, out=out)
        assert torch.equal(out, want)
        fused = torch.zeros(2, T, 3 * 256, dtype=F16, device=dev)  # beside the queries, row by row
        src, out = (fused[..., i:i + 256].unflatten(2, (4, 64)).transpose(1, 2) for i in (0, 512))
        src.copy_(q)
        cache.attend(src, table, lens, out=out)
        assert torch.equal(out, want) and torch.equal(src, q)


def test_read_refuses_one_output_twice():
    cache, table, lens, q = setup("cpu")
    x = torch.zeros(2, 2, 8, 64, dtype=BF16)
    with pytest.raises(ValueError, match="same memory"):
        cache.read(table, lens, 8, out=(x, x))
    both = torch.zeros(2, 2, 8, 2, 64, dtype=BF16)
    got = cache.read(table, lens, 8, out=(both[..., 0, :], both[..., 1, :]))
    want = cache.read(table, lens, 8, dtype=BF16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_pools_are_plain_tensors():
    """Pools that need a gradient, which no call would give them, and negated views are refused."""
    from kitty.kernels import Cache8
    key, value = (torch.zeros(3, 2, 16, 32, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    scale = torch.ones(3, 2, 2)
    with pytest.raises(RuntimeError, match="gradient"):
        Cache8(key, value, scale.clone().requires_grad_())
    with pytest.raises(ValueError, match="negated"):
        Cache8(key, value, torch._neg_view(scale))
    Cache8(key, value, scale.clone().requires_grad_().detach())


@pytest.mark.gpu
def test_module_steps_are_not_captured(dev):
    """KittyCache8 counts tokens on the host too, so a captured push is refused and leaves
    nothing; Cache8's own calls are captured."""
    from kitty import KittyCache8
    from test_attention8 import config
    cache = KittyCache8(config("cuda:0"), 1)
    x = torch.randn(1, 2, 1, 64, device=dev).half()
    cache.push(0, x, x, [4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            cache.push(0, x, x, [4])
        out = cache.layers[0].attend(x, cache.block_table[:1], cache.lens[0, :1])
    graph.replay()
    assert torch.equal(out, cache.attend(0, x, [4])) and cache.tokens(4) == 1 and cache.lens[0, 0].item() == 1
