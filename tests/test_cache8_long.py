"""attend_shared and attend_weighed over 150,000 tokens of the 8-bit cache, where every few hundred tokens one
carries a share of the softmax that a lost or doubled part of the work would show."""
import pytest
import torch

from test_cache8 import BF16, F16, i32

EVERY = 300      # tokens between two that count, fewer than the work is ever cut into


def marks(n):
    """Positions that count: the first, the last, and one in each EVERY."""
    i = torch.arange(0, n - 1, EVERY)
    return torch.unique(torch.cat([i + i // EVERY % 97, torch.tensor([0, n - 1])])).clamp(max=n - 1)


def tokens(gen, u, n, D):
    """Keys and values (H, n, D) of n tokens: small, but for the marked ones, whose keys are u (H, D) and whose
    values are 4 in a channel of their own."""
    k, v = 0.3 * torch.randn(2, u.shape[0], n, D, generator=gen)
    at = marks(n)
    k[:, at] = u[:, None]
    v[:, at, torch.arange(len(at)) % D] = 4.0
    return k, v, at


def exact(cache, q, pages, n):
    """Queries q (Hq, T, D), the last of n tokens in the places `pages` gives (page * G + row), in float64:
    softmax (Hq, T, n), values (H, n, D) and the largest sum of |q k| of a row."""
    H, G, D = cache.num_kv_heads, cache.page_tokens, cache.head_dim
    kv = []
    for i, pool in enumerate((cache.key, cache.value)):
        x = pool.view(torch.uint8)[pages // G, :, pages % G].view(torch.float8_e4m3fn).double() * cache.scale[pages // G][..., i, None].double()
        kv.append(x.transpose(0, 1))
    Hq, T, _ = q.shape
    rows = q.double().view(H, -1, D) * D ** -0.5
    s = (rows @ kv[0].transpose(1, 2)).view(Hq, T, n)
    mag = (rows.abs() @ kv[0].abs().transpose(1, 2)).view(Hq, T, n).amax(-1)
    s = s.masked_fill(torch.arange(n, device=q.device) > torch.arange(n - T, n, device=q.device)[:, None], -float("inf"))
    return torch.softmax(s, -1), kv[1], mag


# Sums of n weights, and of as many products, are of runs and then of one part a run.  With 256 CUs a run has a 128th
# of a KV head's tokens here at most, 1,172, of which a lane adds a sixteenth or more, and there are 512 parts at most:
# fewer than 2,048 additions behind each other.
ADDS = 2048


def check_out(out, p, v, mag, at, dtype, one):
    """out against p @ v, cache8_ref.tolerance's bound with ADDS in the place of n; that without any one of the marked
    tokens `at` it is beyond it."""
    Hq, T, n = p.shape
    H, _, D = v.shape
    flat = p.view(H, -1, n)
    want, spread = (flat @ v).view(Hq, T, D), (flat @ v.abs()).view(Hq, T, D)
    w = 2 * ((D + 6) * 2.0 ** -24 * mag + 2.0 ** -20 + ADDS * 2.0 ** -24) + (2.0 ** -11 if one else 2.0 ** -16)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + w[..., None] * spread + 2.0 ** -23
    # of one fp16 term what lies below its normal numbers: 2^-25 of the largest weight (times its scale, every code)
    if one:
        tol = tol + 2.0 ** -25 * p.amax(-1, keepdim=True) * v.abs().sum(1).repeat_interleave(Hq // H, 0)[:, None]
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())
    share = p[..., at]
    x = v[:, at].repeat_interleave(Hq // H, 0)[:, None]                                 # (Hq, 1, marks, D)
    moved = (share[..., None] / (1 - share[..., None]) * (want[:, :, None] - x)).abs()   # by leaving it out
    assert ((moved > 3 * tol[:, :, None]).any(-1) | (share == 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,per", [(1, 3), (3, 2), (40, 2), (17, 3)])
def test_every_part_counts(dev, dtype, T, per):
    from kitty.kernels import Cache8
    gen = torch.Generator().manual_seed(T)
    n, Hq, H, D, G = 150016, 4, 2, 64, 64
    W = n // G
    cache = Cache8.empty(W + 12 * per, H, D, G, device=dev)
    order = torch.randperm(W + 12 * per, generator=gen).int().to(dev)
    ptable, table = order[:W].view(1, W), order[W:].view(per, 12)
    u = torch.randint(0, 2, (H, D), generator=gen).float() * 2 - 1
    q = (u.repeat_interleave(Hq // H, 0)[:, None] + 0.2 * torch.randn(per, Hq, T, D, generator=gen)).to(dtype).to(dev)
    before = n - 17                                     # the prefix ends inside a page
    k, v, at = tokens(gen, u, before, D)
    cache.write(k[None].to(dev), v[None].to(dev), ptable, i32([0], dev))
    own = [64 + 130 * b for b in range(per)]
    held = []
    for b, m in enumerate(own):
        k, v, to = tokens(gen, u, m, D)
        held.append(to)
        cache.write(k[None].to(dev), v[None].to(dev), table[b:b + 1], i32([0], dev))
    out = cache.attend_shared(q, ptable, i32([before], dev), table, i32(own, dev))
    weights = torch.zeros(1, H, n, device=dev)
    alone = cache.attend_weighed(q[:1], ptable, i32([before], dev), weights)
    rows = Hq // H * T
    place = lambda t, m: (t.long()[:, None] * G + torch.arange(G, device=dev)).flatten()[:m]  # noqa: E731
    for b, m in enumerate(own):
        p, v, mag = exact(cache, q[b], torch.cat([place(ptable[0], before), place(table[b], m)]), before + m)
        marked = torch.cat([at, before + held[b]])
        check_out(out[b], p, v, mag, marked, dtype, dtype == BF16 and rows * per > 64)
    p, v, mag = exact(cache, q[0], place(ptable[0], before), before)
    check_out(alone[0], p, v, mag, at, dtype, dtype == BF16 and rows > 64)
    # each weight is off by that of its exponents and of the rows' sums, and by adding up the rows
    want = p.view(H, -1, before).sum(1)
    rel = 2 * ((D + 6) * 2.0 ** -24 * float(mag.max()) + 2.0 ** -20 + ADDS * 2.0 ** -24) + rows * 2.0 ** -24
    assert ((weights[0, :, :before].double() - want).abs() <= rel * want).all() and (weights[0, :, before:] == 0).all()
    share = p[..., at].amin((0, 1))
    assert float(share[:-1].min() if T > 1 else share.min()) > 3 * rel        # a part left out of the sums would show
