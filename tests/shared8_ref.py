"""Sequences that share prefixes, for the tests of the 8-bit cache: the two parts of
each in one table of single tokens, over which cache8_ref.Ref attends."""
import numpy as np

from cache8_ref import Ref


def flat(cache):
    """The pools as pages of one token: token r of page p is page p * G + r."""
    ref = Ref(cache)
    out = Ref.__new__(Ref)
    out.P, out.H, out.G, out.D = ref.P * ref.G, ref.H, 1, ref.D
    out.pools = [np.swapaxes(x, 1, 2).reshape(out.P, ref.H, 1, ref.D) for x in ref.pools]
    out.scale = np.repeat(ref.scale, ref.G, 0)
    return out, ref


def token_ids(ref, table, b, n):
    """Single-token pages of the first n tokens of a table's row, -1 where there is none."""
    pages = [ref.page(table, b, i // ref.G) for i in range(n)]
    return [p * ref.G + i % ref.G if p >= 0 else -1 for i, p in enumerate(pages)]


def attend_shared(cache, q, prefix_table, prefix_lens, table, lens, q_lens=None, causal=True, sm_scale=None):
    """Ref.attend's five arrays."""
    one, ref = flat(cache)
    each = len(lens) // len(prefix_lens)
    ids, total = [], []
    for b, n in enumerate(lens):
        f = b // each
        before = prefix_lens[f]
        if not 0 <= n <= table.shape[1] * ref.G or not 0 <= before <= prefix_table.shape[1] * ref.G:
            ids.append([])
            total.append(-1)
            continue
        ids.append(token_ids(ref, prefix_table, f, before) + token_ids(ref, table, b, n))
        total.append(before + n)
    joined = np.full((len(lens), max([len(i) for i in ids] + [1])), -1)
    for b, i in enumerate(ids):
        joined[b, :len(i)] = i
    return one.attend(q, joined, total, q_lens, causal, sm_scale)
