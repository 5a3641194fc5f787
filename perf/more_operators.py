"""The 8-bit paged cache where its size counts: prefixes that many sequences
share, tokens weighed by the attention they get, and the light ones evicted.

A cache holds pages of G tokens: ``key`` and ``value`` (P, H, G, D) in e4m3,
``scale`` (P, H, 2) in float32, one scale per page, head and stream (0 keys, 1
values); a code c stands for c * scale.  ``table`` (B, W) int32 names the pages
of each sequence in order.  Three calls of ``kitty.kernels.Cache8``:

* ``attend_shared(q, prefix_table, prefix_lens, table, lens, q_lens, causal)``:
  sequence b of B is the prefix_lens[f] tokens of prefix f = b // (B / F)
  followed by lens[b] tokens of its own; softmax attention of T >= 1 queries over
  both.  Query i of q_lens[b] is the q_lens[b] - i-th token from the end and sees
  itself and what precedes it, or with causal=False every token.  Rows that see
  nothing are zeros.
* ``attend_weighed(q, table, lens, weights, q_lens, causal)``: softmax attention
  over one sequence each, and to weights[b, h, j] (B, H, N) float32 is added what
  token j of KV head h got: the softmax weights of all rows of the head's group.
* ``evict(table, lens, weights, keep, first, last, into)``: of each sequence and
  KV head the first and last tokens stay, and of the others the heaviest, keep
  tokens in all (all where there are no more; of equal weights the earlier
  stays).  They become tokens 0 .. of the pages that ``into`` names, in their
  order; a page's scale is the largest of the pages that its tokens come from,
  and codes of smaller ones are rounded again.  Returns the new lengths, the
  positions kept (B, H, min(keep, N)) int32 with -1 behind them, and their
  weights (B, H, N), zeros behind them.

Keys have a few channels that are 8 times the others; queries, keys and values
are normal otherwise.  Weights spread over orders of magnitude, some are zero.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # four answers to one short prompt, 8 query / 8 KV heads, where latency counts
        dict(name="shared_samples_b4", op="shared", F=1, B=4, T=1, Hq=8, Hkv=8, D=128, G=128, plo=1000, phi=1000, lo=1,
             hi=40, causal=True, ragged=False, dtype="float16"),
        # a serving batch of chats behind one long system prompt
        dict(name="shared_system_b64", op="shared", F=1, B=64, T=1, Hq=32, Hkv=8, D=128, G=64, plo=16384, phi=16384,
             lo=100, hi=2000, causal=True, ragged=False, dtype="bfloat16"),
        # eight unequal prompts with eight samples each, a 70B model's head layout, small pages
        dict(name="shared_samples_8x8", op="shared", F=8, B=64, T=1, Hq=64, Hkv=8, D=128, G=32, plo=2000, phi=9000, lo=0,
             hi=500, causal=True, ragged=False, dtype="float16"),
        # five draft tokens of sixteen sequences behind one document
        dict(name="shared_draft_b16", op="shared", F=1, B=16, T=5, Hq=32, Hkv=8, D=128, G=128, plo=30000, phi=30000,
             lo=64, hi=4000, causal=True, ragged=False, dtype="bfloat16"),
        # padded questions of up to 300 tokens about two documents, just written behind them
        dict(name="shared_questions_b6", op="shared", F=2, B=6, T=300, Hq=16, Hkv=4, D=64, G=16, plo=5000, phi=8000,
             lo=300, hi=300, causal=True, ragged=True, dtype="float16"),
        # one sequence, 8 query / 8 KV heads, 1K context: latency and launches
        dict(name="weighed_single_1k", op="weighed", B=1, T=1, Hq=8, Hkv=8, D=128, G=128, lo=1024, hi=1024, causal=True,
             ragged=False, dtype="float16"),
        # an 8B model's layer, batch 16 at 32K context
        dict(name="weighed_b16_32k", op="weighed", B=16, T=1, Hq=32, Hkv=8, D=128, G=128, lo=32768, hi=32768, causal=True,
             ragged=False, dtype="float16"),
        # the last 32 queries of eight prompts, by which they are cut down before decoding
        dict(name="weighed_window_b8", op="weighed", B=8, T=32, Hq=32, Hkv=8, D=128, G=32, lo=4000, hi=16000, causal=True,
             ragged=False, dtype="bfloat16"),
        # a 2,048-token chunk of a long prompt behind 16K tokens that are in the cache
        dict(name="weighed_chunk_2k", op="weighed", B=1, T=2048, Hq=32, Hkv=8, D=128, G=128, lo=18000, hi=18000,
             causal=True, ragged=False, dtype="float16"),
        # one sequence back to its budget, as every few tokens of a long chat
        dict(name="evict_single_1k", op="evict", B=1, H=8, D=128, G=128, lo=1100, hi=1100, keep=1024, first=4, last=64),
        # a batch of long prompts to half
        dict(name="evict_b16_32k", op="evict", B=16, H=8, D=128, G=128, lo=32768, hi=32768, keep=16384, first=32,
             last=128),
        # unequal sequences, some within the budget, small pages
        dict(name="evict_ragged", op="evict", B=6, H=4, D=64, G=16, lo=500, hi=5000, keep=777, first=1, last=33),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the ranges above: heads, head sizes, page sizes and types of all
    kinds, one token to long prompts, prefixes and contexts from nothing to 64K tokens."""
    op = rng.choice(("shared", "shared", "weighed", "weighed", "evict"))
    D = rng.choice((64, 64, 80, 96, 128, 128, 128, 192, 256))
    G = rng.choice((16, 32, 64, 128))
    if op == "evict":
        H, B = rng.choice((1, 2, 4, 5, 8, 16)), _log(rng, 1, 48)
        hi = _log(rng, 2, min(65536, 500000000 // (B * H * D)))
        keep = rng.randint(max(1, hi // 4), hi)
        first, last = min(rng.choice((0, 1, 4, 32)), keep // 2), min(rng.choice((0, 16, 61, 128)), keep // 2)
        return dict(op=op, B=B, H=H, D=D, G=G, lo=rng.choice((hi, rng.randint(0, hi))), hi=hi, keep=keep, first=first,
                    last=last)
    Hkv = rng.choice((1, 2, 4, 8, 8, 16))
    gq = rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 12, 16))
    kind = rng.choice(("one", "one", "few", "chunk"))
    T = 1 if kind == "one" else rng.randint(2, 9) if kind == "few" else _log(rng, 10, 1000)
    same = dict(op=op, T=T, Hq=Hkv * gq, Hkv=Hkv, D=D, G=G, causal=rng.random() < 0.8, ragged=T > 1 and rng.random() < 0.4,
                dtype=rng.choice(("float16", "bfloat16")))
    if op == "weighed":
        B = _log(rng, 1, 96 if kind == "one" else 16 if kind == "few" else 6)
        # tokens in the cache: at most a 1 GB of codes, and of the plain form's scores a quarter of the largest case's
        most = max(2, min(65536, 500000000 // (B * Hkv * D), 300000000 // (B * Hkv * gq * T)))
        hi = _log(rng, max(1, min(T, most - 1)), most)
        return dict(same, B=B, lo=rng.choice((hi, rng.randint(0, hi))), hi=hi)
    F = rng.choice((1, 1, 1, 2, 3, 5))
    B = F * _log(rng, 1, 64 if kind == "one" else 16 if kind == "few" else 4)
    rows = B * Hkv * gq * T
    most = max(2, min(65536, 400000000 // (F * Hkv * D), 300000000 // rows))
    phi = _log(rng, 1, most)
    hi = _log(rng, 1, max(2, min(4096, 200000000 // (B * Hkv * D), 300000000 // rows)))
    return dict(same, F=F, B=B, plo=rng.choice((phi, rng.randint(0, phi))), phi=phi, lo=rng.choice((hi, rng.randint(0, hi))),
                hi=hi)


# ------------------------------------------------------------ a case's lengths

def _spread(lo, hi, B):
    """B lengths spread evenly over lo .. hi."""
    return [hi] if B == 1 else [lo + (hi - lo) * b // (B - 1) for b in range(B)]


def _rows(case):
    """Real rows of each sequence of a padded batch: all of them, or T / 3 to T."""
    B, T = case["B"], case["T"]
    return _spread(max(1, T // 3), T, B)[::-1] if case["ragged"] else [T] * B


def _width(case):
    """Positions that a weight is kept for: what the longest table row holds."""
    return max(1, -(-case["hi"] // case["G"])) * case["G"]


def _seen(n, t, causal):
    """Tokens that the t last queries of n tokens see, summed."""
    return sum(max(0, n - t + 1 + i) for i in range(t)) if causal else t * n


def work(case):
    B, D, G = case["B"], case["D"], case["G"]
    lens = _spread(case["lo"], case["hi"], B)
    if case["op"] == "evict":
        H, N = case["H"], _width(case)
        kept = [min(n, case["keep"]) for n in lens]
        codes = 2 * sum(kept) * H * D
        pages = sum(-(-n // G) + -(-m // G) for n, m in zip(lens, kept))
        return {"bytes": 2 * codes + 8 * pages * H + 4 * H * (sum(lens) + B * N + B * min(case["keep"], N)),
                "flops": H * sum(lens)}
    Hq, Hkv = case["Hq"], case["Hkv"]
    rows = _rows(case)
    held = list(lens)
    if case["op"] == "shared":
        prefix = _spread(case["plo"], case["phi"], case["F"])
        each = B // case["F"]
        seen = sum(_seen(n + prefix[b // each], t, case["causal"]) for b, (n, t) in enumerate(zip(lens, rows)))
        held += prefix
        more = 0
    else:
        seen = sum(_seen(n, t, case["causal"]) for n, t in zip(lens, rows))
        more = 8 * Hkv * sum(lens)
    return {"bytes": sum(2 * n * Hkv * D + 8 * -(-n // G) * Hkv for n in held) + 4 * sum(rows) * Hq * D + more,
            "flops": 4 * D * Hq * seen}


# --------------------------------------------------------------------- inputs

def _pages(gen, n, H, G, D, keys, dev):
    """n filled pages: codes, and for each the smallest power of two as a scale with which they stay within 448."""
    x = torch.randn(n, H, G, D, generator=gen, device=dev)
    if keys:
        x[..., 5::16] *= 8.0
    m, e = torch.frexp(x.abs().amax((2, 3)))
    s = (torch.where(m <= 0.875, e - 9, e - 8) + 127 << 23).view(torch.float32)     # 448 = 0.875 * 2^9
    return (x / s[..., None, None]).to(E4M3), s


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(dev).manual_seed(seed)
    op, B, D, G = case["op"], case["B"], case["D"], case["G"]
    H = case.get("H") or case["Hkv"]
    lens = _spread(case["lo"], case["hi"], B)
    prefix = _spread(case["plo"], case["phi"], case["F"]) if op == "shared" else []
    target = [min(n, case["keep"]) for n in lens] if op == "evict" else []
    W = _width(case) // G
    counts = [-(-n // G) for n in lens]
    others = [-(-n // G) for n in (prefix or target)]
    P = sum(counts) + sum(others) + 3
    key, ks = _pages(gen, P, H, G, D, True, dev)
    value, vs = _pages(gen, P, H, G, D, False, dev)
    order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)     # pages lie anywhere in the pool
    at = 0

    def table(counts, width):
        nonlocal at
        t = torch.zeros(len(counts), width, dtype=torch.int32, device=dev)
        for b, n in enumerate(counts):
            t[b, :n] = order[at:at + n]
            at += n
        return t

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    state = dict(case=case, key=key, value=value, scale=torch.stack((ks, vs), -1).contiguous(), table=table(counts, W),
                 lens=i32(lens))
    if op == "evict":
        state["into"] = table(others, max(1, -(-min(case["keep"], W * G) // G)))
        w = torch.randn(B, H, W * G, generator=gen, device=dev).mul_(2.5).exp_()
        w = torch.where(w < 0.03, torch.zeros_like(w), w)           # a tenth of them never got any
        state["weights"] = w * (torch.arange(W * G, device=dev) < state["lens"][:, None, None])
    else:
        T, rows = case["T"], _rows(case)
        state["q"] = torch.randn(B, case["Hq"], T, D, generator=gen, device=dev).to(DTYPES[case["dtype"]])
        state["q_lens"] = i32(rows) if rows != [T] * B else None
        if op == "shared":
            state["prefix_table"], state["prefix_lens"] = table(others, max(others + [1])), i32(prefix)
        else:       # as much as a call adds, from those before it
            state["weights"] = torch.rand(B, H, W * G, generator=gen, device=dev) * (case["Hq"] // H * T / max(1, case["hi"]))
    if own:     # the handle that a program keeps with its pools
        pkg = os.path.join(os.getcwd(), "kitty-kv_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from kitty.kernels import Cache8
        state["cache"] = Cache8(state["key"], state["value"], state["scale"])
    return state


# ------------------------------------------------------------------ the passes

def run(state):
    case = state["case"]
    if case["op"] == "shared":
        if own:
            return state["cache"].attend_shared(state["q"], state["prefix_table"], state["prefix_lens"], state["table"],
                                                state["lens"], q_lens=state["q_lens"], causal=case["causal"])
        return _shared(state)
    if case["op"] == "weighed":
        if own:
            out = state["cache"].attend_weighed(state["q"], state["table"], state["lens"], state["weights"],
                                                q_lens=state["q_lens"], causal=case["causal"])
        else:
            out = _weighed(state)
        return {"out": out, "weights": state["weights"]}
    if own:
        lens, kept, weights = state["cache"].evict(state["table"], state["lens"], state["weights"], case["keep"],
                                                   first=case["first"], last=case["last"], into=state["into"])
    else:
        lens, kept, weights = _evict(state)
    return {"key": state["key"], "value": state["value"], "scale": state["scale"], "lens": lens, "kept": kept,
            "weights": weights}


def _tokens(state, table):
    """Keys and values of the tables' pages in float32, (B, H, W G, D) each."""
    B, W = table.shape
    H, G, D = state["key"].shape[1:]
    table = table.long()
    both = []
    for i, pool in enumerate((state["key"], state["value"])):
        x = pool.view(torch.uint8)[table].view(E4M3).float() * state["scale"][table][..., i, None, None]
        both.append(x.transpose(1, 2).reshape(B, H, W * G, D))
    return both


def _ends(state, n, before):
    """(B, T, 1): tokens that each row sees of sequences of n tokens, `before` of them in front of those in question."""
    case = state["case"]
    T = case["T"]
    rows = torch.full_like(n, T) if state["q_lens"] is None else state["q_lens"]
    i = torch.arange(T, device=n.device)
    end = n[:, None] - rows[:, None] + i + 1 if case["causal"] else n[:, None].expand(-1, T)
    return torch.where(i < rows[:, None], end - before[:, None], torch.zeros_like(end))[..., None]


def _softmax(s):
    """exp(s - max) and what it sums to, over the last axis; a row of -inf sums to 0."""
    top = s.amax(-1, keepdim=True)
    return top, s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()


def _shared(st):
    case, q = st["case"], st["q"]
    B, Hq, T, D = q.shape
    F, H = case["F"], case["Hkv"]
    m, gq, dev = B // F, Hq // H, q.device
    pk, pv = _tokens(st, st["prefix_table"])
    k, v = _tokens(st, st["table"])
    L, N = pk.shape[2], k.shape[2]
    before = st["prefix_lens"].repeat_interleave(m)
    total = before + st["lens"]
    qs = q.float().view(F, m, H, gq, T, D)
    # scores over the prefix, its rows those of all its sequences, and over what is theirs: (B, H, gq, T, tokens)
    s = (qs.transpose(1, 2).reshape(F, H, m * gq * T, D) @ pk.transpose(2, 3)).view(F, H, m, gq, T, L).transpose(1, 2)
    s = s.reshape(B, H, gq, T, L)
    s = torch.cat((s, (qs.reshape(B, H, gq * T, D) @ k.transpose(2, 3)).view(B, H, gq, T, N)), -1).div_(math.sqrt(D))
    j, zero = torch.arange(L, device=dev), torch.zeros_like(before)
    sees = torch.cat((j < torch.minimum(_ends(st, total, zero), before[:, None, None]),
                      torch.arange(N, device=dev) < _ends(st, total, before)), -1)
    _, p = _softmax(s.masked_fill_(~sees[:, None, None], -math.inf))
    sums = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(sums == 0, torch.ones_like(sums), sums))
    out = (p[..., :L].view(F, m, H, gq, T, L).transpose(1, 2).reshape(F, H, m * gq * T, L) @ pv).view(F, H, m, gq, T, D)
    out = out.transpose(1, 2).reshape(B, H, gq * T, D) + p[..., L:].reshape(B, H, gq * T, N) @ v
    return out.reshape(B, Hq, T, D).to(q.dtype)


def _weighed(st):
    q = st["q"]
    B, Hq, T, D = q.shape
    k, v = _tokens(st, st["table"])
    H, N = k.shape[1:3]
    gq = Hq // H
    sees = torch.arange(N, device=q.device) < _ends(st, st["lens"], torch.zeros_like(st["lens"]))
    s = (q.float().reshape(B, H, gq * T, D) @ k.transpose(2, 3)).view(B, H, gq, T, N) / math.sqrt(D)
    _, p = _softmax(s.masked_fill_(~sees[:, None, None], -math.inf))
    sums = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(sums == 0, torch.ones_like(sums), sums)).view(B, H, gq * T, N)
    st["weights"] += p.sum(2)
    return (p @ v).view(B, Hq, T, D).to(q.dtype)


def _evict(st):
    case, w, n = st["case"], st["weights"], st["lens"].long()
    B, H, N = w.shape
    G, dev = case["G"], w.device
    K = min(case["keep"], N)
    pos = torch.arange(N, device=dev)
    held = pos < n[:, None]
    stays = held & ((pos < case["first"]) | (pos >= n[:, None] - case["last"]))
    # by class (stays, may go, not there), then weight, then position
    kind = (held.int() + stays.int())[:, None].expand(B, H, N)
    order = w.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(2, kind.gather(2, order).sort(dim=-1, descending=True, stable=True).indices)
    count = n.clamp(max=case["keep"])
    here = torch.arange(K, device=dev) < count[:, None, None]                       # (B, 1, K)
    kept = torch.where(here, order[..., :K], torch.full_like(order[..., :K], N)).sort(-1).values
    here = here.expand(B, H, K)
    source = torch.where(here, kept, torch.zeros_like(kept))
    weights = torch.zeros_like(w)
    weights[..., :K] = torch.where(here, w.gather(2, source), torch.zeros_like(w[..., :K]))
    # a row of tokens for every page of `into`
    pages = st["into"].shape[1]
    pad = lambda x: torch.nn.functional.pad(x, (0, pages * G - K)).view(B, H, pages, G)  # noqa: E731
    source, here = pad(source), pad(here)
    b, h = torch.arange(B, device=dev)[:, None, None, None], torch.arange(H, device=dev)[:, None, None]
    page = st["table"].long()[b, source // G]
    b, h, at, row = (x.expand_as(here)[here] for x in (b, h, st["into"].long()[:, None, :, None], torch.arange(G, device=dev)))
    filled = here.any(-1)
    to = st["into"].long()[:, None].expand(B, H, pages)[filled]
    heads = torch.arange(H, device=dev)[:, None].expand(B, H, pages)[filled]
    for i, pool in enumerate((st["key"], st["value"])):
        was = st["scale"][page, torch.arange(H, device=dev)[:, None, None], i]       # (B, H, pages, G)
        s = torch.where(here, was, torch.zeros_like(was)).amax(-1, keepdim=True)
        factor = (was / s)[here][:, None]
        codes = pool.view(torch.uint8)[page[here], h, (source % G)[here]].view(E4M3).float() * factor
        pool.view(torch.uint8)[at, h, row] = codes.to(E4M3).view(torch.uint8)
        st["scale"][to, heads, i] = s[filled][:, 0]
    return count.int(), torch.where(kept == N, torch.full_like(kept, -1), kept).int(), weights


# ---------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(st)
    dev, G, T = st["key"].device, case["G"], case["T"]
    q = st["q"].double()
    H, gq = case["Hkv"], case["Hq"] // case["Hkv"]
    lens = _spread(case["lo"], case["hi"], case["B"])
    rows = _rows(case)

    def tokens(table, n):
        """The n tokens of a table's row, (H, n, D) twice in float64."""
        ids = table[:-(-n // G)].long()
        both = []
        for i, pool in enumerate((st["key"], st["value"])):
            x = pool.view(torch.uint8)[ids].view(E4M3).double() * st["scale"][ids][..., i, None, None].double()
            both.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
        return both

    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    weights = st["weights"].double() if case["op"] == "weighed" else None
    for b in range(case["B"]):
        parts, t = [tokens(st["table"][b], lens[b])], rows[b]
        if case["op"] == "shared":
            f = b // (case["B"] // case["F"])
            parts = [tokens(st["prefix_table"][f], _spread(case["plo"], case["phi"], case["F"])[f])] + parts
        k, v = (torch.cat([p[i] for p in parts], 1) for i in range(2))
        n = k.shape[1]
        if n == 0:
            continue
        hidden = None
        if case["causal"]:      # row i is token n - t + i
            hidden = torch.arange(n, device=dev) > torch.arange(n - t, n, device=dev)[:, None]
        for h in range(H):
            x = q[b, h * gq:(h + 1) * gq, :t].reshape(gq * t, -1) @ k[h].t() * case["D"] ** -0.5
            x = x.view(gq, t, n)
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
            out[b, h * gq:(h + 1) * gq, :t] = (p.view(gq * t, n) @ v[h]).view(gq, t, -1)
            if weights is not None:
                weights[b, h, :n] += p.sum((0, 1))
    return out if weights is None else {"out": out, "weights": weights}


def _round_e4m3(y):
    """y (float64, |y| <= 448) to the nearest e4m3 value, ties to the even one: steps of
    2^(e - 3) for 2^e <= |y| < 2^(e + 1), of 2^-9 below 2^-6."""
    e = (torch.frexp(y)[1] - 1).clamp(min=-6) - 3
    step = (e.long() + 1023 << 52).view(torch.float64)
    return torch.round(y / step) * step


def _exact_evict(st):
    case = st["case"]
    G, H, dev = case["G"], case["H"], st["key"].device
    w = st["weights"].double()
    N = w.shape[2]
    lens = _spread(case["lo"], case["hi"], case["B"])
    kept = torch.full((case["B"], H, min(case["keep"], N)), -1, dtype=torch.int32, device=dev)
    weights = torch.zeros_like(w)
    pools = [st["key"].double(), st["value"].double()]
    scale = st["scale"].double()
    new = [x.clone() for x in pools], scale.clone()
    heads = torch.arange(H, device=dev)[:, None]
    for b, n in enumerate(lens):
        m = min(n, case["keep"])
        stay = torch.ones(H, n, dtype=torch.bool, device=dev)
        if n > m:
            # positions in the order in which they would go: by weight, the later of equals first
            mid = w[b, :, case["first"]:n - case["last"]].flip(-1)
            gone = mid.sort(dim=-1, stable=True).indices[:, :n - m]
            stay[heads, n - case["last"] - 1 - gone] = False
        at = stay.nonzero()[:, 1].view(H, m)
        kept[b, :, :m] = at.int()
        weights[b, :, :m] = w[b].gather(1, at)
        for page in range(-(-m // G)):
            src = at[:, page * G:(page + 1) * G]
            ids, to = st["table"][b].long()[src // G], int(st["into"][b, page])
            for i in range(2):
                was = scale[ids, heads, i]
                top = was.amax(1)
                new[0][i][to, :, :src.shape[1]] = _round_e4m3(pools[i][ids, heads, src % G] * (was / top[:, None])[..., None])
                new[1][to, :, i] = top
    return {"key": new[0][0], "value": new[0][1], "scale": new[1],
            "lens": torch.tensor([min(n, case["keep"]) for n in lens], dtype=torch.int32, device=dev), "kept": kept,
            "weights": weights}
