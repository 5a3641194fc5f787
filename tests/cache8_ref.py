"""The 8-bit paged cache in float64 numpy, straight from its definition, for its
tests: e4m3 by its 256 values, pages and scales token by token, attention row by
row."""
import numpy as np
import torch

NAN = 0x7F


def _value(c):
    e, m = c >> 3 & 15, c & 7
    if e == 15 and m == 7:
        return np.nan
    x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    return -x if c & 0x80 else x


VALUES = np.array([_value(c) for c in range(256)])
_POS = VALUES[:127]              # 0 .. 448, ascending; odd index = odd mantissa


def encode(y):
    """Nearest e4m3 code of float64 values within +-448, ties to the even code; NaN and infinities -> NAN."""
    y = np.asarray(y, np.float64)
    a = np.where(np.isfinite(y), np.abs(y), 0.0)
    hi = np.searchsorted(_POS, a).clip(0, 126)
    lo = (hi - 1).clip(0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(np.signbit(y), c | 0x80, c)
    return np.where(np.isfinite(y), c, NAN).astype(np.uint8)


def scale_for(m):
    s = 2.0 ** -64
    while m > 448.0 * s:
        s *= 2
    return s


class Ref:
    """numpy copy of a cache's pools."""

    def __init__(self, cache):
        self.pools = [t.view(torch.uint8).cpu().numpy().copy() for t in (cache.key, cache.value)]
        self.scale = cache.scale.cpu().numpy().astype(np.float64)
        self.P, self.H, self.G, self.D = self.pools[0].shape

    def page(self, table, b, number):
        if not 0 <= number < table.shape[1]:
            return -1
        p = int(table[b, number])
        return p if 0 <= p < self.P else -1

    def write(self, k, v, table, start, lens=None):
        B, H, T, D = k.shape
        for st, x in enumerate((k, v)):
            for b in range(B):
                n = T if lens is None else min(max(int(lens[b]), 0), T)
                t = 0 if start[b] >= 0 else n
                while t < n:
                    number, row = divmod(int(start[b]) + t, self.G)
                    m = min(self.G - row, n - t)
                    p = self.page(table, b, number)
                    if p >= 0:
                        for h in range(H):
                            self._rows(st, p, h, row, x[b, h, t:t + m])
                    t += m

    def _rows(self, st, p, h, row, x):
        fin = np.abs(x[np.isfinite(x)])
        s = scale_for(fin.max() if fin.size else 0.0)
        pool, was = self.pools[st][p, h], self.scale[p, h, st]
        if row:
            s = max(s, was)
            if s != was:
                pool[:row] = encode(VALUES[pool[:row]] * np.float64(np.float32(was / s)))
        pool[row:row + len(x)] = encode(x / s)
        self.scale[p, h, st] = s

    def tokens(self, table, b, first, end):
        """Tokens first .. end - 1 of sequence b: (2, H, n, D), NaN without a page."""
        out = np.full((2, self.H, max(end - first, 0), self.D), np.nan)
        for i in range(out.shape[2]):
            p = self.page(table, b, (first + i) // self.G)
            if p >= 0 and first + i >= 0:
                for st in range(2):
                    out[st, :, i] = VALUES[self.pools[st][p, :, (first + i) % self.G]] * self.scale[p, :, st, None]
        return out

    def read(self, table, lens, tokens, start=None):
        B = len(lens)
        out = np.zeros((2, B, self.H, tokens, self.D))
        for b in range(B):
            s = 0 if start is None else int(start[b])
            n = min(max(int(lens[b]) - s, 0), tokens)
            out[:, b, :, :n] = self.tokens(table, b, s, s + n)
        return out

    def attend(self, q, table, lens, q_lens=None, causal=True, sm_scale=None):
        """(out, lse, spread, mag, small): spread = softmax @ |v|, the size of what the sums
        add up; mag the largest sum of |q k| * sm_scale of a row; small = the largest weight
        times value scale, times the sum of |code|, of a channel."""
        B, Hq, T, D = q.shape
        sm = D ** -0.5 if sm_scale is None else sm_scale
        gq = Hq // self.H
        out, spread, small = np.zeros((3, B, Hq, T, D))
        lse = np.full((B, Hq, T), -np.inf)
        mag = np.zeros((B, Hq, T))
        for b in range(B):
            n, t = int(lens[b]), T if q_lens is None else int(q_lens[b])
            if n < 0 or n > table.shape[1] * self.G or not 0 <= t <= T:
                out[b], lse[b] = np.nan, np.nan
                continue
            kv = self.tokens(table, b, 0, n)
            ids = [self.page(table, b, i // self.G) for i in range(n)]
            for h in range(Hq):
                k, v, vs = kv[0, h // gq], kv[1, h // gq], self.scale[ids, h // gq, 1]
                for i in range(t):
                    e = n - t + i + 1 if causal else n
                    if e <= 0:
                        continue
                    with np.errstate(invalid="ignore"):
                        s = k[:e] @ q[b, h, i] * sm
                        w = np.exp(s - s.max())
                        lse[b, h, i] = s.max() + np.log(w.sum())
                        w /= w.sum()
                        out[b, h, i] = w @ v[:e]
                        spread[b, h, i] = w @ np.abs(v[:e])
                        small[b, h, i] = np.max(w * vs[:e]) * (np.abs(v[:e]) / vs[:e, None]).sum(0)
                        mag[b, h, i] = np.nanmax(np.abs(k[:e]) @ np.abs(q[b, h, i]) * sm, initial=0.0)
        return out, lse, spread, mag, small


def tolerance(dtype, ref, spread, mag, small, rows, D, n):
    """How far an attention output may be off: half a step of its type, and of what the
    sums add up the errors of the weights:
    * twice (weight and total) fp32's: scores of D products and sums and 6 factors, 2^-24
      of `mag` each, an exponent's absolute error being the weight's relative one; exp2 and
      the logarithm of a scale, 2^-20 together (log2 is exact for powers of two, and off by
      2^-24 of 8 at most for the others here); sums of n weights, n 2^-24;
    * the weights' own: two bf16 terms, the first off by half a step, 2^-8 of the weight,
      the second by 2^-8 of that rest: 2^-16; for bf16 and more than 64 rows of a KV head
      (32 at more than 128 channels) one fp16 term, 2^-11, and where a weight lies below
      fp16's normal numbers 2^-25 of the largest weight times its scale, on every code."""
    half = torch.finfo(dtype).eps / 2
    one = dtype == torch.bfloat16 and rows > (64 if D <= 128 else 32)
    w = 2 * ((D + 6) * 2.0 ** -24 * mag + 2.0 ** -20 + n * 2.0 ** -24) + (2.0 ** -11 if one else 2.0 ** -16)
    return (half * np.abs(ref) + w[..., None] * spread + (2.0 ** -25 * small if one else 0.0)
            + float(torch.finfo(dtype).smallest_normal) * half * 2)


def numpy(t):
    return t.detach().cpu().double().numpy()
