// Attention of few query rows over the 8-bit paged cache, on gfx950: the
// decode step, and the few tokens of a draft.
//
// Bound by HBM: every code is read once for all the query rows of its KV head
// (head of the group fastest, up to 16 RT rows), at two bytes per token and
// channel.  The work of a batch is its (sequence, KV head) pairs in units of
// 128 tokens, cut into equal runs of units for the workgroups by lengths read
// on the device, so ragged batches stay even.  A workgroup's four waves take 32
// tokens of a unit each, independently (codes HBM -> registers, one step
// ahead), and join in LDS at the end of a pair's run; runs that are not the
// whole of a pair leave a partial that cache8_merge_kernel joins.
//
//  S^T = K Q^T, 16x16x32 MFMAs: A row = token, reduction slot (g, j) of step
//  2c + u = channel 64c + 16g + 8u + j, so a lane reads 16 contiguous codes per
//  64 channels, widened to q's type (exact).  Lane (n = query l & 15, g = l / 16)
//  ends with its query's scores of tokens 4g .. 4g + 3 of each 16-token half.
//  O^T += V^T P^T: the scores' registers are the B operand as they stand, slot
//  8g + e standing for token 4g + e (e < 4) of the first half, 4g + e - 4 of the
//  second.  A lane reads those eight tokens' rows at D / 16 contiguous channels,
//  so A row m of product dt is channel (D / 16) m + dt, and a byte permute
//  pairs two tokens' codes before they are widened to bf16.
//
// Scales: the key's is a factor of the scores, the value's of the weights,
// which go in two bf16 terms: 16 bits (error at most 2^-16) with fp32's range, as
// a page's scale may be anything.  The running maximum is raised only when a score passes it
// by 2^8.
//
// Measured: 16 x 32,768 tokens, 32 query / 8 KV heads of 128, fp16: 168 us, 6.4
// TB/s (the arithmetic alone takes 64, the loads alone as long as both); 64 x
// 512-16,384, 64 / 8, bf16, pages of 32: 187 us, 5.9 TB/s; five queries of 8 x
// 4-20K: 44 us.  Streaming loads were worth 5 % of the first, a second step in
// flight 4 %; a third and fourth, 3 or 4 workgroups a CU, runs per wave instead of
// interleaved steps and lanes that read 1 KB runs nothing or less.
#pragma once
#include "attend8.h"

namespace kitty {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;

template <int DP, int RT>
struct RowBuf {
    u32x4 k[2][DP / 64];
    unsigned v[8][DP / 64];
    float2 sc[2];
};

template <int DP, int RT>
struct RowState {
    u32x4 q[RT][DP / 32];
    f32x4 o[RT][DP / 16];
    float m[RT], l[RT];
    int vis[RT];
};

// Max and sum over the four lanes of one query (16 apart).
__device__ __forceinline__ float quad_max(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, (int)a[0]), __builtin_bit_cast(float, (int)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
}
__device__ __forceinline__ float quad_sum(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return __builtin_bit_cast(float, (int)b[0]) + __builtin_bit_cast(float, (int)b[1]);
}

// Value operand of product dt: the lane's eight tokens at channel dt of its
// D / 16, each byte picked by (tokens 2e, 2e + 1) pairs and widened.  COUNT: 1
// in the place of NaN codes and 0 elsewhere.
template <int DP, bool COUNT>
__device__ __forceinline__ u32x4 value_operand(const unsigned (&v)[8][DP / 64], int dt)
{
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned a = v[2 * e][dt >> 2], b = v[2 * e + 1][dt >> 2];
        // bytes (a.c, b.c, a.c + 1, b.c + 1) with c = dt & 2; both channels of the pair share the permute
        unsigned w = __builtin_amdgcn_perm(b, a, dt & 2 ? 0x07030602u : 0x05010400u);
        if constexpr (COUNT)
            w = (nan_codes(w) >> 7) * 0x38u;
        r[e] = dt & 1 ? widen<true, true>(w) : widen<true, false>(w);
    }
    return r;
}

// 32 tokens from `tok` on, in `buf`, folded into the wave's rows.  mask: some
// row may not see all of them.
// LEAVE: the scores go as well, at byte `at` plus `step` for every 16 tokens, to `out` (1),
// where the store itself drops what is beyond its end (lanes without a row, tokens that
// have no weight): a branch around it would make every wait one for all loads; or to
// `stage` (2).
template <int DP, int RT, bool BF16, int LEAVE>
__device__ __forceinline__ void row_step(RowState<DP, RT> &W, RowBuf<DP, RT> &buf, int tok, int vis_max, float cs, int g, bool mask,
                                         __amdgpu_buffer_rsrc_t out, unsigned char *stage, uint32_t at, uint32_t step)
{
    f32x4 S[RT][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            S[rt][hf] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned w0 = buf.k[hf][c][2 * u], w1 = buf.k[hf][c][2 * u + 1];
                const u32x4 a = {widen<BF16, false>(w0), widen<BF16, true>(w0), widen<BF16, false>(w1), widen<BF16, true>(w1)};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    S[rt][hf] = mfma16<BF16>(a, W.q[rt][2 * c + u], S[rt][hf]);
            }
    }
    // a token's row in the registers: half e / 4, token 4g + e % 4 of it
    bool odd = false;
    if (mask) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int t = tok + 16 * (e >> 2) + 4 * g + (e & 3);
#pragma unroll
            for (int w = 0; w < DP / 64; ++w) {
                buf.v[e][w] = t < vis_max ? buf.v[e][w] : 0;   // rows no query sees hold anything
                odd |= nan_codes(buf.v[e][w]) != 0;
            }
        }
        odd = __ballot(odd) != 0;
    }
    u32x4 hi[RT], lo[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            s[e] = S[rt][e >> 2][e & 3] * (cs * buf.sc[e >> 2].x);
        if (mask)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                s[e] = tok + 16 * (e >> 2) + 4 * g + (e & 3) < W.vis[rt] ? s[e] : -__builtin_inff();
        if constexpr (LEAVE == 2) {
            if (at < 1u << 31)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    *(float4 *)(stage + at + hf * step) = make_float4(s[4 * hf], s[4 * hf + 1], s[4 * hf + 2], s[4 * hf + 3]);
        }
        if constexpr (LEAVE == 1) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                __builtin_amdgcn_raw_buffer_store_b128(
                    u32x4{__builtin_bit_cast(unsigned, s[4 * hf]), __builtin_bit_cast(unsigned, s[4 * hf + 1]),
                          __builtin_bit_cast(unsigned, s[4 * hf + 2]), __builtin_bit_cast(unsigned, s[4 * hf + 3])},
                    out, at + hf * step, 0, 0);
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 8; ++e)
            mx = fmaxf(mx, s[e]);
        if (__ballot(mx > W.m[rt] + 8.0f)) {
            mx = quad_max(mx);
            const float mn = mx > W.m[rt] + 8.0f ? mx : W.m[rt], alpha = __builtin_amdgcn_exp2f(W.m[rt] - mn);
            W.m[rt] = mn;
            W.l[rt] *= alpha;
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt)
                W.o[rt][dt] *= alpha;
        }
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] - W.m[rt]);
            sum += s[e];
            s[e] *= buf.sc[e >> 2].y;
        }
        W.l[rt] += sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            unsigned h, l;
            split_bf16(s[2 * e], s[2 * e + 1], h, l);
            hi[rt][e] = h, lo[rt][e] = l;
        }
    }
    if (odd) {
        // NaN values that not every row sees: count them by row and channel
        // (products of 0 / 1), give those rows NaN and take them out of the codes.
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            u32x4 see;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = tok + 16 * (e >> 1) + 4 * g + 2 * (e & 1);
                see[e] = (t < W.vis[rt] ? 0x3f80u : 0u) | (t + 1 < W.vis[rt] ? 0x3f800000u : 0u);
            }
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                const f32x4 cnt = mfma16<true>(value_operand<DP, true>(buf.v, dt), see, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    W.o[rt][dt][i] = cnt[i] > 0.0f ? __builtin_nanf("") : W.o[rt][dt][i];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int w = 0; w < DP / 64; ++w)
                buf.v[e][w] &= ~((nan_codes(buf.v[e][w]) >> 7) * 0xffu);
    }
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
        const u32x4 vf = value_operand<DP, false>(buf.v, dt);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            W.o[rt][dt] = mfma16<true>(vf, hi[rt], W.o[rt][dt]);
            W.o[rt][dt] = mfma16<true>(vf, lo[rt], W.o[rt][dt]);
        }
    }
}

// Tiles of kUnit tokens of a sequence.
__device__ __forceinline__ int tiles8(const Seq8 &s) { return s.bad ? 0 : (s.n + kUnit - 1) / kUnit; }

// Units of one (KV head, row block) of a sequence: its tiles, and what beginning it
// costs a run that has another part already, `start` tiles' time: 2 (64 ragged
// sequences 206 -> 199 us, 8 with five queries 54.6 -> 52.4; 1, 3 and 4 take 199.2,
// 199.5, 200.9 and 53.1, 52.2, 52.3), 0 where the runs end with the pairs anyway.
constexpr int kStart = 2;
__device__ __forceinline__ int units8(int tiles, int start) { return tiles ? tiles + start : 0; }

// This workgroup's run of the batch's units.
struct Run8 {
    int total, N;      // all units, workgroups that share them
    int u, u1;         // the run's next unit and its end
    int b, pre;        // the sequence of unit u and its first unit
    int start;         // units that beginning a (KV head, row block) counts
};

// First unit of workgroup w: total units shared evenly, the first total % N
// workgroups taking one more.
__device__ __forceinline__ int run_start(int total, int N, int w)
{
    const int each = total / N, more = total - each * N;
    return w * each + min(w, more);
}

// The workgroup that has unit u.
__device__ __forceinline__ int run_of(int total, int N, int u)
{
    const int each = total / N, more = total - each * N, cut = more * (each + 1);
    return u < cut ? u / (each + 1) : more + (u - cut) / each;
}

// (KV head, row block)s of an entry, and the number of its first among all.
template <bool SHARED>
__device__ __forceinline__ int items8(const Attend8 &p, int i)
{
    return p.c.H * (SHARED && p.e0 + i >= p.F ? 1 : p.nrb);
}
__device__ __forceinline__ int first_item8(const Attend8 &p, int i)   // SHARED
{
    return p.e0 + i >= p.F ? p.item0 + (p.e0 + i - p.F) * p.c.H : i * p.c.H * p.nrb;
}

template <bool SHARED>
__device__ __forceinline__ bool find_run(const Attend8 &p, Run8 &R, int wg, int n_wg)
{
    const int lane = threadIdx.x & 63;
    const int B = SHARED ? p.entries : p.B;
    // 64 sequences at a time: tiles of each, units of each and the sum up to it
    auto tiles = [&](int b0) { return b0 + lane < B ? tiles8(entry8<SHARED>(p, b0 + lane)) : 0; };
    auto sums = [&](int b0, int t, int &x) {
        x = units8(t, R.start) * items8<SHARED>(p, b0 + lane);
        int inc = x;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int y = __shfl_up(inc, off);
            inc += lane >= off ? y : 0;
        }
        return inc;
    };
    // equal sequences whose pairs the workgroups divide evenly: no run begins a second one
    int t = tiles(0);
    const int each = __builtin_amdgcn_readlane(t, 0), items = B * p.c.H * p.nrb;
    const int N0 = (int)min((int64_t)n_wg, (int64_t)each * items);
    R.start = kStart;
    if (!SHARED && B <= 64 && N0 > 0 && N0 % items == 0 && !__ballot(lane < B && t != each))
        R.start = 0;
    int x, inc = sums(0, t, x), total = __builtin_amdgcn_readlane(inc, 63);
    for (int b0 = 64; b0 < B; b0 += 64) {
        int y;
        total += __builtin_amdgcn_readlane(sums(b0, tiles(b0), y), 63);
    }
    R.total = total;
    R.N = min(n_wg, total);
    if (wg >= R.N)
        return false;
    R.u = run_start(total, R.N, wg);
    R.u1 = run_start(total, R.N, wg + 1);
    // (the bounds here and below are for lengths that another stream changes under the
    // call: it then gives anything, and ends)
    for (int b0 = 0, base = 0; b0 < B;) {
        const unsigned long long past = __ballot(base + inc > R.u);
        if (past) {
            const int l = __builtin_ctzll(past);
            R.b = b0 + l;
            R.pre = base + __builtin_amdgcn_readlane(inc - x, l);
            return true;
        }
        base += __builtin_amdgcn_readlane(inc, 63);
        b0 += 64;
        inc = sums(b0, tiles(b0), x);
    }
    return false;
}

// Waves of the row kernel's workgroup: 4 for the runs of the split; where it takes the
// whole of one (pair, row block) (DIRECT), 16 of one block of rows, each with one step's
// codes in its 128 registers (8 waves with two steps: 1 x 512 tokens 7.9 us against 7.0,
// 64 x 512 18.0 against 16.1), 8 of two.
constexpr int row_waves(int RT, bool direct) { return !direct ? kWaves : RT == 1 ? 16 : 8; }

// Whether two workgroups' registers and LDS fit a CU.
constexpr bool two_per_cu(int DP, int RT) { return DP <= 128 && DP * RT <= 256; }

// Adds to the weights of tokens tok .. tok + 3 (tok a multiple of four) the sum over up to
// 16 rows of 2^(score - top) / sum, from the scores that a kScores launch left.  vis: how
// many tokens each row sees, 0 behind the last row.  Four rows' scores at a time: read one
// by one the loads' latency was half of a short call (16 rows of 1,024 tokens 15.8 us / 13.0
// in one launch, 27.7 / 14.7 split; four rows of 16 x 32,768 250.7 / 245.6).
__device__ __forceinline__ void weigh_scores4(const float *scores, int rows, const float2 *stat, const int *vis, int tok, int tokens,
                                              float *weights)
{
    const float *s = scores + (int64_t)(tok >> 4) * 16 * rows + (tok & 15);
    float was[4], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        was[e] = tok + e < tokens ? weights[tok + e] : 0.0f;
    for (int r0 = 0; r0 < rows; r0 += 4) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = *(const float4 *)(s + 16 * min(r0 + i, rows - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 st = stat[r0 + i];
            const int v = vis[r0 + i];
            const float xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float with = __builtin_fmaf(__builtin_amdgcn_exp2f(xs[e] - st.x), st.y, sum[e]);
                sum[e] = tok + e < v ? with : sum[e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (tok + e < tokens)
            weights[tok + e] = was[e] + sum[e];
}

// CUT: D is below DP, and the lanes beyond it read nothing.  DIRECT: a workgroup takes
// the whole of one (pair, row block) and writes its rows, so that no merge follows.
// MODE kShared: the entries are prefixes and sequences, the latter of one row block each,
// and all parts are left to cache8_join_kernel; with DIRECT the entries are sequences, and
// each reads its prefix itself.
//
// Workgroup wg of the n_wg that share the work.
// kScores: a stream of reads with writes in it runs at a copy's rate, though the scores of
// four rows are a sixteenth of its bytes: 16 x 32,768 tokens 229 us, 168 with the stores
// dropped (all of a pair's to the same 4 KB: 5 more; cache hints change nothing).  So a
// wave's scores wait in LDS, in what is its part of o afterwards, and leave in bursts, which
// workgroups with equal runs have at about the same time: 203 us.  Bytes that wait: the
// whole call 217 us at 20,064 (what two workgroups a CU allow), 218 at 16,896, 228 at
// 12,288, 234 at 8,448 and 246 unless they wait (another card: 222 and 249).
constexpr int kStage = 16896;

// Rows of a wave's part of o.
constexpr int row_lines(int DP, int RT, bool direct, int mode)
{
    return mode == kScores && !direct && kStage > 64 * RT * (DP + 4) ? (kStage + 4 * (DP + 4) - 1) / (4 * (DP + 4)) : 16 * RT;
}

template <int DP, int RT, bool DIRECT, int MODE>
struct RowLds {
    float o[row_waves(RT, DIRECT)][row_lines(DP, RT, DIRECT, MODE)][DP + 4];
    float2 ml[row_waves(RT, DIRECT)][16 * RT];
    float2 stat[DIRECT && RT == 1 ? 16 : 1];
    int vis[DIRECT && RT == 1 ? 16 : 1];
};

template <int DP, int RT, bool BF16, bool CUT, bool DIRECT, int MODE>
__device__ __forceinline__ void rows_run(const Attend8 &p, int wg, int n_wg, RowLds<DP, RT, DIRECT, MODE> &lds)
{
    constexpr bool SHARED = MODE == kShared, SCORES = MODE == kScores;
    constexpr int RM = 16 * RT, CB = DP / 16, NW = row_waves(RT, DIRECT), NB = NW == 16 ? 1 : 2, STRIDE = 32 * NW;
    auto &lds_o = lds.o;
    auto &lds_ml = lds.ml;
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_seq = p.c.H * p.nrb;   // SHARED: of a prefix
    Run8 R;
    if constexpr (DIRECT) {
        R.b = wg / per_seq;
        R.pre = 0, R.start = 0, R.u = wg - R.b * per_seq, R.u1 = R.u + 1;
    } else {
        if (!find_run<SHARED>(p, R, wg, n_wg))
            return;
    }
    const int u0 = R.u, u1 = R.u1;
    int u = R.u, b = R.b, pre = R.pre;

    while (u < u1 && b < (SHARED ? p.entries : p.B)) {
        const Seq8 sq = entry8<SHARED>(p, b);
        const int tiles = tiles8(sq), units = DIRECT ? tiles : units8(tiles, R.start);
        int item = u, seg = units, tile = 0, tile1 = tiles;                     // seg: units of this run's part
        bool first = true, last_part = true;                                    // whether it has the first and last tile
        if constexpr (!DIRECT) {
            if constexpr (SHARED) {
                const int items = items8<true>(p, b);
                if (u >= pre + units * items) {
                    pre += units * items;
                    ++b;
                    continue;
                }
            } else if (u >= pre + units * per_seq) {
                pre += units * per_seq;
                ++b;
                continue;
            }
            item = (u - pre) / units;
            const int off = (u - pre) - item * units;
            seg = min(units - off, u1 - u);
            if (off + seg <= R.start) {   // none of its tiles
                u += seg;
                continue;
            }
            first = off <= R.start, last_part = off + seg == units;
            tile = max(off - R.start, 0), tile1 = off + seg - R.start;
        }
        int nrb = p.nrb;
        if constexpr (SHARED)
            nrb = sq.prefix ? nrb : 1;
        const int kh = item / nrb, rb = item - kh * nrb, r0 = rb * RM;
        const int t_lo = r0 / p.gq, t_hi = min((r0 + RM - 1) / p.gq, sq.tq - 1);   // query tokens of the block
        int vis_min = visible8(p, sq, t_lo), vis_max = sq.bad || t_hi < t_lo ? 0 : visible8(p, sq, t_hi);

        RowState<DP, RT> W;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const Row8 row = row8<SHARED>(p, sq, b, kh, r0 + 16 * rt + n);
            W.vis[rt] = row.vis;
            if constexpr (SHARED) {
                if (sq.prefix) {
                    vis_min = rt == 0 ? sq.n : vis_min;
                    vis_min = row.real ? min(vis_min, row.vis) : vis_min;
                }
            }
            W.m[rt] = kLowest;
            W.l[rt] = 0.0f;
            const uint16_t *q = p.q + row.b * p.q_s_seq + row.h * p.q_s_head + row.t * p.q_s_tok;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const int ch = 64 * (c >> 1) + 16 * g + 8 * (c & 1);
                W.q[rt][c] = u32x4{0, 0, 0, 0};
                if (row.there && (!CUT || ch < p.c.D))
                    W.q[rt][c] = *(const u32x4 *)(q + ch);
            }
#pragma unroll
            for (int dt = 0; dt < CB; ++dt)
                W.o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if constexpr (SHARED) {
            if (sq.prefix) {
                vis_max = sq.bad ? 0 : sq.n;
#pragma unroll
                for (int off = 1; off < 16; off <<= 1)
                    vis_min = min(vis_min, __shfl_xor(vis_min, off));
                vis_min = __builtin_amdgcn_readfirstlane(vis_min);
            }
        }
        const int lg = p.c.lg;
        const uint8_t *kp = p.c.key + kh * p.c.key_s_head, *vp = p.c.value + kh * p.c.value_s_head;
        const float *sp = p.c.scale + kh * p.c.scale_s_head;
        const uint32_t k_lane = (uint32_t)n * p.c.key_s_tok + 16 * g;
        const uint32_t v_ch = CUT && CB * n >= p.c.D ? 0 : CB * n;
        const uint32_t v_lane = (uint32_t)(4 * g) * p.c.value_s_tok + v_ch;
        auto load = [&](int tok, const int (&id)[2], RowBuf<DP, RT> &buf) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const bool bad = bad_page(p.c, id[hf]);
                const int64_t page = bad ? 0 : id[hf];
                const uint32_t row = (uint32_t)(tok + 16 * hf) & ((1u << lg) - 1);
                const uint8_t *k = kp + page * p.c.key_s_page + (row * p.c.key_s_tok + k_lane);
#pragma unroll
                for (int c = 0; c < DP / 64; ++c)
                    buf.k[hf][c] = CUT && 64 * c + 16 * g >= p.c.D ? u32x4{0, 0, 0, 0} : __builtin_nontemporal_load((const u32x4 *)(k + 64 * c));
                const uint8_t *v = vp + page * p.c.value_s_page + (row * p.c.value_s_tok + v_lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t *src = v + (uint32_t)e * p.c.value_s_tok;
                    unsigned(&d)[DP / 64] = buf.v[4 * hf + e];
                    if constexpr (DP == 64) {
                        d[0] = __builtin_nontemporal_load((const unsigned *)src);
                    } else if constexpr (DP == 128) {
                        const u32x2 x = __builtin_nontemporal_load((const u32x2 *)src);
                        d[0] = x[0], d[1] = x[1];
                    } else {
                        const u32x4 x = __builtin_nontemporal_load((const u32x4 *)src);
                        d[0] = x[0], d[1] = x[1], d[2] = x[2], d[3] = x[3];
                    }
                }
                const uint64_t sc = uniform_load((const uint64_t *)(sp + page * p.c.scale_s_page));
                buf.sc[hf] = make_float2(bad ? __builtin_nanf("") : __builtin_bit_cast(float, (uint32_t)sc),
                                         bad ? 1.0f : __builtin_bit_cast(float, (uint32_t)(sc >> 32)));   // page 0's may be no number
            }
        };
        // The wave's steps.  A ring of NB steps' codes, NB - 1 in flight while one is computed;
        // the page ids of the next load are fetched a step before it.  Loads past the wave's
        // last step repeat that step's: a branch around them would make every wait one for
        // all loads.
        const int rows_all = p.gq * p.T;
        Seq8 before{};
        auto in_prefix = [&](int t) {   // DIRECT and SHARED: tokens of the prefix that row t sees
            if (before.bad || sq.bad || t >= sq.tq)
                return 0;
            return p.causal ? max(before.n + min(sq.n - sq.tq + t + 1, 0), 0) : before.n;
        };
        if constexpr (MODE == kPlain) {
            // (written out: as the lambda below, with the test for stat in the epilogue, calls that are
            // split took 0.3 to 0.8 us more: 4 x 38,933 tokens of 8 / 2 heads 25.4 us / 24.9)
            const int32_t *table = p.table + b * p.bt_stride;
            const int last = (sq.n - 1) >> lg, end = min(tile1 * kUnit, vis_max);
            auto ids = [&](int tok, int (&id)[2]) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    id[hf] = uniform_load(table + min((tok + 16 * hf) >> lg, last));
            };
            int tok = tile * kUnit + 32 * wave;
            if (tok < end) {
                const int final = tok + (end - 1 - tok) / STRIDE * STRIDE;
                RowBuf<DP, RT> ring[NB];
                int id[NB][2];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    ids(min(tok + j * STRIDE, final), id[j]);
#pragma unroll
                for (int j = 0; j < NB - 1; ++j)
                    load(min(tok + j * STRIDE, final), id[j], ring[j]);
                bool more = true;
                while (more) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        if (!more)
                            break;
                        load(min(tok + (NB - 1) * STRIDE, final), id[NB - 1], ring[(j + NB - 1) % NB]);
                        ids(min(tok + NB * STRIDE, final), id[NB - 1]);
                        row_step<DP, RT, BF16, 0>(W, ring[j], tok, vis_max, p.cs, g, tok + 32 > vis_min, __builtin_amdgcn_make_buffer_rsrc(nullptr, 0, 0, 0), nullptr, 0, 0);
                        tok += STRIDE;
                        more = tok < end;
                    }
                }
            }
        } else {
            // a KV head's scores are at most 1 GiB
            const uint32_t sc_step = 64 * rows_all, sc_bytes = SCORES ? (uint32_t)(p.sc_cap * rows_all * 4) : 0;
            const __amdgpu_buffer_rsrc_t scores = __builtin_amdgcn_make_buffer_rsrc(
                SCORES ? (void *)(p.scores + (int64_t)(b * p.c.H + kh) * rows_all * p.sc_cap) : nullptr, 0, sc_bytes, 0x00027000);
            // from token `tok` to `end`, of pages table[0 .. last]
            auto stream = [&](const int32_t *table, int last, int vis_min, int vis_max, int tok, int end) {
                if (tok >= end)
                    return;
                auto ids = [&](int tok, int (&id)[2]) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf)
                        id[hf] = uniform_load(table + min((tok + 16 * hf) >> lg, last));
                };
                const int final = tok + (end - 1 - tok) / STRIDE * STRIDE;
                RowBuf<DP, RT> ring[NB];
                int id[NB][2];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    ids(min(tok + j * STRIDE, final), id[j]);
#pragma unroll
                for (int j = 0; j < NB - 1; ++j)
                    load(min(tok + j * STRIDE, final), id[j], ring[j]);
                bool more = true;
                // LEAVE: scores go to memory as they come (1) or in bursts (2); `held` steps wait
                constexpr int LEAVE = !SCORES ? 0 : DIRECT ? 1 : 2;
                unsigned char *stage = (unsigned char *)&lds_o[wave][0][0];
                const int each = 2 * sc_step, most = (int)sizeof(lds_o[0]) / each;
                int held = 0;
                auto burst = [&](int tok) {    // tok: where the step behind them begins
                    __builtin_amdgcn_wave_barrier();
                    const int per = each / 16, first = tok - held * STRIDE;
                    for (int c = lane; c < held * per; c += 64) {
                        const int s = c / per, from = first + s * STRIDE;
                        __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4 *)(stage + 16 * c), scores,
                                                               from < p.sc_cap ? (uint32_t)(from >> 4) * sc_step + 16 * (c - s * per) : 1u << 31,
                                                               0, 0);
                    }
                    __builtin_amdgcn_wave_barrier();
                    held = 0;
                };
                while (more) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        if (!more)
                            break;
                        load(min(tok + (NB - 1) * STRIDE, final), id[NB - 1], ring[(j + NB - 1) % NB]);
                        ids(min(tok + NB * STRIDE, final), id[NB - 1]);
                        uint32_t at = 0;
                        if constexpr (LEAVE == 1)
                            at = n < rows_all && tok < p.sc_cap ? (uint32_t)(tok >> 4) * sc_step + 64 * n + 16 * g : 1u << 31;
                        else if constexpr (LEAVE == 2)
                            at = n < rows_all ? held * each + 64 * n + 16 * g : 1u << 31;
                        row_step<DP, RT, BF16, LEAVE>(W, ring[j], tok, vis_max, p.cs, g, tok + 32 > vis_min, scores, stage, at, sc_step);
                        tok += STRIDE;
                        more = tok < end;
                        if constexpr (LEAVE == 2) {
                            if (++held == most || !more)
                                burst(tok);
                        }
                    }
                }
            };
            if constexpr (DIRECT && SHARED) {
                const int f = b / p.per;
                before.n = p.prefix_lens[f];
                before.bad = before.n < 0 || before.n > (int64_t)p.prefix_pages << lg || (before.n > 0 && p.c.num_pages == 0);
                int own[RT], least = max(before.n, 0);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int t = (16 * rt + n) / p.gq;
                    own[rt] = W.vis[rt];
                    W.vis[rt] = in_prefix(t);
                    least = t < sq.tq ? min(least, W.vis[rt]) : least;
                }
#pragma unroll
                for (int off = 1; off < 16; off <<= 1)
                    least = min(least, __shfl_xor(least, off));
                const int most = before.bad || sq.bad || sq.tq <= 0 ? 0 : before.n;
                stream(p.prefix_table + f * p.pt_stride, (before.n - 1) >> lg, __builtin_amdgcn_readfirstlane(least), most, 32 * wave, most);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    W.vis[rt] = own[rt];
            }
            stream(table8<SHARED>(p, sq, b), (sq.n - 1) >> lg, vis_min, vis_max, tile * kUnit + 32 * wave, min(tile1 * kUnit, vis_max));
        }

        // the waves' rows joined
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float l = quad_sum(W.l[rt]);
            if (g == 0)
                lds_ml[wave][16 * rt + n] = make_float2(W.m[rt], l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d4 = 0; d4 < CB / 4; ++d4)
                    *(float4 *)&lds_o[wave][16 * rt + n][CB * (4 * g + i) + 4 * d4] =
                        make_float4(W.o[rt][4 * d4][i], W.o[rt][4 * d4 + 1][i], W.o[rt][4 * d4 + 2][i], W.o[rt][4 * d4 + 3][i]);
        }
        __syncthreads();
        const bool whole = first && last_part;
        // a run may hold the whole of any number of items, and has a part of at most two others
        int slot = 2 * wg + (u == u0 ? 0 : 1), rows = min(RM, p.gq * p.T - r0), at = b * per_seq + item;
        if constexpr (SHARED) {
            at = first_item8(p, b) + item;
            slot = whole ? 2 * p.n_wg + at : slot;
            rows = min(RM, rows8<true>(p, sq, b) - r0);
        }
        if (!DIRECT && first && threadIdx.x == 0)
            p.ws_tab[at] =
                whole ? make_int2(SHARED ? slot : -1, SHARED ? -1 : 0)
                      : make_int2(slot, run_of(R.total, R.N, pre + (item + 1) * units - 1));
        for (int i = threadIdx.x; i < rows * (DP / 4); i += 64 * NW) {
            const int r = i / (DP / 4), ch = 4 * (i - r * (DP / 4));
            float m = kLowest, l = 0.0f;
            float2 ml[NW];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                ml[w] = lds_ml[w][r];
                m = fmaxf(m, ml[w].x);
            }
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[w].x - m);
                const float4 x = *(const float4 *)&lds_o[w][r][ch];
                l += f * ml[w].y;
                acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
            }
            if ((SHARED && !DIRECT) || !whole) {
                *(float4 *)(p.ws_o + ((int64_t)slot * RM + r) * DP + ch) = acc;
                if (ch == 0)
                    p.ws_ml[slot * RM + r] = make_float2(m, l);
                continue;
            }
            const int t = (r0 + r) / p.gq, h = kh * p.gq + (r0 + r) - t * p.gq;
            bool bad = sq.bad, sees = visible8(p, sq, t) != 0;
            if constexpr (DIRECT && SHARED)
                bad |= before.bad, sees |= in_prefix(t) > 0;
            const bool none = !bad && !sees;
            const float inv = bad ? __builtin_nanf("") : none ? 0.0f : 1.0f / l;
            if (none)   // steps that no row masks went into its sums too, NaN among them
                acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (!CUT || ch < p.c.D)
                *(uint2 *)(p.out + b * p.o_s_seq + h * p.o_s_head + t * p.o_s_tok + ch) =
                    make_uint2((uint32_t)f2x(acc.x * inv, BF16) | (uint32_t)f2x(acc.y * inv, BF16) << 16,
                               (uint32_t)f2x(acc.z * inv, BF16) | (uint32_t)f2x(acc.w * inv, BF16) << 16);
            if (ch == 0 && p.lse)
                p.lse[((int64_t)b * p.Hq + h) * p.T + t] =
                    bad ? __builtin_nanf("") : none ? -__builtin_inff() : (m + __builtin_log2f(l)) / kLog2e;
            if (MODE != kPlain && ch == 0 && p.stat)
                p.stat[((int64_t)b * p.Hq + h) * p.T + t] = make_float2(m, inv);
            if (SCORES && DIRECT && ch == 0)
                lds.stat[r] = make_float2(m, inv);
        }
        if constexpr (SCORES && DIRECT) {
            // the weights, from the scores that the waves left
            const int tokens = sq.bad ? 0 : min(sq.n, p.w_tokens);
            if (threadIdx.x < 16)
                lds.vis[threadIdx.x] = (int)threadIdx.x < rows_all ? min(visible8(p, sq, threadIdx.x / p.gq), tokens) : 0;
            __syncthreads();
            for (int tok = 4 * threadIdx.x; tok < tokens; tok += 4 * 64 * NW)
                weigh_scores4(p.scores + (int64_t)(b * p.c.H + kh) * rows_all * p.sc_cap, rows_all, lds.stat, lds.vis, tok, tokens,
                              p.weights + b * p.w_s_seq + kh * p.w_s_head);
        }
        if constexpr (DIRECT)
            return;
        __syncthreads();
        u += seg;
    }
}

template <int DP, int RT, bool BF16, bool CUT, bool DIRECT, int MODE>
__global__ __launch_bounds__(64 * row_waves(RT, DIRECT), DIRECT && RT == 1 ? 4 : two_per_cu(DP, RT) ? 2 : 1) void cache8_rows_kernel(Attend8 p)
{
    __shared__ __attribute__((aligned(16))) RowLds<DP, RT, DIRECT, MODE> lds;
    int wg = blockIdx.x;
    if (MODE == kShared && gridDim.x % 8 == 0)   // neighbours of a run on one XCD: they read the same pages
        wg = (wg & 7) * (gridDim.x >> 3) + (wg >> 3);
    rows_run<DP, RT, BF16, CUT, DIRECT, MODE>(p, wg, p.n_wg, lds);
}

} // namespace kitty
