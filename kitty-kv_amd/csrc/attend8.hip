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
#include <algorithm>

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
template <int DP, int RT, bool BF16>
__device__ __forceinline__ void row_step(RowState<DP, RT> &W, RowBuf<DP, RT> &buf, int tok, int vis_max, float cs, int g, bool mask)
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

__device__ __forceinline__ bool find_run(const Attend8 &p, Run8 &R)
{
    const int lane = threadIdx.x & 63, per_seq = p.c.H * p.nrb, wg = blockIdx.x;
    // 64 sequences at a time: tiles of each, units of each and the sum up to it
    auto tiles = [&](int b0) { return b0 + lane < p.B ? tiles8(seq8(p, b0 + lane)) : 0; };
    auto sums = [&](int t, int &x) {
        x = units8(t, R.start) * per_seq;
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
    const int each = __builtin_amdgcn_readlane(t, 0), items = p.B * per_seq;
    const int N0 = (int)min((int64_t)p.n_wg, (int64_t)each * items);
    R.start = kStart;
    if (p.B <= 64 && N0 > 0 && N0 % items == 0 && !__ballot(lane < p.B && t != each))
        R.start = 0;
    int x, inc = sums(t, x), total = __builtin_amdgcn_readlane(inc, 63);
    for (int b0 = 64; b0 < p.B; b0 += 64) {
        int y;
        total += __builtin_amdgcn_readlane(sums(tiles(b0), y), 63);
    }
    R.total = total;
    R.N = min(p.n_wg, total);
    if (wg >= R.N)
        return false;
    R.u = run_start(total, R.N, wg);
    R.u1 = run_start(total, R.N, wg + 1);
    // (the bounds here and below are for lengths that another stream changes under the
    // call: it then gives anything, and ends)
    for (int b0 = 0, base = 0; b0 < p.B;) {
        const unsigned long long past = __ballot(base + inc > R.u);
        if (past) {
            const int l = __builtin_ctzll(past);
            R.b = b0 + l;
            R.pre = base + __builtin_amdgcn_readlane(inc - x, l);
            return true;
        }
        base += __builtin_amdgcn_readlane(inc, 63);
        inc = sums(tiles(b0 += 64), x);
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

// CUT: D is below DP, and the lanes beyond it read nothing.  DIRECT: a workgroup takes
// the whole of one (pair, row block) and writes its rows, so that no merge follows.
template <int DP, int RT, bool BF16, bool CUT, bool DIRECT>
__global__ __launch_bounds__(64 * row_waves(RT, DIRECT), DIRECT && RT == 1 ? 4 : two_per_cu(DP, RT) ? 2 : 1) void cache8_rows_kernel(Attend8 p)
{
    constexpr int RM = 16 * RT, CB = DP / 16, LD = DP + 4, NW = row_waves(RT, DIRECT), NB = NW == 16 ? 1 : 2, STRIDE = 32 * NW;
    __shared__ __attribute__((aligned(16))) float lds_o[NW][RM][LD];
    __shared__ float2 lds_ml[NW][RM];
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_seq = p.c.H * p.nrb, wg = blockIdx.x;
    Run8 R;
    if constexpr (DIRECT) {
        R.b = wg / per_seq;
        R.pre = 0, R.start = 0, R.u = wg - R.b * per_seq, R.u1 = R.u + 1;
    } else {
        if (!find_run(p, R))
            return;
    }
    const int u0 = R.u, u1 = R.u1;
    int u = R.u, b = R.b, pre = R.pre;

    while (u < u1 && b < p.B) {
        const Seq8 sq = seq8(p, b);
        const int tiles = tiles8(sq), units = DIRECT ? tiles : units8(tiles, R.start);
        int item = u, seg = units, tile = 0, tile1 = tiles;                     // seg: units of this run's part
        bool first = true, last_part = true;                                    // whether it has the first and last tile
        if constexpr (!DIRECT) {
            if (u >= pre + units * per_seq) {
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
        const int kh = item / p.nrb, rb = item - kh * p.nrb, r0 = rb * RM;
        const int t_lo = r0 / p.gq, t_hi = min((r0 + RM - 1) / p.gq, sq.tq - 1);   // query tokens of the block
        const int vis_min = visible8(p, sq, t_lo), vis_max = sq.bad || t_hi < t_lo ? 0 : visible8(p, sq, t_hi);
        const int end = min(tile1 * kUnit, vis_max);

        RowState<DP, RT> W;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = r0 + 16 * rt + n, t = r / p.gq, h = kh * p.gq + r - t * p.gq;
            W.vis[rt] = visible8(p, sq, t);
            W.m[rt] = kLowest;
            W.l[rt] = 0.0f;
            const uint16_t *q = p.q + b * p.q_s_seq + h * p.q_s_head + t * p.q_s_tok;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const int ch = 64 * (c >> 1) + 16 * g + 8 * (c & 1);
                W.q[rt][c] = u32x4{0, 0, 0, 0};
                if (!sq.bad && t < sq.tq && (!CUT || ch < p.c.D))
                    W.q[rt][c] = *(const u32x4 *)(q + ch);
            }
#pragma unroll
            for (int dt = 0; dt < CB; ++dt)
                W.o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        const int32_t *table = p.table + b * p.bt_stride;
        const int last = (sq.n - 1) >> p.c.lg, lg = p.c.lg;
        const uint8_t *kp = p.c.key + kh * p.c.key_s_head, *vp = p.c.value + kh * p.c.value_s_head;
        const float *sp = p.c.scale + kh * p.c.scale_s_head;
        const uint32_t k_lane = (uint32_t)n * p.c.key_s_tok + 16 * g;
        const uint32_t v_ch = CUT && CB * n >= p.c.D ? 0 : CB * n;
        const uint32_t v_lane = (uint32_t)(4 * g) * p.c.value_s_tok + v_ch;
        auto ids = [&](int tok, int (&id)[2]) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                id[hf] = uniform_load(table + min((tok + 16 * hf) >> lg, last));
        };
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
        // A ring of NB steps' codes, NB - 1 in flight while one is computed; the page
        // ids of the next load are fetched a step before it.  Loads past the wave's
        // last step repeat that step's: a branch around them would make every wait
        // one for all loads.
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
                    row_step<DP, RT, BF16>(W, ring[j], tok, vis_max, p.cs, g, tok + 32 > vis_min);
                    tok += STRIDE;
                    more = tok < end;
                }
            }
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
        const int slot = 2 * wg + (u == u0 ? 0 : 1), rows = min(RM, p.gq * p.T - r0);
        if (!DIRECT && first && threadIdx.x == 0)
            p.ws_tab[b * per_seq + item] =
                whole ? make_int2(-1, 0) : make_int2(slot, run_of(R.total, R.N, pre + (item + 1) * units - 1));
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
            if (!whole) {
                *(float4 *)(p.ws_o + ((int64_t)slot * RM + r) * DP + ch) = acc;
                if (ch == 0)
                    p.ws_ml[slot * RM + r] = make_float2(m, l);
                continue;
            }
            const int t = (r0 + r) / p.gq, h = kh * p.gq + (r0 + r) - t * p.gq;
            const bool none = !sq.bad && visible8(p, sq, t) == 0;
            const float inv = sq.bad ? __builtin_nanf("") : none ? 0.0f : 1.0f / l;
            if (none)   // steps that no row masks went into its sums too, NaN among them
                acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (!CUT || ch < p.c.D)
                *(uint2 *)(p.out + b * p.o_s_seq + h * p.o_s_head + t * p.o_s_tok + ch) =
                    make_uint2((uint32_t)f2x(acc.x * inv, BF16) | (uint32_t)f2x(acc.y * inv, BF16) << 16,
                               (uint32_t)f2x(acc.z * inv, BF16) | (uint32_t)f2x(acc.w * inv, BF16) << 16);
            if (ch == 0 && p.lse)
                p.lse[((int64_t)b * p.Hq + h) * p.T + t] =
                    sq.bad ? __builtin_nanf("") : none ? -__builtin_inff() : (m + __builtin_log2f(l)) / kLog2e;
        }
        if constexpr (DIRECT)
            return;
        __syncthreads();
        u += seg;
    }
}

// Joins the partials of each row; also, after the row kernel, the rows no
// workgroup touched: of sequences without tokens (0) and of broken lengths (NaN).
// DP / 4 lanes take a row, four channels each.  ALONE: a workgroup per row, whose
// lane groups share its partials and join in LDS (few rows, many partials);
// otherwise a row per lane group.  TILES: the partials are the tile kernel's
// p.splits parts.
template <int DP, bool BF16, bool TILES, bool ALONE>
__global__ __launch_bounds__(64 * kWaves) void cache8_merge_kernel(Attend8 p, int RM)
{
    constexpr int LPR = DP / 4, GROUPS = 64 * kWaves / LPR, STEP = ALONE ? GROUPS : 1;
    const int group = threadIdx.x / LPR, ch = 4 * (threadIdx.x % LPR);
    const int rows = p.gq * p.T, all = ALONE ? blockIdx.x : blockIdx.x * GROUPS + group;
    const int pair = all / rows, row = all - pair * rows;
    if (!ALONE && pair >= p.B * p.c.H)
        return;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, rb = row / RM, r = row - rb * RM;
    const int t = row / p.gq, h = kh * p.gq + row - t * p.gq, item = pair * p.nrb + rb;
    int2 tab = make_int2(0, 0);
    if constexpr (!TILES)
        tab = p.ws_tab[item];   // of a sequence without tokens it holds anything and is not used
    const Seq8 sq = seq8(p, b);
    float m = kLowest, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fold = [&](float m1, float l1, float4 x) {
        const float mn = fmaxf(m, m1);
        const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(m1 - mn);
        m = mn;
        l = f0 * l + f1 * l1;
        o.x = f0 * o.x + f1 * x.x, o.y = f0 * o.y + f1 * x.y, o.z = f0 * o.z + f1 * x.z, o.w = f0 * o.w + f1 * x.w;
    };
    if (sq.bad) {
        l = __builtin_nanf("");
    } else if (sq.n > 0) {
        if (tab.x < 0)
            return;
        tab.x = min(tab.x, 2 * p.n_wg - 1);
        const int first = tab.x >> 1, count = TILES ? p.splits : min(tab.y, p.n_wg - 1) - first + 1;
        for (int i = ALONE ? group : 0; i < count; i += 4 * STEP) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = min(i + j * STEP, count - 1);
                const int64_t s = TILES ? ((int64_t)item * p.splits + k) * RM + r
                                        : (int64_t)(k == 0 ? tab.x : 2 * (first + k)) * RM + r;
                ml[j] = p.ws_ml[s];
                x[j] = *(const float4 *)(p.ws_o + s * DP + ch);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * STEP < count)
                    fold(ml[j].x, ml[j].y, x[j]);
        }
    }
    if constexpr (ALONE) {
        __shared__ __attribute__((aligned(16))) float lds_o[GROUPS][DP];
        __shared__ float2 lds_ml[GROUPS];
        *(float4 *)&lds_o[group][ch] = o;
        if (ch == 0)
            lds_ml[group] = make_float2(m, l);
        __syncthreads();
        if (group != 0)
            return;
#pragma unroll
        for (int k = 1; k < GROUPS; ++k)
            fold(lds_ml[k].x, lds_ml[k].y, *(const float4 *)&lds_o[k][ch]);
    }
    if (ch >= p.c.D)
        return;
    const bool none = !sq.bad && visible8(p, sq, t) == 0;
    if (none)   // steps that no row masks went into its sums too, NaN among them
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float inv = none ? 0.0f : 1.0f / l;
    *(uint2 *)(p.out + b * p.o_s_seq + h * p.o_s_head + t * p.o_s_tok + ch) =
        make_uint2((uint32_t)f2x(o.x * inv, BF16) | (uint32_t)f2x(o.y * inv, BF16) << 16,
                   (uint32_t)f2x(o.z * inv, BF16) | (uint32_t)f2x(o.w * inv, BF16) << 16);
    if (ch == 0 && p.lse)
        p.lse[((int64_t)b * p.Hq + h) * p.T + t] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) / kLog2e;
}

static int device_cus()
{
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
        cus = 256;
    return cus;
}

static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// Which kernel takes a call, by its sizes alone (rows: of a KV head, its group's
// heads times the queries; tokens: of the longest sequence, as far as the host knows).
//
// 1. The row kernel on whole (pair, row block)s, one launch, where a stream of a pair
// is at most kDirectBytes and there are at most kDirectItems of them, or a workgroup
// a CU where a pair has several row blocks.  It saves the merge (on the host too) and
// reads lengths less often, and loses where its few workgroups leave the device idle.
// (The rule has no least number of items: one sequence near the bound would be up to 1.6
// us faster split, as the first row and the 64 channels' have it.)
// us, one launch / split and merge, 8 KV heads, one query, groups of 4, fp16:
//   channels 128, tokens    128          512          1,024        2,048
//   1 sequence              5.0 /  8.5   7.0 /  9.6    9.9 /  9.6  15.8 / 10.0
//   16 sequences            5.2 /  9.0   7.6 / 12.2   11.4 / 14.5  20.0 / 20.1
//   64 sequences            9.1 / 10.6  16.2 / 18.4   26.9 / 28.6  46.6 / 48.7
//   256 sequences          34.8 / 34.1  61.2 / 62.2   99.9 / 101.4
//   channels 64: 1 sequence 512 tokens 5.8 / 9.1, 2,048 10.8 / 9.2; 16 of 2,048 12.4 / 15.0
//   channels 256 (its registers would spill): 1 sequence 512 tokens 13.3 / 11.8
// and of several row blocks against the tile kernel, bf16:
//   128 rows, 128 channels, 1 sequence of 1,024 15.6 / 17.0, 8 (256 items) 19.1 / 26.1, 32 75.5 / 44.3
//   100 rows, 64 channels, 1 sequence of 1,500 13.8 / 14.6, 8 (256 items) 14.5 / 21.5, 32 55.0 / 35.7
//   256 rows, 128 channels, 8 sequences of 512 (512 items) 27.0 / 26.8
//
// 2. The row kernel's split, up to four blocks of 16 rows (two at 256 channels), whose
// codes are read once: beyond 32 rows its registers allow one wave a SIMD, which still
// beats the tile kernel's half-empty workgroups.  us, row / tile kernel, 32 sequences
// of 8,192 tokens, 8 KV heads, fp16:
//   128 channels, 36 rows 141 / 195, 64 rows 175 / 199;  64 channels, 64 rows 97 / 153
//   256 channels, 20 rows 281 in two blocks / 331 in one at a time
// 8 sequences: 49 / 62, 62 / 61, 39 / 48.
//
// 3. The tile kernel beyond.
constexpr int64_t kDirectBytes = 1024 * 128, kDirectItems = 4096;

struct Plan8 {
    bool tiles, direct;
    int DP, RT, nrb, n_wg, splits;
    size_t o_bytes, ml_bytes, bytes;
};

// Rows from which the merge gives each a lane group instead of a workgroup (12,800
// rows of four parts 5.6 us / 9.0 with a wave a row; 1,280 rows of nine 6.5 / 4.6).
constexpr int64_t kMergeRows = 2048;

static int plan8(const Cache8 &c, const kitty_cache8_attention_args &a, Plan8 &pl)
{
    const int64_t rows = (int64_t)a.num_q_heads / c.H * a.tokens, pairs = (int64_t)a.batch * c.H;
    const int64_t cap = (int64_t)a.table_pages << c.lg, units = kStart + (cap + kUnit - 1) / kUnit;
    if (rows > kMaxBlocks || pairs > kMaxBlocks || pairs * rows > kMaxBlocks)
        return fail(KITTY_E_UNSUPPORTED, "too many rows for one launch");
    const int64_t tokens = a.plan_tokens > 0 ? std::min<int64_t>(a.plan_tokens, cap) : cap;
    const int cus = device_cus();
    pl.DP = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    pl.direct = pl.DP <= 128 && tokens * pl.DP <= kDirectBytes &&
                (rows <= 32 ? pairs <= kDirectItems : pairs * ((rows + 31) / 32) <= cus);
    pl.tiles = !pl.direct && rows > (pl.DP == 256 ? 32 : 64);
    pl.RT = rows <= 16 ? 1 : rows <= 32 || pl.direct || pl.DP == 256 ? 2 : rows <= 48 ? 3 : 4;
    const int RM = pl.tiles ? kTileRows : 16 * pl.RT;
    const int64_t nrb = (rows + RM - 1) / RM, items = pairs * nrb;
    if (items * units > 0x7fffffff)
        return fail(KITTY_E_UNSUPPORTED, "too many rows and pages for one launch");
    pl.nrb = (int)nrb;
    pl.n_wg = pl.splits = 1;
    int64_t slots = 0;
    if (pl.tiles) {
        // parts of at least four tiles, until there are two workgroups a CU (one at 256 channels)
        const int64_t want = (pl.DP == 256 ? 1 : 2) * (int64_t)cus / std::max<int64_t>(items, 1);
        pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, tokens / 256));
        slots = pl.splits > 1 ? items * pl.splits : 0;
    } else if (!pl.direct) {
        pl.n_wg = (int)std::max<int64_t>(1, std::min<int64_t>((two_per_cu(pl.DP, pl.RT) ? 2 : 1) * cus, items * units));
        slots = 2 * pl.n_wg;
    }
    pl.o_bytes = up16((size_t)slots * RM * pl.DP * 4);
    pl.ml_bytes = up16((size_t)slots * RM * 8);
    pl.bytes = pl.o_bytes + pl.ml_bytes + (pl.tiles || pl.direct ? 0 : up16((size_t)items * 8));
    return KITTY_OK;
}

static int check_attend8(const kitty_cache8 *cache, const kitty_cache8_attention_args *args, Cache8 &c)
{
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, c))
        return rc;
    const kitty_cache8_attention_args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.table_pages < 0 || a.plan_tokens < 0)
        return fail(KITTY_E_INVALID, "batch, tokens, table_pages and plan_tokens must not be negative");
    if (a.num_q_heads <= 0 || a.num_q_heads % c.H)
        return fail(KITTY_E_INVALID, "num_q_heads must be a positive multiple of num_kv_heads");
    if (a.dtype != KITTY_DTYPE_F16 && a.dtype != KITTY_DTYPE_BF16)
        return fail(KITTY_E_INVALID, "dtype must be KITTY_DTYPE_F16 or KITTY_DTYPE_BF16");
    if (!(a.sm_scale > 0.0f) || a.sm_scale > 1e30f)
        return fail(KITTY_E_INVALID, "sm_scale must be positive and finite");
    if ((int64_t)a.table_pages << c.lg > 1 << 30)
        return fail(KITTY_E_UNSUPPORTED, "a block table is limited to 2^30 tokens a sequence");
    return KITTY_OK;
}

} // namespace kitty

using namespace kitty;

extern "C" int kitty_cache8_attention_workspace_size(const kitty_cache8 *cache, const kitty_cache8_attention_args *args,
                                                     size_t *bytes)
{
    Cache8 c;
    Plan8 pl;
    if (!bytes)
        return fail(KITTY_E_INVALID, "bytes is NULL");
    if (const int rc = check_attend8(cache, args, c))
        return rc;
    if (const int rc = plan8(c, *args, pl))
        return rc;
    *bytes = pl.bytes;
    return KITTY_OK;
}

extern "C" int kitty_cache8_attention(const kitty_cache8 *cache, const kitty_cache8_attention_args *args,
                                      kitty_stream_t stream)
{
    Attend8 p;
    Plan8 pl;
    if (const int rc = check_attend8(cache, args, p.c))
        return rc;
    const kitty_cache8_attention_args &a = *args;
    if (a.batch == 0 || a.tokens == 0)
        return KITTY_OK;
    if (!a.q || !a.out || !a.lens || (!a.block_table && a.table_pages))
        return fail(KITTY_E_INVALID, "NULL q, out, lens or block_table");
    if (!aligned(a.q, 16) || !aligned(a.out, 16))
        return fail(KITTY_E_INVALID, "q and out must be 16-byte aligned");
    for (int64_t s : {a.q_s_seq, a.q_s_head, a.q_s_tok, a.o_s_seq, a.o_s_head, a.o_s_tok})
        if (s % 8)
            return fail(KITTY_E_INVALID, "strides of q and out must be multiples of 8 elements (16-byte rows)");
    if (const int rc = plan8(p.c, a, pl))
        return rc;
    if ((!a.workspace && pl.bytes) || !aligned(a.workspace, 16) || a.workspace_bytes < pl.bytes)
        return fail(KITTY_E_INVALID, "workspace is NULL, misaligned or smaller than kitty_cache8_attention_workspace_size");
    p.q = a.q, p.out = a.out, p.lse = a.lse;
    p.q_s_seq = a.q_s_seq, p.q_s_head = a.q_s_head, p.q_s_tok = a.q_s_tok;
    p.o_s_seq = a.o_s_seq, p.o_s_head = a.o_s_head, p.o_s_tok = a.o_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.lens = a.lens, p.q_lens = a.q_lens;
    p.B = a.batch, p.Hq = a.num_q_heads, p.T = a.tokens, p.gq = a.num_q_heads / p.c.H;
    p.table_pages = a.table_pages, p.causal = a.causal ? 1 : 0;
    p.nrb = pl.nrb, p.n_wg = pl.n_wg, p.splits = pl.splits;
    p.cs = a.sm_scale * kLog2e;
    char *ws = (char *)a.workspace;
    p.ws_o = (float *)ws, p.ws_ml = (float2 *)(ws + pl.o_bytes), p.ws_tab = (int2 *)(ws + pl.o_bytes + pl.ml_bytes);

    const hipStream_t st = (hipStream_t)stream;
    const bool bf16 = a.dtype == KITTY_DTYPE_BF16;
    const dim3 block(64 * kWaves);
    auto merge = [&](auto dp, auto bf, auto tiles) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value, TILES = decltype(tiles)::value;
        const int64_t rows = (int64_t)p.B * p.Hq * p.T;
        const int RM = TILES ? kTileRows : 16 * pl.RT;
        if (rows < kMergeRows) {
            hipLaunchKernelGGL((cache8_merge_kernel<DP, BF, TILES, true>), dim3((unsigned)rows), block, 0, st, p, RM);
        } else {
            const int64_t groups = 256 * kWaves / DP;
            hipLaunchKernelGGL((cache8_merge_kernel<DP, BF, TILES, false>), dim3((unsigned)((rows + groups - 1) / groups)), block,
                               0, st, p, RM);
        }
    };
    auto rows = [&](auto dp, auto rt, auto bf) {
        constexpr int DP = decltype(dp)::value, RT = decltype(rt)::value;
        constexpr bool BF = decltype(bf)::value;
        const dim3 pairs((unsigned)(p.B * p.c.H * p.nrb)), runs((unsigned)p.n_wg), waves(64 * row_waves(RT, true));
        if constexpr (DP <= 128 && RT <= 2) {
            if (pl.direct && p.c.D == DP)
                hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, true>), pairs, waves, 0, st, p);
            else if (pl.direct)
                hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, true>), pairs, waves, 0, st, p);
            if (pl.direct)
                return;
        }
        if (p.c.D == DP)
            hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, false>), runs, block, 0, st, p);
        else
            hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, false>), runs, block, 0, st, p);
    };
    auto go = [&](auto dp, auto bf) {
        constexpr int DP = decltype(dp)::value;
        if (pl.tiles) {
            launch_tiles(p, DP, bf16, st);
            if (p.splits > 1)
                merge(dp, bf, std::true_type{});
            return;
        }
        if (pl.RT == 1)
            rows(dp, std::integral_constant<int, 1>{}, bf);
        else if (pl.RT == 2)
            rows(dp, std::integral_constant<int, 2>{}, bf);
        else if constexpr (DP <= 128) {
            if (pl.RT == 3)
                rows(dp, std::integral_constant<int, 3>{}, bf);
            else
                rows(dp, std::integral_constant<int, 4>{}, bf);
        }
        if (!pl.direct)
            merge(dp, bf, std::false_type{});
    };
    auto by_type = [&](auto dp) {
        if (bf16)
            go(dp, std::true_type{});
        else
            go(dp, std::false_type{});
    };
    if (pl.DP == 64)
        by_type(std::integral_constant<int, 64>{});
    else if (pl.DP == 128)
        by_type(std::integral_constant<int, 128>{});
    else
        by_type(std::integral_constant<int, 256>{});
    return check_launch("8-bit cache attention");
}
