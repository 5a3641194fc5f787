// Attention of many query rows over the 8-bit paged cache, on gfx950: a
// prompt's chunk behind what the cache holds, or decoder rows over an encoder's
// states.
//
// Bound by the matrix cores and the softmax's vector instructions.  One wave
// takes 32 query rows (head of the group fastest), a 256-thread workgroup four
// waves of one (sequence, KV head) pair, and each tile of 64 tokens is widened
// once for all of them: codes HBM -> registers (the next tile's, while one is
// computed) -> 16-bit floats in one of two LDS stages, keys in q's type and
// values in bf16, both exact.  Chunks are swizzled so that neither the key reads
// nor the transposing value reads conflict.
//
//  S^T = K Q^T with 32x32x16 MFMAs: lane (n = query row l & 31, g = l / 32) ends
//  with its row's scores of tokens 8j + 4g + 0..3, so the softmax needs one
//  exchange between lanes l and l + 32 per tile.
//  O^T += V^T P^T: the scores' registers are the B operand as they stand; slots
//  8g + e of a 16-token step stand for tokens 4g + e (e < 4) and 8 + 4g + e - 4,
//  and ds_read_b64_tr_b16 fetches the value rows in that order.
//
// Scales belong to 16-token steps (a page holds 16 tokens or more): the key's is a
// factor of the scores, the value's of the weights.
// Weights: for fp16 results two bf16 terms of weight times scale (16 bits, error at
// most 2^-16, with fp32's range), as a third of the products' time buys the error of
// fp32 weights.  For bf16 results, which keep 8 bits, one fp16 term (11 bits: 2^-11 of
// a weight, 2^-25 of the largest where that is more), as long as the value scales met
// lie close enough for its range; the logarithm of the scale is then added to the
// scores, so that the running maximum m is that of weight times scale, the exponential
// gives w = p * scale in one step (at most 2^8, the largest at least 1), and p's sum is
// that of w by 1 / scale.  From the first tile with a scale beyond (a page of zeros has
// 2^-64) the two terms.  The maximum is raised only when a tile passes it by 2^8.
// Where the row blocks are too few for the device, the tokens of each are split
// evenly, and cache8_merge_kernel joins the parts.
//
// Measured, 32 query / 8 KV heads of 128, 2,048 queries at 18,000 tokens (785 to 940 by
// card and data; the same card for all of these): 851 us fp16 (665 TFLOP/s of the plain
// product, 995 of those executed, where a library product of 8,192^3 reaches 1,170 at
// the clock that the power limit leaves), 665 us bf16, 830 from a far value scale on;
// heads of 64 fp16 581, bf16 469 us, of 256 2,087 and 1,928 us; 8 x 33-100 queries over
// 1,500 states, 16 heads of 64, bf16: 25 us with the merge.  Of the bf16 figures the look
// at the value scales is 1 to 5 % (64 channels 460 without, 256 1,840).  Of the 851: page
// ids a tile ahead 20, NaN values handled behind the loop 75 (the branch in it split the
// products); wave priorities around the products cost 4 %, and two fp16 terms instead of
// bf16, a sixth fewer vector instructions, 2 % (their products draw more power; at 64
// channels they are worth 3 %).  Eight waves a workgroup gain 1 to 5 % where their row
// blocks fill the device exactly, and lose up to 19 elsewhere.
#include <type_traits>

#include "attend8.h"

namespace kitty {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64, kTileWaves = kTileRows / 32;

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// max / sum of a value with the lane 32 apart
__device__ __forceinline__ float other_max(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (int)s[0]), __builtin_bit_cast(float, (int)s[1]));
}
__device__ __forceinline__ float other_sum(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return __builtin_bit_cast(float, (int)s[0]) + __builtin_bit_cast(float, (int)s[1]);
}

// Where 16-byte chunk c of a tile's row lies in the row's DP / 8 chunks.
template <int DP>
__device__ __forceinline__ int key_slot(int row, int c) { return c ^ (row & (DP == 64 ? 7 : 15)); }
template <int DP>
__device__ __forceinline__ int value_slot(int row, int c) { return c ^ (4 * (DP == 64 ? row >> 1 & 1 : row & 3)); }

// 16 codes as two chunks of 16-bit floats.
template <bool BF16>
__device__ __forceinline__ void widen16(u32x4 w, u32x4 (&r)[2])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r[e >> 1][2 * (e & 1)] = widen<BF16, false>(w[e]);
        r[e >> 1][2 * (e & 1) + 1] = widen<BF16, true>(w[e]);
    }
}

// (a, b) as fp16, rounded to nearest.
__device__ __forceinline__ unsigned pack_f16(float a, float b)
{
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    half2v h;
    h[0] = (_Float16)a, h[1] = (_Float16)b;
    return __builtin_bit_cast(unsigned, h);
}

template <int DP>
struct TileState {
    u32x4 q[DP / 16];    // k-step s: channels 16s + 8g .. + 7
    f32x16 o[DP / 32];   // O^T: channels 32dt + 8 (i / 4) + 4g + i % 4
    float m, l;          // running maximum of score (one term: + log2(value scale)), this lane's half of the sum
    int vis;             // tokens the row sees
    int k_base, v_base[DP / 32];
};

// One fp16 term takes value scales (as bits of positive floats) within 2^12 of each
// other, so that its 2^-25 of the largest product of weight and scale is at most 2^-13
// of a weight near 1, and from 2^-64 to 2^32, so that neither the reciprocals nor the
// sum of weights leave fp32's range.
constexpr uint32_t kLeastScale = (127 - 64) << 23, kMostScale = (127 + 32) << 23, kSpan = 12 << 23;

// Scales of a 16-token step: the key's times sm_scale * log2(e); of the value's the
// scale itself (two terms) or the logarithm and the reciprocal (one term).
struct StepScale {
    float key, value, inv_v;
};

// Tokens t0 .. t0 + 63 in a stage folded into the wave's rows.  mask: some row does
// not see them all.  Sums and outputs are relative to 2^m, whatever m was taken from:
// a wave may go over from one term to two at any tile.
template <int DP, bool BF16, int TERMS>
__device__ __forceinline__ void tile_step(TileState<DP> &W, const unsigned char *kst, const unsigned char *vst, int t0,
                                          StepScale (&sc)[4], int lane, bool mask)
{
    const int g = lane >> 5, n = lane & 31;
    f32x16 S[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            S[mt][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int off = W.k_base + 16 * key_slot<DP>(n, 2 * s + g);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
            S[mt] = mfma32<BF16>(*(const u32x4 *)(kst + off + 64 * DP * mt), W.q[s], S[mt]);
    }
    if (mask) {
        asm volatile("");   // a branch, not 32 selects in every tile
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                S[mt][i] = t0 + 32 * mt + 8 * (i >> 2) + 4 * g + (i & 3) < W.vis ? S[mt][i] : -__builtin_inff();
#pragma unroll
        for (int st = 0; st < 4; ++st)   // above 0 as a factor of -infinity; the scores are 0 either way
            sc[st].key = sc[st].key < 1.175494351e-38f ? 1.175494351e-38f : sc[st].key;
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int st = 0; st < 4; ++st) {
        float a = S[st >> 1][8 * (st & 1)];
#pragma unroll
        for (int i = 1; i < 8; ++i)
            a = fmaxf(a, S[st >> 1][8 * (st & 1) + i]);
        mx = fmaxf(mx, TERMS == 2 ? a * sc[st].key : __builtin_fmaf(a, sc[st].key, sc[st].value));
    }
    mx = other_max(mx);
    const bool raise = mx > W.m + 8.0f;
    if (__ballot(raise)) {
        const float mn = raise ? mx : W.m;
        const float alpha = __builtin_amdgcn_exp2f(W.m - mn);
        W.m = mn;
        W.l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                W.o[dt][i] *= alpha;
    }
    unsigned pt[TERMS][2][8];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
        const float add = TERMS == 2 ? -W.m : sc[st].value - W.m;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 4 * (st & 1); i < 4 * (st & 1) + 4; ++i) {
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(S[st >> 1][2 * i], sc[st].key, add));
            const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(S[st >> 1][2 * i + 1], sc[st].key, add));
            sum[0] += a;
            sum[1] += b;
            if constexpr (TERMS == 1)
                pt[0][st >> 1][i] = pack_f16(a, b);
            else
                split_bf16(a * sc[st].value, b * sc[st].value, pt[0][st >> 1][i], pt[1][st >> 1][i]);
        }
        W.l = TERMS == 2 ? W.l + (sum[0] + sum[1]) : __builtin_fmaf(sum[0] + sum[1], sc[st].inv_v, W.l);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int mt = s >> 1, r = 4 * (s & 1);
        u32x4 vf[DP / 32];
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const unsigned char *src = vst + W.v_base[dt] + 32 * DP * s;
            const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)src);
            const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(src + 16 * DP));
            const uint2 a = __builtin_bit_cast(uint2, v0), b = __builtin_bit_cast(uint2, v1);
            vf[dt] = u32x4{a.x, a.y, b.x, b.y};
        }
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
            const u32x4 w = {pt[k][mt][r], pt[k][mt][r + 1], pt[k][mt][r + 2], pt[k][mt][r + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
                W.o[dt] = mfma32<TERMS == 2>(vf[dt], w, W.o[dt]);
        }
    }
}

template <int DP, bool BF16, bool CUT>
__global__ __launch_bounds__(64 * kTileWaves, DP <= 128 ? 2 : 1) void cache8_tile_kernel(Attend8 p)
{
    constexpr int RM = kTileRows, TPR = DP / 16, PASS = 64 * kTileWaves / TPR, NP = kTile / PASS;
    __shared__ __attribute__((aligned(16))) unsigned char ks[2][kTile * DP * 2], vs[2][kTile * DP * 2];
    __shared__ int met_nan;
    const int lane = threadIdx.x & 63, g = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // pairs vary fastest, so with a multiple of eight pairs a pair's pages stay in
    // one XCD's L2; the last row blocks, with the most tokens, start first
    const int pairs = p.B * p.c.H, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int split = rest % p.splits, rb = p.nrb - 1 - rest / p.splits;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, r0 = rb * RM;
    const Seq8 sq = seq8(p, b);
    const int rows = min(RM, p.gq * p.T - r0);
    const int t_lo = r0 / p.gq, t_hi = min((r0 + rows - 1) / p.gq, sq.tq - 1);
    const int vis_max = sq.bad || t_hi < t_lo ? 0 : visible8(p, sq, t_hi), vis_min = visible8(p, sq, t_lo);
    const int nt = (vis_max + kTile - 1) / kTile;
    const int first = (int)((int64_t)nt * split / p.splits), end = (int)((int64_t)nt * (split + 1) / p.splits);

    TileState<DP> W;
    const int w0 = r0 + 32 * wave, r = w0 + n, t = r / p.gq, h = kh * p.gq + r - t * p.gq;
    const bool row = r < p.gq * p.T;
    W.vis = sq.bad ? 0 : visible8(p, sq, t);
    const int w_lo = w0 / p.gq, w_hi = min((w0 + 31) / p.gq, sq.tq - 1);
    const int wave_min = visible8(p, sq, w_lo), wave_max = sq.bad || w_hi < w_lo ? 0 : visible8(p, sq, w_hi);
    {
        const uint16_t *q = p.q + b * p.q_s_seq + h * p.q_s_head + t * p.q_s_tok;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            W.q[s] = u32x4{0, 0, 0, 0};
            if (!sq.bad && t < sq.tq && (!CUT || 16 * s < p.c.D))
                W.q[s] = *(const u32x4 *)(q + 16 * s + 8 * g);
        }
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            W.o[dt][i] = 0.0f;
    W.m = kLowest;
    W.l = 0.0f;
    W.k_base = n * 2 * DP;
    {
        const int i = lane & 15, hs = lane >> 4 & 1, tr = 4 * g + (i >> 2);   // the lane's token row of a 16-token step
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
            W.v_base[dt] = tr * 2 * DP + 16 * value_slot<DP>(tr, 4 * dt + 2 * hs) + 8 * (i & 3);
    }

    // loads: thread x brings chunk x % TPR (16 codes) of rows x / TPR + PASS j; the rows
    // of a wave and j lie in one 16-token step, so their page is the wave's
    const int32_t *table = p.table + b * p.bt_stride;
    const int lg = p.c.lg, last = (sq.n - 1) >> lg;
    const int lr = threadIdx.x / TPR, lc = threadIdx.x % TPR;
    const bool cut = CUT && 16 * lc >= p.c.D;
    const uint8_t *kp = p.c.key + kh * p.c.key_s_head + (cut ? 0 : 16 * lc);
    const uint8_t *vp = p.c.value + kh * p.c.value_s_head + (cut ? 0 : 16 * lc);
    const float *sp = p.c.scale + kh * p.c.scale_s_head;
    u32x4 kr[NP], vr[NP];
    StepScale sc[4];
    uint64_t raw[4];         // the next tile's scales
    int ids[4];              // page ids of the tile that load() takes
    unsigned lost = 0;       // bits of the next tile's steps that have no page
    uint32_t least = kMostScale, most = 0;   // value scales met, as bits
    bool far = false;        // whether one fp16 term does not take them
    auto fetch_ids = [&](int tile) {
#pragma unroll
        for (int st = 0; st < 4; ++st)
            ids[st] = uniform_load(table + min((tile * kTile + 16 * st) >> lg, last));
    };
    auto load = [&](int tile) {
        int64_t page[4];
        lost = 0;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const bool bad = bad_page(p.c, ids[st]);
            page[st] = bad ? 0 : ids[st];
            lost |= (bad ? 1u : 0u) << st;
            raw[st] = uniform_load((const uint64_t *)(sp + page[st] * p.c.scale_s_page));
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            // step of this wave's rows in pass j
            const int st = (64 / TPR * wave + PASS * j) >> 4;
            const int64_t pg = st == 0 ? page[0] : st == 1 ? page[1] : st == 2 ? page[2] : page[3];
            const uint32_t rw = (uint32_t)(tile * kTile + lr + PASS * j) & ((1u << lg) - 1);
            kr[j] = *(const u32x4 *)(kp + pg * p.c.key_s_page + rw * p.c.key_s_tok);
            vr[j] = *(const u32x4 *)(vp + pg * p.c.value_s_page + rw * p.c.value_s_tok);
        }
        fetch_ids(tile + 1);   // a step ahead: the loads above wait for no scalar load of their own
    };
    auto store = [&](int tile, int stage, auto terms) {
        constexpr int TERMS = decltype(terms)::value;
        if (lost) {   // scales 1 for the steps without a page: page 0's may be no numbers
#pragma unroll
            for (int st = 0; st < 4; ++st)
                raw[st] = lost >> st & 1 ? 0x3f8000003f800000ull : raw[st];
        }
        if constexpr (TERMS == 1) {
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                least = min(least, (uint32_t)(raw[st] >> 32));
                most = max(most, (uint32_t)(raw[st] >> 32));
            }
            far = least < kLeastScale || most > kMostScale || most > least + kSpan;
        }
        bool odd = false;
        const bool ragged = (tile + 1) * kTile > vis_min;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int rw = lr + PASS * j;
            if (ragged) {
                // tokens that not every row sees: rows no query sees hold anything, and
                // a NaN would reach the others as 0 * NaN (it is put back at the end)
                if (tile * kTile + rw >= vis_max)
                    vr[j] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned nn = nan_codes(vr[j][e]);
                    odd |= nn != 0;
                    vr[j][e] &= ~((nn >> 7) * 0xffu);
                }
            }
            u32x4 x[2];
            if (lost) {   // keys of a missing page are NaN: so are the scores of rows that see them
                const unsigned c = lost >> ((64 / TPR * wave + PASS * j) >> 4) & 1 ? 0x7f7f7f7fu : 0u;
                kr[j] = kr[j] | c;
            }
            widen16<BF16>(cut ? u32x4{0, 0, 0, 0} : kr[j], x);
            unsigned char *k = ks[stage] + rw * 2 * DP;
            *(u32x4 *)(k + 16 * key_slot<DP>(rw, 2 * lc)) = x[0];
            *(u32x4 *)(k + 16 * key_slot<DP>(rw, 2 * lc + 1)) = x[1];
            widen16<TERMS == 2>(vr[j], x);
            unsigned char *v = vs[stage] + rw * 2 * DP;
            *(u32x4 *)(v + 16 * value_slot<DP>(rw, 2 * lc)) = x[0];
            *(u32x4 *)(v + 16 * value_slot<DP>(rw, 2 * lc + 1)) = x[1];
        }
        if (odd)
            met_nan = 1;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const float vs = __builtin_bit_cast(float, (uint32_t)(raw[st] >> 32));
            sc[st] = StepScale{__builtin_bit_cast(float, (uint32_t)raw[st]) * p.cs, TERMS == 2 ? vs : __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs)};
        }
    };
    if (threadIdx.x == 0)
        met_nan = 0;
    __syncthreads();
    typedef std::integral_constant<int, BF16 ? 1 : 2> Terms;
    int tile = first;
    if (first < end) {
        fetch_ids(first);
        load(first);
        store(first, 0, Terms{});
    }
    for (; tile < end && (!BF16 || !far); ++tile) {
        const int stage = (tile - first) & 1, t0 = tile * kTile;
        __syncthreads();   // the tile is in its stage; every wave is done with the other one
        const bool more = tile + 1 < end;
        if (more)
            load(tile + 1);
        if (t0 < wave_max)
            tile_step<DP, BF16, Terms::value>(W, ks[stage], vs[stage], t0, sc, lane, t0 + kTile > wave_min);
        if (more)
            store(tile + 1, stage ^ 1, Terms{});
    }
    if constexpr (BF16) {
        // from the first tile whose value scales one term does not take: nothing is fetched
        // ahead, which keeps the loop above in its registers
        for (; tile < end; ++tile) {
            __syncthreads();
            fetch_ids(tile);
            load(tile);
            store(tile, 0, std::integral_constant<int, 2>{});
            __syncthreads();
            if (tile * kTile < wave_max)
                tile_step<DP, BF16, 2>(W, ks[0], vs[0], tile * kTile, sc, lane, (tile + 1) * kTile > wave_min);
        }
    }

    __syncthreads();
    if (met_nan) {
        // the NaN values taken out above, to the rows that see them
        for (int tok = max(first, vis_min / kTile) * kTile; tok < min(end * kTile, vis_max); ++tok) {
            const int id = uniform_load(table + (tok >> lg));
            if (bad_page(p.c, id))
                continue;   // its rows' scores are NaN already
            const uint8_t *v = p.c.value + id * p.c.value_s_page + kh * p.c.value_s_head +
                               ((uint32_t)tok & ((1u << lg) - 1)) * p.c.value_s_tok;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int ch = 32 * dt + 8 * j + 4 * g;
                    if (CUT && ch >= p.c.D)
                        continue;
                    const unsigned nn = nan_codes(*(const unsigned *)(v + ch));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (nn >> (8 * e + 7) & 1 && tok < W.vis)
                            W.o[dt][4 * j + e] = __builtin_nanf("");
                }
        }
    }

    const float l = other_sum(W.l);
    if (!row)
        return;
    if (p.splits > 1) {
        const int64_t at = ((int64_t)(pair * p.nrb + rb) * p.splits + split) * RM + 32 * wave + n;
        if (g == 0)
            p.ws_ml[at] = make_float2(W.m, l);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(float4 *)(p.ws_o + at * DP + 32 * dt + 8 * j + 4 * g) =
                    make_float4(W.o[dt][4 * j], W.o[dt][4 * j + 1], W.o[dt][4 * j + 2], W.o[dt][4 * j + 3]);
        return;
    }
    const bool none = !sq.bad && W.vis == 0;
    const float inv = sq.bad ? __builtin_nanf("") : none ? 0.0f : 1.0f / l;
    auto result = [&](float x) -> uint32_t { return f2x(none ? 0.0f : x * inv, BF16); };   // none: tiles that no row masks went into x too
    uint16_t *o = p.out + b * p.o_s_seq + h * p.o_s_head + t * p.o_s_tok;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int ch = 32 * dt + 8 * j + 4 * g;
            if (!CUT || ch < p.c.D)
                *(uint2 *)(o + ch) = make_uint2(result(W.o[dt][4 * j]) | result(W.o[dt][4 * j + 1]) << 16,
                                                result(W.o[dt][4 * j + 2]) | result(W.o[dt][4 * j + 3]) << 16);
        }
    if (g == 0 && p.lse)
        p.lse[((int64_t)b * p.Hq + h) * p.T + t] =
            sq.bad ? __builtin_nanf("") : none ? -__builtin_inff() : (W.m + __builtin_log2f(l)) / kLog2e;
}

void launch_tiles(const Attend8 &p, int DP, bool bf16, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.B * p.c.H * p.nrb * p.splits)), block(64 * kTileWaves);
    auto go = [&](auto dp, auto bf) {
        constexpr int N = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value;
        if (p.c.D == N)
            hipLaunchKernelGGL((cache8_tile_kernel<N, BF, false>), grid, block, 0, stream, p);
        else
            hipLaunchKernelGGL((cache8_tile_kernel<N, BF, true>), grid, block, 0, stream, p);
    };
    auto by_size = [&](auto bf) {
        if (DP == 64)
            go(std::integral_constant<int, 64>{}, bf);
        else if (DP == 128)
            go(std::integral_constant<int, 128>{}, bf);
        else
            go(std::integral_constant<int, 256>{}, bf);
    };
    if (bf16)
        by_size(std::true_type{});
    else
        by_size(std::false_type{});
}

} // namespace kitty
