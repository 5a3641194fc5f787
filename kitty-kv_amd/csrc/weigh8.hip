// What tokens of the 8-bit paged cache are worth, on gfx950: attention (attend8.hip) that
// also adds to every token's weight what it got of the rows' softmax.
//
// The attention leaves each row's maximum and 1 / sum (rather than their log-sum-exp,
// whose rounding would be the weights' largest error).  Up to 16 rows of a KV head it
// leaves the scores as well, and makes the weights from them (attend8.hip).
// Of more rows a second pass over the keys makes p = 2^(score - top) / sum again and sums
// it over the rows of the KV head's group: S = Q K^T with
// 32x32x16 MFMAs: A row = query, column = token, so a lane (n = token l & 31, g = l / 32)
// ends with 16 of 32 queries' scores of its token, and the sum over queries stays in the
// lane until the last row tile; then the two halves of the wave are added.  Query rows
// go head slowest, so that the rows that see a block of tokens are the last queries of
// each head.  A token (and part of the rows) has one owner, and parts are added in their
// order: the sums repeat bit for bit.
//
// The second pass costs one product and an exponential a score where the attention has
// two or three products and the same exponentials: its wave has the keys in registers and
// no running maximum.  Measured, 32 query / 8 KV heads of 128: 2,048 queries at 18,000
// tokens, fp16, 321 to 343 us of 1,190 (830 to 890 TFLOP/s of its product, where a library
// product of 8,192^3 reaches 1,290; rows addressed by divisions instead of additions 371),
// and 5 for the parts; 32 queries of 8 x 4-16K, bf16, 53 of 133 us.  With the rows of the
// latter held in LDS at once and no barriers 60.
#include <type_traits>

#include "attend8_tiles.h"

namespace kitty {

struct Weigh8 {
    Attend8 a;
    float *weights;
    int64_t w_s_seq, w_s_head;
    int N, blocks, parts;   // tokens that have a weight, workgroups of a pair and part, parts of the rows
    float *ws;              // (pair, part, tokens up to cap) where there are parts
    int64_t cap;
};

// 64 tokens a wave, whose keys stay in its registers; 32 rows a tile, which goes through
// LDS for all four waves, the next one's loads in flight while one is computed.
constexpr int kWeighWaves = 4, kWeighTokens = 64 * kWeighWaves, kWeighRows = 32;

template <int DP, bool BF16, bool CUT>
__global__ __launch_bounds__(64 * kWeighWaves, DP <= 128 ? 3 : 1) void cache8_weigh_kernel(Weigh8 w)
{
    constexpr int CPR = DP / 8, PASS = 64 * kWeighWaves / CPR, NP = kWeighRows / PASS;   // 16-byte chunks of a row, rows a pass
    const Attend8 &p = w.a;
    __shared__ __attribute__((aligned(16))) unsigned char lds_q[2][kWeighRows * DP * 2];
    __shared__ __attribute__((aligned(16))) float lds_top[2][kWeighRows], lds_inv[2][kWeighRows];
    __shared__ __attribute__((aligned(16))) int lds_vis[2][kWeighRows];
    const int lane = threadIdx.x & 63, g = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // pairs vary fastest, so with a multiple of eight a pair's rows stay in one XCD's L2
    const int pairs = p.B * p.c.H, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int part = rest % w.parts, block = rest / w.parts;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, lg = p.c.lg;
    const Seq8 sq = seq8(p, b);
    if (sq.bad || sq.n == 0)
        return;
    const int32_t *table = p.table + b * p.bt_stride;
    const float2 *stat = p.stat + ((int64_t)b * p.Hq + kh * p.gq) * p.T;
    const uint16_t *qb = p.q + b * p.q_s_seq + kh * p.gq * p.q_s_head;
    const int tokens = min(sq.n, w.N);
    for (int64_t first = (int64_t)block * kWeighTokens; first < tokens; first += (int64_t)w.blocks * kWeighTokens) {
        // rows that see any of the block's tokens: queries t0 .. tq - 1 of every head
        const int t0 = p.causal ? max((int)first - (sq.n - sq.tq), 0) : 0, each = max(sq.tq - t0, 0), rows = each * p.gq;
        const int tiles = (rows + kWeighRows - 1) / kWeighRows;
        const int begin = (int)((int64_t)tiles * part / w.parts), end = (int)((int64_t)tiles * (part + 1) / w.parts);
        const int tok0 = (int)first + 64 * wave;
        // the thread's rows of the next tile to load: each tile is 32 rows on, by additions
        const int step_h = each ? kWeighRows / each : 0, step_t = kWeighRows - step_h * each;
        const int64_t q_step = step_h * p.q_s_head + step_t * p.q_s_tok, q_wrap = p.q_s_head - each * p.q_s_tok;
        const int ch = 8 * (threadIdx.x % CPR);
        int lr = begin * kWeighRows, lt[NP], nt = 0;
        const uint16_t *src[NP];
        const float2 *from = stat;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = lr + (int)threadIdx.x / CPR + PASS * j, h = each ? r / each : 0;
            lt[j] = r - h * each;
            src[j] = qb + h * p.q_s_head + (t0 + lt[j]) * p.q_s_tok + ch;
        }
        if (wave == 0) {
            const int h = each ? (lr + n) / each : 0;
            nt = lr + n - h * each;
            from = stat + (int64_t)h * p.T + t0 + nt;
        }
        u32x4 buf[NP];
        float2 buf_stat = make_float2(0.0f, 0.0f);
        int buf_vis = 0;
        auto load = [&]() {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                buf[j] = u32x4{0, 0, 0, 0};
                if (lr + (int)threadIdx.x / CPR + PASS * j < rows && (!CUT || ch < p.c.D))
                    buf[j] = *(const u32x4 *)src[j];
                lt[j] += step_t;
                src[j] += q_step;
                if (lt[j] >= each)
                    lt[j] -= each, src[j] += q_wrap;
            }
            if (wave == 0) {
                const bool in = lr + n < rows;
                buf_stat = in ? *from : make_float2(0.0f, 0.0f);
                buf_vis = in ? visible8(p, sq, t0 + nt) : 0;
                nt += step_t;
                from += step_h * p.T + step_t;
                if (nt >= each)
                    nt -= each, from += p.T - each;
            }
            lr += kWeighRows;
        };
        auto store = [&](int stage) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int r = (int)threadIdx.x / CPR + PASS * j;
                *(u32x4 *)(lds_q[stage] + r * 2 * DP + 16 * key_slot<DP>(r, ch / 8)) = buf[j];
            }
            if (threadIdx.x < kWeighRows)
                lds_top[stage][n] = buf_stat.x, lds_inv[stage][n] = buf_stat.y, lds_vis[stage][n] = buf_vis;
        };
        if (begin < end)
            load();
        // the block's keys, behind the first rows' loads
        u32x4 k[2][DP / 16];
        float ks[2], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int tok = tok0 + 32 * h + n, id = table[min(tok, sq.n - 1) >> lg];
            const bool bad = bad_page(p.c, id);
            const int64_t page = bad ? 0 : id;
            const uint8_t *key = p.c.key + page * p.c.key_s_page + kh * p.c.key_s_head + ((uint32_t)tok & ((1u << lg) - 1)) * p.c.key_s_tok + 16 * g;
            ks[h] = bad ? __builtin_nanf("") : p.c.scale[page * p.c.scale_s_page + kh * p.c.scale_s_head] * p.cs;
            u32x4 raw[DP / 32];
#pragma unroll
            for (int c = 0; c < DP / 32; ++c)
                raw[c] = CUT && 32 * c + 16 * g >= p.c.D ? u32x4{0, 0, 0, 0} : *(const u32x4 *)(key + 32 * c);
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                u32x4 y[2];
                widen16<BF16>(raw[c], y);
                k[h][2 * c] = y[0], k[h][2 * c + 1] = y[1];
            }
        }
        __syncthreads();   // of the block before
        if (begin < end)
            store(0);
        for (int i = begin; i < end; ++i) {
            const int stage = (i - begin) & 1;
            __syncthreads();
            if (i + 1 < end)
                load();
            const int vis = lds_vis[stage][n];
            if (__ballot(vis > tok0)) {
                const bool mask = __ballot(vis < tok0 + 64) != 0;
                f32x16 S[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        S[h][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) {
                    const u32x4 q = *(const u32x4 *)(lds_q[stage] + n * 2 * DP + 16 * key_slot<DP>(n, 4 * (s >> 1) + 2 * g + (s & 1)));
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        S[h] = mfma32<BF16>(q, k[h][s], S[h]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 m = *(const float4 *)&lds_top[stage][8 * j + 4 * g];
                    const float top[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            S[h][4 * j + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[h][4 * j + e], ks[h], -top[e]));
                }
                if (mask) {
                    asm volatile("");   // a branch, not 32 selects in every tile
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int4 v = *(const int4 *)&lds_vis[stage][8 * j + 4 * g];
                        const int vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float inv = lds_inv[stage][8 * j + 4 * g + e];
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                sum[h] += tok0 + 32 * h + n < vs[e] ? S[h][4 * j + e] * inv : 0.0f;
                        }
                    }
                } else {
                    float a[2][4] = {};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 v = *(const float4 *)&lds_inv[stage][8 * j + 4 * g];
                        const float inv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                a[h][e] = __builtin_fmaf(S[h][4 * j + e], inv[e], a[h][e]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        sum[h] += (a[h][0] + a[h][1]) + (a[h][2] + a[h][3]);
                }
            }
            if (i + 1 < end)
                store(stage ^ 1);
        }
        const float x = other_sum(sum[0]), y = other_sum(sum[1]), total = g ? y : x;
        const int tok = tok0 + lane;
        if (tok < tokens) {
            if (w.parts > 1)
                w.ws[((int64_t)pair * w.parts + part) * w.cap + tok] = total;
            else
                w.weights[b * w.w_s_seq + kh * w.w_s_head + tok] += total;
        }
    }
}

// The parts' sums into the weights, in their order.
__global__ __launch_bounds__(256) void cache8_weigh_sum_kernel(Weigh8 w)
{
    const Attend8 &p = w.a;
    const int pairs = p.B * p.c.H, pair = blockIdx.x % pairs, block = blockIdx.x / pairs;
    const int b = pair / p.c.H, kh = pair - b * p.c.H;
    const Seq8 sq = seq8(p, b);
    const int tokens = sq.bad ? 0 : min(sq.n, w.N);
    const float *ws = w.ws + (int64_t)pair * w.parts * w.cap;
    for (int64_t tok = (int64_t)block * 256 + threadIdx.x; tok < tokens; tok += (int64_t)w.blocks * 256) {
        float sum = 0.0f;
        for (int i = 0; i < w.parts; ++i)
            sum += ws[i * w.cap + tok];
        w.weights[b * w.w_s_seq + kh * w.w_s_head + tok] += sum;
    }
}

// How the second pass is cut: workgroups of kWeighTokens tokens, and the rows of each in
// parts until there are twelve workgroups a CU, of at least eight tiles (three workgroups
// a CU run at once, and causal rows make them unequal).
//
// Up to 16 rows the scores are kept instead: reading and writing them is 8 bytes a row and
// token where reading the keys again is head_dim, and costs products as well.  A gibibyte
// of them at most, or of the parts' sums.  Where one launch of the row kernel has all of a
// head's rows and tokens, it adds to the weights itself (4 rows of 16 sequences of 512 tokens
// 8.5 us, 14.9 split, of 1,000 13.6 / 18.1; one sequence of 512 8.1 / 11.3, of 1,024 11.4 / 11.4).
struct WeighPlan8 {
    bool scores;
    int64_t cap;
    int blocks, parts;
    size_t bytes;
};

constexpr int64_t kMostScores = 1ll << 30;

static WeighPlan8 plan_weigh(const Cache8 &c, const kitty_cache8_attention_args &a, int weight_tokens)
{
    WeighPlan8 pl{};
    pl.cap = std::min<int64_t>((int64_t)a.table_pages << c.lg, weight_tokens);
    const int64_t pairs = (int64_t)a.batch * c.H, rows = (int64_t)a.num_q_heads / c.H * a.tokens;
    const int64_t sc_bytes = pairs * rows * ((pl.cap + 15) & ~15ll) * 4;
    // (merge and weights are one grid)
    pl.scores = rows <= 16 && sc_bytes <= kMostScores && pairs <= kMaxBlocks / 2;
    if (pl.scores) {
        pl.bytes = up16((size_t)sc_bytes);
        return pl;
    }
    const int64_t known = a.plan_tokens > 0 ? std::min<int64_t>(a.plan_tokens, pl.cap) : pl.cap;
    const int64_t blocks = (known + kWeighTokens - 1) / kWeighTokens, want = 12 * (int64_t)device_cus() / std::max<int64_t>(1, pairs * blocks);
    pl.parts = (int)std::max<int64_t>(1, std::min<int64_t>({want, rows / (8 * kWeighRows), 64, kMostScores / (pairs * std::max<int64_t>(pl.cap, 1) * 4)}));
    pl.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((pl.cap + kWeighTokens - 1) / kWeighTokens, 65536 / (pairs * pl.parts)));
    pl.bytes = pl.parts > 1 ? up16((size_t)pairs * pl.parts * pl.cap * 4) : 0;
    return pl;
}

} // namespace kitty

using namespace kitty;

static int check_weights(const kitty_cache8_attention_args *args, const kitty_cache8_weights *weights)
{
    if (!weights || !args)
        return fail(KITTY_E_INVALID, "args or weights is NULL");
    if (weights->tokens < 0 || (!weights->weights && weights->tokens && args->batch && args->tokens))
        return fail(KITTY_E_INVALID, "weights->tokens must not be negative and weights->weights not NULL");
    if (!aligned(weights->weights, 4))
        return fail(KITTY_E_INVALID, "weights must be 4-byte aligned");
    return KITTY_OK;
}

extern "C" int kitty_cache8_weighed_attention_workspace_size(const kitty_cache8 *cache, const kitty_cache8_attention_args *args,
                                                             const kitty_cache8_weights *weights, size_t *bytes)
{
    if (const int rc = check_weights(args, weights))
        return rc;
    Cache8 c;
    if (!bytes)
        return fail(KITTY_E_INVALID, "bytes is NULL");
    if (const int rc = check_cache8(cache, c))
        return rc;
    if (const int rc = attend8_bytes(cache, args, false, *bytes))   // the checks
        return rc;
    *bytes = 0;
    if (args->batch == 0 || args->tokens == 0)
        return KITTY_OK;
    const WeighPlan8 pl = plan_weigh(c, *args, weights->tokens);
    if (const int rc = attend8_bytes(cache, args, pl.scores && pl.cap, *bytes))
        return rc;
    *bytes = up16(*bytes) + up16((size_t)args->batch * args->num_q_heads * args->tokens * 8) + pl.bytes;
    return KITTY_OK;
}

extern "C" int kitty_cache8_weighed_attention(const kitty_cache8 *cache, const kitty_cache8_attention_args *args,
                                              const kitty_cache8_weights *weights, kitty_stream_t stream)
{
    size_t need;
    if (const int rc = kitty_cache8_weighed_attention_workspace_size(cache, args, weights, &need))
        return rc;
    kitty_cache8_attention_args a = *args;
    if (a.batch == 0 || a.tokens == 0)
        return KITTY_OK;
    if (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < need)
        return fail(KITTY_E_INVALID,
                    "workspace is NULL, misaligned or smaller than kitty_cache8_weighed_attention_workspace_size");
    Weigh8 w{};
    Attend8 &p = w.a;
    if (const int rc = check_cache8(cache, p.c))
        return rc;
    const WeighPlan8 pl = plan_weigh(p.c, a, weights->tokens);
    const size_t rows = up16((size_t)a.batch * a.num_q_heads * a.tokens * 8);
    char *ws = (char *)a.workspace;
    p.stat = (float2 *)ws;
    w.ws = p.scores = (float *)(ws + rows);
    p.sc_cap = (pl.cap + 15) & ~15ll;
    a.workspace = ws + rows + pl.bytes;
    a.workspace_bytes -= rows + pl.bytes;
    const hipStream_t st = (hipStream_t)stream;
    Leave8 leave = {p.stat, pl.scores && pl.cap ? p.scores : nullptr, p.sc_cap,
                    weights->weights, weights->s_seq, weights->s_head, weights->tokens, false};
    if (const int rc = attend8(cache, &a, st, leave))
        return rc;
    if (pl.cap == 0 || leave.weighed)
        return KITTY_OK;
    p.q = a.q;
    p.q_s_seq = a.q_s_seq, p.q_s_head = a.q_s_head, p.q_s_tok = a.q_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.lens = a.lens, p.q_lens = a.q_lens;
    p.B = a.batch, p.Hq = a.num_q_heads, p.T = a.tokens, p.gq = a.num_q_heads / p.c.H;
    p.table_pages = a.table_pages, p.causal = a.causal ? 1 : 0;
    p.cs = a.sm_scale * kLog2e;
    w.weights = weights->weights, w.w_s_seq = weights->s_seq, w.w_s_head = weights->s_head, w.N = weights->tokens;
    w.blocks = pl.blocks, w.parts = pl.parts, w.cap = pl.cap;
    const unsigned pairs = (unsigned)(p.B * p.c.H);
    const dim3 grid(pairs * (unsigned)(pl.blocks * pl.parts)), block(64 * kWeighWaves);
    auto go = [&](auto dp, auto bf) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value;
        if (p.c.D == DP)
            hipLaunchKernelGGL((cache8_weigh_kernel<DP, BF, false>), grid, block, 0, st, w);
        else
            hipLaunchKernelGGL((cache8_weigh_kernel<DP, BF, true>), grid, block, 0, st, w);
    };
    auto by_size = [&](auto bf) {
        if (p.c.D <= 64)
            go(std::integral_constant<int, 64>{}, bf);
        else if (p.c.D <= 128)
            go(std::integral_constant<int, 128>{}, bf);
        else
            go(std::integral_constant<int, 256>{}, bf);
    };
    if (a.dtype == KITTY_DTYPE_BF16)
        by_size(std::true_type{});
    else
        by_size(std::false_type{});
    if (pl.parts > 1)
        hipLaunchKernelGGL(cache8_weigh_sum_kernel, dim3(pairs * (unsigned)pl.blocks), dim3(256), 0, st, w);
    return check_launch("cache8_weigh_kernel");
}
