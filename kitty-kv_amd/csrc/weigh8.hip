// What tokens of the 8-bit paged cache are worth, on gfx950: attention (attend8.hip) that
// also adds to every token's weight what it got of the rows' softmax.
//
// The attention leaves each row's log-sum-exp; a second pass over the keys makes
// p = exp(score - lse) and sums it over the rows of the KV head's group.  S = Q K^T with
// 32x32x16 MFMAs: A row = query, column = token, so a lane (n = token l & 31, g = l / 32)
// ends with 16 of 32 queries' scores of its token, and the sum over queries stays in the
// lane until the last row block; then the two halves of the wave are added.  Query rows
// go head slowest, so that a head's log-sum-exps lie in a run.  A token has one owner:
// its weight is read and written once, in a fixed order of sums.
#include <type_traits>

#include "attend8_tiles.h"

namespace kitty {

struct Weigh8 {
    Attend8 a;
    float *weights;
    int64_t w_s_seq, w_s_head;
    int N, blocks;      // tokens that have a weight, workgroups of a pair
};

constexpr int kWeighWaves = 4, kWeighTokens = 32 * kWeighWaves;

template <int DP, bool BF16, bool CUT>
__global__ __launch_bounds__(64 * kWeighWaves) void cache8_weigh_kernel(Weigh8 w)
{
    const Attend8 &p = w.a;
    __shared__ __attribute__((aligned(16))) float lds_lse[kWeighWaves][32];
    __shared__ __attribute__((aligned(16))) int lds_vis[kWeighWaves][32];
    const int lane = threadIdx.x & 63, g = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = p.B * p.c.H, pair = blockIdx.x % pairs, part = blockIdx.x / pairs;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, rows = p.gq * p.T, lg = p.c.lg;
    const Seq8 sq = seq8(p, b);
    if (sq.bad || sq.n == 0)
        return;
    const int32_t *table = p.table + b * p.bt_stride;
    const float *lse = p.lse + ((int64_t)b * p.Hq + kh * p.gq) * p.T;
    const int tokens = min(sq.n, w.N);
    for (int64_t first = (int64_t)part * kWeighTokens; first < tokens; first += (int64_t)w.blocks * kWeighTokens) {
        const int tok0 = (int)first + 32 * wave, tok = tok0 + n;   // the wave's first token, the lane's
        const int id = table[min(tok, sq.n - 1) >> lg];
        const bool bad = bad_page(p.c, id);
        const int64_t page = bad ? 0 : id;
        const uint8_t *key = p.c.key + page * p.c.key_s_page + kh * p.c.key_s_head + ((uint32_t)tok & ((1u << lg) - 1)) * p.c.key_s_tok + 16 * g;
        const float ks = bad ? __builtin_nanf("") : p.c.scale[page * p.c.scale_s_page + kh * p.c.scale_s_head] * p.cs;
        u32x4 k[DP / 16];
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            const u32x4 x = CUT && 32 * c + 16 * g >= p.c.D ? u32x4{0, 0, 0, 0} : *(const u32x4 *)(key + 32 * c);
            u32x4 y[2];
            widen16<BF16>(x, y);
            k[2 * c] = y[0], k[2 * c + 1] = y[1];
        }
        float sum = 0.0f;
        for (int r0 = 0; r0 < rows; r0 += 32) {
            const int r = r0 + n, hq = r / p.T, t = r - hq * p.T;
            const bool real = r < rows && t < sq.tq;
            const int vis = real ? visible8(p, sq, t) : 0;
            if (!__ballot(vis > tok0))
                continue;   // none of them sees any of the wave's tokens
            const bool mask = __ballot(vis < tok0 + 32) != 0;
            u32x4 q[DP / 16];
            const uint16_t *src = p.q + b * p.q_s_seq + (kh * p.gq + hq) * p.q_s_head + t * p.q_s_tok + 16 * g;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                q[s] = u32x4{0, 0, 0, 0};
                if (real && (!CUT || 32 * (s >> 1) + 16 * g < p.c.D))
                    q[s] = *(const u32x4 *)(src + 32 * (s >> 1) + 8 * (s & 1));
            }
            if (g == 0) {
                lds_lse[wave][n] = real ? lse[r] * kLog2e : 0.0f;
                lds_vis[wave][n] = vis;
            }
            f32x16 S;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                S[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
                S = mfma32<BF16>(q[s], k[s], S);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own rows of the LDS
            float part_sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 l = *(const float4 *)&lds_lse[wave][8 * j + 4 * g];
                const int4 v = *(const int4 *)&lds_vis[wave][8 * j + 4 * g];
                const float ls[4] = {l.x, l.y, l.z, l.w};
                const int vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(S[4 * j + e], ks, -ls[e]));
                    part_sum += mask ? tok < vs[e] ? x : 0.0f : x;
                }
            }
            sum += part_sum;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        sum = other_sum(sum);
        if (g == 0 && tok < tokens)
            w.weights[b * w.w_s_seq + kh * w.w_s_head + tok] += sum;
    }
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
    if (const int rc = kitty_cache8_attention_workspace_size(cache, args, bytes))
        return rc;
    *bytes = up16(*bytes) + up16((size_t)args->batch * args->num_q_heads * args->tokens * 4);
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
    const size_t rows = up16((size_t)a.batch * a.num_q_heads * a.tokens * 4);
    if (!a.lse)
        a.lse = (float *)a.workspace;
    a.workspace = (char *)a.workspace + rows;
    a.workspace_bytes -= rows;
    if (const int rc = kitty_cache8_attention(cache, &a, stream))
        return rc;
    Weigh8 w{};
    Attend8 &p = w.a;
    if (const int rc = check_cache8(cache, p.c))
        return rc;
    p.q = a.q, p.lse = a.lse;
    p.q_s_seq = a.q_s_seq, p.q_s_head = a.q_s_head, p.q_s_tok = a.q_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.lens = a.lens, p.q_lens = a.q_lens;
    p.B = a.batch, p.Hq = a.num_q_heads, p.T = a.tokens, p.gq = a.num_q_heads / p.c.H;
    p.table_pages = a.table_pages, p.causal = a.causal ? 1 : 0;
    p.cs = a.sm_scale * kLog2e;
    w.weights = weights->weights, w.w_s_seq = weights->s_seq, w.w_s_head = weights->s_head, w.N = weights->tokens;
    const int64_t cap = std::min<int64_t>((int64_t)a.table_pages << p.c.lg, w.N), pairs = (int64_t)p.B * p.c.H;
    if (cap == 0)
        return KITTY_OK;
    // a workgroup's tokens, or as many of them as leave enough workgroups to fill the device
    w.blocks = (int)std::min<int64_t>((cap + kWeighTokens - 1) / kWeighTokens, std::max<int64_t>(1, 16384 / pairs));
    const dim3 grid((unsigned)(pairs * w.blocks)), block(64 * kWeighWaves);
    const hipStream_t st = (hipStream_t)stream;
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
    return check_launch("cache8_weigh_kernel");
}
