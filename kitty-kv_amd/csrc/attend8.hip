// Attention over the 8-bit paged cache, on gfx950: which kernel takes a call, its
// launches, and the kernel that joins the parts of rows whose tokens were split and, for
// calls that weigh tokens by the scores of a few rows, makes the weights.
#include "attend8_rows.h"

namespace kitty {

// Joins the partials of each row; also, after the row kernel, the rows no
// workgroup touched: of sequences without tokens (0) and of broken lengths (NaN).
// DP / 4 lanes take a row, four channels each.  ALONE: a workgroup per row, whose
// lane groups share its partials and join in LDS (few rows, many partials);
// otherwise a row per lane group.  TILES: the partials are the tile kernel's
// p.splits parts.
template <int DP, bool BF16, bool TILES, bool ALONE, bool STAT>
__device__ __forceinline__ void merge_rows(const Attend8 &p, int RM)
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
    if (STAT && ch == 0 && p.stat)
        p.stat[((int64_t)b * p.Hq + h) * p.T + t] = make_float2(m, inv);
}

template <int DP, bool BF16, bool TILES, bool ALONE, bool STAT>
__global__ __launch_bounds__(64 * kWaves) void cache8_merge_kernel(Attend8 p, int RM)
{
    merge_rows<DP, BF16, TILES, ALONE, STAT>(p, RM);
}

// The weights of a launch of the row kernel that left its scores.  The rows' tops and sums
// are joined here again, a wave a row, so that merge and weights are one launch (4 rows of
// one sequence of 4,096 tokens, 8 KV heads 13.6 us, 16.2 with a launch of their own).  Bound
// by HBM where the scores are many: 67 MB of them for 16 x 32,768 tokens.
__device__ __forceinline__ void weigh_scores(const Attend8 &p, int index, int blocks)
{
    __shared__ float2 stats[16];
    __shared__ int vis[16];
    const int pairs = p.B * p.c.H, pair = index % pairs, block = index / pairs;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, rows = p.gq * p.T;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tab = p.ws_tab[pair];   // of a sequence without tokens it holds anything and is not used
    const Seq8 sq = seq8(p, b);
    const int tokens = sq.bad ? 0 : min(sq.n, p.w_tokens);
    if ((int64_t)block * 1024 >= tokens)
        return;
    const int slot = min(tab.x, 2 * p.n_wg - 1), begin = slot >> 1, count = min(tab.y, p.n_wg - 1) - begin + 1;
    if (threadIdx.x < 16)
        vis[threadIdx.x] = (int)threadIdx.x < rows ? min(visible8(p, sq, threadIdx.x / p.gq), tokens) : 0;
    for (int r = wave; r < rows; r += kWaves) {
        if (slot < 0) {
            const int t = r / p.gq, h = r - t * p.gq;
            if (lane == 0)
                stats[r] = p.stat[((int64_t)b * p.Hq + kh * p.gq + h) * p.T + t];
            continue;
        }
        float m = kLowest, l = 0.0f;
        for (int k = lane; k < count; k += 64) {
            const float2 ml = p.ws_ml[(int64_t)(k == 0 ? slot : 2 * (begin + k)) * 16 + r];
            const float mn = fmaxf(m, ml.x);
            l = __builtin_amdgcn_exp2f(m - mn) * l + __builtin_amdgcn_exp2f(ml.x - mn) * ml.y;
            m = mn;
        }
        float top = m;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
            top = fmaxf(top, __shfl_xor(top, off));
        l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
            l += __shfl_xor(l, off);
        if (lane == 0)
            stats[r] = make_float2(top, 1.0f / l);
    }
    __syncthreads();
    for (int64_t tok = (int64_t)block * 1024 + 4 * threadIdx.x; tok < tokens; tok += (int64_t)blocks * 1024)
        weigh_scores4(p.scores + (int64_t)pair * rows * p.sc_cap, rows, stats, vis, (int)tok, tokens, p.weights + b * p.w_s_seq + kh * p.w_s_head);
}

// Both, `merges` workgroups of the first and `blocks` for each pair of the second.
template <int DP, bool BF16, bool ALONE>
__global__ __launch_bounds__(64 * kWaves) void cache8_merge_weigh_kernel(Attend8 p, int merges, int blocks)
{
    if ((int)blockIdx.x < merges)
        merge_rows<DP, BF16, false, ALONE, true>(p, 16);
    else
        weigh_scores(p, (int)blockIdx.x - merges, blocks);
}

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
// 3. The tile kernel beyond.  Where a weighed call (kitty_cache8_weighed_attention) would split the
// tokens of each row block, cache8_shared_kernel's runs take them (32 queries of 8 sequences of
// 4,000 to 16,000 tokens: 79 and 10 for the join, against 97 and 8.5 us in equal parts of each).
constexpr int64_t kDirectBytes = 1024 * 128, kDirectItems = 4096;

struct Plan8 {
    bool tiles, direct, runs;
    int DP, RT, nrb, n_wg, splits;
    size_t o_bytes, ml_bytes, bytes;
};

// weighed: a call that leaves its rows' maxima and sums, and scores, the scores as well.
static int plan8(const Cache8 &c, const kitty_cache8_attention_args &a, bool weighed, bool scores, Plan8 &pl)
{
    const int64_t rows = (int64_t)a.num_q_heads / c.H * a.tokens, pairs = (int64_t)a.batch * c.H;
    const int64_t cap = (int64_t)a.table_pages << c.lg, units = kStart + (cap + kUnit - 1) / kUnit;
    if (rows > kMaxBlocks || pairs > kMaxBlocks || pairs * rows > kMaxBlocks)
        return fail(KITTY_E_UNSUPPORTED, "too many rows for one launch");
    const int64_t tokens = a.plan_tokens > 0 ? std::min<int64_t>(a.plan_tokens, cap) : cap;
    const int cus = device_cus();
    pl.DP = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    pl.direct = pl.DP <= 128 && tokens * pl.DP <= kDirectBytes &&
                (rows <= 32 ? pairs <= kDirectItems : pairs * ((rows + 31) / 32) <= cus) && !(weighed && !scores && rows <= 16);
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
    pl.runs = weighed && pl.tiles && pl.splits > 1 && items * (cap / 64 + 4) <= 0x7fffffff;   // its units of 64 tokens
    if (pl.runs) {
        pl.bytes = tile_runs_bytes(c, a);
        return KITTY_OK;
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

int attend8_bytes(const kitty_cache8 *cache, const kitty_cache8_attention_args *args, bool scores, size_t &bytes)
{
    Cache8 c;
    Plan8 pl;
    if (const int rc = check_attend8(cache, args, c))
        return rc;
    if (const int rc = plan8(c, *args, true, scores, pl))
        return rc;
    bytes = pl.bytes;
    return KITTY_OK;
}

int attend8(const kitty_cache8 *cache, const kitty_cache8_attention_args *args, hipStream_t stream, Leave8 &leave)
{
    Attend8 p{};
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
    if (const int rc = plan8(p.c, a, leave.stat != nullptr, leave.scores != nullptr, pl))
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

    p.stat = leave.stat, p.scores = leave.scores, p.sc_cap = leave.sc_cap;
    p.weights = leave.weights, p.w_s_seq = leave.w_s_seq, p.w_s_head = leave.w_s_head, p.w_tokens = leave.w_tokens;
    leave.weighed = leave.scores != nullptr;
    const hipStream_t st = stream;
    const bool bf16 = a.dtype == KITTY_DTYPE_BF16;
    const dim3 block(64 * kWaves);
    auto merge = [&](auto dp, auto bf, auto tiles) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value, TILES = decltype(tiles)::value;
        const int64_t rows = (int64_t)p.B * p.Hq * p.T;
        const int RM = TILES ? kTileRows : 16 * pl.RT;
        if constexpr (!TILES) {
            if (p.scores) {
                const int64_t pairs = (int64_t)p.B * p.c.H, groups = 256 * kWaves / DP;
                const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((p.sc_cap + 1023) / 1024, 65536 / pairs));
                const int64_t merges = rows < kMergeRows ? rows : (rows + groups - 1) / groups;
                const dim3 grid((unsigned)(merges + pairs * blocks));
                if (rows < kMergeRows)
                    hipLaunchKernelGGL((cache8_merge_weigh_kernel<DP, BF, true>), grid, block, 0, st, p, (int)merges, (int)blocks);
                else
                    hipLaunchKernelGGL((cache8_merge_weigh_kernel<DP, BF, false>), grid, block, 0, st, p, (int)merges, (int)blocks);
                return;
            }
        }
        auto launch = [&](auto stat) {
            constexpr bool STAT = decltype(stat)::value;
            const int64_t groups = 256 * kWaves / DP;
            if (rows < kMergeRows)
                hipLaunchKernelGGL((cache8_merge_kernel<DP, BF, TILES, true, STAT>), dim3((unsigned)rows), block, 0, st, p, RM);
            else
                hipLaunchKernelGGL((cache8_merge_kernel<DP, BF, TILES, false, STAT>), dim3((unsigned)((rows + groups - 1) / groups)), block,
                                   0, st, p, RM);
        };
        if (p.stat)
            launch(std::true_type{});
        else
            launch(std::false_type{});
    };
    auto rows = [&](auto dp, auto rt, auto bf) {
        constexpr int DP = decltype(dp)::value, RT = decltype(rt)::value;
        constexpr bool BF = decltype(bf)::value;
        const dim3 pairs((unsigned)(p.B * p.c.H * p.nrb)), runs((unsigned)p.n_wg), waves(64 * row_waves(RT, true));
        if constexpr (RT == 1) {
            if (p.scores) {
                if constexpr (DP <= 128) {
                    if (pl.direct && p.c.D == DP)
                        hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, true, kScores>), pairs, waves, 0, st, p);
                    else if (pl.direct)
                        hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, true, kScores>), pairs, waves, 0, st, p);
                    if (pl.direct)
                        return;
                }
                if (p.c.D == DP)
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, false, kScores>), runs, block, 0, st, p);
                else
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, false, kScores>), runs, block, 0, st, p);
                return;
            }
        }
        auto launch = [&](auto mode) {
            constexpr int MODE = decltype(mode)::value;
            if constexpr (DP <= 128 && RT <= 2 && !(RT == 1 && MODE == kStat)) {   // (plan8: those are split)
                if (pl.direct && p.c.D == DP)
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, true, MODE>), pairs, waves, 0, st, p);
                else if (pl.direct)
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, true, MODE>), pairs, waves, 0, st, p);
                if (pl.direct)
                    return;
            }
            if (p.c.D == DP)
                hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, false, false, MODE>), runs, block, 0, st, p);
            else
                hipLaunchKernelGGL((cache8_rows_kernel<DP, RT, BF, true, false, MODE>), runs, block, 0, st, p);
        };
        if (p.stat)
            launch(std::integral_constant<int, kStat>{});
        else
            launch(std::integral_constant<int, kPlain>{});
    };
    auto go = [&](auto dp, auto bf) {
        constexpr int DP = decltype(dp)::value;
        if (pl.tiles) {
            if (pl.runs) {
                launch_tile_runs(p, bf16, ws, st);
                return;
            }
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
    if (const int rc = plan8(c, *args, false, false, pl))
        return rc;
    *bytes = pl.bytes;
    return KITTY_OK;
}

extern "C" int kitty_cache8_attention(const kitty_cache8 *cache, const kitty_cache8_attention_args *args,
                                      kitty_stream_t stream)
{
    Leave8 none{};
    return attend8(cache, args, (hipStream_t)stream, none);
}
