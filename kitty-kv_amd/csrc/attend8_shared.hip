// Attention over the 8-bit paged cache for sequences that share prefixes, on gfx950.
//
// A prefix's codes are read once for the rows of all its sequences: each (prefix, KV
// head) is an entry with per * T * group query rows, each (sequence, KV head) another
// with its own tokens and T * group rows.  A row's softmax over both is joined from
// parts, each a maximum m, a sum l of 2^(s - m) and the weighted values o relative to m:
// with M the largest m, sum 2^(m - M) o / sum 2^(m - M) l.  cache8_join_kernel does that
// for the parts of both entries at once.
//
// Up to 64 rows of a prefix (32 at more than 128 channels) its entries and the
// sequences' go through the row kernel together (attend8_rows.h): one launch shares the
// units of all entries evenly.  More rows go through the tile kernel (attend8_tiles.h),
// and the sequences' own tokens through whichever takes their rows.
#include "attend8_rows.h"
#include "attend8_tiles.h"

namespace kitty {

// The parts that a launch left of its entries.
struct Part8 {
    const float *o;
    const float2 *ml;
    const int2 *tab;    // row kernel, by (entry, KV head): first slot, last workgroup (-1: all in one slot)
    int e0, nrb, RM;    // its first entry, row blocks of an entry, rows of a block
    int splits, n_wg;   // parts of a row block (tile kernel; 0: row kernel), workgroups (row kernel)
};

// Joins the parts of each row, of its prefix and of its own tokens.  DP / 4 lanes take a
// row, four channels each; ALONE: a workgroup per row, whose lane groups share its parts.
template <int DP, bool BF16, bool ALONE>
__global__ __launch_bounds__(64 * kWaves) void cache8_join_kernel(Attend8 p, Part8 of_prefix, Part8 of_own)
{
    constexpr int LPR = DP / 4, GROUPS = 64 * kWaves / LPR, STEP = ALONE ? GROUPS : 1;
    const int group = threadIdx.x / LPR, ch = 4 * (threadIdx.x % LPR);
    const int rows = p.gq * p.T, all = ALONE ? blockIdx.x : blockIdx.x * GROUPS + group;
    const int pair = all / rows, row = all - pair * rows;
    if (!ALONE && pair >= p.B * p.c.H)
        return;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, f = b / p.per;
    const int t = row / p.gq, h = kh * p.gq + row - t * p.gq;
    const Seq8 own = seq8(p, b);
    const int before = p.prefix_lens[f];
    const bool bad = own.bad || before < 0 || before > (int64_t)p.prefix_pages << p.c.lg || (before > 0 && p.c.num_pages == 0);
    float m = kLowest, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fold = [&](float m1, float l1, float4 x) {
        const float mn = fmaxf(m, m1);
        const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(m1 - mn);
        m = mn;
        l = f0 * l + f1 * l1;
        o.x = f0 * o.x + f1 * x.x, o.y = f0 * o.y + f1 * x.y, o.z = f0 * o.z + f1 * x.z, o.w = f0 * o.w + f1 * x.w;
    };
    auto parts = [&](const Part8 &s, int e, int r, int tokens) {
        if (tokens <= 0)
            return;   // the row kernel left nothing of it
        const int rb = r / s.RM, rr = r - rb * s.RM, item = ((e - s.e0) * p.c.H + kh) * s.nrb + rb;
        int slot = 0, first = 0, count = s.splits;
        if (s.splits == 0) {
            const int2 tab = s.tab[item];
            // (bounds for lengths that another stream changes under the call)
            slot = min(max(tab.x, 0), tab.y < 0 ? 2 * s.n_wg + item : 2 * s.n_wg - 1), first = slot >> 1;
            count = tab.y < 0 ? 1 : min(tab.y, s.n_wg - 1) - first + 1;
        }
        for (int i = ALONE ? group : 0; i < count; i += 4 * STEP) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = min(i + j * STEP, count - 1);
                const int64_t at = s.splits ? ((int64_t)item * s.splits + k) * s.RM + rr
                                            : (int64_t)(k == 0 ? slot : 2 * (first + k)) * s.RM + rr;
                ml[j] = s.ml[at];
                x[j] = *(const float4 *)(s.o + at * DP + ch);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * STEP < count)
                    fold(ml[j].x, ml[j].y, x[j]);
        }
    };
    if (!bad) {
        parts(of_prefix, f, (b - f * p.per) * rows + row, before);
        parts(of_own, p.F + b, row, own.n);
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
    // rows that see nothing: padding's parts hold what the real rows of their blocks see
    const bool none = !bad && (t >= own.tq || (p.causal ? before + (own.n - own.tq + t + 1) <= 0 : before == 0 && own.n == 0));
    if (none)
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float inv = bad ? __builtin_nanf("") : none ? 0.0f : 1.0f / l;
    *(uint2 *)(p.out + b * p.o_s_seq + h * p.o_s_head + t * p.o_s_tok + ch) =
        make_uint2((uint32_t)f2x(o.x * inv, BF16) | (uint32_t)f2x(o.y * inv, BF16) << 16,
                   (uint32_t)f2x(o.z * inv, BF16) | (uint32_t)f2x(o.w * inv, BF16) << 16);
    if (ch == 0 && p.lse)
        p.lse[((int64_t)b * p.Hq + h) * p.T + t] =
            bad ? __builtin_nanf("") : none ? -__builtin_inff() : (m + __builtin_log2f(l)) / kLog2e;
}

// One launch over entries e0 .. e0 + entries - 1, and its part of the workspace.
struct Launch8 {
    bool tiles;
    int RT, e0, entries, nrb, n_wg, splits;
    size_t o_at, ml_at, tab_at;
};

struct SharedPlan8 {
    int DP;
    bool together;        // one launch of the row kernel for prefixes and sequences
    Launch8 prefix, own;
    size_t bytes;
};

static int row_blocks(int64_t rows, int DP)
{
    return rows <= 16 ? 1 : rows <= 32 || DP == 256 ? 2 : rows <= 48 ? 3 : 4;
}

static int plan_shared(const Cache8 &c, const kitty_cache8_shared_args &a, SharedPlan8 &pl)
{
    const int64_t own_rows = (int64_t)a.num_q_heads / c.H * a.tokens, rows = (int64_t)a.batch * a.num_q_heads * a.tokens;
    if (own_rows > kMaxBlocks || rows > kMaxBlocks || (int64_t)a.batch * c.H > kMaxBlocks)
        return fail(KITTY_E_UNSUPPORTED, "too many rows for one launch");
    const int64_t prefix_rows = own_rows * (a.batch / a.prefixes);
    const int64_t prefix_cap = (int64_t)a.prefix_pages << c.lg, own_cap = (int64_t)a.table_pages << c.lg;
    const int cus = device_cus();
    pl.DP = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    pl.bytes = 0;
    const int most = pl.DP == 256 ? 32 : 64;   // rows of an entry that the row kernel takes
    // row launches share at most `units` units
    auto plan = [&](Launch8 &la, bool tiles, int64_t n, int e0, int entries, int64_t tokens, int64_t units) {
        la.tiles = tiles, la.e0 = e0, la.entries = entries;
        la.RT = row_blocks(n, pl.DP);
        const int RM = tiles ? kTileRows : 16 * la.RT;
        const int64_t nrb = (n + RM - 1) / RM, items = entries * (int64_t)c.H * nrb;
        int64_t slots;
        la.nrb = (int)nrb, la.n_wg = la.splits = 0;
        if (tiles) {
            const int64_t want = (pl.DP == 256 ? 1 : 2) * (int64_t)cus / std::max<int64_t>(items, 1);
            la.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, tokens / 256));
            slots = items * la.splits;
            if (slots > kMaxBlocks)
                return fail(KITTY_E_UNSUPPORTED, "too many rows for one launch");
        } else {
            if (units > 0x7fffffff)
                return fail(KITTY_E_UNSUPPORTED, "too many rows and pages for one launch");
            la.n_wg = (int)std::max<int64_t>(1, std::min<int64_t>((two_per_cu(pl.DP, la.RT) ? 2 : 1) * cus, units));
            slots = 2 * la.n_wg + items;
        }
        la.o_at = pl.bytes;
        la.ml_at = la.o_at + up16((size_t)slots * RM * pl.DP * 4);
        la.tab_at = la.ml_at + up16((size_t)slots * RM * 8);
        pl.bytes = la.tab_at + (tiles ? 0 : up16((size_t)items * 8));
        return KITTY_OK;
    };
    const int64_t prefix_tokens = a.plan_prefix > 0 ? std::min<int64_t>(a.plan_prefix, prefix_cap) : prefix_cap;
    const int64_t own_tokens = a.plan_tokens > 0 ? std::min<int64_t>(a.plan_tokens, own_cap) : own_cap;
    const int64_t prefix_units = (int64_t)a.prefixes * c.H * (kStart + (prefix_cap + kUnit - 1) / kUnit);
    const int64_t own_units = (int64_t)a.batch * c.H * (kStart + (own_cap + kUnit - 1) / kUnit);
    pl.together = prefix_rows <= most;
    if (pl.together) {
        const int rc = plan(pl.prefix, false, prefix_rows, 0, a.prefixes + a.batch, 0, prefix_units + own_units);
        pl.own = pl.prefix;
        return rc;
    }
    if (const int rc = plan(pl.prefix, true, prefix_rows, 0, a.prefixes, prefix_tokens, 0))
        return rc;
    return plan(pl.own, own_rows > most, own_rows, a.prefixes, a.batch, own_tokens, own_units);
}

static int check_shared(const kitty_cache8 *cache, const kitty_cache8_shared_args *args, Cache8 &c)
{
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, c))
        return rc;
    const kitty_cache8_shared_args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.table_pages < 0 || a.prefix_pages < 0 || a.plan_tokens < 0 || a.plan_prefix < 0)
        return fail(KITTY_E_INVALID, "batch, tokens, table_pages, prefix_pages, plan_tokens and plan_prefix must not be negative");
    if (a.prefixes <= 0 || a.batch % a.prefixes)
        return fail(KITTY_E_INVALID, "batch must be a multiple of a positive number of prefixes");
    if (a.num_q_heads <= 0 || a.num_q_heads % c.H)
        return fail(KITTY_E_INVALID, "num_q_heads must be a positive multiple of num_kv_heads");
    if (a.dtype != KITTY_DTYPE_F16 && a.dtype != KITTY_DTYPE_BF16)
        return fail(KITTY_E_INVALID, "dtype must be KITTY_DTYPE_F16 or KITTY_DTYPE_BF16");
    if (!(a.sm_scale > 0.0f) || a.sm_scale > 1e30f)
        return fail(KITTY_E_INVALID, "sm_scale must be positive and finite");
    if ((int64_t)a.table_pages << c.lg > 1 << 30 || (int64_t)a.prefix_pages << c.lg > 1 << 30)
        return fail(KITTY_E_UNSUPPORTED, "a block table is limited to 2^30 tokens a sequence");
    return KITTY_OK;
}

} // namespace kitty

using namespace kitty;

extern "C" int kitty_cache8_shared_attention_workspace_size(const kitty_cache8 *cache, const kitty_cache8_shared_args *args,
                                                            size_t *bytes)
{
    Cache8 c;
    SharedPlan8 pl;
    if (!bytes)
        return fail(KITTY_E_INVALID, "bytes is NULL");
    if (const int rc = check_shared(cache, args, c))
        return rc;
    *bytes = 0;
    if (args->batch == 0 || args->tokens == 0)
        return KITTY_OK;
    if (const int rc = plan_shared(c, *args, pl))
        return rc;
    *bytes = pl.bytes;
    return KITTY_OK;
}

extern "C" int kitty_cache8_shared_attention(const kitty_cache8 *cache, const kitty_cache8_shared_args *args,
                                             kitty_stream_t stream)
{
    Attend8 p{};
    SharedPlan8 pl;
    if (const int rc = check_shared(cache, args, p.c))
        return rc;
    const kitty_cache8_shared_args &a = *args;
    if (a.batch == 0 || a.tokens == 0)
        return KITTY_OK;
    if (!a.q || !a.out || !a.lens || !a.prefix_lens || (!a.block_table && a.table_pages) || (!a.prefix_table && a.prefix_pages))
        return fail(KITTY_E_INVALID, "NULL q, out, lens, prefix_lens, block_table or prefix_table");
    if (!aligned(a.q, 16) || !aligned(a.out, 16))
        return fail(KITTY_E_INVALID, "q and out must be 16-byte aligned");
    for (int64_t s : {a.q_s_seq, a.q_s_head, a.q_s_tok, a.o_s_seq, a.o_s_head, a.o_s_tok})
        if (s % 8)
            return fail(KITTY_E_INVALID, "strides of q and out must be multiples of 8 elements (16-byte rows)");
    if (const int rc = plan_shared(p.c, a, pl))
        return rc;
    if (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < pl.bytes)
        return fail(KITTY_E_INVALID,
                    "workspace is NULL, misaligned or smaller than kitty_cache8_shared_attention_workspace_size");
    p.q = a.q, p.out = a.out, p.lse = a.lse;
    p.q_s_seq = a.q_s_seq, p.q_s_head = a.q_s_head, p.q_s_tok = a.q_s_tok;
    p.o_s_seq = a.o_s_seq, p.o_s_head = a.o_s_head, p.o_s_tok = a.o_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.lens = a.lens, p.q_lens = a.q_lens;
    p.prefix_table = a.prefix_table, p.pt_stride = a.pt_stride, p.prefix_lens = a.prefix_lens;
    p.B = a.batch, p.Hq = a.num_q_heads, p.T = a.tokens, p.gq = a.num_q_heads / p.c.H;
    p.F = a.prefixes, p.per = a.batch / a.prefixes, p.prefix_pages = a.prefix_pages;
    p.table_pages = a.table_pages, p.causal = a.causal ? 1 : 0;
    p.cs = a.sm_scale * kLog2e;

    const hipStream_t st = (hipStream_t)stream;
    const dim3 block(64 * kWaves);
    char *ws = (char *)a.workspace;
    auto with = [&](const Launch8 &la) {
        Attend8 x = p;
        x.e0 = la.e0, x.entries = la.entries, x.nrb = la.nrb, x.n_wg = la.n_wg, x.splits = la.splits;
        x.ws_o = (float *)(ws + la.o_at), x.ws_ml = (float2 *)(ws + la.ml_at), x.ws_tab = (int2 *)(ws + la.tab_at);
        return x;
    };
    auto part = [&](const Launch8 &la) {
        return Part8{(const float *)(ws + la.o_at), (const float2 *)(ws + la.ml_at), (const int2 *)(ws + la.tab_at), la.e0,
                     la.nrb, la.tiles ? kTileRows : 16 * la.RT, la.splits, la.n_wg};
    };
    auto launch = [&](const Launch8 &la, auto dp, auto bf, auto cut) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value, CUT = decltype(cut)::value;
        const Attend8 x = with(la);
        if (la.tiles) {
            const dim3 grid((unsigned)(la.entries * p.c.H * la.nrb * la.splits));
            hipLaunchKernelGGL((cache8_tile_kernel<DP, BF, CUT, true>), grid, dim3(64 * kTileWaves), 0, st, x);
            return;
        }
        const dim3 runs((unsigned)la.n_wg);
        if (la.RT == 1)
            hipLaunchKernelGGL((cache8_rows_kernel<DP, 1, BF, CUT, false, kShared>), runs, block, 0, st, x);
        else if (la.RT == 2)
            hipLaunchKernelGGL((cache8_rows_kernel<DP, 2, BF, CUT, false, kShared>), runs, block, 0, st, x);
        else if constexpr (DP <= 128) {
            if (la.RT == 3)
                hipLaunchKernelGGL((cache8_rows_kernel<DP, 3, BF, CUT, false, kShared>), runs, block, 0, st, x);
            else
                hipLaunchKernelGGL((cache8_rows_kernel<DP, 4, BF, CUT, false, kShared>), runs, block, 0, st, x);
        }
    };
    auto go = [&](auto dp, auto bf, auto cut) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value;
        launch(pl.prefix, dp, bf, cut);
        if (!pl.together)
            launch(pl.own, dp, bf, cut);
        const int64_t rows = (int64_t)p.B * p.Hq * p.T, groups = 256 * kWaves / DP;
        const Part8 x = part(pl.prefix), y = part(pl.own);
        if (rows < kMergeRows)
            hipLaunchKernelGGL((cache8_join_kernel<DP, BF, true>), dim3((unsigned)rows), block, 0, st, p, x, y);
        else
            hipLaunchKernelGGL((cache8_join_kernel<DP, BF, false>), dim3((unsigned)((rows + groups - 1) / groups)), block, 0, st, p, x, y);
    };
    auto by_type = [&](auto dp) {
        const bool cut = p.c.D != decltype(dp)::value, bf16 = a.dtype == KITTY_DTYPE_BF16;
        if (bf16)
            cut ? go(dp, std::true_type{}, std::true_type{}) : go(dp, std::true_type{}, std::false_type{});
        else
            cut ? go(dp, std::false_type{}, std::true_type{}) : go(dp, std::false_type{}, std::false_type{});
    };
    if (pl.DP == 64)
        by_type(std::integral_constant<int, 64>{});
    else if (pl.DP == 128)
        by_type(std::integral_constant<int, 128>{});
    else
        by_type(std::integral_constant<int, 256>{});
    return check_launch("8-bit cache attention over shared prefixes");
}
