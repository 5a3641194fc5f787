// Attention over the 8-bit paged cache for sequences that share prefixes, on gfx950.
//
// A prefix's codes are read once for the rows of all its sequences: each (prefix, KV
// head) is an entry with per * T * group query rows, each (sequence, KV head) another
// with its own tokens and T * group rows.  A row's softmax over both is joined from
// parts, each a maximum m, a sum l of 2^(s - m) and the weighted values o relative to m:
// with M the largest m, sum 2^(m - M) o / sum 2^(m - M) l.  cache8_join_kernel does that
// for the parts of both entries at once.
//
// Few rows of a prefix: its entries and the sequences' go through the row kernel together
// (attend8_rows.h), whose one launch shares the units of all entries evenly.
// More: cache8_shared_kernel, one launch for both kinds of work.  Some workgroups share
// the prefixes' tiles (attend8_tiles.h), bound by the matrix cores and the softmax, the
// others the sequences' own tokens, by the row kernel's body and bound by HBM; each kind
// is cut evenly by lengths read on the device, and so are the workgroups between them.
// The first half of a launch fills every CU once and the second half again, so that in
// the middle of the range a CU holds one of each.  Sequences with more rows than the row
// kernel's body takes go through tiles as well.
//
// Measured, fp16 and 8 KV heads of 128 unless said: 64 sequences of 100-2,000 tokens
// behind 16,384 shared ones, 32 query heads, bf16: 69 us, of them 8 for the join (the
// tiles alone 51 of the kernel's 64, the rows alone 50, its beginning 5); eight samples of
// each of 8 prompts of 2,000-9,000, 64 query heads: 61, of them 7; five draft tokens of 16
// sequences behind 30,000, bf16: 97; six padded questions of up to 300 tokens about two
// documents of 5,000-8,000, 16 / 4 heads of 64: 97; four samples of a prompt of 1,000,
// 8 query heads: 11, one launch.  attend over the first in joined tables, whose pages it
// reads for every sequence, takes 4.1 times as long, over the second and third 1.7.
// The matrix cores' and the vector instructions' phases of a tile's waves stand one after
// the other: three workgroups a CU at 64 channels, a third tile in flight and wave
// priorities gained nothing.
#include "attend8_rows.h"
#include "attend8_tiles.h"

namespace kitty {

// The parts that a launch left of its entries.
struct Part8 {
    const float *o;
    const float2 *ml;
    const int2 *tab;        // by item: first slot, last workgroup (-1: all in one slot)
    int e0, nrb, RM, n_wg;  // its first entry, row blocks of an entry, rows of a block, workgroups
    int item0;              // the first entry's first item
};

// Joins the parts of each row, of its prefix and of its own tokens.  DP / 4 lanes take a
// row, four channels each; ALONE: a workgroup per row, whose lane groups share its parts.
// 19 MB of parts in 8.4 us for 2,048 rows of a prefix in 18 parts: 8 or 16 parts in flight
// take 8.4 and 10.1, a workgroup per row 8.7 there, and 13.0 where it is 6.6 for 4,096 rows
// of few parts.
template <int DP, bool BF16, bool ALONE>
__global__ __launch_bounds__(64 * kWaves) void cache8_join_kernel(Attend8 p, Part8 of_prefix, Part8 of_own)
{
    constexpr int LPR = DP / 4, GROUPS = 64 * kWaves / LPR, STEP = ALONE ? GROUPS : 1;
    const int group = threadIdx.x / LPR, ch = 4 * (threadIdx.x % LPR);
    const int rows = p.gq * p.T, all = ALONE ? blockIdx.x : blockIdx.x * GROUPS + group;
    const int pair = all / rows, row = all - pair * rows;
    if (!ALONE && pair >= p.B * p.c.H)
        return;
    const int b = pair / p.c.H, kh = pair - b * p.c.H, f = p.F ? b / p.per : 0;
    const int t = row / p.gq, h = kh * p.gq + row - t * p.gq;
    // an item's table entry is loaded before its lengths are known; where nothing is left it holds anything
    auto place = [&](const Part8 &s, int e, int r, int &rr) {
        const int rb = r / s.RM;
        rr = r - rb * s.RM;
        return s.item0 + ((e - s.e0) * p.c.H + kh) * s.nrb + rb;
    };
    int rr_p, rr_o;
    const int q = p.row_map ? min(p.row_first[b] + t, p.per * p.T - 1) : (b - f * p.per) * p.T + t;
    const int item_p = place(of_prefix, f, q * p.gq + h - kh * p.gq, rr_p), item_o = place(of_own, p.F + b, row, rr_o);
    const int2 tab_p = of_prefix.tab[p.F ? item_p : 0], tab_o = of_own.tab[item_o];
    const Seq8 own = seq8(p, b);
    const int before = p.F ? p.prefix_lens[f] : 0;   // F: 0 for launch_tile_runs
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
    auto parts = [&](const Part8 &s, int item, int rr, int2 tab, int tokens) {
        if (tokens <= 0)
            return;
        // (bounds for lengths that another stream changes under the call)
        const int slot = min(max(tab.x, 0), tab.y < 0 ? 2 * s.n_wg + item : 2 * s.n_wg - 1), first = slot >> 1;
        const int count = tab.y < 0 ? 1 : min(tab.y, s.n_wg - 1) - first + 1;
        for (int i = ALONE ? group : 0; i < count; i += 4 * STEP) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = min(i + j * STEP, count - 1);
                const int64_t at = (int64_t)(k == 0 ? slot : 2 * (first + k)) * s.RM + rr;
                ml[j] = s.ml[at];
                x[j] = *(const float4 *)(s.o + at * DP + ch);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * STEP < count)
                    fold(ml[j].x, ml[j].y, x[j]);
        }
    };
    if (!bad && t < own.tq) {
        parts(of_prefix, item_p, rr_p, tab_p, before);
        parts(of_own, item_o, rr_o, tab_o, own.n);
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
    if (ch == 0 && p.stat)
        p.stat[((int64_t)b * p.Hq + h) * p.T + t] = make_float2(m, inv);
}

// The prefixes' real queries where they are padded, a wave per prefix.
__global__ __launch_bounds__(64 * kWaves) void cache8_shared_queries_kernel(Attend8 p)
{
    const int lane = threadIdx.x & 63, f = blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (f >= p.F)
        return;
    int count = 0;
    int32_t *map = p.row_map + (int64_t)f * p.per * p.T;
    for (int q0 = 0; q0 < p.per; q0 += 64) {
        int mine = 0;
        if (q0 + lane < p.per) {
            const Seq8 own = seq8(p, f * p.per + q0 + lane);
            mine = own.bad ? 0 : own.tq;
        }
        int inc = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int y = __shfl_up(inc, off);
            inc += lane >= off ? y : 0;
        }
        if (q0 + lane < p.per)
            p.row_first[f * p.per + q0 + lane] = count + inc - mine;
        for (int q = 0; q < min(64, p.per - q0); ++q) {
            const int n = __builtin_amdgcn_readlane(mine, q), first = count + __builtin_amdgcn_readlane(inc, q) - n;
            for (int t = lane; t < n; t += 64)
                map[first + t] = (q0 + q) * p.T + t;
        }
        count += __builtin_amdgcn_readlane(inc, 63);
    }
    if (lane == 0)
        p.row_count[f] = count;
}

// Units of tiles: kTile tokens for kTileRows rows, and kTileStart for what beginning an
// item costs (its queries' loads and the leaving of its part).
constexpr int kTileStart = 2;

struct Entry8 {
    Seq8 sq;
    int nrb, tiles, units;   // row blocks, tiles and units of an item
};

__device__ __forceinline__ Entry8 tile_entry(const Attend8 &p, int i)
{
    Entry8 e;
    e.sq = entry8<true>(p, i);
    e.nrb = (rows8<true>(p, e.sq, i) + kTileRows - 1) / kTileRows;
    e.tiles = e.sq.bad ? 0 : (e.sq.n + kTile - 1) / kTile;
    e.units = e.tiles && e.nrb ? e.tiles + kTileStart : 0;
    return e;
}

// The sum over the lanes up to this one.
__device__ __forceinline__ int lanes_sum(int v, int lane)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(v, off);
        v += lane >= off ? y : 0;
    }
    return v;
}

// All units of a launch's tile entries and of its row entries: their loads go together.
__device__ __forceinline__ int2 all_units(const Attend8 &a, const Attend8 &own, bool rows)
{
    const int lane = threadIdx.x & 63, most = rows ? max(a.entries, own.entries) : a.entries;
    int x = 0, y = 0;
    for (int i = lane; i - lane < most; i += 64) {
        const Entry8 e = tile_entry(a, min(i, a.entries - 1));
        const int n = rows ? units8(tiles8(seq8(own, min(i, own.entries - 1))), kStart) : 0;
        x += i < a.entries ? e.units * e.nrb * a.c.H : 0;
        y += i < own.entries ? n * own.c.H : 0;
    }
    return make_int2(__builtin_amdgcn_readlane(lanes_sum(x, lane), 63), rows ? __builtin_amdgcn_readlane(lanes_sum(y, lane), 63) : 0);
}

// Workgroup wg of n_wg's run of the `total` units of the tile entries, by item: KV head
// slowest, then row block, then tiles.
template <int DP, bool BF16, bool CUT>
__device__ __forceinline__ void tiles_run(const Attend8 &p, int wg, int n_wg, int total, unsigned char *lds)
{
    const int lane = threadIdx.x & 63, N = min(n_wg, total);
    if (wg >= N)
        return;
    const int u0 = run_start(total, N, wg), u1 = run_start(total, N, wg + 1);
    int i = -1, pre = 0;
    for (int i0 = 0, base = 0; i0 < p.entries; i0 += 64) {
        int x = 0;
        if (i0 + lane < p.entries) {
            const Entry8 e = tile_entry(p, i0 + lane);
            x = e.units * e.nrb * p.c.H;
        }
        const int inc = lanes_sum(x, lane);
        const unsigned long long past = __ballot(base + inc > u0);
        if (past) {
            const int l = __builtin_ctzll(past);
            i = i0 + l;
            pre = base + __builtin_amdgcn_readlane(inc - x, l);
            break;
        }
        base += __builtin_amdgcn_readlane(inc, 63);
    }
    // (the bounds are for lengths that another stream changes under the call)
    for (int u = u0; u < u1 && i >= 0 && i < p.entries;) {
        const Entry8 e = tile_entry(p, i);
        if (e.units == 0 || u >= pre + e.units * e.nrb * p.c.H) {
            pre += e.units * e.nrb * p.c.H;
            ++i;
            continue;
        }
        const int item = (u - pre) / e.units, off = (u - pre) - item * e.units, seg = min(e.units - off, u1 - u);
        if (off + seg > kTileStart) {
            const bool first = off <= kTileStart, whole = first && off + seg == e.units;
            const int kh = item / e.nrb, rb = item - kh * e.nrb;
            const int at = (p.e0 + i < p.F ? (p.e0 + i) * p.c.H * p.nrb : p.item0 + (p.e0 + i - p.F) * p.c.H * p.own_nrb) +
                           kh * (p.e0 + i < p.F ? p.nrb : p.own_nrb) + rb;
            const int slot = whole ? 2 * p.n_wg + at : 2 * wg + (u == u0 ? 0 : 1);
            if (first && threadIdx.x == 0)
                p.ws_tab[at] = make_int2(slot, whole ? -1 : run_of(total, N, pre + (item + 1) * e.units - 1));
            tile_part<DP, BF16, CUT, true>(p, e.sq, i, kh, rb, 0, max(off - kTileStart, 0), off + seg - kTileStart,
                                           (int64_t)slot * kTileRows, lds);
            __syncthreads();
        }
        u += seg;
    }
}

// What a unit of each kind costs, relative to each other (tile, row): a CU's workgroups of
// either kind slow the other's.  us of calls at tile : row, 32 / 8 heads, fp16 / bf16:
//   channels, sequences x queries, tokens shared, own   3:4        1:1        5:4        3:2        2:1
//    64   64 x 1  16,384  1,000                        59 / 54    53 / 49    52 / 47    59 / 50    56 / 51
//    64   32 x 5  16,384  1,000                        85 / 76    82 / 74    80 / 72    77 / 74    87 / 85
//   128   64 x 1   4,000  1,000                        64 / 61    53 / 51    49 / 49    49 / 50    52 / 53
//   128   32 x 5  16,384  1,000                       118 / 99   113 / 97   112 / 93   108 / 96   119 / 109
//   128   64 x 4 (two prefixes)  8,000  3,000         157 / 148  140 / 133  131 / 129  135 / 138  132 / 119
//   256   64 x 1   4,000  1,000                       161 / 136  129 / 112  115 / 100  102 / 91    87 / 86
//   256   64 x 4 (two prefixes)  8,000  3,000         461 / 374  381 / 311  340 / 279  318 / 263  272 / 267
//   256   32 x 5  16,384  1,000 (1:2 281 / 237)       266 / 267  359 / 361  416 / 417  417 / 417  499 / 498
template <int DP, int RT>
constexpr int2 unit_cost() { return DP <= 128 ? int2{5, 4} : RT == 1 ? int2{2, 1} : int2{2, 3}; }

// RT: the row blocks of a sequence's own rows; 0: they go through tiles, and `a` has all entries.
template <int DP, bool BF16, bool CUT, int RT>
__global__ __launch_bounds__(64 * kWaves, DP <= 128 ? 2 : 1) void cache8_shared_kernel(Attend8 a, Attend8 own)
{
    static_assert(kWaves == kTileWaves, "both kinds of work are of one workgroup's size");
    typedef RowLds<DP, RT ? RT : 1, false, kShared> Rows;
    constexpr int LDS = (int)sizeof(Rows) > kTileLds<DP> ? (int)sizeof(Rows) : kTileLds<DP>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[LDS];
    // workgroup i runs on XCD i % 8: neighbours of a run share one
    const int W = gridDim.x, xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    const int2 units = all_units(a, own, RT != 0);
    const int tiles = units.x, rows = units.y;
    if constexpr (RT == 0) {
        tiles_run<DP, BF16, CUT>(a, xcd * (W >> 3) + j, W, tiles, lds);
    } else {
        int n = 0;   // of an XCD's workgroups, those that take tiles
        if (tiles > 0) {
            const int64_t x = (int64_t)tiles * unit_cost<DP, RT>().x, y = (int64_t)rows * unit_cost<DP, RT>().y;
            n = rows == 0 ? W >> 3 : min(max((int)(((W >> 3) * x + (x + y) / 2) / (x + y)), 1), (W >> 3) - 1);
        }
        const int m = (W >> 3) - n;
        if (j < n)
            tiles_run<DP, BF16, CUT>(a, xcd * n + j, 8 * n, tiles, lds);
        else
            rows_run<DP, RT, BF16, CUT, false, kShared>(own, xcd * m + j - n, 8 * m, *(Rows *)lds);
    }
}

// What takes a call, by its sizes.
// 1. Whole sequences, prefix and all, a workgroup for each and KV head, where a stream of
//    both is at most kSharedDirectBytes and the workgroups at most the CUs: one launch.
//    It reads a prefix once for each sequence, from L2 mostly, and saves the join.  The
//    bound is where it begins to lose for few sequences (up to 1 us within it, 4 samples
//    with 8 query heads); more of them or more rows would gain up to twice as far.  us, one
//    launch / the other ways, fp16, 8 KV heads, one prefix, tokens of both together (64 own):
//      channels, sequences x queries, heads  512          1,024        1,280        2,048        4,096
//      128   4 x 1   8                       8.9 / 11.7  12.2 / 11.7  13.0 / 12.0  18.1 / 12.0  35.4 / 13.9
//      128   8 x 1  32                       8.4 / 13.8  12.5 / 16.2  14.1 / 16.6  21.8 / 17.0  39.6 / 18.3
//      128  32 x 1  32                       9.2 / 20.9  13.0 / 22.0  14.8 / 22.4  21.8 / 25.2  39.5 / 29.3
//      128   8 x 8  32                      12.8 / 23.5  18.1 / 30.6  19.4 / 32.4  25.7 / 35.7  44.2 / 38.5
//       64   4 x 1   8                       7.3 / 11.5   9.0 / 11.5   9.6 / 11.5  11.9 / 11.5  19.8 / 12.9
//       64   8 x 1  32                       7.9 / 12.9  10.0 / 14.2  10.0 / 14.3  14.4 / 14.8  22.4 / 15.3
//       64   8 x 8  32                       9.4 / 18.3  12.3 / 24.0  13.4 / 26.2  17.9 / 29.7  28.6 / 33.2
// 2. The row kernel for prefixes and sequences together: up to 64 rows of a prefix, in
//    blocks of 32, and 32 of a sequence.  64 rows of each of 8 prefixes of 2,000-9,000
//    tokens: 57.6 us in two blocks of 32, 64 by way 3, 74 in one block of 64 (its registers leave
//    one wave a SIMD), 78 in four of 16.  Beyond, codes would be read a third time.
// 3. cache8_shared_kernel.
constexpr int64_t kSharedDirectBytes = 1280 * 128;

struct SharedPlan8 {
    int DP, RT;               // RT: own row blocks, 0 where they are tiles
    bool direct;              // one launch of the row kernel on whole sequences
    bool together;            // one launch of the row kernel for prefixes and sequences, RT blocks
    int W, nrb, own_nrb;      // workgroups; row blocks of a prefix and of a sequence
    int64_t items, own_items; // of the prefixes, of the sequences
    size_t o_at, ml_at, tab_at, own_o_at, own_ml_at, own_tab_at, map_at, bytes;
};

static int plan_shared(const Cache8 &c, const kitty_cache8_shared_args &a, SharedPlan8 &pl)
{
    const int64_t own_rows = (int64_t)a.num_q_heads / c.H * a.tokens, rows = (int64_t)a.batch * a.num_q_heads * a.tokens;
    if (own_rows > kMaxBlocks || rows > kMaxBlocks || (int64_t)a.batch * c.H > kMaxBlocks)
        return fail(KITTY_E_UNSUPPORTED, "too many rows for one launch");
    const int64_t prefix_rows = own_rows * (a.batch / a.prefixes);
    const int64_t prefix_cap = (int64_t)a.prefix_pages << c.lg, own_cap = (int64_t)a.table_pages << c.lg;
    const int64_t F = a.prefixes, B = a.batch, H = c.H;
    const int cus = device_cus();
    pl.DP = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
    const bool by_rows = own_rows <= 32;
    pl.direct = by_rows && pl.DP <= 128 && (prefix_cap + own_cap) * pl.DP <= kSharedDirectBytes && B * H <= cus;
    if (pl.direct) {
        pl.RT = own_rows <= 16 ? 1 : 2;
        return KITTY_OK;
    }
    pl.together = prefix_rows <= 64 && by_rows;
    pl.RT = by_rows ? (pl.together ? prefix_rows : own_rows) <= 16 ? 1 : 2 : 0;
    const int RM = by_rows ? 16 * pl.RT : kTileRows;
    pl.nrb = (int)((prefix_rows + (pl.together ? RM : kTileRows) - 1) / (pl.together ? RM : kTileRows));
    pl.own_nrb = by_rows ? 1 : (int)((own_rows + kTileRows - 1) / kTileRows);
    pl.items = F * H * pl.nrb, pl.own_items = B * H * pl.own_nrb;
    // units as the kernels count them
    const int64_t tile = pl.items * (kTileStart + (prefix_cap + kTile - 1) / kTile);
    const int64_t own = pl.own_items * (by_rows ? kStart + (own_cap + kUnit - 1) / kUnit : kTileStart + (own_cap + kTile - 1) / kTile);
    const int64_t together = pl.items * (kStart + (prefix_cap + kUnit - 1) / kUnit) + own;
    if (tile > 0x7fffffff || own > 0x7fffffff || together > 0x7fffffff || (!by_rows && tile + own > 0x7fffffff))
        return fail(KITTY_E_UNSUPPORTED, "too many rows and pages for one launch");
    // workgroups: what the device holds at once, a multiple of eight; no more than there are units
    const int64_t fit = (pl.together ? two_per_cu(pl.DP, pl.RT) : pl.DP <= 128) ? 2 * cus : cus;
    pl.W = (int)std::min<int64_t>(fit, pl.together ? std::max<int64_t>(together, 1) : tile + own + 16);
    if (!pl.together)
        pl.W = std::max(pl.W / 8 * 8, 16);
    size_t at = 0;
    auto area = [&](int64_t slots, int rm, int64_t items, size_t &o, size_t &ml, size_t &tab) {
        o = at;
        ml = o + up16((size_t)slots * rm * pl.DP * 4);
        tab = ml + up16((size_t)slots * rm * 8);
        at = tab + up16((size_t)items * 8);
    };
    if (pl.together || pl.RT == 0) {
        const int64_t all = pl.items + pl.own_items;
        area(2 * pl.W + all, pl.together ? RM : kTileRows, all, pl.o_at, pl.ml_at, pl.tab_at);
        pl.own_o_at = pl.o_at, pl.own_ml_at = pl.ml_at, pl.own_tab_at = pl.tab_at;
    } else {
        area(2 * pl.W + pl.items, kTileRows, pl.items, pl.o_at, pl.ml_at, pl.tab_at);
        area(2 * pl.W + pl.own_items, RM, pl.own_items, pl.own_o_at, pl.own_ml_at, pl.own_tab_at);
    }
    pl.map_at = at;
    pl.bytes = at + (pl.together ? 0 : up16((size_t)(B * a.tokens + B + F) * 4));   // (the size does not go by q_lens)
    return KITTY_OK;
}

// Every row has a part in the workspace for its prefix and one for its own tokens, in fp32: a
// call for which they are more than kMostParts runs in pieces that use one workspace after
// each other, of whole prefixes, then of one prefix's sequences, then of one sequence's KV
// heads.  64 x 2,048 queries behind four prefixes of 2,000 tokens, 32 / 8 heads of 128:
// 4.1 GiB and 18.2 ms in one, 0.57 GiB and 16.3 ms in eight pieces.
constexpr size_t kMostParts = 1ull << 30;

struct Pieces8 {
    int prefixes, seqs, heads;   // of each: prefixes, sequences of a prefix, KV heads
    bool one;
    SharedPlan8 plan;            // of the one
    size_t bytes;
};

// A piece's sizes.
static void piece_sizes(int prefixes, int seqs, int heads, Cache8 &c, kitty_cache8_shared_args &a)
{
    a.num_q_heads = a.num_q_heads / c.H * heads, c.H = heads;
    a.prefixes = prefixes, a.batch = prefixes * seqs;
}

static int plan_pieces(const Cache8 &c, const kitty_cache8_shared_args &a, Pieces8 &pc)
{
    if (const int rc = plan_shared(c, a, pc.plan))
        return rc;
    const int F = a.prefixes, per = a.batch / a.prefixes;
    pc.prefixes = F, pc.seqs = per, pc.heads = c.H, pc.bytes = pc.plan.bytes;
    pc.one = pc.bytes <= kMostParts;
    if (pc.one)
        return KITTY_OK;
    auto bytes = [&](int prefixes, int seqs, int heads) {
        Cache8 d = c;
        kitty_cache8_shared_args b = a;
        SharedPlan8 pl{};
        piece_sizes(prefixes, seqs, heads, d, b);
        return plan_shared(d, b, pl) ? 0 : pl.bytes;   // what fits one launch whole does in pieces
    };
    for (int *n : {&pc.prefixes, &pc.seqs, &pc.heads})
        while (*n > 1 && bytes(pc.prefixes, pc.seqs, pc.heads) > kMostParts)
            *n = (*n + 1) / 2;
    // the last pieces are smaller and may go another way
    pc.bytes = 0;
    for (int f : {pc.prefixes, F % pc.prefixes})
        for (int s : {pc.seqs, per % pc.seqs})
            for (int h : {pc.heads, c.H % pc.heads})
                if (f && s && h)
                    pc.bytes = std::max(pc.bytes, bytes(f, s, h));
    return KITTY_OK;
}

// Sizes of launch_tile_runs: slots of 128 rows for two parts a workgroup and one an item.
struct TileRuns8 {
    int DP, W, nrb;
    int64_t items;
    size_t ml_at, tab_at, bytes;
};

static TileRuns8 plan_tile_runs(int D, int H, int64_t batch, int64_t rows)
{
    TileRuns8 r;
    r.DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    r.W = std::max((r.DP <= 128 ? 2 : 1) * device_cus() / 8 * 8, 16);
    r.nrb = (int)((rows + kTileRows - 1) / kTileRows);
    r.items = batch * H * r.nrb;
    const size_t slots = 2 * r.W + (size_t)r.items;
    r.ml_at = up16(slots * kTileRows * r.DP * 4);
    r.tab_at = r.ml_at + up16(slots * kTileRows * 8);
    r.bytes = r.tab_at + up16((size_t)r.items * 8);
    return r;
}

size_t tile_runs_bytes(const Cache8 &c, const kitty_cache8_attention_args &a)
{
    return plan_tile_runs(c.D, c.H, a.batch, (int64_t)a.num_q_heads / c.H * a.tokens).bytes;
}

template <int DP, bool BF16>
static void join(const Attend8 &p, const Part8 &of_prefix, const Part8 &of_own, hipStream_t st)
{
    const int64_t rows = (int64_t)p.B * p.c.H * p.gq * p.T, groups = 256 * kWaves / DP;
    if (rows < kMergeRows)
        hipLaunchKernelGGL((cache8_join_kernel<DP, BF16, true>), dim3((unsigned)rows), dim3(64 * kWaves), 0, st, p, of_prefix, of_own);
    else
        hipLaunchKernelGGL((cache8_join_kernel<DP, BF16, false>), dim3((unsigned)((rows + groups - 1) / groups)), dim3(64 * kWaves), 0,
                           st, p, of_prefix, of_own);
}

void launch_tile_runs(const Attend8 &args, bool bf16, void *workspace, hipStream_t st)
{
    Attend8 p = args;
    const TileRuns8 r = plan_tile_runs(p.c.D, p.c.H, p.B, (int64_t)p.gq * p.T);
    p.F = 0, p.per = 1, p.e0 = 0, p.entries = p.B, p.item0 = 0, p.nrb = p.own_nrb = r.nrb, p.n_wg = r.W;
    p.ws_o = (float *)workspace, p.ws_ml = (float2 *)((char *)workspace + r.ml_at), p.ws_tab = (int2 *)((char *)workspace + r.tab_at);
    const Part8 part = {p.ws_o, p.ws_ml, p.ws_tab, 0, r.nrb, kTileRows, r.W, 0};
    auto go = [&](auto dp, auto bf) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value;
        if (p.c.D == DP)
            hipLaunchKernelGGL((cache8_shared_kernel<DP, BF, false, 0>), dim3(r.W), dim3(64 * kWaves), 0, st, p, p);
        else
            hipLaunchKernelGGL((cache8_shared_kernel<DP, BF, true, 0>), dim3(r.W), dim3(64 * kWaves), 0, st, p, p);
        join<DP, BF>(p, part, part, st);
    };
    auto by_size = [&](auto bf) {
        if (r.DP == 64)
            go(std::integral_constant<int, 64>{}, bf);
        else if (r.DP == 128)
            go(std::integral_constant<int, 128>{}, bf);
        else
            go(std::integral_constant<int, 256>{}, bf);
    };
    if (bf16)
        by_size(std::true_type{});
    else
        by_size(std::false_type{});
}

static int check_shared(const kitty_cache8 *cache, const kitty_cache8_shared_args *args, Cache8 &c)
{
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, c))
        return rc;
    const kitty_cache8_shared_args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.table_pages < 0 || a.prefix_pages < 0)
        return fail(KITTY_E_INVALID, "batch, tokens, table_pages and prefix_pages must not be negative");
    if (a.prefixes <= 0 || a.batch % a.prefixes)
        return fail(KITTY_E_INVALID, "batch must be a multiple of a positive number of prefixes");
    if (a.num_q_heads <= 0 || a.num_q_heads % c.H)
        return fail(KITTY_E_INVALID, "num_q_heads must be a positive multiple of num_kv_heads");
    if (a.dtype != KITTY_DTYPE_F16 && a.dtype != KITTY_DTYPE_BF16)
        return fail(KITTY_E_INVALID, "dtype must be KITTY_DTYPE_F16 or KITTY_DTYPE_BF16");
    if (!(a.sm_scale > 0.0f) || a.sm_scale > 1e30f)
        return fail(KITTY_E_INVALID, "sm_scale must be positive and finite");
    if (((int64_t)a.table_pages + a.prefix_pages) << c.lg > 1 << 30)   // a row's place is an int
        return fail(KITTY_E_UNSUPPORTED, "a sequence and its prefix are limited to 2^30 tokens together");
    return KITTY_OK;
}

// One call, or a piece of one whose rows' log-sum-exps are lse_heads heads apart.
static void launch_shared(const Cache8 &c, const kitty_cache8_shared_args &a, const SharedPlan8 &pl, int lse_heads, hipStream_t st)
{
    Attend8 p{};
    p.c = c;
    p.q = a.q, p.out = a.out, p.lse = a.lse;
    p.q_s_seq = a.q_s_seq, p.q_s_head = a.q_s_head, p.q_s_tok = a.q_s_tok;
    p.o_s_seq = a.o_s_seq, p.o_s_head = a.o_s_head, p.o_s_tok = a.o_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.lens = a.lens, p.q_lens = a.q_lens;
    p.prefix_table = a.prefix_table, p.pt_stride = a.pt_stride, p.prefix_lens = a.prefix_lens;
    p.B = a.batch, p.Hq = lse_heads, p.T = a.tokens, p.gq = a.num_q_heads / p.c.H;
    p.F = a.prefixes, p.per = a.batch / a.prefixes, p.prefix_pages = a.prefix_pages;
    p.table_pages = a.table_pages, p.causal = a.causal ? 1 : 0;
    p.cs = a.sm_scale * kLog2e;

    const dim3 block(64 * kWaves);
    char *ws = (char *)a.workspace;
    if (a.q_lens && !pl.together && !pl.direct) {
        p.row_map = (int32_t *)(ws + pl.map_at), p.row_first = p.row_map + (int64_t)p.B * p.T, p.row_count = p.row_first + p.B;
        hipLaunchKernelGGL(cache8_shared_queries_kernel, dim3((unsigned)((p.F + kWaves - 1) / kWaves)), block, 0, st, p);
    }
    p.nrb = pl.nrb, p.own_nrb = pl.own_nrb, p.n_wg = pl.W, p.item0 = (int)pl.items;
    Attend8 x = p, y = p;     // the launch's tile entries, or all of them; its row entries
    x.e0 = 0, x.entries = pl.together || pl.RT == 0 ? p.F + p.B : p.F;
    x.ws_o = (float *)(ws + pl.o_at), x.ws_ml = (float2 *)(ws + pl.ml_at), x.ws_tab = (int2 *)(ws + pl.tab_at);
    y.e0 = p.F, y.entries = p.B, y.item0 = 0, y.nrb = pl.direct ? 1 : y.nrb;
    y.ws_o = (float *)(ws + pl.own_o_at), y.ws_ml = (float2 *)(ws + pl.own_ml_at), y.ws_tab = (int2 *)(ws + pl.own_tab_at);
    const bool apart = !pl.together && pl.RT != 0;
    const int tile_rows = pl.together ? 16 * pl.RT : kTileRows, own_rows = pl.RT ? 16 * pl.RT : kTileRows;
    const Part8 of_prefix = {x.ws_o, x.ws_ml, x.ws_tab, 0, pl.nrb, tile_rows, pl.W, 0};
    const Part8 of_own = {y.ws_o, y.ws_ml, y.ws_tab, p.F, pl.own_nrb, own_rows, pl.W, apart ? 0 : (int)pl.items};
    const dim3 grid((unsigned)pl.W);
    auto go = [&](auto dp, auto bf, auto cut) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value, CUT = decltype(cut)::value;
        if constexpr (DP <= 128) {
            if (pl.direct) {
                const dim3 pairs((unsigned)(p.B * p.c.H));
                if (pl.RT == 1)
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, 1, BF, CUT, true, kShared>), pairs, dim3(64 * row_waves(1, true)), 0, st, y);
                else
                    hipLaunchKernelGGL((cache8_rows_kernel<DP, 2, BF, CUT, true, kShared>), pairs, dim3(64 * row_waves(2, true)), 0, st, y);
                return;
            }
        }
        if (pl.together) {
            if (pl.RT == 1)
                hipLaunchKernelGGL((cache8_rows_kernel<DP, 1, BF, CUT, false, kShared>), grid, block, 0, st, x);
            else
                hipLaunchKernelGGL((cache8_rows_kernel<DP, 2, BF, CUT, false, kShared>), grid, block, 0, st, x);
        } else if (pl.RT == 0) {
            hipLaunchKernelGGL((cache8_shared_kernel<DP, BF, CUT, 0>), grid, block, 0, st, x, y);
        } else if (pl.RT == 1) {
            hipLaunchKernelGGL((cache8_shared_kernel<DP, BF, CUT, 1>), grid, block, 0, st, x, y);
        } else {
            hipLaunchKernelGGL((cache8_shared_kernel<DP, BF, CUT, 2>), grid, block, 0, st, x, y);
        }
        join<DP, BF>(p, of_prefix, of_own, st);
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
}

} // namespace kitty

using namespace kitty;

extern "C" int kitty_cache8_shared_attention_workspace_size(const kitty_cache8 *cache, const kitty_cache8_shared_args *args,
                                                            size_t *bytes)
{
    Cache8 c;
    Pieces8 pc{};
    if (!bytes)
        return fail(KITTY_E_INVALID, "bytes is NULL");
    if (const int rc = check_shared(cache, args, c))
        return rc;
    *bytes = 0;
    if (args->batch == 0 || args->tokens == 0)
        return KITTY_OK;
    if (const int rc = plan_pieces(c, *args, pc))
        return rc;
    *bytes = pc.bytes;
    return KITTY_OK;
}

extern "C" int kitty_cache8_shared_attention(const kitty_cache8 *cache, const kitty_cache8_shared_args *args,
                                             kitty_stream_t stream)
{
    Cache8 c;
    Pieces8 pc{};
    if (const int rc = check_shared(cache, args, c))
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
    if (const int rc = plan_pieces(c, a, pc))
        return rc;
    if ((!a.workspace && pc.bytes) || !aligned(a.workspace, 16) || a.workspace_bytes < pc.bytes)
        return fail(KITTY_E_INVALID,
                    "workspace is NULL, misaligned or smaller than kitty_cache8_shared_attention_workspace_size");
    if (pc.one) {
        launch_shared(c, a, pc.plan, a.num_q_heads, (hipStream_t)stream);
        return check_launch("8-bit cache attention over shared prefixes");
    }
    const int per = a.batch / a.prefixes, gq = a.num_q_heads / c.H;
    for (int f = 0; f < a.prefixes; f += pc.prefixes)
        for (int s = 0; s < per; s += pc.seqs)
            for (int h = 0; h < c.H; h += pc.heads) {
                Cache8 d = c;
                kitty_cache8_shared_args b = a;
                piece_sizes(std::min(pc.prefixes, a.prefixes - f), std::min(pc.seqs, per - s), std::min(pc.heads, c.H - h), d, b);
                const int64_t first = (int64_t)f * per + s;   // sequence
                b.q += first * a.q_s_seq + h * gq * a.q_s_head, b.out += first * a.o_s_seq + h * gq * a.o_s_head;
                if (b.lse)
                    b.lse += (first * a.num_q_heads + h * gq) * a.tokens;
                if (b.prefix_table)
                    b.prefix_table += f * a.pt_stride;
                if (b.block_table)
                    b.block_table += first * a.bt_stride;
                b.prefix_lens += f, b.lens += first;
                if (b.q_lens)
                    b.q_lens += first;
                if (c.num_pages) {
                    d.key += h * c.key_s_head, d.value += h * c.value_s_head;
                    d.scale += h * c.scale_s_head;
                }
                SharedPlan8 pl{};
                if (const int rc = plan_shared(d, b, pl))
                    return rc;
                launch_shared(d, b, pl, a.num_q_heads, (hipStream_t)stream);
            }
    return check_launch("8-bit cache attention over shared prefixes");
}
