// Attention over the 8-bit paged cache: what its two kernels share.
#pragma once
#include <algorithm>

#include "cache8.h"

namespace kitty {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -3.402823466e38f;   // running maximum of rows that have seen no score above -inf
constexpr int kUnit = 128;                    // tokens of a work unit of the row kernel

struct Attend8 {
    Cache8 c;
    const uint16_t *q;
    uint16_t *out;
    float *lse;
    int64_t q_s_seq, q_s_head, q_s_tok, o_s_seq, o_s_head, o_s_tok;
    const int32_t *table, *lens, *q_lens;
    int64_t bt_stride;
    int B, Hq, T, gq, table_pages, causal;
    int nrb;            // row blocks per (sequence, KV head)
    int n_wg;           // row kernel: workgroups that share the work
    int splits;         // tile kernel: parts of a row block's tokens
    float cs;           // sm_scale * log2(e)
    float *ws_o;        // partials: (slots, rows of a block, D padded)
    float2 *ws_ml;      // (slots, rows of a block): maximum (log2 units) and sum
    int2 *ws_tab;       // row kernel, (items): first slot (-1: written whole), last workgroup
    // Sequences that share prefixes: a launch works on `entries` entries from entry e0 on.
    // Entry f < F is prefix f with the query rows of its `per` sequences, F + b what is
    // sequence b's own.
    const int32_t *prefix_table, *prefix_lens;
    int64_t pt_stride;
    int F, per, prefix_pages, e0, entries;
    int own_nrb, item0;   // row blocks of a sequence's own rows in tiles, the number of their first item
    // Padded queries of SHARED launches, or NULL: a prefix's real queries by their number
    // (sequence of the prefix times T plus query), how many each prefix has, and the
    // number of each sequence's first.
    int32_t *row_map, *row_count, *row_first;
    // For a second pass over the tokens: each row's maximum (log2 units) and 1 / sum, like
    // lse; of kScores launches also the scores (log2 units, -inf where masked) of a KV
    // head's up to 16 rows and sc_cap (a multiple of 16) tokens, (16 tokens, row, token).
    float2 *stat;
    float *scores;
    int64_t sc_cap;
    // Weights (of the first w_tokens tokens), added to by the launch that leaves the scores
    // where it has the whole of a KV head's rows and tokens, else by the merge's.
    float *weights;
    int64_t w_s_seq, w_s_head;
    int w_tokens;
};

// What a row kernel does beside plain attention: nothing, leave all parts of prefixes and
// sequences, leave the rows' maxima and sums and the scores, or those without the scores.
constexpr int kPlain = 0, kShared = 1, kScores = 2, kStat = 3;

// kitty_cache8_attention that also leaves stat and, where given, the scores; weighed: the
// weights are done as well.
struct Leave8 {
    float2 *stat;
    float *scores;
    int64_t sc_cap;
    float *weights;
    int64_t w_s_seq, w_s_head;
    int w_tokens;
    bool weighed;
};
int attend8(const kitty_cache8 *cache, const kitty_cache8_attention_args *args, hipStream_t stream, Leave8 &leave);
// Its workspace, with scores or without.
int attend8_bytes(const kitty_cache8 *cache, const kitty_cache8_attention_args *args, bool scores, size_t &bytes);

// The tile kernel's work on sequences of unequal lengths, cut evenly by what they hold
// (attend8_shared.hip): p with its queries, tables and outputs, in `bytes` of workspace.
size_t tile_runs_bytes(const Cache8 &c, const kitty_cache8_attention_args &args);
void launch_tile_runs(const Attend8 &p, bool bf16, void *workspace, hipStream_t stream);

constexpr int kTileRows = 128;   // query rows of the tile kernel's workgroup

// The tile kernel (attend8_tile.hip) on row blocks of kTileRows, p.splits parts each.
void launch_tiles(const Attend8 &p, int DP, bool bf16, hipStream_t stream);

// Reads that are the same for a wave and that no kernel of the call writes:
// through the scalar unit, so that waits for them do not wait for the vector
// loads in flight.
template <typename T>
__device__ __forceinline__ T uniform_load(const T *p)
{
    return *(const __attribute__((address_space(4))) T *)p;
}

// A sequence of the batch as the kernels read it.
struct Seq8 {
    int n, tq;      // tokens in the cache, query rows
    bool bad;       // lengths that break the rules: NaN rows, no pages read
    bool prefix;    // SHARED: a prefix; tq then is what its sequences have together, padding included
};

__device__ __forceinline__ Seq8 seq8(const Attend8 &p, int b)
{
    Seq8 s;
    s.n = p.lens[b];
    s.tq = p.q_lens ? p.q_lens[b] : p.T;
    s.bad = s.n < 0 || s.n > (int64_t)p.table_pages << p.c.lg || s.tq < 0 || s.tq > p.T || (s.n > 0 && p.c.num_pages == 0);
    s.prefix = false;
    return s;
}

// Entry i of a launch: sequence i, or of SHARED launches a prefix or a sequence.
template <bool SHARED>
__device__ __forceinline__ Seq8 entry8(const Attend8 &p, int i)
{
    if constexpr (SHARED) {
        const int e = p.e0 + i;
        if (e < p.F) {
            Seq8 s;
            s.n = p.prefix_lens[e];
            s.tq = p.per * p.T;
            s.bad = s.n < 0 || s.n > (int64_t)p.prefix_pages << p.c.lg || (s.n > 0 && p.c.num_pages == 0);
            s.prefix = true;
            return s;
        }
        return seq8(p, e - p.F);
    }
    return seq8(p, i);
}

template <bool SHARED>
__device__ __forceinline__ const int32_t *table8(const Attend8 &p, const Seq8 &s, int i)
{
    if constexpr (SHARED)
        return s.prefix ? p.prefix_table + (p.e0 + i) * p.pt_stride : p.table + (p.e0 + i - p.F) * p.bt_stride;
    return p.table + i * p.bt_stride;
}

// Tokens that query row t of a sequence sees: those below the result.
__device__ __forceinline__ int visible8(const Attend8 &p, const Seq8 &s, int t)
{
    if (t >= s.tq)
        return 0;
    return p.causal ? max(s.n - s.tq + t + 1, 0) : s.n;
}

// Query rows of an entry and KV head.
template <bool SHARED>
__device__ __forceinline__ int rows8(const Attend8 &p, const Seq8 &s, int i)
{
    if (SHARED && s.prefix)
        return p.gq * (p.row_map ? p.row_count[p.e0 + i] : p.per * p.T);
    return p.gq * p.T;
}

// Query row r of an entry and KV head: sequence, head and token, the entry's tokens that
// it sees, whether it is a row of the call (no padding) and whether it may be loaded (of
// SHARED prefixes padding too, whose sums no one reads: the loads wait for no length).
struct Row8 {
    int b, h, t, vis;
    bool real, there;
};

template <bool SHARED>
__device__ __forceinline__ Row8 row8(const Attend8 &p, const Seq8 &s, int i, int kh, int r)
{
    Row8 w;
    w.t = r / p.gq;
    w.h = kh * p.gq + r - w.t * p.gq;
    w.b = i;
    if constexpr (SHARED) {
        w.b = p.e0 + i - p.F;
        if (s.prefix) {
            const int f = p.e0 + i;
            if (p.row_map)
                w.t = w.t < p.row_count[f] ? p.row_map[(int64_t)f * p.per * p.T + w.t] : p.per * p.T;
            const int q = w.t / p.T;
            w.t -= q * p.T;
            w.b = f * p.per + q;
            w.real = false, w.vis = 0;
            w.there = !s.bad && q < p.per;
            if (w.there) {
                // rows that are tokens of the prefix itself see it up to themselves
                const Seq8 own = seq8(p, w.b);
                w.real = !own.bad && w.t < own.tq;
                if (w.real)
                    w.vis = p.causal ? max(s.n + min(own.n - own.tq + w.t + 1, 0), 0) : s.n;
            }
            return w;
        }
    }
    w.real = w.there = !s.bad && w.t < s.tq;
    w.vis = visible8(p, s, w.t);
    return w;
}

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Codes 2 HI and 2 HI + 1 of four as a pair of 16-bit floats (exact).
template <bool BF16, bool HI>
__device__ __forceinline__ unsigned widen(unsigned codes)
{
    if constexpr (BF16)
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HI));
    else
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HI));
}

// (a, b) as packed bf16 terms hi + lo: 16 bits of each (a rounding to bf16 is off by
// 2^-8 at most, that of the rest by as much of it), fp32's range.
__device__ __forceinline__ void split_bf16(float a, float b, unsigned &hi, unsigned &lo)
{
    bf16x2 h, r;
    h[0] = (__bf16)a, h[1] = (__bf16)b;
    hi = __builtin_bit_cast(unsigned, h);
    r[0] = (__bf16)(a - __builtin_bit_cast(float, hi << 16));
    r[1] = (__bf16)(b - __builtin_bit_cast(float, hi & 0xffff0000u));
    lo = __builtin_bit_cast(unsigned, r);
}

// The four bytes of w that hold a NaN code, as 0x80 each.
__device__ __forceinline__ unsigned nan_codes(unsigned w)
{
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// Rows from which the merge gives each a lane group instead of a workgroup (12,800
// rows of four parts 5.6 us / 9.0 with a wave a row; 1,280 rows of nine 6.5 / 4.6).
constexpr int64_t kMergeRows = 2048;

inline int device_cus()
{
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
        cus = 256;
    return cus;
}

} // namespace kitty
