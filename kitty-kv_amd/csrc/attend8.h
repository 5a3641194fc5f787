// Attention over the 8-bit paged cache: what its two kernels share.
#pragma once
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
};

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
};

__device__ __forceinline__ Seq8 seq8(const Attend8 &p, int b)
{
    Seq8 s;
    s.n = p.lens[b];
    s.tq = p.q_lens ? p.q_lens[b] : p.T;
    s.bad = s.n < 0 || s.n > (int64_t)p.table_pages << p.c.lg || s.tq < 0 || s.tq > p.T || (s.n > 0 && p.c.num_pages == 0);
    return s;
}

// Tokens that query row t of a sequence sees: those below the result.
__device__ __forceinline__ int visible8(const Attend8 &p, const Seq8 &s, int t)
{
    if (t >= s.tq)
        return 0;
    return p.causal ? max(s.n - s.tq + t + 1, 0) : s.n;
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

} // namespace kitty
