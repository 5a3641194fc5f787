// Writing the 8-bit paged cache and reading it back, on gfx950.
//
// write: a workgroup takes the new rows of one (page, head, stream), so that a
// page's scale has one owner.  It loads its rows once (up to 8 pieces of 8
// channels a thread stay in registers), takes the largest finite magnitude,
// and stores codes x * 2^-e: with powers of two the quotient is exact, and so
// is the rescale of codes that were there, which would otherwise round twice.
// Power-of-two scales cost e4m3 no relative precision (its steps are relative);
// the largest code lies in (224, 448].
// read: a thread takes 16 bytes of output in each of four rows; the codes' fp32
// products with the scale round once.
// Both are bound by memory, and by launch latency where few tokens are written.
// Measured: 4 x 8,192 tokens of 8 x 128 fp16 written in 39.8 us (5.05 TB/s; a copy
// reaches 4.9; 46 without streaming loads), one token of one sequence or of 64 in
// 4.2; pages of more than 128 x 128 elements, whose later rows are read twice (the
// second time mostly from the L2): 128 channels and 256 tokens 46.5 us (4.3 TB/s, 41.4 at
// 128 tokens on the same card), 256 and 128 44 us, 256 and 256 55 us; 8 x 8,192 read back in 82 us (4.3 TB/s, three quarters of it stores; 93 with
// 32 bytes of output a thread and row).
#include "cache8.h"

namespace kitty {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kKeep = 8;       // pieces of a thread that stay in registers between the two passes
constexpr int kReadRows = 4;   // rows per thread of the read kernel
// Codes of a thread and row: 16 bytes of output, so that a wave stores 1 KB in a run.
constexpr int read_codes(int out) { return out == KITTY_SRC_F32 ? 4 : 8; }

int check_cache8(const kitty_cache8 *cache, Cache8 &c)
{
    if (!cache)
        return fail(KITTY_E_INVALID, "cache is NULL");
    const kitty_cache8 &a = *cache;
    if (a.num_kv_heads <= 0 || a.num_pages < 0)
        return fail(KITTY_E_INVALID, "num_kv_heads must be positive and num_pages not negative");
    if (a.head_dim <= 0 || a.head_dim % 16)
        return fail(KITTY_E_INVALID, "head_dim must be a multiple of 16");
    if (a.head_dim > 256)
        return fail(KITTY_E_UNSUPPORTED, "the 8-bit cache is built for head_dim up to 256");
    int lg = 4;
    while (lg < 8 && 1 << lg != a.page_tokens)
        ++lg;
    if (1 << lg != a.page_tokens)
        return fail(KITTY_E_INVALID, "page_tokens must be 16, 32, 64, 128 or 256");
    if (a.num_pages && (!a.key || !a.value || !a.scale))
        return fail(KITTY_E_INVALID, "NULL key, value or scale pool");
    if (!aligned(a.key, 16) || !aligned(a.value, 16) || !aligned(a.scale, 8))
        return fail(KITTY_E_INVALID, "code pools must be 16-byte and scales 8-byte aligned");
    for (int64_t s : {a.key_s_page, a.key_s_head, a.key_s_tok, a.value_s_page, a.value_s_head, a.value_s_tok})
        if (s < 0 || s % 16)
            return fail(KITTY_E_INVALID, "code strides must be non-negative multiples of 16");
    for (int64_t s : {a.key_s_tok, a.value_s_tok})
        if (s < a.head_dim || s * a.page_tokens >= (int64_t)1 << 31)
            return fail(KITTY_E_INVALID, "token strides must be at least head_dim and a page's rows span less than 2 GiB");
    if (a.scale_s_page < 0 || a.scale_s_head < 0 || a.scale_s_page % 2 || a.scale_s_head % 2)
        return fail(KITTY_E_INVALID, "scale strides must be non-negative and even");
    c.key = a.key, c.value = a.value, c.scale = a.scale;
    c.key_s_page = a.key_s_page, c.key_s_head = a.key_s_head, c.key_s_tok = (uint32_t)a.key_s_tok;
    c.value_s_page = a.value_s_page, c.value_s_head = a.value_s_head, c.value_s_tok = (uint32_t)a.value_s_tok;
    c.scale_s_page = a.scale_s_page, c.scale_s_head = a.scale_s_head;
    c.num_pages = a.num_pages, c.H = a.num_kv_heads, c.D = a.head_dim, c.lg = lg;
    return KITTY_OK;
}

struct WriteParams {
    Cache8 c;
    const void *src[2];
    int64_t s_seq[2], s_head[2], s_tok[2];
    const int32_t *table, *start, *lens;
    int64_t bt_stride;
    int tokens, table_pages, slots;   // slots: pages that `tokens` tokens can touch
};

// 8 consecutive channels as they come from memory.
template <int SRC>
struct Piece {
    u32x4 w[SRC == KITTY_SRC_F32 ? 2 : 1];

    // ONCE: not read again, and kept from displacing what is
    template <bool VEC, bool ONCE>
    __device__ __forceinline__ void load(const void *base, int64_t off)
    {
        if constexpr (VEC) {
            const u32x4 *s = (const u32x4 *)((const char *)base + off * (SRC == KITTY_SRC_F32 ? 4 : 2));
            w[0] = ONCE ? __builtin_nontemporal_load(s) : s[0];
            if constexpr (SRC == KITTY_SRC_F32)
                w[1] = ONCE ? __builtin_nontemporal_load(s + 1) : s[1];
        } else if constexpr (SRC == KITTY_SRC_F32) {
            const uint32_t *s = (const uint32_t *)base + off;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                w[e >> 2][e & 3] = s[e];
        } else {
            const uint16_t *s = (const uint16_t *)base + off;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[0][e] = (uint32_t)s[2 * e] | (uint32_t)s[2 * e + 1] << 16;
        }
    }
    __device__ __forceinline__ float at(int e) const
    {
        if constexpr (SRC == KITTY_SRC_F32)
            return __builtin_bit_cast(float, (uint32_t)w[e >> 2][e & 3]);   // of an element itself, it takes the first
        else
            return x2f((uint16_t)(w[0][e >> 1] >> (16 * (e & 1))), SRC == KITTY_SRC_BF16);
    }
    // the largest finite |x|, not below m
    __device__ __forceinline__ float top(float m) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = __builtin_fabsf(at(e));
            m = a < __builtin_inff() ? fmaxf(m, a) : m;
        }
        return m;
    }
};

__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d)
{
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// The smallest power of two s >= 2^-64 with m <= 448 s.  m = f 2^k with f in
// [1/2, 1): 448 = 0.875 * 2^9, so s = 2^(k - 9), or 2^(k - 8) where f > 0.875.
__device__ __forceinline__ float scale_for(float m)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, m);
    const int e = max((int)(u >> 23) - 126 - 9 + ((u & 0x7fffff) > 0x600000 ? 1 : 0), -64);
    return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// Codes of a piece: x * inv where the scale is a power of two (exact), else the
// correctly rounded quotient.  The quotients lie within 448.
template <int SRC>
__device__ __forceinline__ uint2 encode(const Piece<SRC> &x, float s, float inv, bool pow2)
{
    float y[8];
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = x.at(e);
        odd |= !(__builtin_fabsf(v) < __builtin_inff());
        y[e] = v * inv;
    }
    if (!pow2) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[e] = x.at(e) / s;
    }
    uint2 r = make_uint2(pack4(y[0], y[1], y[2], y[3]), pack4(y[4], y[5], y[6], y[7]));
    if (odd) {   // NaN and infinities: the NaN code
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!(__builtin_fabsf(x.at(e)) < __builtin_inff())) {
                uint32_t &w = e < 4 ? r.x : r.y;
                w = (w & ~(0xffu << (8 * (e & 3)))) | 0x7fu << (8 * (e & 3));
            }
    }
    return r;
}

template <int SRC, bool VEC, int NT>
__global__ __launch_bounds__(NT) void cache8_write_kernel(WriteParams p)
{
    uint32_t i = blockIdx.x;
    const int slot = (int)(i % (uint32_t)p.slots);
    i /= (uint32_t)p.slots;
    const int st = (int)(i & 1);
    i >>= 1;
    const int h = (int)(i % (uint32_t)p.c.H), b = (int)(i / (uint32_t)p.c.H);
    const int lg = p.c.lg, start = p.start[b];
    const int n = p.lens ? min(max(p.lens[b], 0), p.tokens) : p.tokens;
    if (start < 0)
        return;
    const int64_t page = (int64_t)(start >> lg) + slot, end = (int64_t)start + n;
    if (page << lg >= end || page >= p.table_pages || n == 0)
        return;
    const int id = p.table[b * p.bt_stride + page];
    if (bad_page(p.c, id))
        return;
    // new rows row0 .. row1 - 1 of the page, the first of them row t0 of the source
    const int row0 = slot == 0 ? start & ((1 << lg) - 1) : 0;
    const int row1 = (int)min((int64_t)1 << lg, end - (page << lg));
    const int64_t t0 = slot == 0 ? 0 : (page << lg) - start;
    const int rows = row1 - row0;
    float *scale = p.c.scale + id * p.c.scale_s_page + h * p.c.scale_s_head + st;
    const float old = row0 > 0 ? *scale : 0.0f;

    const int cpr = p.c.D >> 3, rpp = NT / cpr;      // pieces per row, rows per pass
    const int r0 = (int)threadIdx.x / cpr, ch = 8 * ((int)threadIdx.x - r0 * cpr);
    const bool in = r0 < rpp;
    const int64_t s_tok = st ? p.s_tok[1] : p.s_tok[0];
    const void *src = st ? p.src[1] : p.src[0];
    const int64_t src0 = b * (st ? p.s_seq[1] : p.s_seq[0]) + h * (st ? p.s_head[1] : p.s_head[0]) + t0 * s_tok + ch;
    const uint32_t d_tok = st ? p.c.value_s_tok : p.c.key_s_tok;
    uint8_t *dst = st ? p.c.value + id * p.c.value_s_page + h * p.c.value_s_head
                      : p.c.key + id * p.c.key_s_page + h * p.c.key_s_head;

    Piece<SRC> keep[kKeep];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
        if (in && r0 + j * rpp < rows)
            keep[j].template load<VEC, true>(src, src0 + (r0 + j * rpp) * s_tok);
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
        if (in && r0 + j * rpp < rows)
            m = keep[j].top(m);
    if (in)
        for (int r = r0 + kKeep * rpp; r < rows; r += rpp) {
            Piece<SRC> x;
            x.template load<VEC, false>(src, src0 + r * s_tok);
            m = x.top(m);
        }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        m = fmaxf(m, __shfl_xor(m, off));
    if constexpr (NT > 64) {
        __shared__ float part[NT / 64];
        if ((threadIdx.x & 63) == 0)
            part[threadIdx.x >> 6] = m;
        __syncthreads();   // also: every thread has read the old scale before it is replaced
#pragma unroll
        for (int w = 0; w < NT / 64; ++w)
            m = fmaxf(m, part[w]);
    }
    const float s = fmaxf(scale_for(m), old), inv = 1.0f / s;   // old NaN: the new rows' scale
    const bool pow2 = (__builtin_bit_cast(uint32_t, s) & 0x7fffff) == 0;
    uint8_t *out = dst + (uint32_t)row0 * d_tok + ch;
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
        if (in && r0 + j * rpp < rows)
            *(uint2 *)(out + (uint32_t)(r0 + j * rpp) * d_tok) = encode(keep[j], s, inv, pow2);
    if (in)
        for (int r = r0 + kKeep * rpp; r < rows; r += rpp) {
            Piece<SRC> x;
            x.template load<VEC, false>(src, src0 + r * s_tok);
            *(uint2 *)(out + (uint32_t)r * d_tok) = encode(x, s, inv, pow2);
        }
    if (row0 > 0 && s != old && in) {   // the codes of earlier tokens, at the raised scale
        const float f = old / s;
        for (int r = r0; r < row0; r += rpp) {
            uint2 *at = (uint2 *)(dst + (uint32_t)r * d_tok + ch);
            const uint2 v = *at;
            uint2 o;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int w = (int)(e ? v.y : v.x);
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
                (e ? o.y : o.x) = pack4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
            }
            *at = o;
        }
    }
    if (threadIdx.x == 0)
        *scale = s;
}

struct ReadParams {
    Cache8 c;
    void *out[2];
    int64_t s_seq[2], s_head[2], s_tok[2];
    const int32_t *table, *start, *lens;
    int64_t bt_stride;
    int tokens, table_pages, tiles;   // tiles: workgroups per (sequence, head, stream)
};

template <int OUT>
__global__ __launch_bounds__(256) void cache8_read_kernel(ReadParams p)
{
    constexpr int CPT = read_codes(OUT), NW = CPT / 4;
    uint32_t i = blockIdx.x;
    const int tile = (int)(i % (uint32_t)p.tiles);
    i /= (uint32_t)p.tiles;
    const int st = (int)(i & 1);
    i >>= 1;
    const int h = (int)(i % (uint32_t)p.c.H), b = (int)(i / (uint32_t)p.c.H);
    const int cpr = p.c.D / CPT, rpp = 256 / cpr;
    const int r0 = (int)threadIdx.x / cpr, ch = CPT * ((int)threadIdx.x - r0 * cpr);
    if (r0 >= rpp)
        return;
    const int lg = p.c.lg, mask = (1 << lg) - 1;
    const int64_t first = p.start ? p.start[b] : 0, len = p.lens[b];
    const uint8_t *pool = (st ? p.c.value + h * p.c.value_s_head : p.c.key + h * p.c.key_s_head) + ch;
    const int64_t s_page = st ? p.c.value_s_page : p.c.key_s_page;
    const uint32_t s_tok = st ? p.c.value_s_tok : p.c.key_s_tok;
    uint32_t code[kReadRows][NW];
    float s[kReadRows];
#pragma unroll
    for (int j = 0; j < kReadRows; ++j) {
        const int t = (tile * kReadRows + j) * rpp + r0;
        const int64_t pos = first + t;
#pragma unroll
        for (int e = 0; e < NW; ++e)
            code[j][e] = 0;
        s[j] = 0.0f;
        if (t < p.tokens && pos < len) {
            const int64_t page = pos >> lg;
            int id = -1;
            if (pos >= 0 && page < p.table_pages)
                id = p.table[b * p.bt_stride + page];
            if (bad_page(p.c, id)) {
                s[j] = __builtin_nanf("");
            } else {
                s[j] = p.c.scale[id * p.c.scale_s_page + h * p.c.scale_s_head + st];
                const uint8_t *src = pool + id * s_page + (uint32_t)(pos & mask) * s_tok;
                if constexpr (NW == 2) {
                    const u32x2 x = __builtin_nontemporal_load((const u32x2 *)src);
                    code[j][0] = x[0], code[j][1] = x[1];
                } else {
                    code[j][0] = __builtin_nontemporal_load((const uint32_t *)src);
                }
            }
        }
    }
    const int64_t o_tok = st ? p.s_tok[1] : p.s_tok[0];
    const int64_t o0 = b * (st ? p.s_seq[1] : p.s_seq[0]) + h * (st ? p.s_head[1] : p.s_head[0]) + ch;
    void *out = st ? p.out[1] : p.out[0];
#pragma unroll
    for (int j = 0; j < kReadRows; ++j) {
        const int t = (tile * kReadRows + j) * rpp + r0;
        if (t >= p.tokens)
            continue;
        float x[CPT];
#pragma unroll
        for (int e = 0; e < NW; ++e) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[j][e], false);
            const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[j][e], true);
            x[4 * e] = lo[0] * s[j], x[4 * e + 1] = lo[1] * s[j];
            x[4 * e + 2] = hi[0] * s[j], x[4 * e + 3] = hi[1] * s[j];
        }
        const int64_t o = o0 + t * o_tok;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (OUT == KITTY_SRC_F32)
                w[e] = __builtin_bit_cast(uint32_t, x[e]);
            else
                w[e] = (uint32_t)f2x(x[2 * e], OUT == KITTY_SRC_BF16) | (uint32_t)f2x(x[2 * e + 1], OUT == KITTY_SRC_BF16) << 16;
        }
        __builtin_nontemporal_store(w, (u32x4 *)((char *)out + o * (OUT == KITTY_SRC_F32 ? 4 : 2)));
    }
}

} // namespace kitty

using namespace kitty;

extern "C" int kitty_cache8_write(const kitty_cache8 *cache, const kitty_cache8_write_args *args, kitty_stream_t stream)
{
    WriteParams p;
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, p.c))
        return rc;
    const kitty_cache8_write_args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.table_pages < 0)
        return fail(KITTY_E_INVALID, "batch, tokens and table_pages must not be negative");
    if (a.src_dtype < KITTY_SRC_F16 || a.src_dtype > KITTY_SRC_F32)
        return fail(KITTY_E_INVALID, "src_dtype must be KITTY_SRC_F16, KITTY_SRC_BF16 or KITTY_SRC_F32");
    if (a.batch == 0 || a.tokens == 0)
        return KITTY_OK;
    if (!a.key || !a.value || (!a.block_table && a.table_pages) || !a.start)
        return fail(KITTY_E_INVALID, "NULL key, value, block_table or start");
    const int size = a.src_dtype == KITTY_SRC_F32 ? 4 : 2;
    if (!aligned(a.key, size) || !aligned(a.value, size))
        return fail(KITTY_E_INVALID, "key and value must be aligned to their elements");
    const int G = cache->page_tokens;
    const int64_t slots = ((int64_t)a.tokens + G - 2) / G + 1, blocks = (int64_t)a.batch * p.c.H * 2 * slots;
    if (blocks > kMaxBlocks || a.tokens > 1 << 30)
        return fail(KITTY_E_UNSUPPORTED, "too many pages for one launch");
    p.src[0] = a.key, p.src[1] = a.value;
    p.s_seq[0] = a.key_s_seq, p.s_head[0] = a.key_s_head, p.s_tok[0] = a.key_s_tok;
    p.s_seq[1] = a.value_s_seq, p.s_head[1] = a.value_s_head, p.s_tok[1] = a.value_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.start = a.start, p.lens = a.lens;
    p.tokens = a.tokens, p.table_pages = a.table_pages, p.slots = (int)slots;
    bool vec = aligned(a.key, 16) && aligned(a.value, 16);
    for (int st = 0; st < 2; ++st)
        for (int64_t s : {p.s_seq[st], p.s_head[st], p.s_tok[st]})
            vec = vec && s * size % 16 == 0;
    // one wave where a page gets at most two pieces a lane (a decode step), four where there is more to spread
    const bool wave = (int64_t)(a.tokens < G ? a.tokens : G) * p.c.D / 8 <= 128;
    const dim3 grid((unsigned)blocks);
    auto launch = [&](auto src, auto v) {
        constexpr int S = decltype(src)::value;
        constexpr bool V = decltype(v)::value;
        if (wave)
            hipLaunchKernelGGL((cache8_write_kernel<S, V, 64>), grid, dim3(64), 0, (hipStream_t)stream, p);
        else
            hipLaunchKernelGGL((cache8_write_kernel<S, V, 256>), grid, dim3(256), 0, (hipStream_t)stream, p);
    };
    auto by_align = [&](auto src) {
        if (vec)
            launch(src, std::true_type{});
        else
            launch(src, std::false_type{});
    };
    if (a.src_dtype == KITTY_SRC_F16)
        by_align(std::integral_constant<int, KITTY_SRC_F16>{});
    else if (a.src_dtype == KITTY_SRC_BF16)
        by_align(std::integral_constant<int, KITTY_SRC_BF16>{});
    else
        by_align(std::integral_constant<int, KITTY_SRC_F32>{});
    return check_launch("cache8_write_kernel");
}

extern "C" int kitty_cache8_read(const kitty_cache8 *cache, const kitty_cache8_read_args *args, kitty_stream_t stream)
{
    ReadParams p;
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, p.c))
        return rc;
    const kitty_cache8_read_args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.table_pages < 0)
        return fail(KITTY_E_INVALID, "batch, tokens and table_pages must not be negative");
    if (a.out_dtype < KITTY_SRC_F16 || a.out_dtype > KITTY_SRC_F32)
        return fail(KITTY_E_INVALID, "out_dtype must be KITTY_SRC_F16, KITTY_SRC_BF16 or KITTY_SRC_F32");
    if (a.batch == 0 || a.tokens == 0)
        return KITTY_OK;
    if (!a.key || !a.value || (!a.block_table && a.table_pages) || !a.lens)
        return fail(KITTY_E_INVALID, "NULL key, value, block_table or lens");
    const int size = a.out_dtype == KITTY_SRC_F32 ? 4 : 2;
    bool vec = aligned(a.key, 16) && aligned(a.value, 16);
    for (int64_t s : {a.key_s_seq, a.key_s_head, a.key_s_tok, a.value_s_seq, a.value_s_head, a.value_s_tok})
        vec = vec && s * size % 16 == 0;
    if (!vec)
        return fail(KITTY_E_INVALID, "key and value rows must be 16-byte aligned");
    const int rows = kReadRows * (256 / (p.c.D / read_codes(a.out_dtype)));
    const int64_t tiles = ((int64_t)a.tokens + rows - 1) / rows, blocks = (int64_t)a.batch * p.c.H * 2 * tiles;
    if (blocks > kMaxBlocks || a.tokens > 1 << 30)
        return fail(KITTY_E_UNSUPPORTED, "too many tokens for one launch");
    p.out[0] = a.key, p.out[1] = a.value;
    p.s_seq[0] = a.key_s_seq, p.s_head[0] = a.key_s_head, p.s_tok[0] = a.key_s_tok;
    p.s_seq[1] = a.value_s_seq, p.s_head[1] = a.value_s_head, p.s_tok[1] = a.value_s_tok;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.start = a.start, p.lens = a.lens;
    p.tokens = a.tokens, p.table_pages = a.table_pages, p.tiles = (int)tiles;
    const dim3 grid((unsigned)blocks), block(256);
    if (a.out_dtype == KITTY_SRC_F16)
        hipLaunchKernelGGL(cache8_read_kernel<KITTY_SRC_F16>, grid, block, 0, (hipStream_t)stream, p);
    else if (a.out_dtype == KITTY_SRC_BF16)
        hipLaunchKernelGGL(cache8_read_kernel<KITTY_SRC_BF16>, grid, block, 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(cache8_read_kernel<KITTY_SRC_F32>, grid, block, 0, (hipStream_t)stream, p);
    return check_launch("cache8_read_kernel");
}
