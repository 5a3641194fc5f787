// Eviction from the 8-bit paged cache by weight, on gfx950: which tokens of a sequence
// and KV head stay, and their move together.
//
// cache8_select_kernel, a workgroup per (sequence, KV head): the weights between the
// first and last tokens, which stay, map to unsigned keys in the floats' order; three
// passes over 11, 11 and 10 bits, counted in LDS, find the key of the lightest token that
// stays and how many of its equals do (it ends where all of a bin stay, for weights
// without equals mostly after two).  Positions and weights are written in order: a token's
// place is the count of heavier ones before it plus that of its equals, as far as they
// stay, by ballots of a wave over its run of tokens and the waves' counts.  Counts are
// integers: any order of additions gives the same.  Further workgroups of the launch find
// the sequences that name a page twice (new_lengths).
// cache8_pack_kernel, a workgroup per (page, KV head, stream) of the result: the page's
// scale is the largest of the pages that its tokens come from, and codes of smaller
// scales are multiplied by the quotient and rounded again (exact but for subnormals
// where scales are powers of two).  In place the codes go through the workspace, as a
// page of the result may hold tokens that another page of the result needs; sequences
// within the budget are left alone.
//
// The selection is bound by latency: passes, each of counting, a scan and three barriers,
// and a workgroup a CU at most where there are few sequences; the move by HBM.  Measured,
// 8 heads of 128: 16 sequences of 32,768 tokens cut to 16,384 into other pages 254 us: 31
// for the selection and 223 for 1,077 MB read and written (4.83 TB/s, where a copy reaches
// 5.13); one sequence of 1,100 cut to 1,024 14.0, of which the kernels are 8.1 and 4.6
// and the host's call, alongside, 14.6.  Small evictions in one launch, each selecting
// workgroup moving its tokens: 21 to 24 where these are 12.7 (a CU alone moves 0.5 MB in
// 12 us).
#include <algorithm>

#include "cache8.h"

namespace kitty {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Evict8 {
    Cache8 c;
    const float *weights;
    int64_t w_s_seq, w_s_head;
    const int32_t *table, *lens, *into;
    int64_t bt_stride, into_stride;
    int32_t *out_lens, *kept;
    float *out_weights;
    uint8_t *ws_codes;    // in place: (sequence, KV head, stream, K, D)
    float *ws_scale;      //           (sequence, KV head, stream, K)
    int B, N, K, keep, first, last, table_pages, into_pages, tiles;
    int in_place, most_pages;   // pages that a sequence may write
    int group, lanes;           // new_lengths
    unsigned slots;             // cache8_named_kernel's, 0: new_lengths
};

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64;
constexpr int kBins = 2048, kCopies = 4;   // counters of a pass; copies, so that fewer lanes meet at one

// A weight as an unsigned key in the floats' order: both zeros alike, NaN above all.  0
// and 0xffffffff are no weight's: of places behind the sequence and of tokens that stay.
__device__ __forceinline__ uint32_t weight_key(float x)
{
    const uint32_t u = x == 0.0f ? 0u : __builtin_bit_cast(uint32_t, x);
    return x != x ? 0xfffffffeu : u >> 31 ? ~u : u | 0x80000000u;
}

// Tokens of sequence b that stay, -1 where its length breaks the rules.
__device__ __forceinline__ int kept8(const Evict8 &p, int n)
{
    return n < 0 || n > (int64_t)p.table_pages << p.c.lg || n > p.N ? -1 : min(n, p.keep);
}

// Of them, those that are written: in place none of a sequence that is not cut, whose pages
// stay as they are.
__device__ __forceinline__ int written8(const Evict8 &p, int n)
{
    return p.in_place && n <= p.keep ? 0 : kept8(p, n);
}

// Pages of n tokens, 0 of a length that breaks the rules.
__device__ __forceinline__ int pages8(const Evict8 &p, int n) { return n <= 0 ? 0 : ((n - 1) >> p.c.lg) + 1; }

// The sum of a value over the lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned add_dpp(unsigned v)
{
    return v + (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ unsigned scan64(unsigned v)
{
    v = add_dpp<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
    v = add_dpp<0x112, 0xf>(v);
    v = add_dpp<0x114, 0xf>(v);
    v = add_dpp<0x118, 0xf>(v);
    v = add_dpp<0x142, 0xa>(v);   // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    return add_dpp<0x143, 0xc>(v);
}

// The sum of the waves' values before this one's.
__device__ __forceinline__ unsigned sum_before(const unsigned *v, int wave)
{
    unsigned s = 0;
#pragma unroll
    for (int k = 0; k < kSelectWaves; ++k)
        s += k < wave ? v[k] : 0;
    return s;
}

// Lengths after the call: -1 also where a page that a sequence writes is named once more, as
// one that another needs or writes, as it would be lost or written by two workgroups at
// once.  (A page that is read alone may be named often.)  The written pages' ids go into a
// table of open addressing with the number of their entry; then every page that the call
// names is looked up.
//
// Up to kNamed written pages in all, and kLooks in the tables: a workgroup of the selection's
// launch does it, its table in LDS, half full, `lanes` threads for each sequence's pages;
// beside the selection its time is not seen (1 x 1,100 tokens 14 us, 16 x 32,768 in pages of
// 128 254, with and without).  More: three launches of 5 to 10 us before the selection, the
// table in the memory of the weights that come out (cache8_named_kernel): 48 x 65,536 tokens
// of one head of 64 in pages of 16 to half 397 us, where workgroups of the selection with
// several tables take 753; 2,000 x 100 tokens, 2 heads of 64, 107 and 129; 16 x 65,536
// tokens, 8 heads of 128 in pages of 128 602 and 581.  Where the memory is too small
// (thousands of sequences of a few tokens) LDS again, for `group` sequences at a time.
constexpr int kNamed = 2048, kSlots = 2 * kNamed;
constexpr unsigned kFree = 0xffffffffu;   // no page's id
constexpr int64_t kLooks = 1 << 17;       // pages of the tables, beyond which one workgroup would look too long

// In the counters' LDS (with 16 KB more of it a select of 2,000 short sequences took 74 us, 52 without).
struct Named8 {
    unsigned ids[kSlots];
    unsigned short entry[kSlots];
    unsigned twice[kNamed / 32];   // a bit for each sequence of the group
};
static_assert(sizeof(Named8) <= kCopies * kBins * 4, "they share LDS");

__device__ __forceinline__ unsigned slot_of(int id, unsigned slots)   // a power of two
{
    return (unsigned)id * 2654435769u >> (__builtin_clz(slots) + 1);
}

// Pages that a sequence of n tokens writes.
__device__ __forceinline__ int written_pages8(const Evict8 &p, int n) { return min(pages8(p, written8(p, n)), p.into_pages); }

// Pages of its table that a sequence of n tokens needs while others are written: in place
// those that it keeps, as all that moves is read before.
__device__ __forceinline__ int needed8(const Evict8 &p, int n)
{
    const int m = kept8(p, n);
    return m < 0 ? 0 : pages8(p, p.in_place ? m : n);
}

__device__ __forceinline__ void new_lengths(const Evict8 &p, int number, Named8 &named)
{
    unsigned *slots = named.ids;
    const int tid = threadIdx.x, b0 = number * p.group, b1 = min(b0 + p.group, p.B), span = p.most_pages;
    auto flag = [&](int seq) { atomicOr(&named.twice[seq >> 5], 1u << (seq & 31)); };
    if (tid < kNamed / 32)
        named.twice[tid] = 0;
    for (int i = tid; i < kSlots; i += kSelect)
        slots[i] = kFree;
    __syncthreads();
    for (int e = tid; e < (b1 - b0) * span; e += kSelect) {   // kNamed at most
        const int seq = e / span, i = e - seq * span;
        const int id = i < written_pages8(p, p.lens[b0 + seq]) ? p.into[(b0 + seq) * p.into_stride + i] : -1;
        if (bad_page(p.c, id))
            continue;
        for (unsigned s = slot_of(id, kSlots);; s = (s + 1) & (kSlots - 1)) {   // ends: half the slots are free
            const unsigned was = atomicCAS(&slots[s], kFree, (unsigned)id);
            if (was == kFree)
                named.entry[s] = (unsigned short)e;
            if (was == kFree || was == (unsigned)id)
                break;
        }
    }
    __syncthreads();
    // a row's first `count` pages, of which the first `own` are entries from `base` on
    auto look = [&](const int32_t *row, int count, int own, int base) {
        for (int i0 = tid % p.lanes; i0 < count; i0 += 4 * p.lanes) {
            int id[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                id[j] = i0 + j * p.lanes < count ? row[i0 + j * p.lanes] : -1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (bad_page(p.c, id[j]))
                    continue;
                unsigned s = slot_of(id[j], kSlots);
                while (slots[s] != kFree && slots[s] != (unsigned)id[j])
                    s = (s + 1) & (kSlots - 1);
                if (slots[s] == kFree)
                    continue;
                const int i = i0 + j * p.lanes, mine = i < own ? base + i : -1, e = named.entry[s];
                if (e != mine) {
                    flag(e / span);
                    if (mine >= 0)
                        flag(mine / span);
                }
            }
        }
    };
    for (int b = span ? tid / p.lanes : p.B; b < p.B; b += kSelect / p.lanes) {
        const int n = p.lens[b], w = min(written_pages8(p, n), span);
        const int own = b >= b0 && b < b1 ? w : 0, base = (b - b0) * span;
        look(p.table + b * p.bt_stride, needed8(p, n), p.in_place ? own : 0, base);
        if (!p.in_place)
            look(p.into + b * p.into_stride, w, own, base);
    }
    __syncthreads();
    for (int b = b0 + tid; b < b1; b += kSelect)
        p.out_lens[b] = named.twice[(b - b0) >> 5] >> ((b - b0) & 31) & 1 ? -1 : kept8(p, p.lens[b]);
}

// The same in three launches: 0 empties the table, 1 enters the written pages, 2 looks.  A
// wave for 256 pages of a sequence, or more where it has many.
template <int STEP>
__global__ __launch_bounds__(64) void cache8_named_kernel(Evict8 p, int parts)
{
    unsigned *ids = (unsigned *)p.out_weights;
    int *entries = (int *)p.out_weights + p.slots;
    if constexpr (STEP == 0) {
        for (int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x; i < p.slots; i += (int64_t)gridDim.x * 64)
            ids[i] = kFree;
        for (int b = blockIdx.x * 64 + threadIdx.x; b < p.B; b += gridDim.x * 64)
            p.out_lens[b] = kept8(p, p.lens[b]);
        return;
    }
    const int b = blockIdx.x / parts, part = blockIdx.x - b * parts;
    const int n = p.lens[b], written = min(written_pages8(p, n), p.most_pages);
    const int32_t *to = p.into + b * p.into_stride;
    if constexpr (STEP == 1) {
        for (int i = part * 64 + threadIdx.x; i < written; i += parts * 64) {
            const int id = to[i];
            if (bad_page(p.c, id))
                continue;
            for (unsigned s = slot_of(id, p.slots);; s = (s + 1) & (p.slots - 1)) {   // ends: at most half the slots are taken
                const unsigned was = atomicCAS(&ids[s], kFree, (unsigned)id);
                if (was == kFree)
                    entries[s] = b * p.most_pages + i;
                if (was == kFree || was == (unsigned)id)
                    break;
            }
        }
        return;
    }
    auto look = [&](const int32_t *row, int count, int own) {
        for (int i = part * 64 + threadIdx.x; i < count; i += parts * 64) {
            const int id = row[i];
            if (bad_page(p.c, id))
                continue;
            unsigned s = slot_of(id, p.slots);
            while (ids[s] != kFree && ids[s] != (unsigned)id)
                s = (s + 1) & (p.slots - 1);
            if (ids[s] == kFree)
                continue;
            const int mine = i < own ? b * p.most_pages + i : -1, e = entries[s];
            if (e != mine) {
                p.out_lens[e / p.most_pages] = -1;
                if (mine >= 0)
                    p.out_lens[b] = -1;
            }
        }
    };
    look(p.table + b * p.bt_stride, needed8(p, n), p.in_place ? written : 0);
    if (!p.in_place)
        look(to, written, written);
}

// A wave takes a run of 64 j tokens; EACH: j at most, the weights then stay in registers
// (0: any j, they are read again in every pass).  Kept in registers rather than read again:
// 16 x 32,768 tokens, 8 heads 31 us, 73 read again.
template <int EACH>
__global__ __launch_bounds__(kSelect) void cache8_select_kernel(Evict8 p)
{
    __shared__ __attribute__((aligned(16))) unsigned hist[kCopies][kBins], sums[2][kSelectWaves];
    __shared__ unsigned found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pairs = p.B * p.c.H;
    if ((int)blockIdx.x >= pairs) {
        new_lengths(p, blockIdx.x - pairs, *(Named8 *)hist);
        return;
    }
    const int b = blockIdx.x / p.c.H, h = blockIdx.x - b * p.c.H;
    const int n = p.lens[b], m = kept8(p, n);
    const float *w = p.weights + b * p.w_s_seq + h * p.w_s_head;
    int32_t *kept = p.kept + (int64_t)blockIdx.x * p.K;
    float *out = p.out_weights + (int64_t)blockIdx.x * p.N;
    const int end = m < 0 ? 0 : n, last = end - p.last;
    const int steps = (end + kSelect - 1) / kSelect;           // of 64 tokens, a wave
    const int pos0 = wave * steps * 64 + lane;
    auto key_at = [&](int i, float v) { return i >= end ? 0u : i < p.first || i >= last ? 0xffffffffu : weight_key(v); };
    float x[EACH > 0 ? EACH : 1];
    uint32_t keys[EACH > 0 ? EACH : 1];
    if constexpr (EACH > 0) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            x[j] = pos0 + 64 * j < end && j < steps ? w[pos0 + 64 * j] : 0.0f;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            keys[j] = j < steps ? key_at(pos0 + 64 * j, x[j]) : 0;
    }
    auto each = [&](auto body) {
        if constexpr (EACH > 0) {
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (j < steps)
                    body(pos0 + 64 * j, x[j], keys[j]);
        } else {
            for (int j = 0; j < steps; ++j) {
                const int i = pos0 + 64 * j;
                const float v = i < end ? w[i] : 0.0f;
                body(i, v, key_at(i, v));
            }
        }
    };
    uint32_t key = 0;          // tokens above it stay, and `need` of its equals
    int need = 0;
    if (n > m && m > 0) {
        need = m;
        // 11, 11 and 10 bits: signs, exponents and two bits of the fraction first
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t above = pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10), bins = pass == 2 ? 1023 : 2047;
            for (int i = tid; i < kCopies * kBins / 4; i += kSelect)
                ((u32x4 *)hist)[i] = u32x4{0, 0, 0, 0};
            __syncthreads();
            each([&](int, float, uint32_t k) {
                if (((k ^ key) & above) == 0 && k != 0)
                    atomicAdd(&hist[wave & (kCopies - 1)][k >> shift & bins], 1u);
            });
            __syncthreads();
            // from the heaviest: thread t has bins 2047 - 2 t and 2046 - 2 t
            unsigned c[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
                const uint2 two = *(const uint2 *)&hist[k][kBins - 2 - 2 * tid];
                c[0] += two.y, c[1] += two.x;
            }
            const unsigned inc = scan64(c[0] + c[1]);
            if (lane == 63)
                sums[0][wave] = inc;
            __syncthreads();
            unsigned before = inc - c[0] - c[1] + sum_before(sums[0], wave);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (before < (unsigned)need && before + c[e] >= (unsigned)need)
                    found[0] = kBins - 1 - 2 * tid - e, found[1] = need - before, found[2] = c[e];
                before += c[e];
            }
            __syncthreads();
            key |= found[0] << shift;
            need = (int)found[1];
            if (found[2] == found[1]) {   // all of the bin stay: often but one token is left in it
                key -= key ? 1 : 0;
                need = 0;
                break;
            }
        }
    } else if (m == 0) {
        key = 0xffffffffu;     // none stays (first and last are 0)
    }
    int n_above = 0, n_same = 0;
    each([&](int, float, uint32_t k) {
        n_above += __popcll(__ballot(k > key));
        n_same += __popcll(__ballot(k == key));
    });
    if (lane == 0)
        sums[0][wave] = n_above, sums[1][wave] = n_same;
    __syncthreads();
    n_above = (int)sum_before(sums[0], wave), n_same = (int)sum_before(sums[1], wave);   // of the waves before this one
    each([&](int i, float v, uint32_t k) {
        const uint64_t a = __ballot(k > key), c = __ballot(k == key);
        const int e = n_same + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(c >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)c, 0));
        if (k > key || (k == key && e < need)) {
            const int at = n_above + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(a >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)a, 0)) + min(e, need);
            kept[at] = i;
            out[at] = v;
        }
        n_above += __popcll(a), n_same += __popcll(c);
    });
    for (int i = max(m, 0) + tid; i < p.N; i += kSelect)
        out[i] = 0.0f;
    for (int i = max(m, 0) + tid; i < p.K; i += kSelect)
        kept[i] = -1;
}

// Where a kept token's codes are.
struct Source8 {
    const uint8_t *codes;    // NULL: it has no page
    float scale;
};

__device__ __forceinline__ Source8 source8(const Evict8 &p, int b, int h, int st, int pos)
{
    const int id = pos < 0 ? -1 : p.table[b * p.bt_stride + (pos >> p.c.lg)];
    if (bad_page(p.c, id))
        return Source8{nullptr, 0.0f};
    const uint32_t row = (uint32_t)pos & ((1u << p.c.lg) - 1);
    return Source8{st ? p.c.value + id * p.c.value_s_page + h * p.c.value_s_head + row * p.c.value_s_tok
                      : p.c.key + id * p.c.key_s_page + h * p.c.key_s_head + row * p.c.key_s_tok,
                   p.c.scale[id * p.c.scale_s_page + h * p.c.scale_s_head + st]};
}

// The kept tokens' codes and scales, in their new order, into the workspace.
__global__ __launch_bounds__(256) void cache8_stage_kernel(Evict8 p)
{
    uint32_t i = blockIdx.x;
    const int tile = (int)(i % (uint32_t)p.tiles);
    i /= (uint32_t)p.tiles;
    const int st = (int)(i & 1);
    const int h = (int)((i >> 1) % (uint32_t)p.c.H), b = (int)((i >> 1) / (uint32_t)p.c.H);
    const int cpr = p.c.D >> 4, rows = 256 / cpr, r = threadIdx.x / cpr, c = threadIdx.x - r * cpr;
    const int64_t seq = (int64_t)(b * p.c.H + h), list = (2 * seq + st) * p.K;
    const int at = tile * rows + r;
    if (r >= rows || at >= written8(p, p.lens[b]))
        return;
    const Source8 s = source8(p, b, h, st, p.kept[seq * p.K + at]);
    *(u32x4 *)(p.ws_codes + (list + at) * p.c.D + 16 * c) =
        s.codes ? *(const u32x4 *)(s.codes + 16 * c) : u32x4{0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f};
    if (c == 0)
        p.ws_scale[list + at] = s.codes ? s.scale : -1.0f;
}

__device__ __forceinline__ unsigned times(unsigned w, float f)
{
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, r, true);
}

template <bool STAGED>
__global__ __launch_bounds__(256) void cache8_pack_kernel(Evict8 p)
{
    __shared__ const uint8_t *src[256];
    __shared__ float scale[256], part[4];
    uint32_t i = blockIdx.x;
    const int page = (int)(i % (uint32_t)p.tiles);
    i /= (uint32_t)p.tiles;
    const int st = (int)(i & 1);
    const int h = (int)((i >> 1) % (uint32_t)p.c.H), b = (int)((i >> 1) / (uint32_t)p.c.H);
    const int64_t seq = (int64_t)(b * p.c.H + h), list = (2 * seq + st) * p.K;
    const int lg = p.c.lg, first = page << lg, m = written8(p, p.lens[b]);
    if (p.out_lens[b] < 0) {
        // it stays as it was: what the selection said of it goes
        if (i == 2 * (unsigned)seq && page == 0) {
            for (int j = threadIdx.x; j < p.K; j += 256)
                p.kept[seq * p.K + j] = -1;
            for (int j = threadIdx.x; j < p.N; j += 256)
                p.out_weights[seq * p.N + j] = 0.0f;
        }
        return;
    }
    if (first >= m || page >= p.into_pages)
        return;
    const int id = p.into[b * p.into_stride + page];
    if (bad_page(p.c, id))
        return;
    const int rows = min(1 << lg, m - first);
    float mine = -1.0f;       // of a token without a page
    if ((int)threadIdx.x < rows) {
        const int at = first + threadIdx.x;
        if constexpr (STAGED) {
            mine = p.ws_scale[list + at];
            src[threadIdx.x] = p.ws_codes + (list + at) * p.c.D;
        } else {
            const Source8 s = source8(p, b, h, st, p.kept[seq * p.K + at]);
            mine = s.codes ? s.scale : -1.0f;
            src[threadIdx.x] = s.codes;
        }
        scale[threadIdx.x] = mine;
    }
    float top = mine;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        top = fmaxf(top, __shfl_xor(top, off));
    if ((threadIdx.x & 63) == 0)
        part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    if (top < 0.0f)
        top = 1.0f;           // none of its tokens has a page
    uint8_t *dst = st ? p.c.value + id * p.c.value_s_page + h * p.c.value_s_head
                      : p.c.key + id * p.c.key_s_page + h * p.c.key_s_head;
    const uint32_t d_tok = st ? p.c.value_s_tok : p.c.key_s_tok;
    const int cpr = p.c.D >> 4, rpp = 256 / cpr, r0 = threadIdx.x / cpr, c = threadIdx.x - r0 * cpr;
    if (r0 < rpp)
        for (int r = r0; r < rows; r += rpp) {
            const uint8_t *s = src[r];
            const float was = scale[r];
            u32x4 x = {0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f};
            if (STAGED || s)
                x = *(const u32x4 *)(s + 16 * c);
            if (was != top && was >= 0.0f) {
                const float f = was / top;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = times(x[e], f);
            }
            *(u32x4 *)(dst + (uint32_t)r * d_tok + 16 * c) = x;
        }
    if (threadIdx.x == 0)
        p.c.scale[id * p.c.scale_s_page + h * p.c.scale_s_head + st] = top;
}

static int check_evict(const kitty_cache8 *cache, const kitty_cache8_evict_args *args, Evict8 &p, size_t &need)
{
    if (!args)
        return fail(KITTY_E_INVALID, "args is NULL");
    if (const int rc = check_cache8(cache, p.c))
        return rc;
    const kitty_cache8_evict_args &a = *args;
    if (a.batch < 0 || a.table_pages < 0 || a.into_pages < 0 || a.weight_tokens < 0)
        return fail(KITTY_E_INVALID, "batch, table_pages, into_pages and weight_tokens must not be negative");
    if (a.keep < 0 || a.first < 0 || a.last < 0 || (int64_t)a.first + a.last > a.keep)
        return fail(KITTY_E_INVALID, "first and last must not be negative, and keep at least both together");
    if ((int64_t)a.table_pages << p.c.lg > 1 << 30 || a.weight_tokens > 1 << 30)
        return fail(KITTY_E_UNSUPPORTED, "a sequence is limited to 2^30 tokens");
    p.B = a.batch, p.N = a.weight_tokens, p.K = a.keep < a.weight_tokens ? a.keep : a.weight_tokens;
    p.into_pages = a.into ? a.into_pages : a.table_pages;
    p.most_pages = std::min(p.into_pages, p.K ? ((p.K - 1) >> p.c.lg) + 1 : 0);
    // (the selection's launch has workgroups of 1,024 threads, up to 2,049 of them new_lengths')
    if ((int64_t)p.B * p.c.H > kMaxBlocks / 4 - 2049 || (int64_t)p.B * p.c.H * 2 * (((int64_t)p.K >> 4) + 1) > kMaxBlocks)
        return fail(KITTY_E_UNSUPPORTED, "too many tokens for one launch");
    const int64_t pages = (int64_t)p.B * p.most_pages, room = (int64_t)p.B * p.c.H * p.N / 2;
    p.slots = 1;
    while (p.slots < 2 * pages)
        p.slots *= 2;
    if ((pages <= kNamed && (int64_t)p.B * std::min(p.table_pages, (p.N >> p.c.lg) + 1) <= kLooks) || p.slots > room)
        p.slots = 0;
    p.group = std::max(1, kNamed / std::max(p.most_pages, 1));
    p.lanes = 1;
    while (p.lanes < kSelect && (int64_t)2 * p.lanes * p.B <= kSelect)
        p.lanes *= 2;
    need = a.into ? 0 : up16((size_t)p.B * p.c.H * 2 * p.K * p.c.D) + up16((size_t)p.B * p.c.H * 2 * p.K * 4);
    return KITTY_OK;
}

} // namespace kitty

using namespace kitty;

extern "C" int kitty_cache8_evict_workspace_size(const kitty_cache8 *cache, const kitty_cache8_evict_args *args, size_t *bytes)
{
    Evict8 p{};
    if (!bytes)
        return fail(KITTY_E_INVALID, "bytes is NULL");
    return check_evict(cache, args, p, *bytes);
}

extern "C" int kitty_cache8_evict(const kitty_cache8 *cache, const kitty_cache8_evict_args *args, kitty_stream_t stream)
{
    Evict8 p{};
    size_t need;
    if (const int rc = check_evict(cache, args, p, need))
        return rc;
    const kitty_cache8_evict_args &a = *args;
    if (a.batch == 0)
        return KITTY_OK;
    if (!a.lens || !a.out_lens || (!a.block_table && a.table_pages) || (a.weight_tokens && (!a.weights || !a.out_weights)) ||
        (p.K && !a.kept))
        return fail(KITTY_E_INVALID, "NULL lens, out_lens, block_table, weights, out_weights or kept");
    if (!aligned(a.weights, 4) || !aligned(a.out_weights, 4))
        return fail(KITTY_E_INVALID, "weights and out_weights must be 4-byte aligned");
    if (need && (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < need))
        return fail(KITTY_E_INVALID, "workspace is NULL, misaligned or smaller than kitty_cache8_evict_workspace_size");
    p.weights = a.weights, p.w_s_seq = a.w_s_seq, p.w_s_head = a.w_s_head;
    p.table = a.block_table, p.bt_stride = a.bt_stride, p.table_pages = a.table_pages, p.lens = a.lens;
    p.into = a.into ? a.into : a.block_table, p.into_stride = a.into ? a.into_stride : a.bt_stride;
    p.out_lens = a.out_lens, p.kept = a.kept, p.out_weights = a.out_weights;
    p.keep = a.keep, p.first = a.first, p.last = a.last, p.in_place = !a.into;
    p.ws_codes = (uint8_t *)a.workspace;
    p.ws_scale = (float *)((char *)a.workspace + up16((size_t)p.B * p.c.H * 2 * p.K * p.c.D));
    const hipStream_t st = (hipStream_t)stream;
    const unsigned pairs = (unsigned)(p.B * p.c.H), grid = pairs + (p.slots ? 0 : (unsigned)((p.B - 1) / p.group + 1));
    if (p.slots) {
        const int parts = std::min((std::max(std::min(p.table_pages, (p.N >> p.c.lg) + 1), p.most_pages) + 255) / 256, 64);
        const dim3 waves((unsigned)p.B * (unsigned)parts), block(64);
        hipLaunchKernelGGL(cache8_named_kernel<0>, dim3(std::min(p.slots / 256 + 1, 2048u)), block, 0, st, p, parts);
        hipLaunchKernelGGL(cache8_named_kernel<1>, waves, block, 0, st, p, parts);
        hipLaunchKernelGGL(cache8_named_kernel<2>, waves, block, 0, st, p, parts);
    }
    // by what a sequence can hold: 8 or 32 weights a lane in registers (1,100 tokens 8.2 us
    // with room for 8, 12.1 with room for 32, 8.6 read again; 31 and 73 for 32,768 tokens)
    const int64_t cap = std::min<int64_t>((int64_t)p.table_pages << p.c.lg, p.N);
    if (cap <= 8 * kSelect)
        hipLaunchKernelGGL(cache8_select_kernel<8>, dim3(grid), dim3(kSelect), 0, st, p);
    else if (cap <= 32 * kSelect)
        hipLaunchKernelGGL(cache8_select_kernel<32>, dim3(grid), dim3(kSelect), 0, st, p);
    else
        hipLaunchKernelGGL(cache8_select_kernel<0>, dim3(grid), dim3(kSelect), 0, st, p);
    if (p.K > 0) {
        if (!a.into) {
            const int rows = 256 / (p.c.D >> 4);
            p.tiles = (p.K + rows - 1) / rows;
            hipLaunchKernelGGL(cache8_stage_kernel, dim3(pairs * 2 * (unsigned)p.tiles), dim3(256), 0, st, p);
        }
        p.tiles = ((p.K - 1) >> p.c.lg) + 1;
        if (a.into)
            hipLaunchKernelGGL(cache8_pack_kernel<false>, dim3(pairs * 2 * (unsigned)p.tiles), dim3(256), 0, st, p);
        else
            hipLaunchKernelGGL(cache8_pack_kernel<true>, dim3(pairs * 2 * (unsigned)p.tiles), dim3(256), 0, st, p);
    }
    return check_launch("8-bit cache eviction");
}
