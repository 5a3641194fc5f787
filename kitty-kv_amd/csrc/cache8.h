// The 8-bit paged cache: what its kernels share (cache8.hip, attend8*.hip).
#pragma once
#include "common.h"

namespace kitty {

// kitty_cache8 as the kernels read it.
struct Cache8 {
    uint8_t *key, *value;
    float *scale;
    int64_t key_s_page, key_s_head, value_s_page, value_s_head, scale_s_page, scale_s_head;
    uint32_t key_s_tok, value_s_tok;   // a page's rows of one head span less than 2 GiB
    int64_t num_pages;
    int H, D, lg;                      // heads, head_dim, log2 of the page's tokens
};

// Checks a cache and fills `c`; KITTY_OK or the error's code.
int check_cache8(const kitty_cache8 *cache, Cache8 &c);

// Workgroups of up to 256 threads that one launch takes (a grid has less than 2^32 threads).
constexpr int64_t kMaxBlocks = 0xffffffffll / 256;

inline size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

inline bool aligned(const void *p, unsigned a) { return ((uintptr_t)p & (a - 1)) == 0; }

__device__ __forceinline__ bool bad_page(const Cache8 &c, int id) { return id < 0 || id >= c.num_pages; }

} // namespace kitty
