// Shared pieces of the paged key-value cache kernels (paged.hip,
// paged_attention.hip): exact division by a page size, wave scans, the cache's
// refusals.
#pragma once

#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "../../include/flash.h"
#include "args.hpp"
#include "common.hpp"

namespace bmb {

// n / d and n % d for 0 <= n < 2^31 by one 64-bit product: with
// s = ceil(log2 d) and m = ceil(2^(31+s) / d), m d exceeds 2^(31+s) by e < d
// <= 2^s, so n m / 2^(31+s) exceeds n / d by n e / (d 2^(31+s)) < 1 / d: too
// little to reach the next whole number. m <= 2^32 - 1 since d > 2^(s-1).
struct FastDiv {
    uint32_t d, m;
    int shift;
    __host__ static FastDiv of(int divisor) {
        FastDiv f;
        f.d = (uint32_t)divisor;
        int s = 0;
        while ((1ull << s) < f.d) ++s;
        f.shift = 31 + s;
        f.m = (uint32_t)(((1ull << f.shift) + f.d - 1) / f.d);
        return f;
    }
    __device__ __forceinline__ int quot(int n) const {
        return (int)(((uint64_t)(uint32_t)n * m) >> shift);
    }
};

// Sum of two counts that stays at 2^32 - 1 once it would pass it.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
    const uint32_t s = a + b;
    return s < a ? 0xffffffffu : s;
}

// Inclusive scan over the 64 lanes: four steps inside the rows of 16 lanes,
// then the last lane of row 0 (2) to row 1 (3) and of row 1 to rows 2 and 3.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, false));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, false));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, false));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, false));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false));
    return x;
}

// The cache's own description, checked: nullptr if a call may use it, else why
// not. Without `buffers` its pointers are not looked at.
inline const char *cache_fault(const PagedCache *c, bool buffers) {
    if (c == nullptr || (buffers && (c->k == nullptr || c->v == nullptr))) return "no cache";
    const int size = element_size(c->type);
    if (size == 0) return "unknown element type of the cache";
    if (c->pages < 1 || c->page_size < 1 || c->kv_heads < 1) return "empty cache";
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128)
        return "head size is not 32, 64 or 128";
    if ((long long)c->pages * c->page_size > INT_MAX) return "2^31 or more tokens in the cache";
    const unsigned long long halves = buffers ? (uintptr_t)c->k | (uintptr_t)c->v : 0;
    const unsigned long long bits = halves | (unsigned long long)(c->page_stride * size) |
                                    (unsigned long long)(c->token_stride * size) |
                                    (unsigned long long)(c->head_stride * size);
    if (bits % 16 != 0) return "the cache's buffers and strides are no multiples of 16 bytes";
    if (c->token_stride >= (1ll << 26))  // lanes' offsets: 16 rows in 32 bits
        return "token_stride of the cache is 2^26 elements or more";
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
        return "negative stride of the cache";
    return nullptr;
}

}  // namespace bmb
