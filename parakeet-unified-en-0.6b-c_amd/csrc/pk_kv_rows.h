// pk_kv_rows.h - rows on their way into the key-value cache: what pk_kv_cache.hip and
// pk_rope.hip share.
#pragma once

#include "pk_decode.h"

namespace pkgpu {
namespace decode {

// Index of the cache row of one slot and head, or -1.
__device__ inline long long cache_row(int slot, uint32_t head, uint32_t heads, int page_shift, int n_slots)
{
    if (slot < 0 || slot >= n_slots) return -1;
    const uint32_t page = (uint32_t)slot >> page_shift, off = (uint32_t)slot & ((1u << page_shift) - 1);
    return (((long long)page * heads + head) << page_shift) + off;
}

__device__ inline uint32_t max_bits(const float* x)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    return m;
}

// One row's 8 elements of this lane into the cache at element `at`.
template <int CACHE, int DIM>
__device__ inline void write_part(void* cache, float* scales, long long row, int part, float* x)
{
    if constexpr (CACHE == E2M1) {
        const uint32_t byte = group_byte(max_over<kGroup / 8>(max_bits(x)));
        const uint32_t w = codes_e2m1(x, byte);
        if (row < 0) return;
        if (part % (kGroup / 8) == 0)
            reinterpret_cast<uint8_t*>(scales)[(size_t)row * (DIM / kGroup) + part / (kGroup / 8)] = (uint8_t)byte;
        reinterpret_cast<uint32_t*>(cache)[(size_t)row * (DIM / 8) + part] = w;
        return;
    } else if constexpr (row_scaled(CACHE)) {
        const RowCode c = row_code(max_over<DIM / 8>(max_bits(x)), top_of(CACHE));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = coded(x[i], c);
        if (row >= 0 && part == 0) scales[row] = c.scale;
    }
    if constexpr (CACHE != E2M1)
        if (row >= 0) store8<CACHE>(static_cast<char*>(cache) + ((size_t)row * DIM + 8 * part) * size_of(CACHE), x);
}

}  // namespace decode
}  // namespace pkgpu
