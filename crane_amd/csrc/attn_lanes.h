// attn_lanes.h -- what a wave's lanes say to each other, and its reads of LDS, in the attention
// kernels over pages (shared.hip, f8_attn.hip).
#pragma once

#include "common.h"

namespace crane {

typedef unsigned int u32x4_v __attribute__((ext_vector_type(4)));

// A wave-uniform value the compiler holds in vector registers (a buffer resource made
// of such would be read lane by lane).
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Maximum over the four lane groups of a query row; every lane gets it.  (A row swap of a
// value with itself leaves each row's value in one result and its neighbour's in the
// other.)
__device__ __forceinline__ float groups_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// The same, and the sum, over the two halves of the wave.
__device__ __forceinline__ float halves_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS byte addresses, and reads at them.
__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
}
__device__ __forceinline__ u32x4_v lds_read16(uint32_t at) {
    return *(const __attribute__((address_space(3))) u32x4_v*)(uintptr_t)at;
}

}  // namespace crane
