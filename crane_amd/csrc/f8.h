// f8.h -- shared device helpers of the 8-bit KV cache (include/crane_f8.h): e4m3 codes
// and a power-of-two scale for every 32 rows of a head.
#pragma once

#include "common.h"
#include "../../include/crane_f8.h"

namespace crane {

constexpr int kBlockRows8 = CRANE_F8_BLOCK_ROWS;
// The smallest scale, 2^-100: a code's smallest step times it is 2^-109, so that every
// value and its products with ordinary ones are normal in f32 and bf16.
constexpr int kLeastScale = 27;

typedef float f32x2_v __attribute__((ext_vector_type(2)));

// 2^(byte - 127) of a scale byte in 1 .. 254; 0 for 0.
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }
// 1 over it, subnormal for 254.
__device__ __forceinline__ float inverse_scale(int byte) {
    return byte < 254 ? scale_of(254 - byte) : __uint_as_float(0x400000u);
}

// The byte of the smallest scale 2^e with amax <= 448 2^e (448 = 1.75 2^8, the largest
// code), from the bits of a finite amax >= 0.
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t u = __float_as_uint(amax);
    return max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u), kLeastScale);
}

// Eight values times `inv` (a power of two), rounded to codes.  Values are within 448
// then, or not finite, which the conversion turns into a NaN.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * inv, x[4 * h + 1] * inv, 0, false);
        w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv, r, true);
    }
    return make_uint2(w[0], w[1]);
}
// Four codes' values, at scale 1.
__device__ __forceinline__ void values4(uint32_t w, float* x) {
    const f32x2_v a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = a[0];
    x[1] = a[1];
    x[2] = b[0];
    x[3] = b[1];
}
// Four codes rounded again for a scale 1 / down times theirs.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float down) {
    float x[4];
    values4(w, x);
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * down, x[1] * down, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * down, x[3] * down, r, true);
}

// ---- host
// Quantise rows k, v [B, Hkv, S, D] of `dtype` into rows start[b] .. (start null: 0 ..) of the
// pages, as the append does (f8_cache.hip; for the cache manager, which has checked its
// arguments).
int f8_write_rows(const void* k, const void* v, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                  const PagedRows& rows, const int32_t* start, int B, int64_t S, int Hkv, int dtype, hipStream_t st);

// A grid's threads are 32 bits and a workgroup is 256 of them.
constexpr int64_t kMostUnits8 = 0xffffff;
// The workgroups of f8_write_rows: a block, of k or of v, of a head, for wherever in its first
// block a sequence's S rows begin.
inline int64_t f8_rows_units(int B, int64_t S, int Hkv) {
    return (int64_t)B * 2 * Hkv * ((S + 2 * kBlockRows8 - 2) / kBlockRows8);
}

// A check the launchers share: the pools' addresses.
inline int check_pools8(const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale) {
    if (!k_pool || !v_pool || !k_scale || !v_scale) return CRANE_HIP_E_INVALID;
    return aligned16(k_pool) && aligned16(v_pool) && aligned16(k_scale) && aligned16(v_scale) ? CRANE_HIP_OK
                                                                                              : CRANE_HIP_E_ALIGN;
}
}  // namespace crane
