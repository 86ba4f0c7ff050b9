// pages.hip -- copies of rows between pages of the K/V pools; the C ABI is
// crane_hip_copy_pages in include/crane_shared.h.
//
// A page [Hkv, page_rows, D] of a pool is Hkv runs of page_rows rows, and a copy
// takes the first rows of each run.  The pairs and the pools' addresses go to the
// kernel as arguments: the lists are the host's (page lists live there), so nothing
// is uploaded and nothing waits.
#include <algorithm>
#include <vector>

#include "common.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr int kPools = 128;      // pools per launch: K and V of 64 layers
constexpr int kPairs = 128;      // pairs per launch
constexpr int kBlockBytes = 16384;  // bytes of one head's run per workgroup: 4 loads of 16 bytes per thread

typedef unsigned int u32x4_v __attribute__((ext_vector_type(4)));

struct CopyArgs {
    uint8_t* pool[kPools];
    int32_t src[kPairs], dst[kPairs], rows[kPairs];
};

// grid: (heads x blocks of a run, pairs, pools)
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a, int blocks, int Hkv, int64_t run_bytes,
                                                         int row_bytes) {
    const int head = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const int64_t bytes = (int64_t)a.rows[blockIdx.y] * row_bytes;
    const int64_t at = (int64_t)block * kBlockBytes + 16 * threadIdx.x;
    uint8_t* pool = a.pool[blockIdx.z];
    const uint8_t* src = pool + ((int64_t)a.src[blockIdx.y] * Hkv + head) * run_bytes;
    uint8_t* dst = pool + ((int64_t)a.dst[blockIdx.y] * Hkv + head) * run_bytes;
    if ((int64_t)(block + 1) * kBlockBytes <= bytes) {  // all loads issued before the first store
        u32x4_v x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const u32x4_v*>(src + at + i * 4096);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4_v*>(dst + at + i * 4096) = x[i];
        return;
    }
    for (int i = 0; i < 4; ++i)
        if (at + i * 4096 < bytes)
            *reinterpret_cast<u32x4_v*>(dst + at + i * 4096) = *reinterpret_cast<const u32x4_v*>(src + at + i * 4096);
}

}  // namespace
}  // namespace crane

using namespace crane;

extern "C" int crane_hip_copy_pages(void* const* pools, int n_pools, int64_t n_pages, int page_rows, int Hkv, int D,
                                    const int32_t* src, const int32_t* dst, const int32_t* rows, int n, int dtype,
                                    void* stream) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (n_pools < 0 || n < 0 || Hkv <= 0 || Hkv > 65535) return CRANE_HIP_E_INVALID;
    int32_t dummy = 0;  // no block table here; only the pool sizes are checked
    int rc = check_paged(n_pages, page_rows, &dummy, 1, Hkv);
    if (rc) return rc;
    if (n == 0 || n_pools == 0) return CRANE_HIP_OK;
    if (!pools || !src || !dst) return CRANE_HIP_E_INVALID;
    for (int i = 0; i < n_pools; ++i) {
        if (!pools[i]) return CRANE_HIP_E_INVALID;
        if (!aligned16(pools[i])) return CRANE_HIP_E_ALIGN;
    }
    int max_rows = 0;
    for (int i = 0; i < n; ++i) {
        const int r = rows ? rows[i] : page_rows;
        if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages || r < 0 || r > page_rows)
            return CRANE_HIP_E_INVALID;
        max_rows = std::max(max_rows, r);
    }
    try {
        std::vector<int32_t> to(dst, dst + n);
        std::sort(to.begin(), to.end());
        if (std::adjacent_find(to.begin(), to.end()) != to.end()) return CRANE_HIP_E_INVALID;
        for (int i = 0; i < n; ++i)
            if (std::binary_search(to.begin(), to.end(), src[i])) return CRANE_HIP_E_INVALID;
    } catch (...) {  // no memory for the check
        return CRANE_HIP_E_INVALID;
    }
    if (max_rows == 0) return CRANE_HIP_OK;
    const int row_bytes = kHeadDim * elem_size(dtype);
    const int64_t run = (int64_t)page_rows * row_bytes;
    const int64_t blocks = ((int64_t)max_rows * row_bytes + kBlockBytes - 1) / kBlockBytes;
    if (blocks * Hkv > 0x7fffffffLL) return CRANE_HIP_E_INVALID;
    CopyArgs a;
    for (int p0 = 0; p0 < n_pools; p0 += kPools) {
        const int np = n_pools - p0 < kPools ? n_pools - p0 : kPools;
        for (int i = 0; i < np; ++i) a.pool[i] = (uint8_t*)pools[p0 + i];
        for (int i0 = 0; i0 < n; i0 += kPairs) {
            const int ni = n - i0 < kPairs ? n - i0 : kPairs;
            for (int i = 0; i < ni; ++i) {
                a.src[i] = src[i0 + i];
                a.dst[i] = dst[i0 + i];
                a.rows[i] = rows ? rows[i0 + i] : page_rows;
            }
            hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(blocks * Hkv), (unsigned)ni, (unsigned)np), dim3(256),
                               0, (hipStream_t)stream, a, (int)blocks, Hkv, run, row_bytes);
            rc = launch_status(hipGetLastError());
            if (rc) return rc;
        }
    }
    return CRANE_HIP_OK;
}
