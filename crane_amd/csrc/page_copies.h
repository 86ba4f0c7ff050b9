// page_copies.h -- copies of rows between pages of pools (defined in pages.hip, used by
// crane_hip_copy_pages and the paged cache manager).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace crane {

// crane_hip_copy_pages for rows of `row_bytes`, a multiple of 8 (the pools' alignment is 16
// bytes where it is one of 16, else 8); it checks the pools and the lists, not the sizes.
int copy_page_rows(void* const* pools, int n_pools, int64_t n_pages, int page_rows, int Hkv, int row_bytes,
                   const int32_t* src, const int32_t* dst, const int32_t* rows, int n, hipStream_t stream);

}  // namespace crane
