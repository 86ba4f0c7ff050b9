// f8_cache.hip -- rows into and out of the paged KV cache in 8 bits (gfx950): the fused
// per-head QK-RMSNorm + RoPE append that quantises k and v as it writes them, and the
// read that gives values back.  The C ABI and the format are include/crane_f8.h's.
//
// The append is append.hip's pass over the merged qkv rows with 8 lanes to a head row
// (lane l holds dims [8l, 8l + 8) and [64 + 8l, + 8): the rotation is lane-local), in f32
// from the row to its one rounding.  q heads are independent items.  k and v need the
// largest magnitude of all new rows of a 32-row block before any of them can be written:
// a workgroup takes one block of one head, its 32 lane groups a row each, and holds the
// rows in registers between the maximum and the codes, so every row is read once and
// written once.  With one new token a block has one new row, and its lane group needs
// nobody: those items are independent again.
//
// A scale is a power of two.  Codes are floating point: scaling by 2^k moves their
// exponent and rounds nothing while they stay normal, so a block's common scale costs
// no precision (a value keeps its 4 significant bits down to 2^-14 of the block's
// largest), and a block whose scale grows later has its older codes moved exactly
// (subnormal ones aside).
#include "f8.h"

namespace crane {
namespace {

constexpr int kItems = 32;  // head rows of a 256-thread workgroup

// Sum and maximum over the 8 lanes of a row; every lane gets them.
__device__ __forceinline__ float group8_sum(float x) {
    x += dpp<0xB1>(x);   // quad_perm [1,0,3,2]
    x += dpp<0x4E>(x);   // quad_perm [2,3,0,1]
    x += dpp<0x141>(x);  // row_half_mirror
    return x;
}
__device__ __forceinline__ float group8_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));
    return x;
}

// 16 bytes past the caches.
typedef unsigned int u32x4_v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_streamed(float* p, const float (&x)[4]) {
    const u32x4_v w = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_v*>(p));
}
__device__ __forceinline__ void store_streamed(bf16_t* p, const float (&x)[8]) {
    const u32x4_v w = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                       pack_bf16x2(x[6], x[7])};
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_v*>(p));
}

// 8 elements, past the caches or not.
template <bool STREAM> __device__ __forceinline__ void take8(const bf16_t* p, float (&v)[8]) {
    if constexpr (!STREAM) return load8(p, v);
    const u32x4_v t = __builtin_nontemporal_load(reinterpret_cast<const u32x4_v*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(t[i]);
        v[2 * i + 1] = bf16_hi(t[i]);
    }
}
template <bool STREAM> __device__ __forceinline__ void take8(const float* p, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const u32x4_v* q = reinterpret_cast<const u32x4_v*>(p + 4 * h);
        const u32x4_v t = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = __uint_as_float(t[i]);
    }
}
template <bool STREAM> __device__ __forceinline__ void put8(bf16_t* p, const float (&v)[8]) {
    if constexpr (STREAM) store_streamed(p, v);
    else store8(p, v);
}
template <bool STREAM> __device__ __forceinline__ void put8(float* p, const float (&v)[8]) {
    if constexpr (!STREAM) return store8(p, v);
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    store_streamed(p, a);
    store_streamed(p + 4, b);
}

template <typename T> struct Append {
    const T* qkv;
    int64_t row_stride;
    const T *qw, *kw;
    float eps;
    int order;
    const T *cos, *sin;
    int64_t cs_stride, table_rows;
    const int32_t* positions;
    T* q_out;
    uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
    PagedRows rows;
    const int32_t* cache_len;   // null: 0 for every sequence
    const T *k_rows, *v_rows;   // [B, Hkv, S, D] as they are to be quantised, in place of qkv
    int S, Hq, Hkv;
    int64_t q_items, q_blocks;  // q head rows, and the workgroups that take them
    int64_t units;              // blocks mode: (sequence, block, k or v head)
    int blocks;                 // blocks mode: blocks a sequence's S rows can touch
};

// A lane's 16 values of a head row, normed and rotated in f32.
struct RowValues {
    float a[8], b[8];  // dims 8l .., 64 + 8l ..
};

template <typename T>
__device__ __forceinline__ void norm(RowValues& x, const float (&w1)[8], const float (&w2)[8], float eps) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        ss = __builtin_fmaf(x.a[i], x.a[i], ss);
        ss = __builtin_fmaf(x.b[i], x.b[i], ss);
    }
    const float r = 1.0f / sqrtf(group8_sum(ss) * (1.0f / kHeadDim) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x.a[i] = x.a[i] * r * w1[i];
        x.b[i] = x.b[i] * r * w2[i];
    }
}

template <typename T>
__device__ __forceinline__ void norm_rope(RowValues& x, const Append<T>& p, const T* w, int64_t pos, int l) {
    float c[8], s[8], w1[8], w2[8];
    load8(p.cos + pos * p.cs_stride + 8 * l, c);
    load8(p.sin + pos * p.cs_stride + 8 * l, s);
    if (w) {
        load8(w + 8 * l, w1);
        load8(w + 64 + 8 * l, w2);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w1[i] = w2[i] = 1.f;
    }
    if (p.order == CRANE_HIP_NORM_THEN_ROPE) norm<T>(x, w1, w2, p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float u = x.a[i], v = x.b[i];
        x.a[i] = u * c[i] - v * s[i];
        x.b[i] = u * s[i] + v * c[i];
    }
    if (p.order == CRANE_HIP_ROPE_THEN_NORM) norm<T>(x, w1, w2, p.eps);
}

template <bool STREAM, typename T>
__device__ __forceinline__ void load_row(RowValues& x, const Append<T>& p, int64_t tok, int head, int l) {
    const T* src = p.qkv + tok * p.row_stride + (int64_t)head * kHeadDim;
    take8<STREAM>(src + 8 * l, x.a);
    take8<STREAM>(src + 64 + 8 * l, x.b);
}

// The largest finite magnitude of a lane's values, 0 or more.
__device__ __forceinline__ float largest(const RowValues& x) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x.a[i]), b = fabsf(x.b[i]);
        m = fmaxf(m, fmaxf(a < INFINITY ? a : 0.f, b < INFINITY ? b : 0.f));
    }
    return m;
}

// Rounding to 4 bits takes magnitudes past 1.9375 2^127 to 2^128, which no type holds: under
// scales that reach that far finite values stop at the largest code below it, 1.875 2^127.
constexpr float kMostValue = 0x1.ep127f;
constexpr int kLargeScale = 247;  // 448 times the next smaller scale is finite
__device__ __forceinline__ void hold_finite(float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (fabsf(x[i]) < INFINITY) x[i] = fminf(fmaxf(x[i], -kMostValue), kMostValue);
}
__device__ __forceinline__ void store_codes(uint8_t* row, RowValues& x, int byte, int l) {
    if (byte >= kLargeScale) {
        hold_finite(x.a);
        hold_finite(x.b);
    }
    const float inv = inverse_scale(byte);
    *reinterpret_cast<uint2*>(row + 8 * l) = codes8(x.a, inv);
    *reinterpret_cast<uint2*>(row + 64 + 8 * l) = codes8(x.b, inv);
}

template <bool STREAM, typename T> __device__ __forceinline__ void q_item(const Append<T>& p, int64_t item, int l) {
    if (item >= p.q_items) return;  // whole 8-lane groups leave together
    const int head = (int)(item % p.Hq);
    const int64_t tok = item / p.Hq;
    const int s = (int)(tok % p.S), b = (int)(tok / p.S);
    const int64_t pos = (int64_t)p.positions[b] + s;
    RowValues x;
    load_row<STREAM>(x, p, tok, head, l);
    if (pos < 0 || pos >= p.table_rows) return;
    norm_rope(x, p, p.qw, pos, l);
    T* dst = p.q_out + (((int64_t)b * p.Hq + head) * p.S + s) * kHeadDim;
    put8<STREAM>(dst + 8 * l, x.a);
    put8<STREAM>(dst + 64 + 8 * l, x.b);
}

// S = 1: every head row is an item of 8 lanes (1 sequence 3.6 us, 4.2 through the blocks
// kernel, whose workgroups hold 31 idle rows; 32 sequences at 32 / 8 heads 3.7 for 4.8: a
// launch, and the rows' latency).  grid: q items, then k and v items.
template <typename T> __global__ __launch_bounds__(256) void f8_append_token_kernel(Append<T> p) {
    const int l = threadIdx.x & 7;
    if ((int64_t)blockIdx.x < p.q_blocks) return q_item<false>(p, (int64_t)blockIdx.x * kItems + (threadIdx.x >> 3), l);
    const int64_t item = ((int64_t)blockIdx.x - p.q_blocks) * kItems + (threadIdx.x >> 3);
    if (item >= p.units) return;
    const int hh = (int)(item % (2 * p.Hkv)), b = (int)(item / (2 * p.Hkv));
    const bool is_v = hh >= p.Hkv;
    const int h = is_v ? hh - p.Hkv : hh;
    const int64_t j = p.cache_len[b], pos = p.positions[b];
    RowValues x;
    load_row<false>(x, p, b, p.Hq + hh, l);
    const int64_t off = p.rows.offset(b, p.Hkv, h, j);
    if (off < 0) return;
    const int64_t at = off / kHeadDim / kBlockRows8;
    uint8_t* scale = (is_v ? p.v_scale : p.k_scale) + at;
    uint8_t* block = (is_v ? p.v_pool : p.k_pool) + at * kBlockRows8 * kHeadDim;
    const int held = (int)(j % kBlockRows8);
    if (!is_v) {
        if (pos < 0 || pos >= p.table_rows) {
            // the rows that come after it in the block keep to its scale
            if (l == 0 && !held) *scale = kLeastScale;
            return;
        }
        norm_rope(x, p, p.kw, pos, l);
    }
    const int need = scale_byte(group8_max(largest(x)));
    const int had = held ? *scale : 0, byte = max(need, had);
    if (byte > had && held) {
        const float down = scale_of(max(127 + had - byte, 0));
        uint4* old = reinterpret_cast<uint4*>(block) + l;
#pragma unroll 4
        for (int r = 0; r < held; ++r) {
            uint4 w = old[8 * r];
            w = make_uint4(recode4(w.x, down), recode4(w.y, down), recode4(w.z, down), recode4(w.w, down));
            old[8 * r] = w;
        }
    }
    store_codes(block + held * kHeadDim, x, byte, l);
    if (l == 0 && byte != had) *scale = (uint8_t)byte;
}

// Any S.  ROWS: k_rows and v_rows in place of qkv's.  The rows and q, each touched once, go
// past the caches: 8 prompts of 4096 tokens, 28 / 4 heads (302 MB read, 268 MB written) 105
// us to 98, 5.8 TB/s: the memory is the bound (a large copy reaches 5.2).  grid: q items,
// then one workgroup per (sequence, block, k or v head).
template <typename T, bool ROWS> __global__ __launch_bounds__(256) void f8_append_blocks_kernel(Append<T> p) {
    const int l = threadIdx.x & 7, r = threadIdx.x >> 3;
    if ((int64_t)blockIdx.x < p.q_blocks) return q_item<true>(p, (int64_t)blockIdx.x * kItems + r, l);
    const int64_t unit = (int64_t)blockIdx.x - p.q_blocks;
    const int hh = (int)(unit % (2 * p.Hkv));
    const int64_t x0 = unit / (2 * p.Hkv);
    const int b = (int)(x0 / p.blocks);
    const bool is_v = hh >= p.Hkv;
    const int h = is_v ? hh - p.Hkv : hh;
    const int64_t len = ROWS && !p.cache_len ? 0 : p.cache_len[b];
    const int64_t first = (len & ~(int64_t)(kBlockRows8 - 1)) + (x0 % p.blocks) * kBlockRows8;
    if (first >= len + p.S) return;  // the sequence's rows end before
    const int64_t off = p.rows.offset(b, p.Hkv, h, first);
    if (off < 0) return;
    const int64_t s = first + r - len;
    const bool old = s < 0;
    bool fresh = !old && s < p.S;
    RowValues x;
    if (ROWS && fresh) {
        const T* src = (is_v ? p.v_rows : p.k_rows) + (((int64_t)b * p.Hkv + h) * p.S + s) * kHeadDim;
        take8<true>(src + 8 * l, x.a);
        take8<true>(src + 64 + 8 * l, x.b);
    } else if (fresh) {
        load_row<true>(x, p, (int64_t)b * p.S + s, p.Hq + hh, l);
        if (!is_v) {
            const int64_t pos = (int64_t)p.positions[b] + s;
            fresh = pos >= 0 && pos < p.table_rows;
            if (fresh) norm_rope(x, p, p.kw, pos, l);
        }
    }
    __shared__ float most[4];
    const float m = wave_max(fresh ? largest(x) : -1.f);
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
    const float amax = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    const int64_t at = off / kHeadDim / kBlockRows8;
    uint8_t* scale = (is_v ? p.v_scale : p.k_scale) + at;
    if (amax < 0.f) {  // no row is written: a block that begins with them gets a scale all the same
        if (first >= len && threadIdx.x == 0) *scale = kLeastScale;
        return;
    }
    uint8_t* row = (is_v ? p.v_pool : p.k_pool) + off + r * kHeadDim;
    const int had = first < len ? *scale : 0, byte = max(scale_byte(amax), had);
    if (fresh) store_codes(row, x, byte, l);
    if (old && byte > had) {
        const float down = scale_of(max(127 + had - byte, 0));
        uint4* w = reinterpret_cast<uint4*>(row) + l;
        const uint4 c = *w;
        *w = make_uint4(recode4(c.x, down), recode4(c.y, down), recode4(c.z, down), recode4(c.w, down));
    }
    __syncthreads();  // every wave has read the old scale
    if (threadIdx.x == 0) *scale = (uint8_t)byte;
}

template <typename T> int launch_append(Append<T> p, int B, hipStream_t st) {
    p.q_items = (int64_t)B * p.S * p.Hq;
    p.q_blocks = (p.q_items + kItems - 1) / kItems;
    // S rows from any row of a block on touch at most this many blocks
    p.blocks = (int)(((int64_t)p.S + 2 * kBlockRows8 - 2) / kBlockRows8);
    p.units = (int64_t)B * 2 * p.Hkv * (p.S == 1 ? 1 : p.blocks);
    const int64_t grid = p.q_blocks + (p.S == 1 ? (p.units + kItems - 1) / kItems : p.units);
    if (grid > 0xffffffffLL / 256) return CRANE_HIP_E_INVALID;  // a grid's threads: 32 bits
    if (p.S == 1)
        hipLaunchKernelGGL(f8_append_token_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((f8_append_blocks_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, st, p);
    return launch_status(hipGetLastError());
}

template <typename T> int launch_rows(Append<T> p, int B, hipStream_t st) {
    p.units = f8_rows_units(B, p.S, p.Hkv);
    p.blocks = (int)(p.units / ((int64_t)B * 2 * p.Hkv));
    hipLaunchKernelGGL((f8_append_blocks_kernel<T, true>), dim3((unsigned)p.units), dim3(256), 0, st, p);
    return launch_status(hipGetLastError());
}

// Codes to values.  A workgroup takes 64 rows of a head (two blocks, within one page), a
// thread 16 bytes of values at a time, so that a wave's stores are whole lines side by
// side; all its loads are issued before the first store.  The stores go past the caches.
// 16 sequences of 512 to 4096 rows, 8 heads, to bf16 (347 MB): 48 us, 7.2 TB/s (8-byte
// stores through the caches 75); one of 333 to f32: 4.1, a launch and two dependent loads.
// grid: (row tiles of all heads, k and v)
constexpr int kReadRows = 2 * kBlockRows8;
template <typename T>
__global__ __launch_bounds__(256) void f8_read_kernel(const uint8_t* __restrict__ k_pool,
                                                      const uint8_t* __restrict__ v_pool,
                                                      const uint8_t* __restrict__ k_scale,
                                                      const uint8_t* __restrict__ v_scale, PagedRows rows,
                                                      const int32_t* __restrict__ kv_len, int64_t max_kv, int Hkv,
                                                      T* __restrict__ k_out, T* __restrict__ v_out, int tiles) {
    constexpr int kN = 16 / sizeof(T);                         // codes of a load
    constexpr int kPerRow = kHeadDim / kN, kLoads = kReadRows * kPerRow / 256;
    constexpr int kStep = 256 / kPerRow;                       // rows between a thread's loads
    const int bh = blockIdx.x / tiles, j0 = (blockIdx.x - bh * tiles) * kReadRows;
    const int b = bh / Hkv, h = bh - b * Hkv;
    const int r0 = threadIdx.x / kPerRow, c = kN * (threadIdx.x % kPerRow);
    const uint8_t *pool = blockIdx.y ? v_pool : k_pool, *scales = blockIdx.y ? v_scale : k_scale;
    const int64_t len = kv_len[b], off = j0 < len ? rows.offset(b, Hkv, h, j0) : -1;
    const int n = off < 0 ? 0 : (int)min((int64_t)kReadRows, len - j0);  // rows of the tile that have values
    const int out_rows = (int)min((int64_t)kReadRows, max_kv - j0);
    uint32_t w[kLoads][kN / 4];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = r0 + kStep * i;
#pragma unroll
        for (int x = 0; x < kN / 4; ++x)
            w[i][x] = r < n ? reinterpret_cast<const uint32_t*>(pool + off + r * kHeadDim + c)[x] : 0u;
    }
    float scale[2] = {0.f, 0.f};
    if (n > 0) {
        const uint8_t* s = scales + off / (kHeadDim * kBlockRows8);
        scale[0] = scale_of(s[0]);
        scale[1] = n > kBlockRows8 ? scale_of(s[1]) : 0.f;
    }
    T* out = (blockIdx.y ? v_out : k_out) + ((int64_t)bh * max_kv + j0) * kHeadDim + c;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = r0 + kStep * i;
        float x[kN];
#pragma unroll
        for (int y = 0; y < kN / 4; ++y) values4(w[i][y], x + 4 * y);
#pragma unroll
        for (int y = 0; y < kN; ++y) x[y] *= scale[r / kBlockRows8];
        if (r < out_rows) store_streamed(out + r * kHeadDim, x);
    }
}

}  // namespace

int f8_write_rows(const void* k, const void* v, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                  const PagedRows& rows, const int32_t* start, int B, int64_t S, int Hkv, int dtype, hipStream_t st) {
    if (S > 0x7fffffffLL || f8_rows_units(B, S, Hkv) > kMostUnits8) return CRANE_HIP_E_INVALID;
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        Append<T> p{};
        p.k_rows = (const T*)k;
        p.v_rows = (const T*)v;
        p.k_pool = (uint8_t*)k_pool;
        p.v_pool = (uint8_t*)v_pool;
        p.k_scale = (uint8_t*)k_scale;
        p.v_scale = (uint8_t*)v_scale;
        p.rows = rows;
        p.cache_len = start;
        p.S = (int)S;
        p.Hkv = Hkv;
        return launch_rows(p, B, st);
    };
    return dtype == CRANE_HIP_F32 ? go(float()) : go(bf16_t());
}

}  // namespace crane

using namespace crane;

extern "C" int crane_hip_qknorm_rope_append_paged_f8(const void* qkv, int64_t qkv_row_stride, const void* q_norm_w,
                                                     const void* k_norm_w, float eps, int order, const void* cos,
                                                     const void* sin, int64_t cs_stride, int64_t table_rows,
                                                     const int32_t* positions, void* q_out, void* k_pool, void* v_pool,
                                                     void* k_scale, void* v_scale, int64_t n_pages, int page_rows,
                                                     const int32_t* block_table, int64_t table_stride,
                                                     const int32_t* cache_len, int B, int S, int Hq, int Hkv, int D,
                                                     int dtype, void* stream) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return CRANE_HIP_E_INVALID;
    if (Hq % Hkv != 0) return CRANE_HIP_E_GQA;
    if (order < CRANE_HIP_NORM_THEN_ROPE || order > CRANE_HIP_ROPE_ONLY) return CRANE_HIP_E_INVALID;
    if (!(eps >= 0.0f)) return CRANE_HIP_E_INVALID;
    int rc = check_paged(n_pages, page_rows, block_table, table_stride, Hkv);
    if (rc) return rc;
    if ((int64_t)S > table_stride * page_rows) return CRANE_HIP_E_CAPACITY;
    if (B == 0 || S == 0) return CRANE_HIP_OK;
    if (!qkv || !cos || !sin || !positions || !q_out || !cache_len) return CRANE_HIP_E_INVALID;
    if ((rc = check_pools8(k_pool, v_pool, k_scale, v_scale))) return rc;
    if (cs_stride < D / 2 || table_rows <= 0) return CRANE_HIP_E_INVALID;
    if (qkv_row_stride < ((int64_t)Hq + 2 * (int64_t)Hkv) * D) return CRANE_HIP_E_INVALID;
    const int64_t per16 = dtype == CRANE_HIP_BF16 ? 8 : 4;  // elements per 16 bytes
    if (qkv_row_stride % per16 != 0 || cs_stride % per16 != 0) return CRANE_HIP_E_ALIGN;
    if (!aligned16(qkv) || !aligned16(cos) || !aligned16(sin) || !aligned16(q_out) ||
        (q_norm_w && !aligned16(q_norm_w)) || (k_norm_w && !aligned16(k_norm_w)))
        return CRANE_HIP_E_ALIGN;
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        Append<T> p{};
        p.qkv = (const T*)qkv;
        p.row_stride = qkv_row_stride;
        p.qw = (const T*)q_norm_w;
        p.kw = (const T*)k_norm_w;
        p.eps = eps;
        p.order = order;
        p.cos = (const T*)cos;
        p.sin = (const T*)sin;
        p.cs_stride = cs_stride;
        p.table_rows = table_rows;
        p.positions = positions;
        p.q_out = (T*)q_out;
        p.k_pool = (uint8_t*)k_pool;
        p.v_pool = (uint8_t*)v_pool;
        p.k_scale = (uint8_t*)k_scale;
        p.v_scale = (uint8_t*)v_scale;
        p.rows = PagedRows{block_table, table_stride, n_pages, page_rows};
        p.cache_len = cache_len;
        p.S = S;
        p.Hq = Hq;
        p.Hkv = Hkv;
        return launch_append(p, B, (hipStream_t)stream);
    };
    return dtype == CRANE_HIP_F32 ? go(float()) : go(bf16_t());
}

extern "C" int crane_hip_read_paged_f8(const void* k_pool, const void* v_pool, const void* k_scale,
                                       const void* v_scale, int64_t n_pages, int page_rows,
                                       const int32_t* block_table, int64_t table_stride, const int32_t* kv_len,
                                       int64_t max_kv, int B, int Hkv, int D, void* k_out, void* v_out, int dtype,
                                       void* stream) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (B < 0 || Hkv <= 0 || max_kv < 0) return CRANE_HIP_E_INVALID;
    int rc = check_paged(n_pages, page_rows, block_table, table_stride, Hkv);
    if (rc) return rc;
    if (max_kv > table_stride * page_rows) return CRANE_HIP_E_CAPACITY;
    if (B == 0 || max_kv == 0) return CRANE_HIP_OK;
    if (!kv_len || !k_out || !v_out) return CRANE_HIP_E_INVALID;
    if ((rc = check_pools8(k_pool, v_pool, k_scale, v_scale))) return rc;
    if (!aligned16(k_out) || !aligned16(v_out)) return CRANE_HIP_E_ALIGN;
    const int64_t heads = (int64_t)B * Hkv, tiles = (max_kv + kReadRows - 1) / kReadRows;
    if (heads > 0xffffffLL || tiles > 0xffffffLL / heads) return CRANE_HIP_E_INVALID;  // a grid's threads: 32 bits
    const dim3 grid((unsigned)(heads * tiles), 2);
    const PagedRows rows{block_table, table_stride, n_pages, page_rows};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == CRANE_HIP_F32)
        hipLaunchKernelGGL(f8_read_kernel<float>, grid, dim3(256), 0, st, (const uint8_t*)k_pool,
                           (const uint8_t*)v_pool, (const uint8_t*)k_scale, (const uint8_t*)v_scale, rows, kv_len,
                           max_kv, Hkv, (float*)k_out, (float*)v_out, (int)tiles);
    else
        hipLaunchKernelGGL(f8_read_kernel<bf16_t>, grid, dim3(256), 0, st, (const uint8_t*)k_pool,
                           (const uint8_t*)v_pool, (const uint8_t*)k_scale, (const uint8_t*)v_scale, rows, kv_len,
                           max_kv, Hkv, (bf16_t*)k_out, (bf16_t*)v_out, (int)tiles);
    return launch_status(hipGetLastError());
}
