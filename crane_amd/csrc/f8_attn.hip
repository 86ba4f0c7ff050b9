// f8_attn.hip -- attention over the paged KV cache in 8 bits (gfx950); the C ABI and the
// cache's format are include/crane_f8.h's.
//
// Query i of sequence b sees rows [0, L), L = kv_len[b] - S + 1 + i (causal) or kv_len[b].
// With s_j = scale q . k_j over any set of keys,
//     m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j,
// and disjoint sets join as o = sum w o' / sum w l', w = exp(m' - max m).  The rows of a
// workgroup are (query, head of the GQA group) of one sequence and kv head, which share
// every key they read.
//
// A code times its power-of-two scale has 4 significant bits, so bf16 holds it exactly,
// and one v_cvt_scalef32_pk_bf16_fp8 makes two of them, scale included.  The products run
// on bf16 MFMAs, whose sums are f32's: 8-bit MFMAs would take K and V as they are at twice
// the rate, but q and the probabilities would need two 8-bit parts each (the same time),
// and they align the products of a sum to its largest and cut them at about 2^-13 of
// it (measured: 64 products of mixed magnitudes off by up to 2^-12 of the largest, bf16
// 2^-22).  bf16 calls round the probabilities to bf16; f32 calls split q and the
// probabilities into three bf16 parts, 24 bits in all, and take three products.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "attn_lanes.h"
#include "f8.h"
#include "shared_plan.h"

namespace crane {
namespace {

constexpr float kNoMax = -FLT_MAX;  // m before the first key (finite: exp2(-inf - m) is 0, not NaN)
constexpr float kSlack = 16.f, kMostMax = 0x1p26f;  // see Rows8
// What the rounding of mc = m c leaves of it (0 where nobody counts from mc, see Rows8).
__device__ __forceinline__ float left_of(float m, float mc, float c) {
    return fabsf(mc) <= kMostMax ? __builtin_fmaf(m, c, -mc) : 0.f;
}
constexpr int kTile = 64;           // keys of a tile: two blocks, within one page
constexpr int kRow = kHeadDim;      // bytes of a row of codes
constexpr int kTileBytes = kTile * kRow;

struct Args8 {
    const void* q;
    const uint8_t *k, *v, *k_scale, *v_scale;
    void* out;
    PagedRows rows;
    const int32_t* kv_len;
    int B, S, Hq, Hkv, G;  // G = Hq / Hkv heads per kv head
    int max_kv, causal;
    float c;               // scale log2 e
    int tiles;             // row tiles of a (sequence, kv head)
    int pairs;             // (sequence, chunk) pairs there may be; 0: every sequence is one chunk
    int tile_rows;         // query rows of a tile
    float* ws_o;           // [pairs, Hkv, tiles, tile_rows, D], unnormalised
    float2* ws_ml;         // [pairs, Hkv, tiles, tile_rows] (m, l)
    int4* ws_cut;          // [B] a sequence's chunks, the pair of its second one, rows of a chunk
    __device__ __forceinline__ int len(int b) const { return max(0, min(kv_len[b], max_kv)); }
    // Rows query s of a sequence of n rows sees.
    __device__ __forceinline__ int limit(int n, int s) const { return causal ? n - S + 1 + s : n; }
    // Where the partial results of a tile's row are (in rows of ws_o).
    __device__ __forceinline__ int64_t slot(int pair, int kvh, int tile, int row) const {
        return (((int64_t)pair * Hkv + kvh) * tiles + tile) * tile_rows + row;
    }
    // The row of out [B, S, Hq] that is row `at` of q [B, Hq, S].
    __device__ __forceinline__ int64_t out_row(int at) const {
        if (S == 1) return at;
        const int bh = at / S, s = at - bh * S, b = bh / Hq;
        return ((int64_t)b * S + s) * Hq + (bh - b * Hq);
    }
};

// The sequences' chunks.  All are cut into chunks of the same number of tiles, few enough
// of them that there are no more than `pairs` in all: as many workgroups as the device
// holds at once, whatever the lengths (and however far above them max_kv is, as in a
// captured graph).  Every wave works it out from kv_len, lane x holding sequences x, 64 +
// x, ...  Pair b < B is the first chunk of sequence b, which needs nothing of this to start;
// the others follow, sequence by sequence.
struct Cut {
    int b, chunk;  // a pair's; b = -1 past the last
    int n, rest;   // the sequence's chunks, and the pair of its second one
    int tiles;     // tiles of a chunk
    int len;       // the sequence's rows
    __device__ __forceinline__ int pair(int c) const { return c == 0 ? b : rest + c - 1; }
};
constexpr int kMostCut = 256;   // sequences of a batch that is cut
constexpr int kLeastChunk = 4;  // tiles: every wave of a workgroup has one
// Inclusive sums over the wave's lanes.
__device__ __forceinline__ float wave_scan(float x) {
    x += dpp<0x111>(x);  // row_shr:1
    x += dpp<0x112>(x);
    x += dpp<0x114>(x);
    x += dpp<0x118>(x);
    x += dpp_rows<0x142, 0xa>(x, 0.f);  // row_bcast:15 into rows 1, 3
    x += dpp_rows<0x143, 0xc>(x, 0.f);  // row_bcast:31 into rows 2, 3
    return x;
}
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// ceil(x / d) for x < 2^26 and a quotient below 2^20, r about 1 / d.
__device__ __forceinline__ int ceil_by(int x, int d, float r) {
    int q = (int)((float)x * r);
    q -= q * d > x ? 1 : 0;
    q += (q + 1) * d <= x ? 1 : 0;
    return q + (q * d < x ? 1 : 0);
}
struct Lengths {
    static constexpr int kN = kMostCut / 64;
    int of[kN];
    __device__ __forceinline__ void load(const Args8& a, int lane) {
#pragma unroll
        for (int i = 0; i < kN; ++i) of[i] = 64 * i + lane < a.B ? a.kv_len[64 * i + lane] : 0;
    }
};
__device__ __forceinline__ Cut cut_at(const Args8& a, const Lengths& raw, int pair, int lane) {
    constexpr int kN = Lengths::kN;
    int len[kN], t[kN];
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        len[i] = max(0, min(raw.of[i], a.max_kv));
        t[i] = 64 * i + lane < a.B ? max(1, (len[i] + kTile - 1) / kTile) : 0;
        total += (float)t[i];
    }
    total = wave_sum(total);
    // About half a chunk of every sequence is not filled: start there, and go on until all fit,
    // which is so at the longest sequence's tiles, at the latest.
    const float pairs = (float)a.pairs;
    int c = max(kLeastChunk, (int)(total * __builtin_amdgcn_rcpf(pairs - 0.5f * (float)a.B)));
    float r;
    for (;;) {
        r = __builtin_amdgcn_rcpf((float)c);
        float f = 0.f;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (64 * i < a.B) f += (float)ceil_by(t[i], c, r);
        f = wave_sum(f);
        if (f <= pairs) break;
        c = max(c + 1, (int)((float)c * f * __builtin_amdgcn_rcpf(pairs)));
    }
    Cut x{-1, 0, 0, 0, c, 0};
    float before = (float)a.B;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        if (64 * i >= a.B || x.b >= 0) continue;
        const float n = (float)ceil_by(t[i], c, r), upto = before + wave_scan(n - (64 * i + lane < a.B ? 1.f : 0.f));
        const uint64_t mine = __ballot(pair < a.B ? 64 * i + lane == pair : (float)pair < upto);
        if (mine) {
            const int at = __builtin_ctzll(mine);
            x.b = 64 * i + at;
            x.n = (int)lane_value(n, at);
            x.rest = (int)lane_value(upto, at) - (x.n - 1);
            x.chunk = pair < a.B ? 0 : pair - x.rest + 1;
            x.len = __builtin_amdgcn_readlane(len[i], at);
        }
        before = lane_value(upto, 63);
    }
    return x;
}

// Pages of a sequence, one id per lane: 64 from `page0` on (all of the table's row where it
// has no more: then the first load waits for nothing).
struct Pages8 {
    const int32_t* row;
    int stride, ids, page0, P, lane;
    __device__ __forceinline__ Pages8(const Args8& a, int ln)
        : stride((int)a.rows.stride), P(a.rows.page_rows), lane(ln) {}
    __device__ __forceinline__ void open(const Args8& a, int b, int begin) {
        row = a.rows.table + (int64_t)b * a.rows.stride;
        load(stride <= 64 ? 0 : begin / P);
    }
    __device__ __forceinline__ void load(int from) {
        page0 = from;
        ids = page0 + lane < stride ? row[page0 + lane] : -1;
    }
    // The tile of keys [j, j + 64) of a kv head: its offset in a pool and the bytes of its rows
    // before `end` (0 for a page outside the pool: its rows read as zero).  j never falls.
    struct Tile {
        int64_t off;
        int bytes;
    };
    __device__ __forceinline__ Tile tile(const Args8& a, int kvh, int j, int end) {
        const int p = j / P;
        if (p - page0 >= 64) load(p);
        const int id = __builtin_amdgcn_readlane(ids, p - page0);
        const bool ok = (unsigned)id < (unsigned)a.rows.n_pages;
        const int rows = ok ? max(0, min(kTile, end - j)) : 0;
        const int64_t off = (((int64_t)(ok ? id : 0) * a.Hkv + kvh) * P + (j - p * P)) * kRow;
        return Tile{uniform(off), __builtin_amdgcn_readfirstlane(rows * kRow)};
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint8_t* pool, const Pages8::Tile& t) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(pool) + t.off, (short)0, t.bytes, 0x00020000);
}

// The scales of a tile's two blocks, as f32.  A byte of a block without rows may be
// anything; 254 keeps 0 times it 0.
struct Scales {
    float of[2];
    // The first of them among the pool's: even.
    static __device__ __forceinline__ int64_t at(int64_t tile_off) { return tile_off / (kRow * kBlockRows8); }
    // From the aligned word that they are in.
    __device__ __forceinline__ void set(uint32_t word, int64_t tile_off) {
        const uint32_t w = word >> (8 * (at(tile_off) & 2));
        of[0] = scale_of(min(w & 255u, 254u));
        of[1] = scale_of(min((w >> 8) & 255u, 254u));
    }
    // That word: by one scalar load (through the constant address space) ...
    __device__ __forceinline__ void load(const uint8_t* pool, int64_t tile_off) {
        typedef const __attribute__((address_space(4))) uint32_t* words_t;
        set(((words_t)(uintptr_t)pool)[at(tile_off) >> 2], tile_off);
    }
    // ... or by a vector load, for later.
    static __device__ __forceinline__ uint32_t fetch(const uint8_t* pool, int64_t tile_off) {
        const uint8_t* from = pool + (at(tile_off) & ~(int64_t)3);
        return __builtin_amdgcn_raw_buffer_load_b32(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from), (short)0, 4, 0x00020000), 0, 0, 0);
    }
};

// Eight codes to bf16, times a scale.
__device__ __forceinline__ u32x4_v widen(uint32_t lo, uint32_t hi, float scale) {
    u32x4_v r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return r;
}
// Not 0 where one of four codes is a NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ f32x4_v mfma(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                   0, 0, 0);
}

__device__ __forceinline__ f32x16_v mfma(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                   0, 0, 0);
}

// Eight values as an MFMA operand: bf16 calls round them once, f32 calls carry them in
// three parts, each the rounding of what the ones before leave.
//
// The weights of bf16 calls in one part: results are 0.0017 to 0.0023 off (relative, in the
// norm; 0.00166 is the rounding of the results themselves), against values that a cache in 8
// bits holds to 0.026.  A second part reaches 0.00166 and is a product, two subtractions and
// a conversion more: 8 sequences of 32768 rows 86.3 us to 87.2, 32 of up to 4096 33.4 to
// 34.6, 5 drafted tokens of 16 28.2 to 30.2, 1 of 300 6.2 to 6.7, 1024 tokens of 4 prompts
// over 5000 to 9000 keys 405 to 562.  The sum that divides is of the weights as they are
// rounded, so that what a rounding moves all weights by goes out again.
template <typename T> struct Parts;
template <> struct Parts<bf16_t> {
    static constexpr int kN = 1;
    u32x4_v part[1];
    __device__ __forceinline__ void set(const float* x) {
#pragma unroll
        for (int w = 0; w < 4; ++w) part[0][w] = pack_bf16x2(x[2 * w], x[2 * w + 1]);
    }
    __device__ __forceinline__ void load(const bf16_t* p) { part[0] = *reinterpret_cast<const u32x4_v*>(p); }
};
template <> struct Parts<float> {
    static constexpr int kN = 3;
    u32x4_v part[3];  // the smallest last
    __device__ __forceinline__ void set(const float* x) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float a = x[2 * w], b = x[2 * w + 1];
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const uint32_t u = pack_bf16x2(a, b);
                part[n][w] = u;
                // an infinity leaves a NaN, which the products would make of it anyway
                a -= bf16_lo(u);
                b -= bf16_hi(u);
            }
        }
    }
    __device__ __forceinline__ void load(const float* p) {
        float x[8];
        load8(p, x);
        set(x);
    }
};
// c += a b, the smallest parts first.
template <typename T, typename C> __device__ __forceinline__ C product(u32x4_v a, const Parts<T>& b, C c) {
#pragma unroll
    for (int n = Parts<T>::kN - 1; n >= 0; --n) c = mfma(a, b.part[n], c);
    return c;
}
__device__ __forceinline__ u32x4_v ones() { return u32x4_v{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}; }

typedef int i32x2_v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_v lds_i32x2_v;
// Within 16 lanes, lane x gets column x of the 8 rows x 16 columns of bytes that the lanes
// point at (lane x: 8 columns from 8 (x % 2) on of row x / 2).
__device__ __forceinline__ uint2 lds_read_tr8(uint32_t at) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_v*)(uintptr_t)at));
}

// Wait for the wave's vector memory (or LDS) operations; the other counters at their
// maxima.
__device__ __forceinline__ void wait_memory() { __builtin_amdgcn_s_waitcnt(0x0F70); }
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// A tile of K or V in LDS keeps the pools' rows (128 bytes, half a sweep of the banks) with
// their 16-byte chunks XOR-permuted by permute8(row), so that neither the 16 rows of a K
// read nor the 16 rows of two lane groups' transposed V reads meet in a bank.
//
// v_mfma_f32_16x16x32_bf16, S^T = K Q^T with K rows as A: lane (i, g) = (lane % 16, lane /
// 16) holds, for query row i, rows 4 g + r of the product.  A's row x of product (u, b) is
// key 32 u + 8 (x / 4) + 4 b + x % 4, so that over b the lane holds keys 32 u + 8 g + (0 ..
// 7): as P^T, the B operand of O^T = V^T P^T as they stand, with V's bytes of those keys
// from one transposed read.
__device__ __forceinline__ int permute8(int row) {
    return ((row >> 1) & 1) | ((row >> 2) & 2) | ((((row >> 4) ^ (row >> 2)) & 1) << 2);
}
// The byte of a tile that instruction x of its copy (1 KiB, 8 rows) takes for a lane.
__device__ __forceinline__ int copy_from(int x, int lane) {
    const int row = 8 * x + (lane >> 3);
    return row * kRow + 16 * ((lane & 7) ^ permute8(row));
}
// A lane's reads of a tile that starts at k and v.
struct TileReads {
    uint32_t k, v;
    __device__ __forceinline__ TileReads(uint32_t k_lds, uint32_t v_lds, int lane) {
        const int i = lane & 15, g = lane >> 4, k_row = 8 * (i >> 2) + (i & 3), v_row = 8 * g + (i >> 1);
        k = k_lds + k_row * kRow + 16 * (g ^ permute8(k_row));
        v = v_lds + v_row * kRow + 16 * permute8(v_row) + 8 * (i & 1);
    }
    // Dims 64 half + 16 g .. of the key that is row i of product kt = 2 u + b (4 rows on, or 4
    // chunks, bit 2 of the chunk flips).
    __device__ __forceinline__ u32x4_v key(int kt, int half) const {
        return lds_read16((k ^ (((kt & 1) ^ half) << 6)) + 32 * (kt >> 1) * kRow + 4 * (kt & 1) * kRow);
    }
    // Keys 32 u + 8 g .. of dim 16 n + i.
    __device__ __forceinline__ uint2 value(int u, int n) const { return lds_read_tr8((v ^ (16 * n)) + 32 * u * kRow); }
};

// A wave's 16 RT query rows: their q and their running results.
template <typename T, int RT> struct Rows8 {
    const int i, g;
    Parts<T> q[RT][4];    // dims 16 g .., 16 g + 8 .., 64 + 16 g .., 64 + 16 g + 8 ..
    f32x4_v o[RT][8];     // dims 16 n + 4 g + r of row i
    f32x4_v l[RT];        // the sum over all keys, in all four
    float m[RT], mc[RT];  // the raw score p's exponent counts from, and m c rounded ..
    float left[RT];       // .. and what that leaves: weights are exp2((s - m) c + left)  (all 0 before the first key)
    float limit[RT];      // a score past this moves m
    bool big;             // some m c has lost bits below 1: its row's exponents are (s - m) c

    __device__ __forceinline__ explicit Rows8(int lane) : i(lane & 15), g(lane >> 4), big(false) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[t][n][r] = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) l[t][r] = 0.f;
            m[t] = limit[t] = kNoMax;
            mc[t] = left[t] = 0.f;
        }
    }
    // This lane's rows of those from row0 on: their places in q [B, Hq, S] (-1: none), the keys
    // they see (up to `end`), and q.
    __device__ __forceinline__ void open(const Args8& a, int b, int kvh, int row0, int n, int end, int (&at)[RT],
                                         int (&hi)[RT]) {
        const int R = a.S * a.G;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = row0 + 16 * t + i, s = min(r, R - 1) / a.G, h = min(r, R - 1) - s * a.G;
            at[t] = r < R ? (int)(((int64_t)b * a.Hq + kvh * a.G + h) * a.S + s) : -1;  // fewer than 2^31 query rows
            hi[t] = min(a.limit(n, s), end);
            const T* row = reinterpret_cast<const T*>(a.q) + (int64_t)max(at[t], 0) * kHeadDim;
#pragma unroll
            for (int step = 0; step < 4; ++step) q[t][step].load(row + 64 * (step >> 1) + 16 * g + 8 * (step & 1));
        }
    }
    // s[t][8 u + e]: the raw score of key 32 u + 8 g + e; key(kt, half) as TileReads::key.
    template <class KEY> __device__ __forceinline__ void scores(float (&s)[RT][16], const Scales& ks, KEY key) const {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            f32x4_v acc[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[t][r] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32x4_v w = key(kt, half);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const u32x4_v y = widen(w[2 * x], w[2 * x + 1], ks.of[kt >> 1]);
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[t] = product(y, q[t][2 * half + x], acc[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][4 * kt + r] = acc[t][r];
        }
    }
    // The scores, of keys from j on, that a row does not see vanish.
    __device__ __forceinline__ void mask(float (&s)[RT][16], int j, const int (&hi)[RT]) const {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                s[t][e] = j + 32 * (e >> 3) + 8 * g + (e & 7) < hi[t] ? s[t][e] : -INFINITY;
    }
    // m for these scores.  It moves, and o and l are scaled, only where a score passes it by
    // kSlack (as a power of two): f32 and bf16 hold larger weights as exactly.
    __device__ __forceinline__ void settle(const float (&s)[RT][16], float c) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float mx = s[t][0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
            if (__any(mx > limit[t])) {
                const float to = fmaxf(m[t], groups_max(mx)), was = left[t];
                mc[t] = to == kNoMax ? 0.f : to * c;
                left[t] = to == kNoMax ? 0.f : left_of(to, mc[t], c);
                const float f = fast_exp2(__builtin_fmaf(m[t] - to, c, left[t] - was));
                m[t] = to;
                limit[t] = to == kNoMax ? kNoMax : to + kSlack / c;
                big = __any(big || !(fabsf(mc[t]) <= kMostMax));
#pragma unroll
                for (int r = 0; r < 4; ++r) l[t][r] *= f;
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[t][n][r] *= f;
            }
        }
    }
    // Weights p in place of the scores.  s c - mc is one product with one rounding, which leaves
    // every weight the factor exp2(left), the rounding of m c; o / l takes that out again where
    // one m stays, and where it moves, or results of several m are joined, `left` does (m c of
    // 2^20 has half a step of 2^-5: a factor of 1.02).  It overflows or vanishes where half a
    // step of m c passes a hundred: past kMostMax (`big`) the difference is taken first.
    template <bool BIG> __device__ __forceinline__ void weights(float (&s)[RT][16], float c) const {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                s[t][e] = fast_exp2(BIG ? __builtin_fmaf(s[t][e] - m[t], c, left[t])
                                        : __builtin_fmaf(s[t][e], c, -mc[t]));
    }
    // o += P V, and l with it: a product of ones sums the weights as they are rounded.
    // value(u, n) as TileReads::value.
    template <class VALUE>
    __device__ __forceinline__ void accumulate(const float (&p)[RT][16], const Scales& vs, VALUE value) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            Parts<T> w[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                w[t].set(&p[t][8 * u]);
                l[t] = product(ones(), w[t], l[t]);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint2 y = value(u, n);
                const u32x4_v x = widen(y.x, y.y, vs.of[u]);
#pragma unroll
                for (int t = 0; t < RT; ++t) o[t][n] = product(x, w[t], o[t][n]);
            }
        }
    }
    // Where V holds NaN codes and some rows do not see their keys, 0 times them would reach those
    // rows: the codes become 0, and the dims that held one become NaN for the rows that see
    // the first such key, key j + 32 u + 8 g + e those with a limit past it.
    __device__ __forceinline__ void settle_nan(uint2 (&v)[2][8], int j, const int (&hi)[RT]) {
        uint32_t bad = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < 8; ++n) bad |= nan_codes(v[u][n].x) | nan_codes(v[u][n].y);
        if (!__any(bad != 0)) return;
        constexpr int kNone = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            int first = kNone;  // of dim 16 n + i
#pragma unroll
            for (int u = 1; u >= 0; --u) {
                const uint32_t x = nan_codes(v[u][n].x), y = nan_codes(v[u][n].y);
                const int key = j + 32 * u + 8 * g;
                if (y) first = key + 4 + (__builtin_ctz(y) >> 3);
                if (x) first = key + (__builtin_ctz(x) >> 3);
                v[u][n].x &= ~((x >> 7) * 255u);
                v[u][n].y &= ~((y >> 7) * 255u);
            }
            first = min(first, __shfl_xor(first, 16));
            first = min(first, __shfl_xor(first, 32));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = __shfl(first, 4 * g + r);
#pragma unroll
                for (int t = 0; t < RT; ++t) o[t][n][r] = f < hi[t] ? __builtin_nanf("") : o[t][n][r];
            }
        }
    }
};

// ---- the stream form: 16 RT query rows a wave, every wave walking tiles of its own
//
// A wave copies its next tile of K and V (8 KiB each) into LDS of its own while it works
// on the one in its registers: the copies are asynchronous, take whole 128-byte rows, and
// hold no registers, which the reads could not do for the layouts the products want.
//
// Decode is bound by memory where there is enough of it: 8 sequences of 32768 rows at 64 / 8
// heads (537 MB) 85.6 us, 6.3 TB/s, of which 78 are this kernel's at 6.9; 32 of 512 to 4096
// at 32 / 8 (163 MB) 33.5, of which 4 are the first dependent loads (lengths, page, rows), 24
// the rows at that rate and 4 the join; 1 of 300, whole, 6.3.
template <typename T, int RT> struct Stream : Rows8<T, RT> {
    typedef Rows8<T, RT> Base;
    TileReads reads;
    int from[4];      // copy_from() of instructions x (mod 4)
    u32x4_v k[4][2];  // TileReads::key and value of the tile
    uint2 v[2][8];
    Scales ks, vs;
    __device__ __forceinline__ Stream(int lane, uint8_t* lds)
        : Base(lane), reads(lds_at(lds), lds_at(lds) + kTileBytes, lane) {
#pragma unroll
        for (int x = 0; x < 4; ++x) from[x] = copy_from(x, lane);
    }
    // Start the copies of a tile.
    __device__ __forceinline__ void copy(const Args8& a, const Pages8::Tile& t, uint8_t* lds) const {
        const auto rk = tile_rsrc(a.k, t), rv = tile_rsrc(a.v, t);
#pragma unroll
        for (int x = 0; x < 8; ++x)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, lds + 1024 * x, 16, from[x & 3] + 4096 * (x >> 2), 0, 0, 2);
#pragma unroll
        for (int x = 0; x < 8; ++x)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, lds + kTileBytes + 1024 * x, 16, from[x & 3] + 4096 * (x >> 2),
                                                     0, 0, 2);
    }
    // The copied tile into registers.
    __device__ __forceinline__ void take() {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int half = 0; half < 2; ++half) k[kt][half] = reads.key(kt, half);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < 8; ++n) v[u][n] = reads.value(u, n);
    }
    // The tile in registers, of keys from j on.  Every row sees the keys before min_hi.
    __device__ __forceinline__ void step(const Args8& a, int j, const int (&hi)[RT], int min_hi, int end) {
        float s[RT][16];
        this->scores(s, ks, [&](int kt, int half) __attribute__((always_inline)) { return k[kt][half]; });
        const bool masked = j + kTile > min(min_hi, end);
        if (masked) this->mask(s, j, hi);
        this->settle(s, a.c);
        if (this->big) this->template weights<true>(s, a.c);
        else this->template weights<false>(s, a.c);
        if (masked && min_hi < end) this->settle_nan(v, j, hi);
        this->accumulate(s, vs, [&](int u, int n) __attribute__((always_inline)) { return v[u][n]; });
    }
};

// The LDS of a workgroup: its waves' tiles, then their results.  (8 waves a workgroup where
// no more than one a CU is launched took 6.4 us for 6.2 at 1 token of 300, 10.0 for 9.8 at
// 2 of 1000, 14.1 for 13.1 at 16 times 8 of 1000.)
constexpr int kWaves8 = 4;
template <int RT> union StreamLds {
    static constexpr int kStride = kHeadDim + 4;  // f32 per row: 16 rows at one column hit different banks
    __attribute__((aligned(1024))) uint8_t tile[kWaves8][2 * kTileBytes];
    struct {
        float o[kWaves8][16 * RT][kStride];
        float m[kWaves8][16 * RT], left[kWaves8][16 * RT], l[kWaves8][16 * RT];
    } join;
};

// Workgroup x's item of `units` (pair, kv head) units with `tiles` row tiles each.  Ids that
// are equal mod 8 run on one XCD: where the units come in eights it gets all tiles of a
// unit, one after the other, and reads their keys through its own L2.  Otherwise a unit's
// tiles are on all XCDs (4 units of 66 tiles, 6000 keys: on 4 XCDs 88 us, on all 65).  The
// last tiles, which see most keys of a causal call, go first (8 prompts of 2048 tokens:
// 297 us to 281).
struct Item8 {
    int block, kvh, pair;
    __device__ __forceinline__ Item8(const Args8& a, int x) {
        const int units = (a.pairs ? a.pairs : a.B) * a.Hkv;
        int unit = x / a.tiles;
        block = x - unit * a.tiles;
        if (units % 8 == 0) {
            const int c = x / (8 * a.tiles), rem = x - c * 8 * a.tiles;
            block = rem >> 3;
            unit = 8 * c + (rem & 7);
        }
        block = a.tiles - 1 - block;
        pair = unit / a.Hkv;
        kvh = unit - pair * a.Hkv;
    }
};

template <typename T, int RT>
__global__ __launch_bounds__(64 * kWaves8, 2) void f8_stream_kernel(Args8 a) {
    __shared__ StreamLds<RT> sm;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Item8 x(a, blockIdx.x);
    const int R = a.S * a.G, row0 = x.block * 16 * RT;
    // The tile's first and last queries; the last sees most.
    const int first = row0 / a.G, last = (min(row0 + 16 * RT, R) - 1) / a.G;
    Pages8 pages(a, lane);
    Pages8::Tile tile;
    Stream<T, RT> st(lane, sm.tile[wave]);
    int b = x.pair, n = 0, begin = 0, end = 0, j = wave * kTile;
    Lengths lengths;
    if (a.pairs) lengths.load(a, lane);
    if (b < a.B) {  // a first chunk: its waves' first tiles are in it however the sequence is cut
        n = a.len(b);
        end = a.limit(n, last);
        pages.open(a, b, 0);
        if (j < end) st.copy(a, tile = pages.tile(a, x.kvh, j, end), sm.tile[wave]);
    } else if (!a.pairs) {
        return;
    }
    bool direct = true;
    if (a.pairs) {
        const Cut cut = cut_at(a, lengths, x.pair, lane);
        if (cut.b < 0) return;
        direct = __builtin_amdgcn_readfirstlane(cut.n) == 1;
        const int per = __builtin_amdgcn_readfirstlane(cut.tiles) * kTile;
        begin = __builtin_amdgcn_readfirstlane(cut.chunk) * per;
        if (begin > 0) {
            b = __builtin_amdgcn_readfirstlane(cut.b);
            n = __builtin_amdgcn_readfirstlane(cut.len);
            end = min(begin + per, a.limit(n, last));
            if (begin >= end) return;  // the join reads no chunk past a row's keys
            pages.open(a, b, begin);
            j = begin + wave * kTile;
            if (j < end) st.copy(a, tile = pages.tile(a, x.kvh, j, end), sm.tile[wave]);
        } else if (!direct) {
            end = min(per, end);
            if (x.kvh == 0 && x.block == 0 && tid == 0) a.ws_cut[b] = make_int4(cut.n, cut.rest, per, 0);
        }
        if (direct && x.kvh == 0 && x.block == 0 && tid == 0) a.ws_cut[b] = make_int4(1, 0, 0, 0);
    }
    const int min_hi = a.limit(n, first);

    int at[RT], hi[RT];
    st.open(a, b, x.kvh, row0, n, end, at, hi);
    constexpr int kStride = kWaves8 * kTile;
    for (; j < end; j += kStride) {
        st.ks.load(a.k_scale, tile.off);
        st.vs.load(a.v_scale, tile.off);
        wait_memory();
        __builtin_amdgcn_sched_barrier(0);
        st.take();
        if (j + kStride < end) {
            tile = pages.tile(a, x.kvh, j + kStride, end);
            wait_lds();  // the tile is in registers: its LDS is free
            __builtin_amdgcn_sched_barrier(0);
            st.copy(a, tile, sm.tile[wave]);
            __builtin_amdgcn_sched_barrier(0);
        }
        st.step(a, j, hi, min_hi, end);
    }

    T* out = reinterpret_cast<T*>(a.out);
    __syncthreads();  // every wave's tiles are read
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (st.g == 0) {
            sm.join.m[wave][16 * t + st.i] = st.m[t];
            sm.join.left[wave][16 * t + st.i] = st.left[t];
            sm.join.l[wave][16 * t + st.i] = st.l[t][0];
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = st.o[t][d][r];
            store4(&sm.join.o[wave][16 * t + st.i][16 * d + 4 * st.g], y);
        }
    }
    __syncthreads();
    // 16 threads per row, 8 dims each.
    for (int r = tid >> 4; r < 16 * RT && row0 + r < R; r += 4 * kWaves8) {
        const int s = (row0 + r) / a.G, h = row0 + r - s * a.G, d = 8 * (tid & 15);
        const int place = (int)(((int64_t)b * a.Hq + x.kvh * a.G + h) * a.S + s);
        float top = sm.join.m[0][r];
#pragma unroll
        for (int w = 1; w < kWaves8; ++w) top = fmaxf(top, sm.join.m[w][r]);
        float l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves8; ++w) {
            const float f = fast_exp2(__builtin_fmaf(sm.join.m[w][r] - top, a.c, -sm.join.left[w][r]));
            float z[8];
            load8(&sm.join.o[w][r][d], z);
            l += f * sm.join.l[w][r];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += f * z[e];
        }
        if (direct) {
            const bool none = min(a.limit(n, s), end) <= 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = none ? 0.f : y[e] / l;
            store8(out + a.out_row(place) * kHeadDim + d, y);
        } else {
            const int64_t slot = a.slot(x.pair, x.kvh, x.block, r);
            store8(a.ws_o + slot * kHeadDim + d, y);
            if (d == 0) a.ws_ml[slot] = make_float2(top, l);
        }
    }
}

// ---- the block form: 128 query rows a workgroup, a tile of keys shared by its waves
//
// 32 rows to a wave and every wave on the same tile: the workgroup reads K and V once for
// 128 rows.  Tiles are copied one ahead into the other of two buffers, a quarter of each by
// every wave.  All of a tile's K is read before the first product, all of its V before the
// softmax that hides it, and only then is the next tile's copy started: a transposed read
// waits for every copy under way (the compiler cannot tell them apart).  With reads one
// ahead of their use, copies started first and the scales by scalar loads 12 prompts' 1024
// tokens over 5000 to 9000 keys (28 / 4 heads, 2688 workgroups) took 1239 us, so 1130; with
// the products' phases above the softmax in the CU's priority 1121 (1.0 PFLOP/s, as over
// 9000 keys each), with the weights' sum as a product 0.7% more.  What is left is the issue
// of instructions that are no products: without the conversions of codes (timing only) 11%
// less, without the exponentials 8%.
//
// v_mfma_f32_32x32x16_bf16 (half the instructions and operand reads of the 16-row product
// for the same work): lane (i, h) = (lane % 32, lane / 32) holds, for query row i, rows 8 a
// + 4 h + c of a product (register 4 a + c).  A's row x is key 16 (x / 16)
// + 8 (x / 4 % 2) + 4 (x / 8 % 2) + x % 4 of 32, so that the lane holds keys 16 s + 8 h +
// (0 .. 7), s = 0, 1: P^T of two products with V^T, whose bytes are one transposed read
// each.
struct BlockLds {
    __attribute__((aligned(1024))) uint8_t k[2][kTileBytes];
    __attribute__((aligned(1024))) uint8_t v[2][kTileBytes];
};
// The chunk permutation of these tiles: 16 rows of a K read, and 8 rows x 2 chunks of a V
// read, do not meet in a bank.
__device__ __forceinline__ int permute8_block(int row) { return ((row >> 3) & 1) | (row & 6); }

template <typename T> struct BlockRows {
    const int i, h;
    uint32_t k_at, v_at;  // where this lane's reads of the first tiles start
    Parts<T> q[8];        // [2 x + y]: dims 32 x + 16 h + 8 y ..
    f32x16_v o[4];        // dims 32 d + 8 a + 4 h + c of row i
    // The weights' sum: bf16's of the rounded ones, over all keys, in every register; f32's, whose
    // parts hold all of their bits, over the lane's own keys (a product would spill more).
    static constexpr bool kProductSum = Parts<T>::kN == 1;
    std::conditional_t<kProductSum, f32x16_v, float> l;
    float m, mc, left, limit;  // as Rows8
    bool big;
    __device__ __forceinline__ BlockRows(int lane, const BlockLds& sm)
        : i(lane & 31), h(lane >> 5), l{}, m(kNoMax), mc(0.f), left(0.f), limit(kNoMax), big(false) {
        const int k_row = (i & 16) | ((i & 4) << 1) | ((i & 8) >> 1) | (i & 3), v_row = 8 * h + ((lane & 15) >> 1);
        k_at = lds_at(sm.k) + k_row * kRow + 16 * (h ^ permute8_block(k_row));
        v_at = lds_at(sm.v) + v_row * kRow + 16 * (((lane >> 4) & 1) ^ permute8_block(v_row)) + 8 * (lane & 1);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    }
    __device__ __forceinline__ float sum() const {
        if constexpr (kProductSum) return l[0];
        else return halves_sum(l);
    }
    // Chunk 2 x + h of key block u's row i.
    __device__ __forceinline__ u32x4_v key(int u, int x, uint32_t buf) const {
        return lds_read16((k_at ^ (32 * x)) + buf + 32 * u * kRow);
    }
    // Keys 32 u + 16 s + 8 h .. of dim 32 d + i.
    __device__ __forceinline__ uint2 value(int u, int s, int d, uint32_t buf) const {
        return lds_read_tr8((v_at ^ (32 * d)) + buf + (32 * u + 16 * s) * kRow);
    }
    // s[u][8 t + e]: the raw score of key 32 u + 16 t + 8 h + e.
    __device__ __forceinline__ void scores(f32x16_v (&s)[2], const Scales& ks, uint32_t buf) const {
        u32x4_v k[2][4];
#pragma unroll
        for (int z = 0; z < 8; ++z) k[z >> 2][z & 3] = key(z >> 2, z & 3, buf);
        __builtin_amdgcn_sched_barrier(0);  // all reads under way before the first is waited for
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    s[u] = product(widen(k[u][x][2 * y], k[u][x][2 * y + 1], ks.of[u]), q[2 * x + y], s[u]);
        }
    }
    __device__ __forceinline__ void mask(f32x16_v (&s)[2], int j, int hi) const {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[u][r] = j + 32 * u + 16 * (r >> 3) + 8 * h + (r & 7) < hi ? s[u][r] : -INFINITY;
    }
    __device__ __forceinline__ void settle(const f32x16_v (&s)[2], float c) {
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
        if (__any(mx > limit)) {
            const float to = fmaxf(m, halves_max(mx)), was = left;
            mc = to == kNoMax ? 0.f : to * c;
            left = to == kNoMax ? 0.f : left_of(to, mc, c);
            const float f = fast_exp2(__builtin_fmaf(m - to, c, left - was));
            m = to;
            limit = to == kNoMax ? kNoMax : to + kSlack / c;
            big = __any(big || !(fabsf(mc) <= kMostMax));
            if constexpr (kProductSum) {
#pragma unroll
                for (int r = 0; r < 16; ++r) l[r] *= f;
            } else {
                l *= f;
            }
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
        }
    }
    template <bool BIG> __device__ __forceinline__ void weights(f32x16_v (&s)[2], float c) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = fast_exp2(BIG ? __builtin_fmaf(s[u][r] - m, c, left) : __builtin_fmaf(s[u][r], c, -mc));
                if constexpr (!kProductSum) sum[u] += s[u][r];
            }
        if constexpr (!kProductSum) l += sum[0] + sum[1];
    }
    __device__ __forceinline__ void accumulate(const f32x16_v (&p)[2], const Scales& vs, const uint2 (&v)[2][2][4]) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = p[u][8 * t + e];
                Parts<T> w;
                w.set(x);
                if constexpr (kProductSum) l = product(ones(), w, l);
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] = product(widen(v[u][t][d].x, v[u][t][d].y, vs.of[u]), w, o[d]);
            }
    }
    // As Rows8::settle_nan; key j + 32 u + 16 t + 8 h + e.
    __device__ __forceinline__ void settle_nan(uint2 (&v)[2][2][4], int j, int hi) {
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const uint2 c = v[x >> 3][(x >> 2) & 1][x & 3];
            bad |= nan_codes(c.x) | nan_codes(c.y);
        }
        if (!__any(bad != 0)) return;
        constexpr int kNone = 0x7fffffff;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            int first = kNone;  // of dim 32 d + i
#pragma unroll
            for (int z = 3; z >= 0; --z) {
                uint2& c = v[z >> 1][z & 1][d];
                const uint32_t x = nan_codes(c.x), y = nan_codes(c.y);
                const int key = j + 16 * z + 8 * h;
                if (y) first = key + 4 + (__builtin_ctz(y) >> 3);
                if (x) first = key + (__builtin_ctz(x) >> 3);
                c.x &= ~((x >> 7) * 255u);
                c.y &= ~((y >> 7) * 255u);
            }
            first = min(first, __shfl_xor(first, 32));
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int f = __shfl(first, 8 * (r >> 2) + 4 * h + (r & 3));
                o[d][r] = f < hi ? __builtin_nanf("") : o[d][r];
            }
        }
    }
};

template <typename T>
__global__ __launch_bounds__(64 * kWaves8, 2) void f8_block_kernel(Args8 a) {
    __shared__ BlockLds sm;
    constexpr int kRows = 128;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Item8 x(a, blockIdx.x);
    const int R = a.S * a.G, block0 = x.block * kRows, row0 = block0 + 32 * wave;
    const int b = x.pair, n = a.len(b);
    // What the block's last row and this wave's first and last rows see.
    auto seen = [&](int r) __attribute__((always_inline)) { return a.limit(n, min(r, R - 1) / a.G); };
    const int end = seen(block0 + kRows - 1), min_hi = seen(row0), max_hi = row0 < R ? seen(row0 + 31) : 0;

    Pages8 pages(a, lane);
    pages.open(a, b, 0);
    BlockRows<T> st(lane, sm);
    int from[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const int row = 16 * wave + 8 * y + (lane >> 3);
        from[y] = row * kRow + 16 * ((lane & 7) ^ permute8_block(row));
    }
    auto tile_at = [&](int j) __attribute__((always_inline)) { return pages.tile(a, x.kvh, j, end); };
    auto copy = [&](const Pages8::Tile& t, int buf) __attribute__((always_inline)) {
        const auto rk = tile_rsrc(a.k, t), rv = tile_rsrc(a.v, t);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, sm.k[buf] + 1024 * (2 * wave + y), 16, from[y], 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, sm.v[buf] + 1024 * (2 * wave + y), 16, from[y], 0, 0, 0);
        }
    };
    Pages8::Tile tile{0, 0};
    uint32_t k_scales = 0, v_scales = 0;
    auto start = [&](int j, int buf) __attribute__((always_inline)) {
        if (j >= end) return;
        copy(tile = tile_at(j), buf);
        k_scales = Scales::fetch(a.k_scale, tile.off);
        v_scales = Scales::fetch(a.v_scale, tile.off);
    };
    start(0, 0);
    const int r = row0 + st.i, s_of = min(r, R - 1) / a.G, head = min(r, R - 1) - s_of * a.G;
    const int at = r < R ? (int)(((int64_t)b * a.Hq + x.kvh * a.G + head) * a.S + s_of) : -1;
    const int hi = min(a.limit(n, s_of), end);
#pragma unroll
    for (int y = 0; y < 8; ++y)
        st.q[y].load(reinterpret_cast<const T*>(a.q) + (int64_t)max(at, 0) * kHeadDim + 32 * (y >> 1) + 16 * st.h +
                     8 * (y & 1));
    for (int j = 0, half = 0; j < end; j += kTile, half ^= 1) {
        const uint32_t buf = half * kTileBytes;
        wait_memory();
        __syncthreads();  // the tile is there, and the one before it is used
        Scales ks, vs;
        ks.set(__builtin_amdgcn_readfirstlane(k_scales), tile.off);
        vs.set(__builtin_amdgcn_readfirstlane(v_scales), tile.off);
        if (j >= max_hi) {  // none of the wave's rows
            start(j + kTile, half ^ 1);
            continue;
        }
        f32x16_v s[2];
        uint2 v[2][2][4];
        __builtin_amdgcn_s_setprio(1);
        st.scores(s, ks, buf);
#pragma unroll
        for (int z = 0; z < 16; ++z) v[z >> 3][(z >> 2) & 1][z & 3] = st.value(z >> 3, (z >> 2) & 1, z & 3, buf);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        start(j + kTile, half ^ 1);
        const bool masked = j + kTile > min(min_hi, end);
        if (masked) st.mask(s, j, hi);
        st.settle(s, a.c);
        if (st.big) st.template weights<true>(s, a.c);
        else st.template weights<false>(s, a.c);
        if (masked && min_hi < end) st.settle_nan(v, j, hi);
        __builtin_amdgcn_s_setprio(1);
        st.accumulate(s, vs, v);
        __builtin_amdgcn_s_setprio(0);
    }

    const float l = st.sum();
    if (at < 0) return;
    T* out = reinterpret_cast<T*>(a.out) + a.out_row(at) * kHeadDim + 4 * st.h;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = hi <= 0 ? 0.f : st.o[d][4 * e + c] / l;
            store4(out + 32 * d + 8 * e, y);
        }
}

// Join a query row's chunks: P waves per row, lane x owns dims 2 x, 2 x + 1, wave p takes
// chunks p, p + P, ...  The first loads (kJoinRegs chunks a wave, m and l of 64) are
// issued at once.
constexpr int kJoinRegs = 8;
template <typename T, int P>
__global__ __launch_bounds__(P == 1 ? 256 : 64 * P) void f8_join_kernel(Args8 a, int n_rows) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = P == 1 ? 0 : wave;
    const int row = __builtin_amdgcn_readfirstlane(P == 1 ? blockIdx.x * 4 + wave : blockIdx.x);
    if (row >= n_rows) return;  // P > 1: the whole workgroup
    const int bh = row / a.S, s = row - bh * a.S, b = bh / a.Hq, head = bh - b * a.Hq, kvh = head / a.G;
    const int4 cut = a.ws_cut[b];
    if (cut.x == 1) return;  // written by the workgroup that had the sequence
    const int keys = a.limit(a.len(b), s), n = keys > 0 ? (keys + cut.z - 1) / cut.z : 0;
    const int r = s * a.G + head - kvh * a.G, tile = r / a.tile_rows;
    // chunk c's results
    const int64_t at = a.slot(0, kvh, tile, r - tile * a.tile_rows), next = (int64_t)a.Hkv * a.tiles * a.tile_rows;
    auto ml = [&](int c) __attribute__((always_inline)) { return a.ws_ml[at + (c == 0 ? b : cut.y + c - 1) * next]; };
    auto o = [&](int c) __attribute__((always_inline)) {
        return reinterpret_cast<const float2*>(a.ws_o + (at + (c == 0 ? b : cut.y + c - 1) * next) * kHeadDim)[lane];
    };
    float2 x[kJoinRegs];
#pragma unroll
    for (int i = 0; i < kJoinRegs; ++i) x[i] = o(min(p + P * i, max(n - 1, 0)));
    const float2 mine = ml(min(lane, max(n - 1, 0)));
    float top = lane < n ? mine.x : kNoMax;
    for (int c = lane + 64; c < n; c += 64) top = fmaxf(top, ml(c).x);
    top = wave_max(top);
    float den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int c0 = 0; c0 < n; c0 += 64) {
        const float2 t = c0 == 0 ? mine : ml(min(c0 + lane, n - 1));
        const float w = c0 + lane < n ? fast_exp2((t.x - top) * a.c) : 0.f;
        den += c0 + lane < n ? w * t.y : 0.f;
        auto add = [&](int c, float2 y) __attribute__((always_inline)) {
            const float wc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), c - c0));
            x0 += wc * y.x;
            x1 += wc * y.y;
        };
        int c = c0 + p;
        if (c0 == 0) {
#pragma unroll
            for (int i = 0; i < kJoinRegs; ++i)
                if (p + P * i < min(n, 64)) add(p + P * i, x[i]);
            c += P * kJoinRegs;
        }
        for (; c < min(n, c0 + 64); c += P) add(c, o(c));
    }
    den = wave_sum(den);
    if constexpr (P > 1) {
        __shared__ float2 part[P - 1][64];
        if (p > 0) part[p - 1][lane] = make_float2(x0, x1);
        __syncthreads();
        if (p > 0) return;
#pragma unroll
        for (int i = 0; i < P - 1; ++i) {
            x0 += part[i][lane].x;
            x1 += part[i][lane].y;
        }
    }
    T* out = reinterpret_cast<T*>(a.out) + a.out_row(row) * kHeadDim + 2 * lane;
    Elem<T>::store(out, n == 0 ? 0.f : x0 / den);
    Elem<T>::store(out + 1, n == 0 ? 0.f : x1 / den);
}

// How a call is launched: its form, the rows of a workgroup, and whether and into how many
// chunks at most the sequences are cut.
struct Plan8 {
    bool block;
    int rows;
    int64_t tiles, pairs, items;
    size_t ml_off, cut_off, total;
};

Plan8 plan8(int64_t max_kv, int B, int S, int Hq, int Hkv, bool bf16) {
    Plan8 p{};
    const int64_t R = (int64_t)S * (Hq / Hkv), slots = 2 * kCus;  // two workgroups a CU, of any form
    // The block form where its workgroups, whose waves all walk all keys, fill the device: bf16,
    // 1024 tokens of 2 prompts of 1024 at 32 / 8 heads (512 of them) 40 us, 45 in the stream form,
    // of 8192 267 for 285; of 1 prompt (256) 28 for 25, 167 for 143; 256 tokens of 7 to 3000 (448)
    // 74 for 74.  f32, whose 16 rows a wave hide more: 1024 tokens of 8 prompts of 1024 at 28 / 4
    // (1792) 210 for 279, 256 tokens of 16 to 3000 (1024) 370 for 360.
    const int64_t blocks = B * Hkv * ceil_div(R, 128);
    p.block = blocks >= (bf16 ? 1 : 3) * slots;
    // Else 16 or 32 rows a wave.  16 leave room for loads under way, 32 widen the codes once for
    // twice the rows.  f32 takes 16: its q has three parts, and 32 rows spill (256 tokens of 4 to
    // 3000 113 us for 151, 9 to 40 tokens of 4 to 4000 22 to 41 for 35 to 56).  bf16 takes 16 up to
    // 16 rows (32 decode steps of 4 rows 34.4 for 36.3); past 32 while that is a workgroup a CU at
    // most (8 sequences of 1000 to 4000 at 32 / 8 heads: 16 tokens, 256 of them, 22.6 for 26.4, 20
    // tokens, 320 of them, 37.6 for 28.2); and from 17 to 32, where it reads the keys twice, while
    // the chunks are short (5 tokens, 28 / 4: 4 sequences of up to 5000 15.7 for 17.1; 32 / 8: 4 of
    // 16000 32.5 for 29.0, 16 of 5000 32.4 for 28.1).
    auto most = [&](int rows) { return slots / (Hkv * ceil_div(R, rows)); };  // chunks that fit at once
    const bool half = !bf16 || R <= 16 ||
                      (R > 32 ? B * Hkv * ceil_div(R, 16) <= kCus : B * max_kv <= 1024 * most(16));
    p.rows = p.block ? 128 : half ? 16 : 32;
    p.tiles = ceil_div(R, p.rows);
    const int64_t heads = Hkv * p.tiles;
    // Cut where the device holds more of them at once, and they are longer than the second kernel is
    // worth (1 sequence of 1000 rows at 32 / 8 heads: 8.7 us whole, 9.2 cut; 4 of 2000: 14.2 and
    // 10.0).  Decode, bound by memory: 40 of up to 4096 (1.6 chunks each fit) 44.7 whole, 37.5 cut,
    // 56 (1.1) 49.6 and 51.9; f32 likewise.  bf16 past 16 rows is bound by instructions, and a
    // workgroup a CU does: 24 tokens of 8 of up to 4000 (2.7) 28.4 whole, 32.0 cut, 5 tokens of 16
    // of up to 5000 (4) 33.4 and 28.1.
    const bool cut = bf16 && R > 16 ? most(p.rows) >= 3 * B : 2 * most(p.rows) > 3 * B;
    if (!p.block && B <= kMostCut && cut && max_kv > 1024) p.pairs = most(p.rows);
    p.items = (p.pairs ? p.pairs : B) * heads;
    const size_t rows = (size_t)(p.pairs * heads * p.rows);
    p.ml_off = rows * kHeadDim * sizeof(float);
    p.cut_off = p.ml_off + rows * sizeof(float2);
    p.total = p.pairs ? p.cut_off + B * sizeof(int4) : 0;
    return p;
}

template <typename T> int launch8(const Args8& a, const Plan8& p, int64_t n_rows, hipStream_t st) {
    const dim3 grid((unsigned)p.items), threads(64 * kWaves8);
    if (p.block) hipLaunchKernelGGL(f8_block_kernel<T>, grid, threads, 0, st, a);
    else if (p.rows == 16) hipLaunchKernelGGL((f8_stream_kernel<T, 1>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((f8_stream_kernel<bf16_t, 2>), grid, threads, 0, st, a);
    int rc = launch_status(hipGetLastError());
    if (rc || !p.pairs) return rc;
    // About a sequence's chunks, a wave for up to kJoinRegs of them: 1 sequence of 32768 rows at 64 /
    // 8 heads (64 chunks) takes 34.0 us in all with 1 wave a row, 21.4 with 4, 19.7 with 16; of 8000
    // at 32 / 8 (32) 13.3, 10.5, 11.0; 4 of 2000 (8) 9.8, 10.2, 10.7; 32 of up to 8192 (2) 33.5,
    // 35.0, 38.2.
    const int64_t chunks = std::min(p.pairs / a.B, ceil_div(a.max_kv, kLeastChunk * kTile));
    if (chunks <= kJoinRegs)
        hipLaunchKernelGGL((f8_join_kernel<T, 1>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, st, a,
                           (int)n_rows);
    else if (chunks <= 4 * kJoinRegs)
        hipLaunchKernelGGL((f8_join_kernel<T, 4>), dim3((unsigned)n_rows), dim3(256), 0, st, a, (int)n_rows);
    else
        hipLaunchKernelGGL((f8_join_kernel<T, 16>), dim3((unsigned)n_rows), dim3(1024), 0, st, a, (int)n_rows);
    return launch_status(hipGetLastError());
}

int check_sizes8(int64_t max_kv, int B, int S, int Hq, int Hkv, int D, int dtype) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return CRANE_HIP_E_INVALID;
    if (Hq % Hkv != 0) return CRANE_HIP_E_GQA;
    if (B > 65535 || (int64_t)B * Hq > 0x7fffffffLL) return CRANE_HIP_E_INVALID;
    if ((int64_t)B * Hq * S > kMostThreads / 64) return CRANE_HIP_E_INVALID;  // a wave each in the join
    if (max_kv > 0x7fffffffLL - (1 << 20)) return CRANE_HIP_E_INVALID;  // a tile's bounds stay within 31 bits
    return CRANE_HIP_OK;
}

}  // namespace
}  // namespace crane

using namespace crane;

extern "C" size_t crane_hip_attn_paged_f8_workspace(int64_t max_kv, int B, int S, int Hq, int Hkv, int D, int dtype) {
    if (check_sizes8(max_kv, B, S, Hq, Hkv, D, dtype) || B == 0 || S == 0 || max_kv <= 0) return 0;
    const Plan8 p = plan8(max_kv, B, S, Hq, Hkv, dtype == CRANE_HIP_BF16);
    return p.items <= kMostThreads / (64 * kWaves8) ? p.total : 0;
}

extern "C" int crane_hip_attn_paged_f8(const void* q, const void* k_pool, const void* v_pool, const void* k_scale,
                                       const void* v_scale, int64_t n_pages, int page_rows,
                                       const int32_t* block_table, int64_t table_stride, const int32_t* kv_len,
                                       int64_t max_kv, int B, int S, int Hq, int Hkv, int D, float scale, int flags,
                                       void* workspace, size_t ws_bytes, void* out, int dtype, void* stream) {
    int rc = check_sizes8(max_kv, B, S, Hq, Hkv, D, dtype);
    if (rc) return rc;
    if (flags & ~CRANE_HIP_PREFILL_CAUSAL) return CRANE_HIP_E_INVALID;
    if (!(scale > 0.0f) || !__builtin_isfinite(scale * kLog2e)) return CRANE_HIP_E_INVALID;
    if ((rc = check_paged(n_pages, page_rows, block_table, table_stride, Hkv))) return rc;
    if (max_kv <= 0) return CRANE_HIP_E_INVALID;
    if (max_kv > table_stride * page_rows) return CRANE_HIP_E_CAPACITY;
    if (B == 0 || S == 0) return CRANE_HIP_OK;
    if (!q || !kv_len || !out) return CRANE_HIP_E_INVALID;
    if ((rc = check_pools8(k_pool, v_pool, k_scale, v_scale))) return rc;
    if (!aligned16(q) || !aligned16(out)) return CRANE_HIP_E_ALIGN;
    const Plan8 p = plan8(max_kv, B, S, Hq, Hkv, dtype == CRANE_HIP_BF16);
    if (p.items > kMostThreads / (64 * kWaves8)) return CRANE_HIP_E_INVALID;
    if (p.total && (!workspace || ws_bytes < p.total || !aligned16(workspace))) return CRANE_HIP_E_WORKSPACE;
    Args8 a;
    a.q = q;
    a.k = (const uint8_t*)k_pool;
    a.v = (const uint8_t*)v_pool;
    a.k_scale = (const uint8_t*)k_scale;
    a.v_scale = (const uint8_t*)v_scale;
    a.out = out;
    a.rows = PagedRows{block_table, table_stride, n_pages, page_rows};
    a.kv_len = kv_len;
    a.B = B;
    a.S = S;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.max_kv = (int)max_kv;
    a.causal = flags & CRANE_HIP_PREFILL_CAUSAL;
    a.c = scale * kLog2e;
    a.tiles = (int)p.tiles;
    a.pairs = (int)p.pairs;
    a.tile_rows = p.rows;
    a.ws_o = (float*)workspace;
    a.ws_ml = (float2*)((char*)workspace + p.ml_off);
    a.ws_cut = (int4*)((char*)workspace + p.cut_off);
    const int64_t n_rows = (int64_t)B * Hq * S;
    const hipStream_t st = (hipStream_t)stream;
    return dtype == CRANE_HIP_F32 ? launch8<float>(a, p, n_rows, st) : launch8<bf16_t>(a, p, n_rows, st);
}
