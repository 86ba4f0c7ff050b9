// shared.hip -- attention over a paged KV cache in which groups of sequences share
// their first rows (gfx950); the C ABI is include/crane_shared.h.
//
// Sequence b has n = kv_len[b] rows; its query i sees rows [0, L), L = n - S + 1 + i
// (causal) or n.  With s_j = scale q . k_j over any set J of keys,
//     m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j,
// and the results of disjoint sets join as o = sum w_J o_J / sum w_J l_J, w_J =
// exp(m_J - max m).  So a group's shared rows are one set for all of its members'
// queries together, every sequence's own rows another, and each is cut into chunks
// for parallelism.  A workgroup (4 waves) takes one chunk for a block of query rows of
// one kv head; rows are (member, query, head of the GQA group) of the whole group for
// shared chunks, (query, head) of one sequence for its own.  A second kernel joins the
// chunks.  Two forms, by the rows there are:
//
// Stream (up to 16 rows: HBM-bound).  Every wave takes 32-key steps of its own, K and V
// from memory to registers two steps ahead, and the waves' m, l, o are joined through
// LDS at the end.  bf16, v_mfma_f32_16x16x32_bf16: S^T = K Q^T with K rows as A and
// query rows as B, so lane (i, g) = (lane % 16, lane / 16) holds, for query row i, keys
// 4 g + r of two 16-key halves.  Those 8 values, rounded to bf16, are the B operand
// P^T of O^T = V^T P^T as they stand: the order of the 32 keys inside the k index is
// free as long as V follows it, so lane group g takes V rows 4 g + r of both halves.
// It reads dims [8 i, 8 i + 8) of each (whole 256-byte rows per 16 lanes) and v_perm
// pairs them into the A operand of eight products, product n giving dims 8 m + n: a
// lane ends with dims [32 g, 32 g + 32) of its query row.
//
// Block (more rows: 128 of bf16, 64 of f32, a share for each wave).  The waves walk the
// same keys, staged in LDS by buffer_load ... lds one tile ahead, so that K and V are
// read from memory once for the block.  bf16, v_mfma_f32_32x32x16_bf16: the same
// products with 32 rows a wave and 64 keys a tile; V^T comes from the row-major tile
// by transposed LDS reads.
//
// f32 runs the stream's layout on v_mfma_f32_16x16x4_f32 in both forms: a k slot takes
// one key (or dim) of every lane group, so no pairing is needed.
//
// l sums p as computed in f32; only the P operand is rounded (bf16).
#include <float.h>

#include <type_traits>

#include "common.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr int kAlign = 64;         // chunk bounds are multiples of it (whole steps of every form)
constexpr int kWaves = 4;
constexpr float kNoMax = -FLT_MAX; // m before the first key (finite: exp2(-inf - m) is 0, not NaN)
constexpr int kMaxChunk = 8192;    // rows per chunk: its pages' ids fit one lane each
constexpr int kMinChunk = 128;
constexpr int kStreamRows = 16;    // query rows of a workgroup
template <typename T> constexpr int kBlockRows = sizeof(T) == 2 ? 128 : 64;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}
typedef unsigned int u32x4_v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4_v buf_load16(__amdgpu_buffer_rsrc_t r, int off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}
__device__ __forceinline__ f32x4_v mfma(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0,
                                                   0, 0);
}
__device__ __forceinline__ f32x4_v mfma(float a, float b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

struct Args {
    const void *q, *k, *v;
    void* out;
    PagedRows rows;
    const int32_t *kv_len, *shared, *groups, *members;
    int n_groups, max_group, max_shared;
    int B, S, Hq, Hkv, G;     // G = Hq / Hkv heads per kv head
    int max_kv, causal;
    float c;                  // scale log2 e
    int shared_chunk, own_chunk;    // rows per chunk
    int shared_splits, own_splits;  // chunks
    int shared_tiles, own_tiles;    // row blocks per (group or sequence, kv head)
    int shared_items;               // workgroups of the shared role, which come first (a multiple of 8)
    float* ws_o;              // [B Hq S, slots, D] f32, unnormalised
    float2* ws_ml;            // [B Hq S, slots] (m, l)
    __device__ __forceinline__ int slots() const { return shared_splits + own_splits; }
    __device__ __forceinline__ int len(int b) const { return max(0, min(kv_len[b], max_kv)); }
    __device__ __forceinline__ int shared_of(int b) const { return shared ? max(0, min(shared[b], max_shared)) : 0; }
    // Rows query s of sequence b sees.
    __device__ __forceinline__ int limit(int b, int s) const { return causal ? len(b) - S + 1 + s : len(b); }
    // First row of own chunk 0: chunk bounds sit on tile bounds.
    __device__ __forceinline__ static int own_base(int shared_rows) { return shared_rows & ~(kAlign - 1); }
};

// A workgroup's item: a segment of keys (a group's shared rows or a sequence's own)
// and the query rows that meet it.
template <bool SHARED> struct Segment {
    const Args& a;
    int table_row, lo, hi;   // block table row; keys [lo, hi) of it (own: up to each query's limit)
    int first, n_rows, R;    // first member; query rows per kv head, in all and per member
    __device__ __forceinline__ Segment(const Args& args, int seg) : a(args), R(args.S * args.G) {
        if constexpr (SHARED) {
            const int4 d = reinterpret_cast<const int4*>(a.groups)[seg];
            first = min(max(d.x, 0), a.B);
            const int members = min(max(d.y, 0), min(a.max_group, a.B - first));
            table_row = d.z;
            lo = 0;
            hi = min(d.w, a.max_shared);
            n_rows = table_row < 0 || table_row >= a.B ? 0 : members * R;
        } else {
            first = 0;
            table_row = seg;
            lo = a.shared_of(seg);
            hi = 0x7fffffff;
            n_rows = R;
        }
    }
    __device__ __forceinline__ int base() const { return SHARED ? 0 : Args::own_base(lo); }
    struct Row {
        int b, s, h;  // sequence (or one outside the batch), query, head of the GQA group
    };
    __device__ __forceinline__ Row row(int r) const {
        const int member = SHARED ? r / R : 0, rem = r - member * R, s = rem / a.G;
        return Row{SHARED ? a.members[first + member] : table_row, s, rem - s * a.G};
    }
    // Row r's place in [B, Hq, S] (-1: none) and the keys it sees: [lo, to).
    __device__ __forceinline__ int64_t query(int r, int kvh, int& to) const {
        to = 0;
        if (r >= n_rows) return -1;
        const Row x = row(r);
        if (x.b < 0 || x.b >= a.B) return -1;
        to = min(hi, a.limit(x.b, x.s));
        return ((int64_t)x.b * a.Hq + kvh * a.G + x.h) * a.S + x.s;
    }
};

// A wave-uniform value the compiler holds in vector registers (a buffer resource made
// of such would be read lane by lane).
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// A chunk's pages, one id per lane: those from the chunk's first on, or the whole table
// row where it fits (then the load waits for nothing).
struct Pages {
    int ids, page0, P;
    __device__ __forceinline__ Pages(const Args& a, int table_row, int begin, int lane) : ids(-1), P(a.rows.page_rows) {
        page0 = a.rows.stride <= 64 ? 0 : begin / P;
        if (page0 + lane < a.rows.stride) ids = a.rows.table[table_row * a.rows.stride + page0 + lane];
    }
    // Rows [j, min(j + n, end)) of a kv head, within one page: their offset in a pool and
    // their bytes.  No rows past `end`, nor of a page outside the pool: they read as zero.
    struct Tile {
        int64_t off;
        int bytes;
    };
    template <typename T>
    __device__ __forceinline__ Tile tile(const Args& a, int kvh, int j, int n, int end) const {
        const int p = j / P;
        const int id = __builtin_amdgcn_readlane(ids, (p - page0) & 63);
        const bool ok = (unsigned)id < (unsigned)a.rows.n_pages;
        const int rows = ok ? max(0, min(n, end - j)) : 0;
        const int64_t off = (((int64_t)(ok ? id : 0) * a.Hkv + kvh) * P + (j - p * P)) * kHeadDim;
        return Tile{uniform(off), __builtin_amdgcn_readfirstlane(rows * kHeadDim * (int)sizeof(T))};
    }
};
template <typename T> __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* pool, const Pages::Tile& t) {
    return make_rsrc(reinterpret_cast<const T*>(pool) + t.off, t.bytes);
}

__device__ __forceinline__ int wave_max_int(int x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = max(x, __shfl_xor(x, d));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_min_int(int x) { return -wave_max_int(-x); }

struct StreamShared {
    static constexpr int kStride = kHeadDim + 4;  // f32 per row: 16 rows at one column hit different banks
    float m[kWaves][kStreamRows];
    float l[kWaves][kStreamRows];
    __attribute__((aligned(16))) float o[kWaves][kStreamRows][kStride];
};
// Tiles of 16 KiB: 64 keys of bf16, 32 of f32.
constexpr int kTileBytes = 16384;
struct BlockShared {
    __attribute__((aligned(1024))) uint8_t k[2][kTileBytes];
    __attribute__((aligned(1024))) uint8_t v[2][kTileBytes];
    int again[kWaves];
};

// One wave step's K or V fragments of a lane: kKeys keys in halves of 16.
template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
    static constexpr int kKeys = 32, kSlots = 8;
    u32x4_v k[2][4];  // [half][32-dim step]: row 16 half + i, dims 32 t + 8 g ..
    u32x4_v v[8];     // [e]: row 16 (e / 4) + 4 g + e % 4, dims 8 i ..
};
template <> struct Frag<float> {
    static constexpr int kKeys = 16, kSlots = 4;
    u32x4_v k[8];     // [16-dim step]: row i, dims 16 t + 4 g ..
    u32x4_v v[4][2];  // [e][d]: row 4 g + e, dims 64 d + 4 i ..
};

__device__ __forceinline__ void load_k(Frag<bf16_t>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t) f.k[h][t] = buf_load16(r, (16 * h + i) * 256 + 64 * t + 16 * g);
}
__device__ __forceinline__ void load_v(Frag<bf16_t>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = buf_load16(r, (16 * (e >> 2) + 4 * g + (e & 3)) * 256 + 16 * i);
}
__device__ __forceinline__ void load_k(Frag<float>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int t = 0; t < 8; ++t) f.k[t] = buf_load16(r, i * 512 + 64 * t + 16 * g);
}
__device__ __forceinline__ void load_v(Frag<float>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < 2; ++d) f.v[e][d] = buf_load16(r, (4 * g + e) * 512 + 256 * d + 16 * i);
}

// A query row's fragment: the K fragment's dims.
template <typename T> struct QFrag {
    static constexpr int kSteps = kHeadDim * (int)sizeof(T) / 64;
    u32x4_v q[kSteps];
    __device__ __forceinline__ void load(const T* row, int g) {
#pragma unroll
        for (int t = 0; t < kSteps; ++t) q[t] = reinterpret_cast<const u32x4_v*>(row)[4 * t + g];
    }
};

// s[4 h + r]: the raw score of key 16 h + 4 g + r for query row i.
__device__ __forceinline__ void scores(const Frag<bf16_t>& f, const QFrag<bf16_t>& q, float (&s)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f32x4_v a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t) a = mfma(f.k[h][t], q.q[t], a);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * h + r] = a[r];
    }
}
__device__ __forceinline__ void scores(const Frag<float>& f, const QFrag<float>& q, float (&s)[4]) {
    f32x4_v a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int d = 0; d < 4; ++d) a = mfma(__uint_as_float(f.k[t][d]), __uint_as_float(q.q[t][d]), a);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = a[r];
}

// The V operand of product n: bf16 keys in pairs, dims 8 m + n; f32 dims 64 (n / 4) +
// 4 m + n % 4.
__device__ __forceinline__ u32x4_v v_operand(const Frag<bf16_t>& f, int n) {
    u32x4_v a;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        a[w] = __builtin_amdgcn_perm(f.v[2 * w + 1][n >> 1], f.v[2 * w][n >> 1], n & 1 ? 0x07060302u : 0x05040100u);
    return a;
}
__device__ __forceinline__ float v_operand(const Frag<float>& f, int e, int n) {
    return __uint_as_float(f.v[e][n >> 2][n & 3]);
}
__device__ __forceinline__ bool any_nonfinite(const Frag<bf16_t>& f) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < 4; ++d)
            bad |= (f.v[e][d] & 0x7f80u) == 0x7f80u || (f.v[e][d] & 0x7f800000u) == 0x7f800000u;
    return bad;
}
__device__ __forceinline__ bool any_nonfinite(const Frag<float>& f) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < 8; ++d) bad |= (f.v[e][d >> 2][d & 3] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

// A query row's running state in a lane: o[n] holds product n's dims for m = 4 g + r;
// l is the sum over the lane's own keys.
template <typename T> struct Row {
    f32x4_v o[8];
    float l, m;
    __device__ __forceinline__ void clear() {
        const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n] = z;
        l = 0.f;
        m = kNoMax;
    }
    // Four consecutive dims from o[n0 .. n0 + 3][r] on (n0 = 0 or 4).
    static __device__ __forceinline__ int dim(int n0, int r, int g) {
        return sizeof(T) == 2 ? 32 * g + 8 * r + n0 : 16 * n0 + 16 * g + 4 * r;
    }
};

// Maximum over the four lane groups of a query row; every lane gets it.  (A row swap
// of a value with itself leaves each row's value in one result and its neighbour's in
// the other.)
__device__ __forceinline__ float groups_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// p = exp2(s c - m) of the step's scores, with m moved to the largest so far and o, l
// scaled to it.  Without a branch: one around the scaling makes the compiler copy o
// on both sides of it, in every step.
template <typename T, int N> __device__ __forceinline__ void softmax_step(Row<T>& st, float (&s)[N], float c) {
    float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    if constexpr (N == 8) mx = fmaxf(mx, fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    const float m = fmaxf(st.m, groups_max(mx) * c);
    const float a = fast_exp2(st.m - m);
    st.m = m;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        s[e] = fast_exp2(__builtin_fmaf(s[e], c, -m));
        sum += s[e];
    }
    st.l = __builtin_fmaf(st.l, a, sum);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[n][r] *= a;
}

// Sum over the four lane groups; every lane gets it.
__device__ __forceinline__ float groups_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// o += P V.
__device__ __forceinline__ void accumulate(Row<bf16_t>& st, const Frag<bf16_t>& f, const float (&p)[8]) {
    u32x4_v b;
#pragma unroll
    for (int w = 0; w < 4; ++w) b[w] = pack_bf16x2(p[2 * w], p[2 * w + 1]);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        st.o[n] = mfma(v_operand(f, n), b, st.o[n]);
        if (n & 1) __builtin_amdgcn_sched_barrier(0);  // two operands paired ahead, not all eight
    }
}
__device__ __forceinline__ void accumulate(Row<float>& st, const Frag<float>& f, const float (&p)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < 8; ++n) st.o[n] = mfma(v_operand(f, e, n), p[e], st.o[n]);
}

// The same where rows do not see every key and V holds an infinity or a NaN: p = 0 times
// it would reach the rows that do not see the key, so the keys are taken one by one and
// added only where they are seen.  The lane's row sees keys [from, to) of the step.
__device__ __forceinline__ void accumulate_each(Row<bf16_t>& st, const Frag<bf16_t>& f, const float (&p)[8], int g,
                                                int from, int to) {
    u32x4_v b;
#pragma unroll
    for (int w = 0; w < 4; ++w) b[w] = pack_bf16x2(p[2 * w], p[2 * w + 1]);
    const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const u32x4_v v = v_operand(f, n);
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {  // key 16 h + 4 g + r is slot 4 h + r of lane group g
            const int e = 4 * (key >> 4) + (key & 3);
            u32x4_v mask;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                mask[w] = g == ((key >> 2) & 3) && w == (e >> 1) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
            const f32x4_v d = mfma(v & mask, b & mask, z);
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] += key >= from && key < to ? d[r] : 0.f;
        }
    }
}
__device__ __forceinline__ void accumulate_each(Row<float>& st, const Frag<float>& f, const float (&p)[4], int g,
                                                int from, int to) {
    const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
            const int mine = g == (key >> 2) ? key & 3 : -1;
            float pk = 0.f, vk = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pk = e == mine ? p[e] : pk;
                vk = e == mine ? v_operand(f, e, n) : vk;
            }
            const f32x4_v d = mfma(vk, pk, z);
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] += key >= from && key < to ? d[r] : 0.f;
        }
    }
}

// A row sees keys [lo, hi) only: the others' scores vanish.
template <int N> __device__ __forceinline__ void mask_step(float (&s)[N], int j, int g, int lo, int hi) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int key = j + 16 * (e >> 2) + 4 * g + (e & 3);
        s[e] = key >= lo && key < hi ? s[e] : -INFINITY;
    }
}

// ---- the stream form

template <typename T, bool SHARED>
__device__ __forceinline__ void attend_stream(const Args& a, StreamShared& sm, int seg, int kvh, int block, int chunk) {
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // uniform: buffer resources are scalar
    constexpr int kKeys = Frag<T>::kKeys, kSlots = Frag<T>::kSlots;
    const Segment<SHARED> sg(a, seg);
    const int row0 = block * kStreamRows;
    if (row0 >= sg.n_rows) return;
    const int per = SHARED ? a.shared_chunk : a.own_chunk, lo = sg.lo, begin = sg.base() + chunk * per;
    const Pages pages(a, sg.table_row, begin, lane);

    int hi;
    const int64_t at = sg.query(row0 + i, kvh, hi);
    QFrag<T> q;
    q.load(reinterpret_cast<const T*>(a.q) + (at < 0 ? 0 : at) * kHeadDim, g);
    const int end = min(begin + per, wave_max_int(hi));
    hi = min(hi, end);  // a step may reach past the chunk's end
    const int min_hi = wave_min_int(at < 0 ? end : hi);
    const bool direct = a.slots() == 1;
    if (begin >= end && !direct) return;  // the join reads no slot past a row's keys

    Row<T> st;
    st.clear();
    auto tile_at = [&](int j) __attribute__((always_inline)) { return pages.tile<T>(a, kvh, j, kKeys, end); };
    auto k_tile = [&](Frag<T>& f, const Pages::Tile& t) __attribute__((always_inline)) {
        load_k(f, tile_rsrc<T>(a.k, t), i, g);
    };
    auto v_tile = [&](Frag<T>& f, const Pages::Tile& t) __attribute__((always_inline)) {
        load_v(f, tile_rsrc<T>(a.v, t), i, g);
    };
    // Two steps' tiles are in flight: a step's K registers are loaded again, for the
    // step after the next, once its scores are taken, its V registers after its
    // product.  A step past the end loads nothing and sees no key.
    constexpr int kStride = kWaves * kKeys;
    const int j0 = begin + wave * kKeys;
    Frag<T> f[2];
    bool again = false;  // a key some rows do not see has an infinity or a NaN in V
    auto step = [&](Frag<T>& f, int j) __attribute__((always_inline)) {
        const Pages::Tile next = tile_at(j + 2 * kStride);
        float s[kSlots];
        scores(f, q, s);
        __builtin_amdgcn_sched_barrier(0);  // the loads take the registers just read, not new ones
        k_tile(f, next);
        if (j < lo || j + kKeys > min_hi) {
            mask_step(s, j, g, lo, hi);
            if (j < lo || min_hi < min(j + kKeys, end)) again = again || __any(any_nonfinite(f));
        }
        softmax_step(st, s, a.c);
        accumulate(st, f, s);
        __builtin_amdgcn_sched_barrier(0);
        v_tile(f, next);
    };
    {
        // In the steps' own order: the loop's first wait has to hold for both.
        const Pages::Tile t0 = tile_at(j0), t1 = tile_at(j0 + kStride);
        __builtin_amdgcn_sched_barrier(0);
        k_tile(f[0], t0);
        __builtin_amdgcn_sched_barrier(0);
        v_tile(f[0], t0);
        __builtin_amdgcn_sched_barrier(0);
        k_tile(f[1], t1);
        __builtin_amdgcn_sched_barrier(0);
        v_tile(f[1], t1);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (int j = j0; j < end; j += 2 * kStride) {
        step(f[0], j);
        step(f[1], j + kStride);
    }
    if (again) {  // the wave's keys once more, each added only to the rows that see it
        st.clear();
        for (int j = j0; j < end; j += kStride) {
            const Pages::Tile tile = tile_at(j);
            k_tile(f[0], tile);
            v_tile(f[0], tile);
            float s[kSlots];
            scores(f[0], q, s);
            mask_step(s, j, g, lo, hi);
            softmax_step(st, s, a.c);
            accumulate_each(st, f[0], s, g, lo - j, hi - j);
        }
    }

    // Join the waves: m first, then o and l at the common m.
    const float l = groups_sum(st.l);
    if (g == 0) sm.m[wave][i] = st.m;
    __syncthreads();
    {
        const float m = fmaxf(fmaxf(sm.m[0][i], sm.m[1][i]), fmaxf(sm.m[2][i], sm.m[3][i]));
        const float w = fast_exp2(st.m - m);
        if (g == 0) sm.l[wave][i] = w * l;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n0 = 0; n0 < 8; n0 += 4) {
                const float x[4] = {w * st.o[n0][r], w * st.o[n0 + 1][r], w * st.o[n0 + 2][r], w * st.o[n0 + 3][r]};
                store4(&sm.o[wave][i][Row<T>::dim(n0, r, g)], x);
            }
    }
    __syncthreads();
    // 16 threads per row, 8 dims each.
    const int r = tid >> 4, d = 8 * (tid & 15);
    int to;
    const int64_t place = sg.query(row0 + r, kvh, to);
    if (place < 0) return;
    float x[8];
    load8(&sm.o[0][r][d], x);
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        float y[8];
        load8(&sm.o[w][r][d], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += y[e];
    }
    const float m = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
    const float sum = (sm.l[0][r] + sm.l[1][r]) + (sm.l[2][r] + sm.l[3][r]);
    if (direct) {
        const typename Segment<SHARED>::Row w = sg.row(row0 + r);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to <= lo ? 0.f : x[e] / sum;
        store8(reinterpret_cast<T*>(a.out) + (((int64_t)w.b * a.S + w.s) * a.Hq + kvh * a.G + w.h) * kHeadDim + d, x);
    } else {
        const int64_t slot = place * a.slots() + (SHARED ? 0 : a.shared_splits) + chunk;
        store8(a.ws_o + slot * kHeadDim + d, x);
        if (d == 0) a.ws_ml[slot] = make_float2(m, sum);
    }
}

// ---- the block form

// LDS tiles keep the pools' rows with their 16-byte chunks XOR-permuted by the row, so
// that neither 16 rows read at one chunk (K) nor whole or transposed rows (V) meet in a
// bank.  bf16 rows of 16 chunks: by the row's two 2-bit halves swapped (transposed
// reads take 4 rows x 4 chunks); f32 rows of 32 chunks: by the row mod 16.
template <typename T> __device__ __forceinline__ int swizzle(int row) {
    return sizeof(T) == 2 ? ((row & 3) << 2) | ((row >> 2) & 3) : row & 15;
}
// The byte of a tile's row its 16-byte chunk c sits at.
template <typename T> __device__ __forceinline__ int chunk_at(int row, int c) {
    return row * kHeadDim * (int)sizeof(T) + 16 * (c ^ swizzle<T>(row));
}

// One tile into LDS: a wave copies 4 KiB of K and of V, 1 KiB an instruction, lane l
// the 16 bytes at 16 l of it.
template <typename T>
__device__ __forceinline__ void stage(const Args& a, const Pages::Tile& t, uint8_t* k, uint8_t* v, int wave, int lane) {
    constexpr int kRow = kHeadDim * (int)sizeof(T);
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc<T>(a.k, t), rv = tile_rsrc<T>(a.v, t);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int at = 4096 * wave + 1024 * x + 16 * lane, row = at / kRow;
        const int from = row * kRow + 16 * (((at % kRow) / 16) ^ swizzle<T>(row));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, k + 4096 * wave + 1024 * x, 16, from, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, v + 4096 * wave + 1024 * x, 16, from, 0, 0, 0);
    }
}
// Wait for the wave's own copies (expcnt and lgkmcnt at their maxima).
__device__ __forceinline__ void wait_copies() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ u32x4_v lds_read16(const uint8_t* p) { return *(const u32x4_v*)p; }
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_v;
typedef __attribute__((address_space(3))) s16x4_v lds_s16x4_v;
// Within 16 lanes, lane x gets column x of the 4 rows x 16 columns of bf16 that the
// lanes point at (lane x: 4 columns from 4 (x % 4) on of row x / 4).
__device__ __forceinline__ uint2 lds_read_tr16(const uint8_t* p) {
    const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_v*)(uintptr_t)at));
}
__device__ __forceinline__ f32x16_v mfma(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0,
                                                   0, 0);
}
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

// A wave's share of a block: Q, o, m and l of its rows, and one tile's work.
template <typename T> struct BlockWave;

// bf16: 32 rows; lane (n, h) = (lane % 32, lane / 32) holds, for row n, keys 32 b +
// 8 (r / 4) + 4 h + r % 4 in register r of score block b, and dims 32 d + 8 (r / 4) +
// 4 h + r % 4 in register r of o[d].
template <> struct BlockWave<bf16_t> {
    static constexpr int kRows = 32, kKeys = 64;
    u32x4_v q[8];
    f32x16_v o[4];
    float m, l;
    int n, h, vrow, vcol;
    __device__ __forceinline__ explicit BlockWave(int lane) : n(lane & 31), h(lane >> 5) {
        vrow = 4 * h + ((lane & 15) >> 2);
        vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
        m = kNoMax;
        l = 0.f;
    }
    __device__ __forceinline__ void load_q(const bf16_t* row) {
#pragma unroll
        for (int t = 0; t < 8; ++t) q[t] = reinterpret_cast<const u32x4_v*>(row)[2 * t + h];
    }
    // V^T, dims 32 d + lane % 32, of keys 16 s + 8 e + 4 h + (0 .. 3), e = 0, 1.
    __device__ __forceinline__ u32x4_v v_frag(const uint8_t* v, int s, int d) const {
        const int r0 = 16 * s + vrow, c = (32 * d + vcol) >> 3, byte = 2 * (vcol & 7);
        const uint2 x = lds_read_tr16(v + chunk_at<bf16_t>(r0, c) + byte);
        const uint2 y = lds_read_tr16(v + chunk_at<bf16_t>(r0 + 8, c) + byte);
        return u32x4_v{x.x, x.y, y.x, y.y};
    }
    template <bool EDGE, bool EACH>
    __device__ __forceinline__ void tile(const uint8_t* k, const uint8_t* v, int j, int lo, int hi, float c) {
        f32x16_v s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[b] = mfma(lds_read16(k + chunk_at<bf16_t>(32 * b + n, 2 * t + h)), q[t], s[b]);
        if constexpr (EDGE) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = j + 32 * b + 8 * (r >> 2) + 4 * h + (r & 3);
                    s[b][r] = key >= lo && key < hi ? s[b][r] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        const float next = fmaxf(m, halves_max(mx) * c);
        const float w = fast_exp2(m - next);
        m = next;
        float sum = 0.f;
        u32x4_v p[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = fast_exp2(__builtin_fmaf(s[b][r], c, -m)), y = fast_exp2(__builtin_fmaf(s[b][r + 1], c, -m));
                sum += x + y;
                p[2 * b + (r >> 3)][(r & 7) >> 1] = pack_bf16x2(x, y);
            }
        l = __builtin_fmaf(l, w, sum);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= w;
        if constexpr (!EACH) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] = mfma(v_frag(v, t, d), p[t], o[d]);
        } else {  // see accumulate_each; key 16 t + 8 e + 4 h + x is slot 4 e + x of half h in step t
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const u32x4_v x = v_frag(v, t, d);
#pragma unroll 1
                    for (int key = 0; key < 16; ++key) {
                        const int e = 4 * (key >> 3) + (key & 3), at = j + 16 * t + key;
                        u32x4_v mask;
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            mask[y] = h == ((key >> 2) & 1) && y == (e >> 1) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
                        f32x16_v z;
#pragma unroll
                        for (int r = 0; r < 16; ++r) z[r] = 0.f;
                        z = mfma(x & mask, p[t] & mask, z);
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] += at >= lo && at < hi ? z[r] : 0.f;
                    }
                }
        }
    }
    __device__ __forceinline__ float sum() const { return halves_sum(l); }
    template <class F> __device__ __forceinline__ void rows4(F f) const {  // f(dim, four consecutive values)
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const float x[4] = {o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
                f(32 * d + 2 * r + 4 * h, x);
            }
    }
    static __device__ __forceinline__ int row(int lane) { return lane & 31; }
    __device__ __forceinline__ bool writes_ml() const { return h == 0; }
};

// f32: 16 rows, the stream's layout with the fragments from LDS.
template <> struct BlockWave<float> {
    static constexpr int kRows = 16, kKeys = 32;
    QFrag<float> q;
    Row<float> st;
    int i, g;
    __device__ __forceinline__ explicit BlockWave(int lane) : i(lane & 15), g(lane >> 4) {}
    __device__ __forceinline__ void clear() { st.clear(); }
    __device__ __forceinline__ void load_q(const float* row) { q.load(row, g); }
    template <bool EDGE, bool EACH>
    __device__ __forceinline__ void tile(const uint8_t* k, const uint8_t* v, int j, int lo, int hi, float c) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Frag<float> f;
#pragma unroll
            for (int t = 0; t < 8; ++t) f.k[t] = lds_read16(k + chunk_at<float>(16 * half + i, 4 * t + g));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < 2; ++d) f.v[e][d] = lds_read16(v + chunk_at<float>(16 * half + 4 * g + e, 16 * d + i));
            float s[4];
            scores(f, q, s);
            if constexpr (EDGE) mask_step(s, j + 16 * half, g, lo, hi);
            softmax_step(st, s, c);
            if constexpr (EACH) accumulate_each(st, f, s, g, lo - j - 16 * half, hi - j - 16 * half);
            else accumulate(st, f, s);
        }
    }
    __device__ __forceinline__ float sum() const { return groups_sum(st.l); }
    template <class F> __device__ __forceinline__ void rows4(F f) const {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n0 = 0; n0 < 8; n0 += 4) {
                const float x[4] = {st.o[n0][r], st.o[n0 + 1][r], st.o[n0 + 2][r], st.o[n0 + 3][r]};
                f(Row<float>::dim(n0, r, g), x);
            }
    }
    static __device__ __forceinline__ int row(int lane) { return lane & 15; }
    __device__ __forceinline__ bool writes_ml() const { return g == 0; }
};
template <typename T> __device__ __forceinline__ float wave_m(const BlockWave<T>& w) {
    if constexpr (sizeof(T) == 2) return w.m;
    else return w.st.m;
}

// Whether a V tile holds an infinity or a NaN (the whole tile, by one wave).
template <typename T> __device__ __forceinline__ bool tile_nonfinite(const uint8_t* v, int lane) {
    constexpr uint32_t kExp = sizeof(T) == 2 ? 0x7f80u : 0;
    bool bad = false;
#pragma unroll 4
    for (int x = 0; x < kTileBytes / 1024; ++x) {
        const u32x4_v u = lds_read16(v + 1024 * x + 16 * lane);
#pragma unroll
        for (int y = 0; y < 4; ++y)
            bad |= (u[y] & 0x7f800000u) == 0x7f800000u || (kExp && (u[y] & kExp) == kExp);
    }
    return __any(bad);
}

template <typename T, bool SHARED>
__device__ __forceinline__ void attend_block(const Args& a, BlockShared& sm, int seg, int kvh, int block, int chunk) {
    typedef BlockWave<T> Wave;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Segment<SHARED> sg(a, seg);
    const int row0 = block * kBlockRows<T>;
    if (row0 >= sg.n_rows) return;
    const int per = SHARED ? a.shared_chunk : a.own_chunk, lo = sg.lo, begin = sg.base() + chunk * per;
    const Pages pages(a, sg.table_row, begin, lane);
    // Keys any row of the block can see: a group's shared rows, or what the block's last
    // query sees.
    int end = begin + per;
    if constexpr (SHARED) end = min(end, sg.hi);
    else end = min(end, a.limit(seg, (min(row0 + kBlockRows<T>, sg.n_rows) - 1) / a.G));
    end = __builtin_amdgcn_readfirstlane(end);
    const bool direct = a.slots() == 1;
    if (begin >= end && !direct) return;

    Wave w(lane);
    int hi;
    const int r = row0 + Wave::kRows * wave + Wave::row(lane);
    const int64_t at = sg.query(r, kvh, hi);
    w.load_q(reinterpret_cast<const T*>(a.q) + (at < 0 ? 0 : at) * kHeadDim);
    w.clear();
    hi = min(hi, end);
    const int max_hi = wave_max_int(hi), min_hi = wave_min_int(at < 0 ? end : hi);

    // Tile t is computed while tile t + 1 comes in: its buffer's last readers passed the
    // barrier before the copies are issued.
    const int n = max(0, (end - begin + Wave::kKeys - 1) / Wave::kKeys);
    auto issue = [&](int t) __attribute__((always_inline)) {
        stage<T>(a, pages.tile<T>(a, kvh, begin + t * Wave::kKeys, Wave::kKeys, end), sm.k[t & 1], sm.v[t & 1], wave, lane);
    };
    auto walk = [&](auto each) __attribute__((always_inline)) {
        constexpr bool kEach = decltype(each)::value;
        bool bad = false;
        if (n > 0) issue(0);
        for (int t = 0; t < n; ++t) {
            wait_copies();
            __syncthreads();
            if (t + 1 < n) issue(t + 1);
            const int j = begin + t * Wave::kKeys;
            const uint8_t *k = sm.k[t & 1], *v = sm.v[t & 1];
            if (j >= max_hi) continue;  // none of the wave's rows sees the tile
            if constexpr (kEach) {
                w.template tile<true, true>(k, v, j, lo, hi, a.c);
            } else if (j < lo || j + Wave::kKeys > min_hi) {
                if (j < lo || min_hi < min(j + Wave::kKeys, end)) bad = bad || tile_nonfinite<T>(v, lane);
                w.template tile<true, false>(k, v, j, lo, hi, a.c);
            } else {
                w.template tile<false, false>(k, v, j, lo, hi, a.c);
            }
        }
        return bad;
    };
    const bool bad = walk(std::false_type());
    sm.again[wave] = bad;
    __syncthreads();
    if (sm.again[0] | sm.again[1] | sm.again[2] | sm.again[3]) {  // once more, keys one by one
        w.clear();
        walk(std::true_type());
    }
    const float l = w.sum();
    if (at < 0) return;
    if (direct) {
        const typename Segment<SHARED>::Row x = sg.row(r);
        T* out = reinterpret_cast<T*>(a.out) + (((int64_t)x.b * a.S + x.s) * a.Hq + kvh * a.G + x.h) * kHeadDim;
        w.rows4([&](int d, const float(&y)[4]) {
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = hi <= lo ? 0.f : y[e] / l;
            store4(out + d, z);
        });
    } else {
        const int64_t slot = at * a.slots() + (SHARED ? 0 : a.shared_splits) + chunk;
        w.rows4([&](int d, const float(&y)[4]) { store4(a.ws_o + slot * kHeadDim + d, y); });
        if (w.writes_ml()) a.ws_ml[slot] = make_float2(wave_m(w), l);
    }
}

// A role's item x of `units` (segment, kv head, chunk) units with `blocks` row blocks
// each: ids that are equal mod 8 run on one XCD, which so gets the blocks of a unit,
// one after the other, and reads their keys through its own L2.
struct Item {
    int block, kvh, seg, chunk;
    bool ok;
    __device__ __forceinline__ Item(int x, int blocks, int Hkv, int segs, int chunks) {
        const int c = x / (8 * blocks), rem = x - c * 8 * blocks;
        block = rem >> 3;
        int unit = 8 * c + (rem & 7);
        ok = unit < segs * Hkv * chunks;
        kvh = unit % Hkv;
        unit /= Hkv;
        seg = unit % segs;
        chunk = unit / segs;
    }
};

// grid: the shared role's items, then the own role's.
template <typename T, bool SHARED_BLOCK, bool OWN_BLOCK>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_attn_kernel(Args a) {
    __shared__ union {
        StreamShared stream;
        typename std::conditional<SHARED_BLOCK || OWN_BLOCK, BlockShared, int>::type block;
    } sm;
    if ((int)blockIdx.x < a.shared_items) {
        const Item x(blockIdx.x, a.shared_tiles, a.Hkv, a.n_groups, a.shared_splits);
        if (!x.ok) return;
        if constexpr (SHARED_BLOCK) attend_block<T, true>(a, sm.block, x.seg, x.kvh, x.block, x.chunk);
        else attend_stream<T, true>(a, sm.stream, x.seg, x.kvh, x.block, x.chunk);
    } else {
        const Item x(blockIdx.x - a.shared_items, a.own_tiles, a.Hkv, a.B, a.own_splits);
        if (!x.ok) return;
        if constexpr (OWN_BLOCK) attend_block<T, false>(a, sm.block, x.seg, x.kvh, x.block, x.chunk);
        else attend_stream<T, false>(a, sm.stream, x.seg, x.kvh, x.block, x.chunk);
    }
}

// Join a query row's chunks: one wave per row, lane l owns dims 2 l, 2 l + 1.
template <typename T> __global__ __launch_bounds__(256) void shared_join_kernel(Args a, int64_t n_rows) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= n_rows) return;
    const int64_t bh = row / a.S;
    const int s = (int)(row - bh * a.S);
    const int b = (int)(bh / a.Hq), h = (int)(bh - (int64_t)b * a.Hq);
    const int limit = a.limit(b, s), shared = a.shared_of(b);
    const int seen = min(shared, limit);
    const int n_shared = seen > 0 ? (seen + a.shared_chunk - 1) / a.shared_chunk : 0;
    const int own = limit - Args::own_base(shared);
    const int n_own = limit > shared ? min((own + a.own_chunk - 1) / a.own_chunk, a.own_splits) : 0;
    const int n = n_shared + n_own;
    const float2* ml = a.ws_ml + row * a.slots();
    const float2* o = reinterpret_cast<const float2*>(a.ws_o + row * a.slots() * kHeadDim) + lane;
    // slot of the c-th chunk the row sees
    auto slot = [&](int c) { return c < n_shared ? c : a.shared_splits + c - n_shared; };
    float mx = kNoMax;
    for (int c = lane; c < n; c += 64) mx = fmaxf(mx, ml[slot(c)].x);
    mx = wave_max(mx);
    float den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int c0 = 0; c0 < n; c0 += 64) {
        float w = 0.f;
        if (c0 + lane < n) {
            const float2 t = ml[slot(c0 + lane)];
            w = fast_exp2(t.x - mx);
            den += w * t.y;
        }
        for (int c = c0; c < min(n, c0 + 64); ++c) {
            const float wc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), c - c0));
            const float2 t = o[(int64_t)slot(c) * (kHeadDim / 2)];
            x0 += wc * t.x;
            x1 += wc * t.y;
        }
    }
    den = wave_sum(den);
    T* out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.S + s) * a.Hq + h) * kHeadDim + 2 * lane;
    Elem<T>::store(out, n ? x0 / den : 0.f);
    Elem<T>::store(out + 1, n ? x1 / den : 0.f);
}

// How a call is cut: the forms, row blocks and key chunks of both roles.
struct Plan {
    bool share, shared_block, own_block;
    int shared_tiles, own_tiles, shared_chunk, own_chunk, shared_splits, own_splits;
    int64_t shared_items, own_items;
    size_t ml_off, total;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool make_plan(int n_groups, int max_group, int64_t max_shared, int64_t max_own, int B, int S, int Hq, int Hkv, int dtype,
               Plan* p) {
    const int64_t R = (int64_t)S * (Hq / Hkv), M = (int64_t)max_group * R;
    const int block_rows = dtype == CRANE_HIP_F32 ? kBlockRows<float> : kBlockRows<bf16_t>;
    // A sequence that fills whole row blocks by itself has nothing to gain.
    p->share = n_groups > 0 && max_shared > 0 && R < block_rows;
    p->shared_block = M > kStreamRows;
    p->own_block = R > kStreamRows;
    const int64_t st = p->share ? ceil_div(M, p->shared_block ? block_rows : kStreamRows) : 0;
    const int64_t ot = ceil_div(R, p->own_block ? block_rows : kStreamRows);
    // own chunk 0 starts on a multiple of kAlign
    const int64_t shared = p->share ? max_shared : 0, own = max_own + (p->share ? kAlign : max_shared);
    // Rows times keys of all items, spread over 1024 workgroups (4 per CU).
    const int64_t total = (int64_t)n_groups * Hkv * st * shared + (int64_t)B * Hkv * ot * own;
    int64_t chunk = ceil_div(ceil_div(total, 1024), kMinChunk) * kMinChunk;
    chunk = chunk < 2 * kMinChunk ? 2 * kMinChunk : chunk > kMaxChunk ? kMaxChunk : chunk;
    p->shared_chunk = p->own_chunk = (int)chunk;
    const int64_t ss = ceil_div(shared, chunk), os = ceil_div(own, chunk);
    p->shared_items = 8 * st * ceil_div((int64_t)n_groups * Hkv * ss, 8);
    p->own_items = 8 * ot * ceil_div((int64_t)B * Hkv * os, 8);
    const int64_t rows = (int64_t)B * Hq * S;
    if (rows > 0x7fffffffLL || st > 0x7fffffffLL || ot > 0x7fffffffLL || p->shared_items + p->own_items > 0x7fffffffLL)
        return false;
    p->shared_tiles = (int)st;
    p->own_tiles = (int)ot;
    p->shared_splits = (int)ss;
    p->own_splits = (int)os;
    const int64_t slots = ss + os;
    const size_t up = 255;
    p->ml_off = ((size_t)rows * slots * kHeadDim * sizeof(float) + up) & ~up;
    p->total = slots > 1 ? p->ml_off + (size_t)rows * slots * sizeof(float2) : 0;
    return true;
}

template <typename T> int launch(Args& a, const Plan& p, int64_t n_rows, hipStream_t st) {
    const dim3 grid((unsigned)(p.shared_items + p.own_items)), threads(64 * kWaves);
    if (p.own_block)
        hipLaunchKernelGGL((shared_attn_kernel<T, true, true>), grid, threads, 0, st, a);
    else if (p.share && p.shared_block)
        hipLaunchKernelGGL((shared_attn_kernel<T, true, false>), grid, threads, 0, st, a);
    else
        hipLaunchKernelGGL((shared_attn_kernel<T, false, false>), grid, threads, 0, st, a);
    int rc = launch_status(hipGetLastError());
    if (rc || p.shared_splits + p.own_splits == 1) return rc;
    hipLaunchKernelGGL((shared_join_kernel<T>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, st, a, n_rows);
    return launch_status(hipGetLastError());
}

// The checks both entry points make of the sizes.
int check_sizes(int n_groups, int max_group, int64_t max_shared, int64_t max_own, int B, int S, int Hq, int Hkv, int D,
                int dtype) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return CRANE_HIP_E_INVALID;
    if (Hq % Hkv != 0) return CRANE_HIP_E_GQA;
    if (B > 65535 || n_groups < 0 || n_groups > B || max_group < 0 || max_group > B) return CRANE_HIP_E_INVALID;
    // a chunk's bounds stay within 31 bits
    if (max_shared < 0 || max_own < 0 || max_shared > 0x7fffffffLL - 2 * kMaxChunk ||
        max_own > 0x7fffffffLL - 2 * kMaxChunk - max_shared)
        return CRANE_HIP_E_INVALID;
    if (n_groups > 0 && max_group == 0) return CRANE_HIP_E_INVALID;
    if (n_groups == 0 && max_shared > 0) return CRANE_HIP_E_INVALID;
    return CRANE_HIP_OK;
}

}  // namespace
}  // namespace crane

using namespace crane;

extern "C" size_t crane_hip_attn_shared_workspace(int n_groups, int max_group, int64_t max_shared, int64_t max_own, int B,
                                                  int S, int Hq, int Hkv, int D, int dtype) {
    if (check_sizes(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, D, dtype) || B == 0 || S == 0) return 0;
    Plan p;
    return make_plan(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, dtype, &p) ? p.total : 0;
}

extern "C" int crane_hip_attn_shared_paged(const void* q, const void* k_pool, const void* v_pool, int64_t n_pages,
                                           int page_rows, const int32_t* block_table, int64_t table_stride,
                                           const int32_t* kv_len, int64_t max_kv, const int32_t* shared_rows,
                                           const int32_t* groups, const int32_t* members, int n_groups, int max_group,
                                           int64_t max_shared, int64_t max_own, int B, int S, int Hq, int Hkv, int D,
                                           float scale, int flags, void* workspace, size_t ws_bytes, void* out,
                                           int dtype, void* stream) {
    int rc = check_sizes(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, D, dtype);
    if (rc) return rc;
    if (flags & ~CRANE_HIP_PREFILL_CAUSAL) return CRANE_HIP_E_INVALID;
    if (!(scale > 0.0f) || !__builtin_isfinite(scale)) return CRANE_HIP_E_INVALID;
    rc = check_paged(n_pages, page_rows, block_table, table_stride, Hkv);
    if (rc) return rc;
    if (max_kv <= 0) return CRANE_HIP_E_INVALID;
    if (max_kv > table_stride * page_rows) return CRANE_HIP_E_CAPACITY;
    if (max_shared > max_kv || max_own > max_kv) return CRANE_HIP_E_CAPACITY;
    if (B == 0 || S == 0) return CRANE_HIP_OK;
    if (!q || !k_pool || !v_pool || !kv_len || !out) return CRANE_HIP_E_INVALID;
    if (n_groups > 0 && (!shared_rows || !groups || !members)) return CRANE_HIP_E_INVALID;
    if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) ||
        (n_groups > 0 && !aligned16(groups)))
        return CRANE_HIP_E_ALIGN;
    Plan p;
    if (!make_plan(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, dtype, &p)) return CRANE_HIP_E_INVALID;
    if (p.total && (!workspace || ws_bytes < p.total || !aligned16(workspace))) return CRANE_HIP_E_WORKSPACE;
    Args a;
    a.q = q;
    a.k = k_pool;
    a.v = v_pool;
    a.out = out;
    a.rows = PagedRows{block_table, table_stride, n_pages, page_rows};
    a.kv_len = kv_len;
    a.shared = p.share ? shared_rows : nullptr;
    a.groups = groups;
    a.members = members;
    a.n_groups = n_groups;
    a.max_group = max_group;
    a.max_shared = (int)max_shared;
    a.B = B;
    a.S = S;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.max_kv = (int)max_kv;
    a.causal = flags & CRANE_HIP_PREFILL_CAUSAL;
    a.c = scale * kLog2e;
    a.shared_chunk = p.shared_chunk;
    a.own_chunk = p.own_chunk;
    a.shared_splits = p.shared_splits;
    a.own_splits = p.own_splits;
    a.shared_tiles = p.shared_tiles;
    a.own_tiles = p.own_tiles;
    a.shared_items = (int)p.shared_items;
    a.ws_o = (float*)workspace;
    a.ws_ml = (float2*)((char*)workspace + p.ml_off);
    const int64_t n_rows = (int64_t)B * Hq * S;
    const hipStream_t st = (hipStream_t)stream;
    return dtype == CRANE_HIP_F32 ? launch<float>(a, p, n_rows, st) : launch<bf16_t>(a, p, n_rows, st);
}
