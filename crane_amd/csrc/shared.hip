// shared.hip -- attention over a paged KV cache in which groups of sequences share
// their first rows (gfx950); the C ABI is include/crane_shared.h.
//
// Sequence b has n = kv_len[b] rows; its query i sees rows [0, L), L = n - S + 1 + i
// (causal) or n.  With s_j = scale q . k_j over any set J of keys,
//     m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j,
// and the results of disjoint sets join as o = sum w_J o_J / sum w_J l_J, w_J =
// exp(m_J - max m).  So a group's shared rows are one set for all of its members'
// queries together, every sequence's own rows another, and each is cut into chunks
// for parallelism.  A workgroup takes one chunk for 16 query rows of one kv head:
//   shared: rows are (member, query, head of the GQA group) of the whole group;
//   own:    rows are (query, head) of one sequence.
// Its 4 waves take the chunk's 32-key tiles in turn, each with its own m, l, o, joined
// through LDS at the end; a second kernel joins the chunks.
//
// A wave's tile (bf16, v_mfma_f32_16x16x32_bf16): S^T = K Q^T with K rows as A and
// query rows as B, so lane (i, g) = (lane % 16, lane / 16) holds, for query row i, keys
// 4 g + r of two 16-key halves.  Those 8 values, rounded to bf16, are the B operand
// P^T of O^T = V^T P^T as they stand: the order of the 32 keys inside the k index is
// free as long as V follows it, so lane group g takes V rows 4 g + r of both halves.
// It reads dims [8 i, 8 i + 8) of each (whole 256-byte rows per 16 lanes) and v_perm
// pairs them into the A operand of eight products, product n giving dims 8 m + n: a
// lane ends with dims [32 g, 32 g + 32) of its query row.  K and V go from memory to
// registers; nothing is staged.  f32 runs the same layout on v_mfma_f32_16x16x4_f32,
// where k = 4 g-slots take one key (or dim) of every lane group and no pairing is
// needed.
//
// The reference m of a row moves lazily: p = exp2(s c - m), c = scale log2 e, against
// the row's current m, and only when some lane's score passes it by kLag (2^8 in p)
// are the four lane groups' maxima joined and o, l scaled.  m cancels between o and l.
// bf16: l sums the rounded p (a product with ones), so numerator and denominator see
// the same weights.
#include <float.h>

#include "common.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr int kTile = 32;          // keys per wave step
constexpr int kWaves = 4;
constexpr float kLag = 8.0f;       // log2 units a row's scores may pass its m before m moves
constexpr float kNoMax = -FLT_MAX; // m before the first key (finite: exp2(-inf - m) is 0, not NaN)
constexpr int kMaxChunk = 8192;    // rows per chunk: its pages' ids fit one lane each
constexpr int kMinChunk = kTile * kWaves;

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
    const int32_t *kv_len, *shared, *group_start, *group_seq;
    int n_groups, max_group, max_shared;
    int B, S, Hq, Hkv, G;     // G = Hq / Hkv heads per kv head
    int max_kv, causal;
    float c;                  // scale log2 e
    int shared_chunk, own_chunk;    // rows per chunk
    int shared_splits, own_splits;  // chunks
    int shared_tiles, own_tiles;    // row blocks per (group or sequence, kv head)
    int shared_items;               // workgroups of the shared role, which come first
    float* ws_o;              // [B Hq S, slots, D] f32, unnormalised
    float2* ws_ml;            // [B Hq S, slots] (m, l)
    __device__ __forceinline__ int slots() const { return shared_splits + own_splits; }
    __device__ __forceinline__ int len(int b) const { return max(0, min(kv_len[b], max_kv)); }
    __device__ __forceinline__ int shared_of(int b) const { return shared ? max(0, min(shared[b], max_shared)) : 0; }
    // Rows query s of sequence b sees.
    __device__ __forceinline__ int limit(int b, int s) const { return causal ? len(b) - S + 1 + s : len(b); }
    // First row of own chunk 0: chunk bounds sit on tile bounds.
    __device__ __forceinline__ static int own_base(int shared_rows) { return shared_rows & ~(kTile - 1); }
};

template <typename T, int RT> struct Shared {
    static constexpr int kStride = kHeadDim + 4;  // f32 per row: 16 rows at one column hit different banks
    float m[kWaves][16 * RT];
    float l[kWaves][16 * RT];
    __attribute__((aligned(16))) float o[kWaves][16 * RT][kStride];
};

// One 32-key tile's K or V fragments of a lane.
template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
    u32x4_v k[2][4];  // [half][32-dim step]: row 16 half + i, dims 32 t + 8 g ..
    u32x4_v v[8];     // [e]: row 16 (e / 4) + 4 g + e % 4, dims 8 i ..
};
template <> struct Frag<float> {
    u32x4_v k[2][8];  // [half][16-dim step]: row 16 half + i, dims 16 t + 4 g ..
    u32x4_v v[8][2];  // [e]: the same rows, dims 8 i ..
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
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 8; ++t) f.k[h][t] = buf_load16(r, (16 * h + i) * 512 + 64 * t + 16 * g);
}
__device__ __forceinline__ void load_v(Frag<float>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < 2; ++d)
            f.v[e][d] = buf_load16(r, (16 * (e >> 2) + 4 * g + (e & 3)) * 512 + 32 * i + 16 * d);
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
__device__ __forceinline__ void scores(const Frag<float>& f, const QFrag<float>& q, float (&s)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f32x4_v a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) a = mfma(__uint_as_float(f.k[h][t][d]), __uint_as_float(q.q[t][d]), a);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * h + r] = a[r];
    }
}

// The V operand of product n (dims 8 m + n): bf16 keys in pairs.
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
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < 8; ++d) bad |= (f.v[e][d >> 2][d & 3] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

// A query row's running state in a lane: o[n] holds dims 32 g + 8 r + n.  l: bf16 the
// full sum in every register, f32 the lane's own keys' part.
template <typename T> struct Row {
    static constexpr bool kBf16 = sizeof(T) == 2;
    f32x4_v o[8];
    f32x4_v l;
    float m;
    __device__ __forceinline__ void clear() {
        const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n] = z;
        l = z;
        m = kNoMax;
    }
    __device__ __forceinline__ float sum() const {
        if constexpr (kBf16) return l[0];
        float x = l[0];
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        return x;
    }
};

// p = exp2(s c - m) of the tile's 8 scores; m moves first where a score passes it by
// more than kLag.
template <typename T> __device__ __forceinline__ void softmax_step(Row<T>& st, float (&s)[8], float c) {
    float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    mx *= c;
    if (__any(mx > st.m + kLag)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m = fmaxf(st.m, mx);
        const float a = fast_exp2(st.m - m);
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] *= a;
#pragma unroll
        for (int r = 0; r < 4; ++r) st.l[r] *= a;
        st.m = m;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = fast_exp2(__builtin_fmaf(s[e], c, -st.m));
}

// o += P V and l += sum p.
__device__ __forceinline__ void accumulate(Row<bf16_t>& st, const Frag<bf16_t>& f, const float (&p)[8]) {
    u32x4_v b, one;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        b[w] = pack_bf16x2(p[2 * w], p[2 * w + 1]);
        one[w] = 0x3f803f80u;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) st.o[n] = mfma(v_operand(f, n), b, st.o[n]);
    st.l = mfma(one, b, st.l);
}
__device__ __forceinline__ void accumulate(Row<float>& st, const Frag<float>& f, const float (&p)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int n = 0; n < 8; ++n) st.o[n] = mfma(v_operand(f, e, n), p[e], st.o[n]);
        st.l[0] += p[e];
    }
}

// The same for a tile in which rows do not see every key and V holds an infinity or a
// NaN: p = 0 times it would reach the rows that do not see the key, so the keys are
// taken one by one and added only where they are seen.  The lane's row sees keys
// [from, to) of the tile.
__device__ __forceinline__ void accumulate_each(Row<bf16_t>& st, const Frag<bf16_t>& f, const float (&p)[8], int g,
                                                int from, int to) {
    u32x4_v b, one;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        b[w] = pack_bf16x2(p[2 * w], p[2 * w + 1]);
        one[w] = 0x3f803f80u;
    }
    const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int key = 0; key < kTile; ++key) {  // key 16 h + 4 g + r is slot 4 h + r of lane group g
        const int e = 4 * (key >> 4) + (key & 3);
        u32x4_v mask;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            mask[w] = g == ((key >> 2) & 3) && w == (e >> 1) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
        const u32x4_v bk = b & mask;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const f32x4_v d = mfma(v_operand(f, n) & mask, bk, z);
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] += key >= from && key < to ? d[r] : 0.f;
        }
    }
    st.l = mfma(one, b, st.l);
}
__device__ __forceinline__ void accumulate_each(Row<float>& st, const Frag<float>& f, const float (&p)[8], int g,
                                                int from, int to) {
    const f32x4_v z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int key = 0; key < kTile; ++key) {
        const int mine = g == ((key >> 2) & 3) ? 4 * (key >> 4) + (key & 3) : -1;
        float pk = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) pk = e == mine ? p[e] : pk;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            float vk = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) vk = e == mine ? v_operand(f, e, n) : vk;
            const f32x4_v d = mfma(vk, pk, z);
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] += key >= from && key < to ? d[r] : 0.f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) st.l[0] += p[e];
}

__device__ __forceinline__ int wave_max_int(int x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = max(x, __shfl_xor(x, d));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_min_int(int x) { return -wave_max_int(-x); }

// One workgroup's item: 16 RT query rows (the `block`-th of the segment's) against
// chunk `chunk` of the segment's keys.
template <typename T, int RT, bool SHARED>
__device__ __forceinline__ void attend(const Args& a, Shared<T, RT>& sm, int seg, int kvh, int block, int chunk) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4;
    const int R = a.S * a.G;  // query rows per (sequence, kv head)
    int first = 0, members = 1, table_row = seg, lo, hi_seg;
    if constexpr (SHARED) {
        first = min(max(a.group_start[seg], 0), a.B);
        members = min(max(a.group_start[seg + 1] - first, 0), min(a.max_group, a.B - first));
        if (members == 0) return;
        table_row = a.group_seq[first];
        if (table_row < 0 || table_row >= a.B) return;
        lo = 0;
        hi_seg = a.shared_of(table_row);
    } else {
        lo = a.shared_of(seg);
        hi_seg = 0x7fffffff;
    }
    const int n_rows = members * R;
    const int row0 = block * 16 * RT;
    if (row0 >= n_rows) return;
    const int base = SHARED ? 0 : Args::own_base(lo);
    const int per = SHARED ? a.shared_chunk : a.own_chunk;
    const int begin = base + chunk * per;

    // This lane's query rows: index into q and the workspace, and the keys they see.
    int64_t at[RT];  // (b Hq + h) S + s, or -1
    int hi[RT], max_hi = 0, min_hi = 0x7fffffff;
    QFrag<T> q[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = row0 + 16 * t + i;
        at[t] = -1;
        hi[t] = 0;
        if (r < n_rows) {
            const int member = r / R, rem = r - member * R, s = rem / a.G, h = rem - s * a.G;
            const int b = SHARED ? a.group_seq[first + member] : seg;
            if (b >= 0 && b < a.B) {
                at[t] = ((int64_t)b * a.Hq + kvh * a.G + h) * a.S + s;
                hi[t] = min(hi_seg, a.limit(b, s));
                max_hi = max(max_hi, hi[t]);
                min_hi = min(min_hi, hi[t]);
            }
        }
        q[t].load(reinterpret_cast<const T*>(a.q) + (at[t] < 0 ? 0 : at[t]) * kHeadDim, g);
    }
    max_hi = wave_max_int(max_hi);
    min_hi = wave_min_int(min_hi);
    const int end = min(begin + per, max_hi);
    const bool direct = a.slots() == 1;
    if (begin >= end && !direct) return;  // the join reads no slot past a row's keys

    Row<T> st[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) st[t].clear();

    // The chunk's page ids, one per lane.
    const int P = a.rows.page_rows;
    const int page0 = begin / P;
    int ids = -1;
    if (begin < end && page0 + lane < a.rows.stride && (int64_t)(page0 + lane) * P < end)
        ids = a.rows.table[table_row * a.rows.stride + page0 + lane];
    // Buffers over rows [j, min(j + 32, end)) of this kv head: rows past the last one
    // any query of the wave sees, and pages outside the pool, read as zero.
    auto tile_offset = [&](int j, int& bytes) __attribute__((always_inline)) {
        const int p = j / P;
        const int id = __builtin_amdgcn_readlane(ids, p - page0);
        const bool ok = id >= 0 && id < a.rows.n_pages;
        bytes = ok ? max(0, min(kTile, end - j)) * kHeadDim * (int)sizeof(T) : 0;
        return ok ? (((int64_t)id * a.Hkv + kvh) * P + (j - p * P)) * kHeadDim : 0;
    };
    Frag<T> f;
    int j = begin + wave * kTile;
    if (j < end) {
        int bytes;
        const int64_t off = tile_offset(j, bytes);
        load_k(f, make_rsrc(reinterpret_cast<const T*>(a.k) + off, bytes), i, g);
        load_v(f, make_rsrc(reinterpret_cast<const T*>(a.v) + off, bytes), i, g);
    }
    while (j < end) {
        const int next = j + kWaves * kTile;
        int bytes = 0;
        int64_t off = 0;
        if (next < end) off = tile_offset(next, bytes);
        float s[RT][8];
#pragma unroll
        for (int t = 0; t < RT; ++t) scores(f, q[t], s[t]);
        if (next < end) load_k(f, make_rsrc(reinterpret_cast<const T*>(a.k) + off, bytes), i, g);
        const bool edge = j < lo || j + kTile > min_hi;
        if (edge) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = j + 16 * (e >> 2) + 4 * g + (e & 3);
                    s[t][e] = key >= lo && key < hi[t] ? s[t][e] : -INFINITY;
                }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) softmax_step(st[t], s[t], a.c);
        if (edge && (j < lo || min_hi < min(j + kTile, end)) && __any(any_nonfinite(f))) {
#pragma unroll
            for (int t = 0; t < RT; ++t) accumulate_each(st[t], f, s[t], g, lo - j, hi[t] - j);
        } else {
#pragma unroll
            for (int t = 0; t < RT; ++t) accumulate(st[t], f, s[t]);
        }
        if (next < end) load_v(f, make_rsrc(reinterpret_cast<const T*>(a.v) + off, bytes), i, g);
        j = next;
    }

    // Join the waves: m first, then o and l at the common m.
    float l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] = st[t].sum();
        if (g == 0) sm.m[wave][16 * t + i] = st[t].m;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = 16 * t + i;
        const float m = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
        const float w = fast_exp2(st[t].m - m);
        if (g == 0) sm.l[wave][r] = w * l[t];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            float x[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = w * st[t].o[n][r4];
            store8(&sm.o[wave][r][32 * g + 8 * r4], x);
        }
    }
    __syncthreads();
    // 16 threads per row, 8 dims each.
    for (int r = tid >> 4; r < 16 * RT; r += 16) {
        const int rr = row0 + r;
        if (rr >= n_rows) break;
        const int member = rr / R, rem = rr - member * R, s = rem / a.G, h = rem - s * a.G;
        const int b = SHARED ? a.group_seq[first + member] : seg;
        if (b < 0 || b >= a.B) continue;
        const int d = 8 * (tid & 15);
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
        const int hq = kvh * a.G + h;
        if (direct) {
            const bool none = min(hi_seg, a.limit(b, s)) <= lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = none ? 0.f : x[e] / sum;
            store8(reinterpret_cast<T*>(a.out) + (((int64_t)b * a.S + s) * a.Hq + hq) * kHeadDim + d, x);
        } else {
            const int64_t slot = (((int64_t)b * a.Hq + hq) * a.S + s) * a.slots() + (SHARED ? 0 : a.shared_splits) + chunk;
            store8(a.ws_o + slot * kHeadDim + d, x);
            if (d == 0) a.ws_ml[slot] = make_float2(m, sum);
        }
    }
}

// grid: the shared role's items (chunk slowest), then the own role's.
template <typename T, int RT>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_attn_kernel(Args a) {
    __shared__ Shared<T, RT> sm;
    int x = blockIdx.x;
    if (x < a.shared_items) {
        const int block = x % a.shared_tiles;
        x /= a.shared_tiles;
        const int kvh = x % a.Hkv;
        x /= a.Hkv;
        attend<T, RT, true>(a, sm, x % a.n_groups, kvh, block, x / a.n_groups);
    } else {
        x -= a.shared_items;
        const int block = x % a.own_tiles;
        x /= a.own_tiles;
        const int kvh = x % a.Hkv;
        x /= a.Hkv;
        attend<T, RT, false>(a, sm, x % a.B, kvh, block, x / a.B);
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

// How a call is cut: row blocks and key chunks of both roles.
struct Plan {
    int rows;  // query rows per workgroup
    int shared_tiles, own_tiles, shared_chunk, own_chunk, shared_splits, own_splits;
    int64_t shared_items, own_items;
    size_t ml_off, total;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool make_plan(int n_groups, int max_group, int64_t max_shared, int64_t max_own, int B, int S, int Hq, int Hkv, Plan* p) {
    const int64_t R = (int64_t)S * (Hq / Hkv);
    p->rows = 16;
    const int64_t st = max_shared > 0 && n_groups > 0 ? ceil_div((int64_t)max_group * R, p->rows) : 0;
    const int64_t ot = ceil_div(R, p->rows);
    const int64_t shared = st ? max_shared : 0, own = max_own + kTile;  // own chunk 0 starts on a tile bound
    // Rows times keys of all items, spread over 1024 workgroups (4 per CU).
    const int64_t total = (int64_t)n_groups * Hkv * st * shared + (int64_t)B * Hkv * ot * own;
    int64_t chunk = ceil_div(ceil_div(total, 1024), kMinChunk) * kMinChunk;
    chunk = chunk < kMinChunk ? kMinChunk : chunk > kMaxChunk ? kMaxChunk : chunk;
    p->shared_chunk = p->own_chunk = (int)chunk;
    const int64_t ss = ceil_div(shared, chunk), os = ceil_div(own, chunk);
    p->shared_items = (int64_t)n_groups * Hkv * st * ss;
    p->own_items = (int64_t)B * Hkv * ot * os;
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
    const int64_t items = p.shared_items + p.own_items;
    hipLaunchKernelGGL((shared_attn_kernel<T, 1>), dim3((unsigned)items), dim3(64 * kWaves), 0, st, a);
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
    return make_plan(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, &p) ? p.total : 0;
}

extern "C" int crane_hip_attn_shared_paged(const void* q, const void* k_pool, const void* v_pool, int64_t n_pages,
                                           int page_rows, const int32_t* block_table, int64_t table_stride,
                                           const int32_t* kv_len, int64_t max_kv, const int32_t* shared_rows,
                                           const int32_t* group_start, const int32_t* group_seq, int n_groups,
                                           int max_group, int64_t max_shared, int64_t max_own, int B, int S, int Hq,
                                           int Hkv, int D, float scale, int flags, void* workspace, size_t ws_bytes,
                                           void* out, int dtype, void* stream) {
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
    if (n_groups > 0 && (!shared_rows || !group_start || !group_seq)) return CRANE_HIP_E_INVALID;
    if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out)) return CRANE_HIP_E_ALIGN;
    Plan p;
    if (!make_plan(n_groups, max_group, max_shared, max_own, B, S, Hq, Hkv, &p)) return CRANE_HIP_E_INVALID;
    if (p.total && (!workspace || ws_bytes < p.total || !aligned16(workspace))) return CRANE_HIP_E_WORKSPACE;
    Args a;
    a.q = q;
    a.k = k_pool;
    a.v = v_pool;
    a.out = out;
    a.rows = PagedRows{block_table, table_stride, n_pages, page_rows};
    a.kv_len = kv_len;
    a.shared = n_groups > 0 ? shared_rows : nullptr;
    a.group_start = group_start;
    a.group_seq = group_seq;
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
