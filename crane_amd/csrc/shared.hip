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
// Stream (16 or 32 rows: HBM-bound).  Every wave takes 32-key steps of its own, K and V
// from memory to registers ahead of their use, and the waves' m, l, o are joined through
// LDS at the end.  bf16, v_mfma_f32_16x16x32_bf16: S^T = K Q^T with K rows as A and
// query rows as B, so lane (i, g) = (lane % 16, lane / 16) holds, for query row i, keys
// 4 g + r of two 16-key halves.  Those 8 values, rounded to bf16, are the B operand
// P^T of O^T = V^T P^T as they stand: the order of the 32 keys inside the k index is
// free as long as V follows it, so lane group g takes V rows 4 g + r of both halves.
// It reads dims [8 i, 8 i + 8) of each (whole 256-byte rows per 16 lanes) and v_perm
// pairs them into the A operand of eight products, product n giving dims 8 m + n: a
// lane ends with dims [32 g, 32 g + 32) of its query row.
//
// f32 runs this layout on v_mfma_f32_16x16x4_f32: a k slot takes one key (or dim) of
// every lane group, so no pairing is needed.
//
// Block (bf16, more rows: 32 for each wave).  The waves walk the same keys, staged in
// LDS by buffer_load ... lds one tile ahead, so that K and V are read from memory once
// for the block.  v_mfma_f32_32x32x16_bf16: the same products with 32 rows a wave and
// 64 keys a tile; V^T comes from the row-major tile by transposed LDS reads.
//
// l sums p as computed in f32; only the P operand is rounded (bf16).
//
// A row's m is settled by the first keys of its walk (two steps, one tile) and then left
// alone: exp2(s - m) of f32 or bf16 stays exact to its own rounding however far s passes
// m, until it overflows.  So the walk takes no maximum and scales nothing (60 of about
// 150 vector instructions of a step), and looks once, at its end, whether l passed
// kMostSum or o is not finite.  That is so after a row's scores rose by 2^60 (41 in
// natural units) over its first keys, or where V holds an infinity or a NaN, even in a
// key the row does not see (0 x inf).  Then the walk is repeated with m moved at every
// step and such keys added to the rows that see them only.  So it is where m itself is past
// kMostMax: s scale log2 e - m is one product with one rounding, which leaves every weight of
// the row the factor exp2(the rounding of m); o / l takes that out again, but it overflows or
// vanishes once half a step of m passes a hundred.  The repeated walk keeps the maximum as
// the scores are, too, and takes (s - max) scale log2 e for such rows, 0 for the largest.
//
// Measured (both kernels, HIP graph): 2 sequences, 512 shared rows, 16 / 8 heads 8.7 us;
// 32 sequences of 32 / 8 heads and 200 to 1500 rows behind 4096 33 us, 140 MB; 64 behind
// 32768 rows 98 us, 69 GFLOP (0.83 PFLOP/s in the block form, bound by MFMAs and
// exponentials in turn); 32 sequences of 200 to 1500 rows that share nothing 25 us, 119 MB
// (4.8 TB/s); 16 of 4000 to 8000 at 8 / 8 heads 72 us, 428 MB (5.9 TB/s).
#include <float.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "attn_lanes.h"
#include "shared_plan.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr float kNoMax = -FLT_MAX; // m before the first key (finite: exp2(-inf - m) is 0, not NaN)
constexpr float kMostSum = 0x1p60f;  // see above
constexpr float kMostMax = 0x1p26f;  // see above: half a step of m is 2 at most
constexpr size_t kHalfLds = 81920;   // half of a CU's LDS

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}
// NT: read once, streamed past the caches.
template <bool NT = false> __device__ __forceinline__ u32x4_v buf_load16(__amdgpu_buffer_rsrc_t r, int off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? 2 : 0);
}
__device__ __forceinline__ f32x4_v mfma(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                   0, 0, 0);
}
__device__ __forceinline__ f32x4_v mfma(float a, float b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

struct Args {
    const void *q, *k, *v;
    void* out;
    PagedRows rows;
    const int32_t *kv_len, *shared, *groups, *members;
    int n_groups, n_members, max_shared;
    int B, S, Hq, Hkv, G;     // G = Hq / Hkv heads per kv head
    int max_kv, causal;
    float c;                  // scale log2 e
    int chunk;    // rows per chunk
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
    // The row of out [B, S, Hq] that is row `at` of q [B, Hq, S].
    __device__ __forceinline__ int64_t out_row(int at) const {
        if (S == 1) return at;
        const int bh = at / S, s = at - bh * S, b = bh / Hq;
        return ((int64_t)b * S + s) * Hq + (bh - b * Hq);
    }
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
            const Members of(d.x, d.y, a.n_members);
            first = of.first;
            table_row = d.z;
            lo = 0;
            hi = min(d.w, a.max_shared);
            n_rows = table_row < 0 || table_row >= a.B ? 0 : of.n * R;
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
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* pool, const Pages::Tile& t) {
    return make_rsrc(reinterpret_cast<const T*>(pool) + t.off, t.bytes);
}

// Maximum over N = 16 or 32 neighbouring lanes, for values that repeat every N lanes of
// the wave; uniform.
template <int CTRL> __device__ __forceinline__ int dpp_int(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false);
}
template <int N> __device__ __forceinline__ int rows_max(int x) {
    x = max(x, dpp_int<0xB1>(x));   // quad_perm [1,0,3,2]
    x = max(x, dpp_int<0x4E>(x));   // quad_perm [2,3,0,1]
    x = max(x, dpp_int<0x124>(x));  // row_ror:4
    x = max(x, dpp_int<0x128>(x));  // row_ror:8
    if constexpr (N == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
        x = max((int)r[0], (int)r[1]);
    }
    return __builtin_amdgcn_readfirstlane(x);
}
template <int N> __device__ __forceinline__ int rows_min(int x) { return -rows_max<N>(-x); }

template <int RT> struct StreamShared {
    static constexpr int kStride = kHeadDim + 4;  // f32 per row: 16 rows at one column hit different banks
    float m[kWaves][16 * RT];
    float l[kWaves][16 * RT];
    int place[16 * RT], to[16 * RT];  // Segment::query of every row
    __attribute__((aligned(16))) float o[kWaves][16 * RT][kStride];
};
// Tiles of 64 keys.
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
template <bool NT>
__device__ __forceinline__ void load_v(Frag<bf16_t>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = buf_load16<NT>(r, (16 * (e >> 2) + 4 * g + (e & 3)) * 256 + 16 * i);
}
__device__ __forceinline__ void load_k(Frag<float>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int t = 0; t < 8; ++t) f.k[t] = buf_load16(r, i * 512 + 64 * t + 16 * g);
}
template <bool NT>
__device__ __forceinline__ void load_v(Frag<float>& f, __amdgpu_buffer_rsrc_t r, int i, int g) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < 2; ++d) f.v[e][d] = buf_load16<NT>(r, (4 * g + e) * 512 + 256 * d + 16 * i);
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

// p = exp2(s c - m) of the step's scores; MOVE: m moved to the largest so far first, and
// o and l scaled to it.
template <bool MOVE, typename T, int N>
__device__ __forceinline__ void softmax_step(Row<T>& st, float (&s)[N], float c) {
    if constexpr (MOVE) {
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        if constexpr (N == 8) mx = fmaxf(mx, fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        const float m = fmaxf(st.m, groups_max(mx) * c), a = fast_exp2(st.m - m);
        st.m = m;
        st.l *= a;
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[n][r] *= a;
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        s[e] = fast_exp2(__builtin_fmaf(s[e], c, -st.m));
        sum += s[e];
    }
    st.l += sum;
}

// The largest score so far as it is and as an m (finite; of no score: no larger than any
// score's), and p's exponent for rows of any m.
struct Largest {
    float raw = kNoMax, m = kNoMax;
    bool big = true;
    // Takes a step's largest score; o's and l's factor.
    __device__ __forceinline__ float move(float score, float c) {
        const float r = fmaxf(raw, score), x = fminf(fmaxf(r * c, kNoMax), FLT_MAX);
        big = fabsf(x) > kMostMax;
        const float a = fast_exp2(big ? (raw - r) * c : m - x);
        raw = r;
        m = x;
        return a;
    }
    __device__ __forceinline__ float exponent(float s, float c) const {
        return big ? (s - raw) * c : __builtin_fmaf(s, c, -m);
    }
};

// softmax_step<true> for rows of any m.
template <typename T, int N>
__device__ __forceinline__ void softmax_step(Row<T>& st, Largest& top, float (&s)[N], float c) {
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, s[e]);
    const float a = top.move(groups_max(mx), c);
    st.m = top.m;
    st.l *= a;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[n][r] *= a;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        s[e] = fast_exp2(top.exponent(s[e], c));
        sum += s[e];
    }
    st.l += sum;
}

// Sum over the four lane groups; every lane gets it.
__device__ __forceinline__ float groups_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// o += P V, every V operand for all row tiles.
template <int RT>
__device__ __forceinline__ void accumulate(Row<bf16_t> (&st)[RT], const Frag<bf16_t>& f, const float (&p)[RT][8]) {
    u32x4_v b[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) b[t][w] = pack_bf16x2(p[t][2 * w], p[t][2 * w + 1]);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const u32x4_v v = v_operand(f, n);
#pragma unroll
        for (int t = 0; t < RT; ++t) st[t].o[n] = mfma(v, b[t], st[t].o[n]);
        if (n & 1) __builtin_amdgcn_sched_barrier(0);  // two operands paired ahead, not all eight
    }
}
template <int RT>
__device__ __forceinline__ void accumulate(Row<float> (&st)[RT], const Frag<float>& f, const float (&p)[RT][4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int t = 0; t < RT; ++t) st[t].o[n] = mfma(v_operand(f, e, n), p[t][e], st[t].o[n]);
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

// Whether a walk that did not move m came out well (a row without keys did).
__device__ __forceinline__ bool sound_sums(float l, float m) {
    return (l <= kMostSum) & ((fabsf(m) <= kMostMax) | (m == kNoMax));
}
template <typename T> __device__ __forceinline__ bool sound(const Row<T>& st) {
    bool ok = sound_sums(st.l, st.m);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) ok = ok && fabsf(st.o[n][r]) < INFINITY;
    return ok;
}

// A row sees keys [lo, hi) only: the others' scores vanish.
template <int N> __device__ __forceinline__ void mask_step(float (&s)[N], int j, int g, int lo, int hi) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int key = j + 16 * (e >> 2) + 4 * g + (e & 3);
        s[e] = key >= lo && key < hi ? s[e] : -INFINITY;
    }
}

// ---- the stream form: 16 RT query rows

template <typename T, int RT, bool NT, bool SHARED>
__device__ __forceinline__ void attend_stream(const Args& a, StreamShared<RT>& sm, int seg, int kvh, int block,
                                              int chunk) {
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // uniform: buffer resources are scalar
    constexpr int kKeys = Frag<T>::kKeys, kSlots = Frag<T>::kSlots;
    const Segment<SHARED> sg(a, seg);
    const int row0 = block * 16 * RT;
    if (row0 >= sg.n_rows) return;
    const int per = a.chunk, lo = sg.lo, begin = sg.base() + chunk * per;
    const Pages pages(a, sg.table_row, begin, lane);

    int hi[RT], at[RT], most = 0;
    QFrag<T> q[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        at[t] = (int)sg.query(row0 + 16 * t + i, kvh, hi[t]);  // fewer than 2^31 query rows
        q[t].load(reinterpret_cast<const T*>(a.q) + (int64_t)max(at[t], 0) * kHeadDim, g);
        most = max(most, hi[t]);
    }
    const int end = min(begin + per, rows_max<16>(most));
    int least = end;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        hi[t] = min(hi[t], end);  // a step may reach past the chunk's end
        least = min(least, at[t] < 0 ? end : hi[t]);
    }
    const int min_hi = rows_min<16>(least);
    const bool direct = a.slots() == 1;
    if (begin >= end && !direct) return;  // the join reads no slot past a row's keys

    Row<T> st[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) st[t].clear();
    auto tile_at = [&](int j) __attribute__((always_inline)) { return pages.tile<T>(a, kvh, j, kKeys, end); };
    auto k_tile = [&](Frag<T>& f, const Pages::Tile& t) __attribute__((always_inline)) {
        load_k(f, tile_rsrc<T>(a.k, t), i, g);
    };
    auto v_tile = [&](Frag<T>& f, const Pages::Tile& t) __attribute__((always_inline)) {
        load_v<NT>(f, tile_rsrc<T>(a.v, t), i, g);
    };
    // One step's tiles are in flight: its K registers are loaded again, for the step on,
    // once its scores are taken, its V registers after its product (two steps in flight
    // leave 16 rows two workgroups a CU in place of three: 32 sequences of 512 to 4096 keys
    // in chunks of 256 76 us for 70, a call of 2 short ones 8.7 for 8.4).  A step past the
    // end loads nothing and sees no key.
    constexpr int kStride = kWaves * kKeys;
    const int j0 = begin + wave * kKeys;
    Frag<T> f;
    auto step = [&](int j, auto move) __attribute__((always_inline)) {
        const Pages::Tile next = tile_at(j + kStride);
        float s[RT][kSlots];
#pragma unroll
        for (int t = 0; t < RT; ++t) scores(f, q[t], s[t]);
        __builtin_amdgcn_sched_barrier(0);  // the loads take the registers just read, not new ones
        k_tile(f, next);
        if (j < lo || j + kKeys > min_hi) {
#pragma unroll
            for (int t = 0; t < RT; ++t) mask_step(s[t], j, g, lo, hi[t]);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) softmax_step<decltype(move)::value>(st[t], s[t], a.c);
        accumulate(st, f, s);
        __builtin_amdgcn_sched_barrier(0);
        v_tile(f, next);
    };
    const Pages::Tile first = tile_at(j0);
    // In the steps' own order: the loop's first wait has to hold for both.
    __builtin_amdgcn_sched_barrier(0);
    k_tile(f, first);
    __builtin_amdgcn_sched_barrier(0);
    v_tile(f, first);
    __builtin_amdgcn_sched_barrier(0);
    // A row that sees any key of the wave's sees one in its first two steps: lo is less
    // than kAlign past the chunk's begin.
    step(j0, std::true_type());
    step(j0 + kStride, std::true_type());
    for (int j = j0 + 2 * kStride; j < end; j += kStride) step(j, std::false_type());
    bool again = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) again = again || (at[t] >= 0 && !sound(st[t]));
    if (__any(again)) {
#pragma unroll
        for (int t = 0; t < RT; ++t) st[t].clear();
        Largest top[RT];
        for (int j = j0; j < end; j += kStride) {
            const Pages::Tile tile = tile_at(j);
            k_tile(f, tile);
            v_tile(f, tile);
            float s[RT][kSlots];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                scores(f, q[t], s[t]);
                mask_step(s[t], j, g, lo, hi[t]);
                softmax_step(st[t], top[t], s[t], a.c);
            }
            if (__any(any_nonfinite(f))) {
#pragma unroll
                for (int t = 0; t < RT; ++t) accumulate_each(st[t], f, s[t], g, lo - j, hi[t] - j);
            } else {
                accumulate(st, f, s);
            }
        }
    }

    // Join the waves: m first, then o and l at the common m.
    float l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] = groups_sum(st[t].l);
        if (g == 0) sm.m[wave][16 * t + i] = st[t].m;
        if (tid < 16) {
            sm.place[16 * t + i] = at[t];
            sm.to[16 * t + i] = hi[t];
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = 16 * t + i;
        const float m = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
        const float w = fast_exp2(st[t].m - m);
        if (g == 0) sm.l[wave][r] = w * l[t];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int n0 = 0; n0 < 8; n0 += 4) {
                const f32x4_v* o = st[t].o + n0;
                const float y[4] = {w * o[0][x], w * o[1][x], w * o[2][x], w * o[3][x]};
                store4(&sm.o[wave][r][Row<T>::dim(n0, x, g)], y);
            }
    }
    __syncthreads();
    // 16 threads per row, 8 dims each.
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = 16 * t + (tid >> 4), d = 8 * (tid & 15), place = sm.place[r];
        if (place < 0) continue;
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
            const bool none = sm.to[r] <= lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = none ? 0.f : x[e] / sum;
            store8(reinterpret_cast<T*>(a.out) + a.out_row(place) * kHeadDim + d, x);
        } else {
            const int64_t slot = (int64_t)place * a.slots() + (SHARED ? 0 : a.shared_splits) + chunk;
            store8(a.ws_o + slot * kHeadDim + d, x);
            if (d == 0) a.ws_ml[slot] = make_float2(m, sum);
        }
    }
}

// ---- the block form

// LDS tiles keep the pools' rows (256 bytes, a full sweep of the banks) with their
// 16-byte chunks XOR-permuted by the row's two low 2-bit halves swapped, so that neither
// 16 rows read at one chunk (K) nor 4 rows x 4 chunks (transposed V) meet in a bank.
constexpr int kRowBytes = kHeadDim * 2;
__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }
// The byte of a tile its row's 16-byte chunk c sits at.
__device__ __forceinline__ int chunk_at(int row, int c) { return row * kRowBytes + 16 * (c ^ swizzle(row)); }

// One tile into LDS: a wave copies 4 KiB, 1 KiB (4 rows) an instruction, lane l the 16
// bytes at 16 l of it.
__device__ __forceinline__ void stage(__amdgpu_buffer_rsrc_t r, uint8_t* to, int wave, int lane) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int row = 16 * wave + 4 * x + (lane >> 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + 4096 * wave + 1024 * x, 16, chunk_at(row, lane & 15), 0, 0, 0);
    }
}
// Wait for the wave's own copies but the last N instructions' (expcnt and lgkmcnt at
// their maxima).
template <int N> __device__ __forceinline__ void wait_copies() {
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_v;
typedef __attribute__((address_space(3))) s16x4_v lds_s16x4_v;
// Within 16 lanes, lane x gets column x of the 4 rows x 16 columns of bf16 that the
// lanes point at (lane x: 4 columns from 4 (x % 4) on of row x / 4).
__device__ __forceinline__ uint2 lds_read_tr16(uint32_t at) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_v*)(uintptr_t)at));
}
__device__ __forceinline__ f32x16_v mfma(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                   0, 0, 0);
}
// A wave's share of a block: Q, o, m and l of its 32 rows, and one tile's work.  Lane
// (n, h) = (lane % 32, lane / 32) holds, for row n, keys 32 b + 8 (r / 4) + 4 h + r % 4 in
// register r of score block b, and dims 32 d + 8 (r / 4) + 4 h + r % 4 in register r of
// o[d].
struct BlockWave {
    static constexpr int kRows = 32, kKeys = 64;
    u32x4_v q[8];
    f32x16_v o[4];
    float m, l;
    int n, h;
    // Byte offsets in a tile, the swizzle of rows 16 apart being the same: ko[t] of row n,
    // chunk 2 t + h; vo[2 d + e] of row 8 e + 4 h + lane % 16 / 4, where the transposed
    // reads of dims 32 d + lane % 32 start.
    uint32_t ko[8], vo[8];
    __device__ __forceinline__ BlockWave(int lane, const BlockShared& sm) : n(lane & 31), h(lane >> 5) {
#pragma unroll
        for (int t = 0; t < 8; ++t) ko[t] = lds_at(sm.k) + chunk_at(n, 2 * t + h);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * e + 4 * h + ((lane & 15) >> 2);
                const int col = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                vo[2 * d + e] = lds_at(sm.v) + chunk_at(row, col >> 3) + 2 * (col & 7);
            }
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
    __device__ __forceinline__ bool sound() const {
        bool ok = sound_sums(l, m);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) ok = ok && fabsf(o[d][r]) < INFINITY;
        return ok;
    }
    // V^T, dims 32 d + lane % 32, of keys 16 s + 8 e + 4 h + (0 .. 3), e = 0, 1.
    __device__ __forceinline__ u32x4_v v_frag(uint32_t buf, int s, int d) const {
        const uint2 x = lds_read_tr16(vo[2 * d] + buf + 16 * s * kRowBytes);
        const uint2 y = lds_read_tr16(vo[2 * d + 1] + buf + 16 * s * kRowBytes);
        return u32x4_v{x.x, x.y, y.x, y.y};
    }
    // A tile's raw scores.
    __device__ __forceinline__ void scores(f32x16_v (&s)[2], uint32_t buf) const {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[b] = mfma(lds_read16(ko[t] + buf + 32 * b * kRowBytes), q[t], s[b]);
    }
    // Row n sees keys [lo, hi) only.
    __device__ __forceinline__ void mask(f32x16_v (&s)[2], int j, int lo, int hi) const {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = j + 32 * b + 8 * (r >> 2) + 4 * h + (r & 3);
                s[b][r] = key >= lo && key < hi ? s[b][r] : -INFINITY;
            }
    }
    // A row's largest score.
    __device__ __forceinline__ float largest(const f32x16_v (&s)[2]) const {
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        return halves_max(mx);
    }
    // p = exp2(exponent of s), rounded and paired: p[t] is the B operand of keys 16 t ..; l.
    template <class EXPONENT>
    __device__ __forceinline__ void weights(const f32x16_v (&s)[2], u32x4_v (&p)[4], EXPONENT exponent) {
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = fast_exp2(exponent(s[b][r])), y = fast_exp2(exponent(s[b][r + 1]));
                sum += x + y;
                p[2 * b + (r >> 3)][(r & 7) >> 1] = pack_bf16x2(x, y);
            }
        l += sum;
    }
    __device__ __forceinline__ void accumulate(const u32x4_v (&p)[4], uint32_t buf) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] = mfma(v_frag(buf, t, d), p[t], o[d]);
    }
    // A step's order: K fragments read four ahead of their MFMAs with the exponentials
    // between, then V fragments two ahead.
    template <class MORE> static __device__ __forceinline__ void schedule(MORE) {
        constexpr int kMfma = 0x8, kRead = 0x100, kValu = 0x2;
        if constexpr (MORE::value) {
            __builtin_amdgcn_sched_group_barrier(kRead, 4, 0);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                if (x < 12) __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kValu, 7, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(kRead, 4, 0);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            if (x < 14) __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
        }
    }
    // As accumulate_each above; key 16 t + 8 e + 4 h + x is slot 4 e + x of half h in step t.
    __device__ __forceinline__ void accumulate_each(const u32x4_v (&p)[4], uint32_t buf, int j, int lo, int hi) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const u32x4_v x = v_frag(buf, t, d);
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
};

// Whether a V tile holds an infinity or a NaN (the whole tile, by one wave).
__device__ __forceinline__ bool tile_nonfinite(const uint8_t* v, int lane) {
    const uint32_t at = lds_at(v) + 16 * lane;
    bool bad = false;
#pragma unroll 4
    for (int x = 0; x < kTileBytes / 1024; ++x) {
        const u32x4_v u = lds_read16(at + 1024 * x);
#pragma unroll
        for (int y = 0; y < 4; ++y) bad |= (u[y] & 0x7f800000u) == 0x7f800000u || (u[y] & 0x7f80u) == 0x7f80u;
    }
    return __any(bad);
}

template <bool SHARED>
__device__ __forceinline__ void attend_block(const Args& a, BlockShared& sm, int seg, int kvh, int block, int chunk) {
    constexpr int kKeys = BlockWave::kKeys;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Segment<SHARED> sg(a, seg);
    const int row0 = block * kBlockRows;
    if (row0 >= sg.n_rows) return;
    const int per = a.chunk, lo = sg.lo, begin = sg.base() + chunk * per;
    const Pages pages(a, sg.table_row, begin, lane);
    // Keys any row of the block can see: a group's shared rows, or what the block's last
    // query sees.
    int end = begin + per;
    if constexpr (SHARED) end = min(end, sg.hi);
    else end = min(end, a.limit(seg, (min(row0 + kBlockRows, sg.n_rows) - 1) / a.G));
    end = __builtin_amdgcn_readfirstlane(end);
    const bool direct = a.slots() == 1;
    if (begin >= end && !direct) return;

    BlockWave w(lane, sm);
    int hi;
    const int64_t at = sg.query(row0 + BlockWave::kRows * wave + w.n, kvh, hi);
    w.load_q(reinterpret_cast<const bf16_t*>(a.q) + (at < 0 ? 0 : at) * kHeadDim);
    w.clear();
    hi = min(hi, end);
    const int max_hi = rows_max<32>(hi), min_hi = rows_min<32>(at < 0 ? end : hi);

    const int n = max(0, (end - begin + kKeys - 1) / kKeys);
    auto tile_at = [&](int t) __attribute__((always_inline)) {
        return pages.tile<bf16_t>(a, kvh, begin + t * kKeys, kKeys, end);
    };
    auto issue_k = [&](int t) __attribute__((always_inline)) {
        stage(tile_rsrc<bf16_t>(a.k, tile_at(t)), sm.k[t & 1], wave, lane);
    };
    auto issue_v = [&](int t) __attribute__((always_inline)) {
        stage(tile_rsrc<bf16_t>(a.v, tile_at(t)), sm.v[t & 1], wave, lane);
    };
    // Step t takes the weights and the V product of tile t and the scores of tile t + 1,
    // whose MFMAs run beside the exponentials, while K of tile t + 2 and V of tile t + 1
    // come in (into the buffers of K(t) and V(t - 1), whose readers passed the barrier).
    // A tile past `max_hi` is seen by none of the wave's rows.
    f32x16_v sa[2], sb[2];
    auto step = [&](int t, f32x16_v(&s)[2], f32x16_v(&next)[2], auto more) __attribute__((always_inline)) {
        wait_copies<0>();
        __syncthreads();
        if (t + 2 < n) issue_k(t + 2);
        if (t + 1 < n) issue_v(t + 1);
        const int j = begin + t * kKeys;
        if (j >= max_hi) return;
        if (j < lo || j + kKeys > min_hi) w.mask(s, j, lo, hi);
        u32x4_v p[4];
        if constexpr (decltype(more)::value) w.scores(next, ((t + 1) & 1) * kTileBytes);
        w.weights(s, p, [&](float x) __attribute__((always_inline)) { return __builtin_fmaf(x, a.c, -w.m); });
        w.accumulate(p, (t & 1) * kTileBytes);
        BlockWave::schedule(more);
    };
    if (n > 0) {
        issue_k(0);
        issue_v(0);
        if (n > 1) issue_k(1);
        if (n > 1) wait_copies<8>();
        else wait_copies<4>();
        __syncthreads();
        w.scores(sa, 0);
        // A row that sees any key of the chunk sees one in its first tile.
        w.mask(sa, begin, lo, hi);
        w.m = fmaxf(w.m, w.largest(sa) * a.c);
    }
    int t = 0;
    for (; t + 2 < n; t += 2) {
        step(t, sa, sb, std::true_type());
        step(t + 1, sb, sa, std::true_type());
    }
    if (t + 2 == n) step(t, sa, sb, std::true_type()), step(t + 1, sb, sa, std::false_type());
    else if (t < n) step(t, sa, sb, std::false_type());
    sm.again[wave] = __any(at >= 0 && !w.sound());
    __syncthreads();
    if (sm.again[0] | sm.again[1] | sm.again[2] | sm.again[3]) {
        w.clear();
        Largest top;
        for (t = 0; t < n; ++t) {
            __syncthreads();
            issue_k(t);
            issue_v(t);
            wait_copies<0>();
            __syncthreads();
            const uint32_t buf = (t & 1) * kTileBytes;
            const int j = begin + t * kKeys;
            w.scores(sa, buf);
            w.mask(sa, j, lo, hi);
            const float x = top.move(w.largest(sa), a.c);
            w.m = top.m;
            w.l *= x;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) w.o[d][r] *= x;
            u32x4_v p[4];
            w.weights(sa, p, [&](float x) __attribute__((always_inline)) { return top.exponent(x, a.c); });
            if (tile_nonfinite(sm.v[t & 1], lane)) w.accumulate_each(p, buf, j, lo, hi);
            else w.accumulate(p, buf);
        }
    }
    const float l = halves_sum(w.l);
    if (at < 0) return;
    const int64_t slot = at * a.slots() + (SHARED ? 0 : a.shared_splits) + chunk;
    bf16_t* out = reinterpret_cast<bf16_t*>(a.out) + a.out_row((int)at) * kHeadDim;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = w.o[d][r + e];
            const int dim = 32 * d + 2 * r + 4 * w.h;
            if (direct) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = hi <= lo ? 0.f : x[e] / l;
                store4(out + dim, x);
            } else {
                store4(a.ws_o + slot * kHeadDim + dim, x);
            }
        }
    if (!direct && w.h == 0) a.ws_ml[slot] = make_float2(w.m, l);
}

// The forms of a role, by its query rows per workgroup.  V, whose loads take whole rows,
// streams past the caches where one workgroup reads it: always for 16 rows (16 sequences
// of 4000 to 8000 keys, 428 MB: 79 us for 73), and for 32 where they are all there are
// (11 sequences in 3 groups of 11776 f32 rows: 65 for 60; groups of two blocks 27 for 30
// the other way).  K's loads take half a line at a time and want the caches (32 sequences
// of 200 to 1500 keys: 25 us, 29 with K streamed too).
template <typename T, int ROWS, bool ONCE, bool SHARED, class SM>
__device__ __forceinline__ void attend(const Args& a, SM& sm, const Item& x) {
    if constexpr (ROWS == kBlockRows) attend_block<SHARED>(a, sm.block, x.seg, x.kvh, x.block, x.chunk);
    else if constexpr (ROWS == 32) attend_stream<T, 2, ONCE, SHARED>(a, sm.stream32, x.seg, x.kvh, x.block, x.chunk);
    else attend_stream<T, 1, true, SHARED>(a, sm.stream16, x.seg, x.kvh, x.block, x.chunk);
}

template <int SHARED_ROWS, int OWN_ROWS> union AttnShared {
    StreamShared<1> stream16;
    typename std::conditional<SHARED_ROWS == 32 || OWN_ROWS == 32, StreamShared<2>, int>::type stream32;
    typename std::conditional<SHARED_ROWS == kBlockRows || OWN_ROWS == kBlockRows, BlockShared, int>::type block;
};

// ONCE: one block of rows covers a group's.
// grid: the shared role's items, then the own role's.
template <typename T, int SHARED_ROWS, int OWN_ROWS, bool ONCE>
__global__ __launch_bounds__(64 * kWaves, SHARED_ROWS == 16 ? 3 : 2) void shared_attn_kernel(Args a) {
    __shared__ AttnShared<SHARED_ROWS, OWN_ROWS> sm;
    if ((int)blockIdx.x < a.shared_items) {
        const Item x(blockIdx.x, a.shared_tiles, a.Hkv, a.n_groups, a.shared_splits);
        if (x.ok) attend<T, SHARED_ROWS, ONCE, true>(a, sm, x);
    } else {
        const Item x(blockIdx.x - a.shared_items, a.own_tiles, a.Hkv, a.B, a.own_splits);
        if (x.ok) attend<T, OWN_ROWS, false, false>(a, sm, x);
    }
}

// Join a query row's chunks: P waves per row, lane l owns dims 2 l, 2 l + 1, wave p takes
// slots p, p + P, ...  Every first load (8 slots a wave, the m and l of 64) is issued
// before the row's lengths are known, so that up to 8 P slots cost one round trip; slots
// past the row's keys hold anything and are left out by selects.
constexpr int kJoinRegs = 8;
template <typename T, int P>
__global__ __launch_bounds__(P == 1 ? 256 : 64 * P) void shared_join_kernel(Args a, int n_rows) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = P == 1 ? 0 : wave;
    const int row = P == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= n_rows) return;  // P > 1: the whole workgroup
    const int slots = a.slots();
    const float2* ml = a.ws_ml + (int64_t)row * slots;
    const float2* o = reinterpret_cast<const float2*>(a.ws_o + (int64_t)row * slots * kHeadDim) + lane;
    float2 x[kJoinRegs];
#pragma unroll
    for (int i = 0; i < kJoinRegs; ++i) x[i] = o[(int64_t)min(p + P * i, slots - 1) * (kHeadDim / 2)];
    const float2 first = ml[min(lane, slots - 1)];
    const int bh = row / a.S, s = row - bh * a.S, b = bh / a.Hq;
    const int n = a.len(b), shared = a.shared_of(b);
#pragma unroll
    for (int i = 0; i < kJoinRegs; ++i) asm volatile("" ::"v"(x[i].x), "v"(x[i].y));  // loaded above the branches below
    asm volatile("" ::"v"(first.x), "v"(first.y));
    const int limit = a.causal ? n - a.S + 1 + s : n;
    const int seen = min(shared, limit), own = limit - Args::own_base(shared);
    const int n_shared = seen > 0 ? (seen + a.chunk - 1) / a.chunk : 0;
    const int n_own = limit > shared ? (own + a.chunk - 1) / a.chunk : 0;
    // the row has keys in the chunk of slot c
    auto has = [&](int c) __attribute__((always_inline)) {
        return c < a.shared_splits ? c < n_shared : c < slots && c - a.shared_splits < n_own;
    };
    float mx = has(lane) ? first.x : kNoMax;
    for (int c = lane + 64; c < slots; c += 64) mx = fmaxf(mx, has(c) ? ml[c].x : kNoMax);
    mx = wave_max(mx);
    float den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int c0 = 0; c0 < slots; c0 += 64) {
        const float2 t = c0 == 0 ? first : ml[min(c0 + lane, slots - 1)];
        const float w = has(c0 + lane) ? fast_exp2(t.x - mx) : 0.f;
        den += has(c0 + lane) ? w * t.y : 0.f;
        auto add = [&](int c, float2 y) __attribute__((always_inline)) {
            if (!has(c)) return;
            const float wc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), c - c0));
            x0 += wc * y.x;
            x1 += wc * y.y;
        };
        int c = c0 + p;
        if (c0 == 0) {
#pragma unroll
            for (int i = 0; i < kJoinRegs; ++i)
                if (p + P * i < 64) add(p + P * i, x[i]);
            c += P * kJoinRegs;
        }
        for (; c < min(slots, c0 + 64); c += P) add(c, o[(int64_t)c * (kHeadDim / 2)]);
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
    const bool none = n_shared + n_own == 0;
    T* out = reinterpret_cast<T*>(a.out) + a.out_row(row) * kHeadDim + 2 * lane;
    Elem<T>::store(out, none ? 0.f : x0 / den);
    Elem<T>::store(out + 1, none ? 0.f : x1 / den);
}

void size_workspace(const Sizes& z, Plan* p) {
    const int64_t slots = p->shared_splits + p->own_splits;
    p->ml_off = ((size_t)z.rows() * slots * kHeadDim * sizeof(float) + 255) & ~(size_t)255;
    p->total = slots > 1 ? p->ml_off + (size_t)z.rows() * slots * sizeof(float2) : 0;
}

// The plan for these sizes.  A thread's last one is kept, by the sizes' values: the
// workspace query, the call and the next layers' calls all ask for the same (1 group: 3.1 us
// to make, 0.1 to find).  Up to 256 groups, which bounds what a thread holds: past them
// every question makes it (257 groups: 44 us, 512: 84, where 256 take 3 to compare).
bool make_plan(const Sizes& z, Plan* p) {
    constexpr int kKept = 256;
    struct Kept {
        bool any;
        Sizes z;
        int32_t groups[4 * kKept];
        Plan p;
    };
    static thread_local Kept kept;
    const size_t bytes = (size_t)z.n_groups * 4 * sizeof(int32_t);
    if (!kept.any || !kept.z.same(z) || (bytes && std::memcmp(kept.groups, z.groups, bytes))) {
        *p = plan_for(z);
        size_workspace(z, p);
        kept.any = z.n_groups <= kKept;
        if (kept.any) {
            kept.z = z;
            kept.p = *p;
            if (bytes) std::memcpy(kept.groups, z.groups, bytes);
        }
    } else {
        *p = kept.p;
    }
    return p->fits;
}

template <typename T> int launch(Args& a, const Plan& p, int64_t n_rows, hipStream_t st) {
    const dim3 grid((unsigned)(p.shared_items + p.own_items)), threads(64 * kWaves);
    // About 240 workgroups with work, or 256 in all, get a CU each, by LDS that lets no
    // second one in: the dispatcher otherwise pairs some and leaves CUs idle (9 sequences,
    // 5 groups of 20000 rows in chunks of 2560, bf16: 80 us for 46; 27 sequences, 5 groups
    // of 6656 rows: 33 for 26).
#define CRANE_SHARED_CASE(s, o, once)                                                                        \
    static_assert(sizeof(AttnShared<s, o>) <= kHalfLds);                                                     \
    if (p.shared_rows == s && p.own_rows == o && (s != 32 || o != 16 || once == (p.shared_tiles == 1)))      \
        hipLaunchKernelGGL((shared_attn_kernel<T, s, o, once>), grid, threads,                               \
                           p.spread ? kHalfLds + 256 - sizeof(AttnShared<s, o>) : 0, st, a);
    CRANE_SHARED_CASE(16, 16, true)
    CRANE_SHARED_CASE(32, 16, true)
    CRANE_SHARED_CASE(32, 16, false)
    CRANE_SHARED_CASE(32, 32, false)
    if constexpr (sizeof(T) == 2) {
        CRANE_SHARED_CASE(128, 16, false)
        CRANE_SHARED_CASE(128, 32, false)
        CRANE_SHARED_CASE(128, 128, false)
    }
#undef CRANE_SHARED_CASE
    int rc = launch_status(hipGetLastError());
    if (rc || p.shared_splits + p.own_splits == 1) return rc;
    const int64_t slots = p.shared_splits + p.own_splits;
    if (slots <= kJoinRegs || n_rows > kMostThreads / 256)
        hipLaunchKernelGGL((shared_join_kernel<T, 1>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, st, a,
                           (int)n_rows);
    else if (slots <= 4 * kJoinRegs || n_rows > kMostThreads / 1024)
        hipLaunchKernelGGL((shared_join_kernel<T, 4>), dim3((unsigned)n_rows), dim3(256), 0, st, a, (int)n_rows);
    else
        hipLaunchKernelGGL((shared_join_kernel<T, 16>), dim3((unsigned)n_rows), dim3(1024), 0, st, a, (int)n_rows);
    return launch_status(hipGetLastError());
}

int64_t mean_of(int64_t mean_own, int64_t max_own) { return std::min(std::max<int64_t>(mean_own, 0), max_own); }

// The checks both entry points make of the sizes.
int check_sizes(const int32_t* groups, int n_groups, int64_t max_own, int B, int S, int Hq, int Hkv, int D, int dtype) {
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return CRANE_HIP_E_INVALID;
    if (Hq % Hkv != 0) return CRANE_HIP_E_GQA;
    if (B > 65535 || n_groups < 0 || n_groups > B || (n_groups > 0 && !groups)) return CRANE_HIP_E_INVALID;
    if ((int64_t)B * Hq > 0x7fffffffLL || (int64_t)B * Hq * S > kMostThreads / 64) return CRANE_HIP_E_INVALID;
    // a chunk's bounds stay within 31 bits
    const int64_t most = 0x7fffffffLL - 2 * kMaxChunk;
    if (max_own < 0 || max_own > most) return CRANE_HIP_E_INVALID;
    for (int g = 0; g < n_groups; ++g) {
        const int32_t* d = groups + 4 * g;
        if (d[0] < 0 || d[1] < 0 || (int64_t)d[0] + d[1] > B || d[2] < 0 || d[2] >= B || d[3] < 0 ||
            d[3] > most - max_own)
            return CRANE_HIP_E_INVALID;
    }
    return CRANE_HIP_OK;
}

}  // namespace
}  // namespace crane

using namespace crane;

extern "C" size_t crane_hip_attn_shared_workspace(const int32_t* groups_host, int n_groups, int64_t max_kv,
                                                  int64_t max_own, int64_t mean_own, int B, int S, int Hq, int Hkv,
                                                  int D, int dtype) {
    if (check_sizes(groups_host, n_groups, max_own, B, S, Hq, Hkv, D, dtype) || B == 0 || S == 0 || max_kv <= 0)
        return 0;
    Plan p;
    const Sizes z{groups_host, n_groups, max_kv, max_own, mean_of(mean_own, max_own), B, S,
                  Hq, Hkv, dtype == CRANE_HIP_BF16};
    return make_plan(z, &p) ? p.total : 0;
}

extern "C" int crane_hip_attn_shared_paged(const void* q, const void* k_pool, const void* v_pool, int64_t n_pages,
                                           int page_rows, const int32_t* block_table, int64_t table_stride,
                                           const int32_t* kv_len, int64_t max_kv, const int32_t* shared_rows,
                                           const int32_t* groups, const int32_t* members, const int32_t* groups_host,
                                           int n_groups, int64_t max_own, int64_t mean_own, int B, int S, int Hq,
                                           int Hkv, int D, float scale, int flags, void* workspace, size_t ws_bytes,
                                           void* out, int dtype, void* stream) {
    int rc = check_sizes(groups_host, n_groups, max_own, B, S, Hq, Hkv, D, dtype);
    if (rc) return rc;
    if (flags & ~CRANE_HIP_PREFILL_CAUSAL) return CRANE_HIP_E_INVALID;
    if (!(scale > 0.0f) || !__builtin_isfinite(scale)) return CRANE_HIP_E_INVALID;
    rc = check_paged(n_pages, page_rows, block_table, table_stride, Hkv);
    if (rc) return rc;
    if (max_kv <= 0) return CRANE_HIP_E_INVALID;
    if (max_kv > table_stride * page_rows || max_own > max_kv) return CRANE_HIP_E_CAPACITY;
    if (B == 0 || S == 0) return CRANE_HIP_OK;
    if (!q || !k_pool || !v_pool || !kv_len || !out) return CRANE_HIP_E_INVALID;
    if (n_groups > 0 && (!shared_rows || !groups || !members)) return CRANE_HIP_E_INVALID;
    if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) ||
        (n_groups > 0 && !aligned16(groups)))
        return CRANE_HIP_E_ALIGN;
    Plan p;
    const Sizes z{groups_host, n_groups, max_kv, max_own, mean_of(mean_own, max_own), B, S,
                  Hq, Hkv, dtype == CRANE_HIP_BF16};
    if (!make_plan(z, &p)) return CRANE_HIP_E_INVALID;
    if (p.max_shared > max_kv) return CRANE_HIP_E_CAPACITY;
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
    a.n_members = p.members;
    a.max_shared = p.max_shared;
    a.B = B;
    a.S = S;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.max_kv = (int)max_kv;
    a.causal = flags & CRANE_HIP_PREFILL_CAUSAL;
    a.c = scale * kLog2e;
    a.chunk = p.chunk;
    a.shared_splits = (int)p.shared_splits;
    a.own_splits = (int)p.own_splits;
    a.shared_tiles = (int)p.shared_tiles;
    a.own_tiles = (int)p.own_tiles;
    a.shared_items = (int)p.shared_items;
    a.ws_o = (float*)workspace;
    a.ws_ml = (float2*)((char*)workspace + p.ml_off);
    const int64_t n_rows = (int64_t)B * Hq * S;
    const hipStream_t st = (hipStream_t)stream;
    return dtype == CRANE_HIP_F32 ? launch<float>(a, p, n_rows, st) : launch<bf16_t>(a, p, n_rows, st);
}
