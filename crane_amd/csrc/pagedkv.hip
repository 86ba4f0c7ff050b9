// pagedkv.hip -- paged KV-cache manager (one layer's K/V pools) over the paged
// attention launchers; the C ABI is include/crane_pkv.h.
//
// Crane keeps one contiguous [B, Hkv, cap, D] buffer per layer and sequence
// group (Attention::update_kv_cache, qwen3/modeling.rs:313-370) and copies
// whole caches to set up and tear down every batched-decode round
// (setup_batch_decode / pad_and_stack_kv_caches :973-1030, 1141-1200;
// extract_batch_kv :1066-1102).  Here rows live in fixed pages of a pool and a
// sequence is a list of page ids: appends fill the last page and then take a
// new one from the free list, and a batch is B rows of a block table, so no KV
// row is ever moved.  Page lists and lengths are kept on the host (the source
// of truth) and mirrored on the device for the current batch only: set_batch
// uploads them, and an append that opens new pages patches the device table
// with a kernel whose arguments carry the new entries (no host buffer, no
// synchronisation on the decode path).
//
// Pages are shared: each counts the sequences that hold it, a fork adds owners to the
// pages its rows fill and copies the page they end in, and a page returns to the free
// list with its last owner.  A shared page is full of rows for each of its owners, and
// every operation keeps it so (fork and truncate copy the page that would be partial,
// write_seq gives its shared pages up first), so an append only ever writes pages of
// one owner and needs no check.  set_batch groups the batch by its shared pages for
// the attention that reads them once.  Calls over several layers' caches plan every
// cache first and change none unless all can go through; caches that need the same
// copies get them in one launch.
#include <algorithm>
#include <new>
#include <vector>

#include "common.h"
#include "page_groups.h"
#include "../../include/crane_pkv.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr int kPatch = 64;  // table entries per patch launch
struct TablePatch {
    int n;
    int32_t idx[kPatch];
    int32_t val[kPatch];
};

__global__ void patch_table_kernel(int32_t* table, TablePatch p) {
    const int i = threadIdx.x;
    if (i < p.n) table[p.idx[i]] = p.val[i];
}

__global__ void pkv_add_lengths_kernel(int32_t* len, int B, int S) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < B) len[i] += S;
}

__global__ void pkv_starts_kernel(const int32_t* len, int32_t* start, int B, int S) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < B) start[i] = len[i] - S;
}

// Contiguous rows [B, Hkv, S, D] -> rows (start[b] or 0) + s of the pages.
// One thread moves 16 bytes; K and V together.
__global__ __launch_bounds__(256) void scatter_rows_kernel(const uint8_t* __restrict__ k, const uint8_t* __restrict__ v,
                                                           uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool,
                                                           PagedRows rows, const int32_t* __restrict__ start, int B,
                                                           int Hkv, int S, int row_bytes, int64_t n_chunks) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= n_chunks) return;
    const int cpr = row_bytes / 16;
    const int64_t row = t / cpr;
    const int chunk = (int)(t % cpr);
    const int s = (int)(row % S);
    const int kvh = (int)((row / S) % Hkv);
    const int b = (int)(row / ((int64_t)S * Hkv));
    const int64_t off = rows.offset(b, Hkv, kvh, (int64_t)(start ? start[b] : 0) + s);
    if (off < 0) return;
    const int64_t dst = off * (row_bytes / kHeadDim) + 16 * chunk;
    const int64_t src = row * row_bytes + 16 * chunk;
    *reinterpret_cast<uint4*>(k_pool + dst) = *reinterpret_cast<const uint4*>(k + src);
    *reinterpret_cast<uint4*>(v_pool + dst) = *reinterpret_cast<const uint4*>(v + src);
}

// Rows [0, len) of sequence (table row) 0 -> contiguous [Hkv, len, D].
__global__ __launch_bounds__(256) void gather_rows_kernel(const uint8_t* __restrict__ k_pool,
                                                          const uint8_t* __restrict__ v_pool, uint8_t* __restrict__ k,
                                                          uint8_t* __restrict__ v, PagedRows rows, int Hkv, int64_t len,
                                                          int row_bytes, int64_t n_chunks) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= n_chunks) return;
    const int cpr = row_bytes / 16;
    const int64_t row = t / cpr;
    const int chunk = (int)(t % cpr);
    const int64_t j = row % len;
    const int kvh = (int)(row / len);
    const int64_t off = rows.offset(0, Hkv, kvh, j);
    const int64_t dst = row * row_bytes + 16 * chunk;
    uint4 zk = make_uint4(0, 0, 0, 0), zv = zk;
    if (off >= 0) {
        const int64_t src = off * (row_bytes / kHeadDim) + 16 * chunk;
        zk = *reinterpret_cast<const uint4*>(k_pool + src);
        zv = *reinterpret_cast<const uint4*>(v_pool + src);
    }
    *reinterpret_cast<uint4*>(k + dst) = zk;
    *reinterpret_cast<uint4*>(v + dst) = zv;
}

int hip_rc(hipError_t e) { return e == hipSuccess ? CRANE_HIP_OK : CRANE_HIP_E_LAUNCH; }

struct Seq {
    bool live = false;
    int64_t len = 0;
    std::vector<int32_t> pages;
};

// Page copies of one cache: rows [0, rows[i]) of page src[i] to page dst[i].
struct Copies {
    std::vector<int32_t> src, dst, rows;
    void add(int32_t s, int32_t d, int64_t r) {
        src.push_back(s);
        dst.push_back(d);
        rows.push_back((int32_t)r);
    }
    bool operator==(const Copies& o) const { return src == o.src && dst == o.dst && rows == o.rows; }
};

}  // namespace

class PagedKv {
  public:
    PagedKv(int Hkv, int D, int dtype, int P, int64_t n_pages, int max_seqs, int max_pps)
        : Hkv_(Hkv), D_(D), dtype_(dtype), es_(elem_size(dtype)), P_(P), n_pages_(n_pages), max_seqs_(max_seqs),
          max_pps_(max_pps), seqs_(max_seqs) {}
    ~PagedKv() { release(); }
    PagedKv(const PagedKv&) = delete;
    PagedKv& operator=(const PagedKv&) = delete;

    int init() {
        const size_t pool = pool_bytes();
        if (hipMalloc(&k_pool_, pool) != hipSuccess || hipMalloc(&v_pool_, pool) != hipSuccess ||
            hipMalloc(&d_table_, sizeof(int32_t) * (size_t)max_seqs_ * max_pps_) != hipSuccess ||
            hipMalloc(&d_len_, sizeof(int32_t) * (size_t)max_seqs_) != hipSuccess ||
            hipMalloc(&d_start_, sizeof(int32_t) * (size_t)max_seqs_) != hipSuccess ||
            hipMalloc(&d_one_, sizeof(int32_t) * (size_t)max_pps_) != hipSuccess ||
            hipMalloc(&d_groups_, sizeof(int32_t) * 4 * (size_t)max_seqs_) != hipSuccess) {
            release();
            return CRANE_HIP_E_LAUNCH;
        }
        refs_.assign((size_t)n_pages_, 0);
        free_.reserve((size_t)n_pages_);
        for (int64_t p = n_pages_ - 1; p >= 0; --p) free_.push_back((int32_t)p);
        return CRANE_HIP_OK;
    }

    size_t row_bytes() const { return (size_t)D_ * es_; }
    size_t pool_bytes() const { return (size_t)n_pages_ * Hkv_ * P_ * row_bytes(); }
    uint64_t bytes() const { return 2ull * pool_bytes(); }
    int64_t free_pages() const { return (int64_t)free_.size(); }
    int B() const { return (int)batch_.size(); }
    int Hkv() const { return Hkv_; }
    int D() const { return D_; }
    int dtype() const { return dtype_; }

    bool live(int id) const { return id >= 0 && id < max_seqs_ && seqs_[id].live; }
    bool in_batch(int id) const { return std::find(batch_.begin(), batch_.end(), id) != batch_.end(); }
    int64_t len(int id) const { return live(id) ? seqs_[id].len : -1; }
    int64_t max_len() const {
        int64_t m = 0;
        for (int id : batch_) m = std::max(m, seqs_[id].len);
        return m;
    }
    PagedRows batch_rows() const { return PagedRows{d_table_, max_pps_, n_pages_, P_}; }

    int seq_add(int* id) {
        for (int i = 0; i < max_seqs_; ++i)
            if (!seqs_[i].live) {
                seqs_[i].live = true;
                seqs_[i].len = 0;
                seqs_[i].pages.clear();
                *id = i;
                return CRANE_HIP_OK;
            }
        return CRANE_HIP_E_CAPACITY;
    }

    int seq_free(int id) {
        if (!live(id) || in_batch(id)) return CRANE_HIP_E_INVALID;
        Seq& s = seqs_[id];
        for (auto it = s.pages.rbegin(); it != s.pages.rend(); ++it) drop(*it);
        s = Seq();
        return CRANE_HIP_OK;
    }

    int set_batch(const int* ids, int B, hipStream_t st) {
        if (B < 0 || B > max_seqs_ || (B > 0 && !ids)) return CRANE_HIP_E_INVALID;
        std::vector<char> seen((size_t)max_seqs_, 0);
        for (int b = 0; b < B; ++b) {
            if (!live(ids[b]) || seen[ids[b]]) return CRANE_HIP_E_INVALID;
            seen[ids[b]] = 1;
        }
        PageGroups groups;
        std::vector<int32_t> table((size_t)B * max_pps_, -1), lens((size_t)B), shared;
        for (int b = 0; b < B; ++b) {
            const Seq& s = seqs_[ids[b]];
            std::copy(s.pages.begin(), s.pages.end(), table.begin() + (size_t)b * max_pps_);
            lens[b] = (int32_t)s.len;
        }
        if (shared_pages_ > 0) {
            std::vector<PageList> lists((size_t)B);
            for (int b = 0; b < B; ++b) lists[b] = {seqs_[ids[b]].pages.data(), seqs_[ids[b]].pages.size()};
            groups = group_pages(lists);
        }
        if (groups.count()) {  // crane_hip_attn_shared_paged's groups, members and shared rows
            for (int i = 0; i < groups.count(); ++i) {
                const int32_t at = groups.start[i], leader = groups.members[at];
                for (int32_t x : {at, groups.start[i + 1] - at, leader, groups.shared[leader] * P_})
                    shared.push_back(x);
            }
            shared.insert(shared.end(), groups.members.begin(), groups.members.end());
            for (int32_t pages : groups.shared) shared.push_back(pages * P_);
        }
        std::vector<int> batch(ids, ids + B);
        batch_.clear();  // no batch if an upload fails
        n_groups_ = 0;
        if (B == 0) return CRANE_HIP_OK;
        int rc = upload(d_table_, table, st);
        if (!rc) rc = upload(d_len_, lens, st);
        if (!rc && !shared.empty()) rc = upload(d_groups_, shared, st);
        if (!rc) rc = hip_rc(hipStreamSynchronize(st));  // the staging vectors go out of scope
        if (rc) return rc;
        batch_.swap(batch);
        n_groups_ = groups.count();
        n_members_ = (int)groups.members.size();
        batch_groups_.swap(shared);
        return CRANE_HIP_OK;
    }

    // Pages for S more rows in every batch sequence: checked first, then taken
    // from the free list, and the new device table entries patched in.
    // added[b] counts the pages batch sequence b received (for unreserve).
    int reserve(int64_t S, hipStream_t st, std::vector<int>* added = nullptr) {
        if (S < 0) return CRANE_HIP_E_INVALID;
        int64_t need_total = 0;
        for (int id : batch_) {
            const Seq& s = seqs_[id];
            const int64_t need = (s.len + S + P_ - 1) / P_;
            if (need > max_pps_ || s.len + S > 0x7fffffffLL) return CRANE_HIP_E_CAPACITY;
            need_total += std::max<int64_t>(0, need - (int64_t)s.pages.size());
        }
        if (need_total > (int64_t)free_.size()) return CRANE_HIP_E_CAPACITY;
        TablePatch patch;
        patch.n = 0;
        if (added) added->assign((size_t)B(), 0);
        for (int b = 0; b < B(); ++b) {
            Seq& s = seqs_[batch_[b]];
            const int64_t need = (s.len + S + P_ - 1) / P_;
            while ((int64_t)s.pages.size() < need) {
                if (added) ++(*added)[b];
                const int32_t page = take();
                patch.idx[patch.n] = (int32_t)((int64_t)b * max_pps_ + (int64_t)s.pages.size());
                patch.val[patch.n] = page;
                ++patch.n;
                s.pages.push_back(page);
                if (patch.n == kPatch) {
                    const int rc = launch_patch(d_table_, patch, st);
                    if (rc) return rc;
                    patch.n = 0;
                }
            }
        }
        return patch.n ? launch_patch(d_table_, patch, st) : CRANE_HIP_OK;
    }

    // Give back the pages a reserve() took when the launch it was for was
    // rejected.  Their device table entries stay, past the sequences' page
    // counts, where no kernel reads them; the next reserve() overwrites them.
    void unreserve(const std::vector<int>& added) {
        for (int b = B() - 1; b >= 0; --b) {
            Seq& s = seqs_[batch_[b]];
            for (int i = 0; i < added[b]; ++i) {
                drop(s.pages.back());
                s.pages.pop_back();
            }
        }
    }

    int grow_lengths(int S, hipStream_t st) {
        for (int id : batch_) seqs_[id].len += S;
        if (batch_.empty()) return CRANE_HIP_OK;
        hipLaunchKernelGGL(pkv_add_lengths_kernel, dim3((B() + 255) / 256), dim3(256), 0, st, d_len_, B(), S);
        return launch_status(hipGetLastError());
    }

    int update(const void* k, const void* v, int S, hipStream_t st) {
        if (S < 0) return CRANE_HIP_E_INVALID;
        if (S == 0 || batch_.empty()) return CRANE_HIP_OK;
        if (!k || !v || !aligned16(k) || !aligned16(v)) return !k || !v ? CRANE_HIP_E_INVALID : CRANE_HIP_E_ALIGN;
        int rc = reserve(S, st);
        if (rc) return rc;
        rc = scatter(k, v, batch_rows(), d_len_, B(), S, st);
        return rc ? rc : grow_lengths(S, st);
    }

    int append_qkv(const void* qkv, int64_t qkv_row_stride, const void* q_norm_w, const void* k_norm_w, float eps,
                   int order, const void* cos, const void* sin, int64_t cs_stride, int64_t table_rows,
                   const int32_t* positions, void* q_out, int S, int Hq, hipStream_t st) {
        if (S < 0 || Hq <= 0) return CRANE_HIP_E_INVALID;
        if (S == 0 || batch_.empty()) return CRANE_HIP_OK;
        std::vector<int> added;
        int rc = reserve(S, st, &added);
        if (rc) return rc;
        rc = crane_hip_qknorm_rope_append_paged(qkv, qkv_row_stride, q_norm_w, k_norm_w, eps, order, cos, sin,
                                                cs_stride, table_rows, positions, q_out, k_pool_, v_pool_, n_pages_,
                                                P_, d_table_, max_pps_, d_len_, B(), S, Hq, Hkv_, D_, dtype_, st);
        if (rc) {  // rejected arguments: nothing ran, the pages go back
            unreserve(added);
            return rc;
        }
        return grow_lengths(S, st);
    }

    int decode(const void* q, int Hq, float scale, int score_mode, void* ws, size_t ws_bytes, void* out,
               hipStream_t st) const {
        if (batch_.empty()) return CRANE_HIP_OK;
        const int64_t m = max_len();
        if (m == 0) return CRANE_HIP_E_INVALID;
        return crane_hip_attn_decode_paged(q, k_pool_, v_pool_, n_pages_, P_, d_table_, max_pps_, d_len_, m, B(), Hq,
                                           Hkv_, D_, scale, score_mode, ws, ws_bytes, out, dtype_, st);
    }

    int prefill(const void* q, int Hq, int S, float scale, int flags, void* out, hipStream_t st) {
        if (S < 0) return CRANE_HIP_E_INVALID;
        if (batch_.empty() || S == 0) return CRANE_HIP_OK;
        for (int id : batch_)
            if (seqs_[id].len < S) return CRANE_HIP_E_INVALID;  // every sequence holds its S new rows
        hipLaunchKernelGGL(pkv_starts_kernel, dim3((B() + 255) / 256), dim3(256), 0, st, d_len_, d_start_, B(), S);
        const int rc = launch_status(hipGetLastError());
        if (rc) return rc;
        return crane_hip_attn_prefill_paged(q, k_pool_, v_pool_, n_pages_, P_, d_table_, max_pps_, d_start_,
                                            max_len() - S, B(), S, Hq, Hkv_, D_, scale, flags, out, dtype_, st);
    }

    int read_seq(int id, void* k, void* v, hipStream_t st) {
        if (!live(id)) return CRANE_HIP_E_INVALID;
        const Seq& s = seqs_[id];
        if (s.len == 0) return CRANE_HIP_OK;
        if (!k || !v) return CRANE_HIP_E_INVALID;
        if (!aligned16(k) || !aligned16(v)) return CRANE_HIP_E_ALIGN;
        int rc = upload_one(s.pages, st);
        if (rc) return rc;
        const int64_t n_chunks = (int64_t)Hkv_ * s.len * (int64_t)(row_bytes() / 16);
        hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)((n_chunks + 255) / 256)), dim3(256), 0, st,
                           (const uint8_t*)k_pool_, (const uint8_t*)v_pool_, (uint8_t*)k, (uint8_t*)v, one_rows(), Hkv_,
                           s.len, (int)row_bytes(), n_chunks);
        return launch_status(hipGetLastError());
    }

    int write_seq(int id, const void* k, const void* v, int64_t len, hipStream_t st) {
        if (!live(id) || in_batch(id) || len < 0) return CRANE_HIP_E_INVALID;
        if (len > 0 && (!k || !v)) return CRANE_HIP_E_INVALID;
        if (len > 0 && (!aligned16(k) || !aligned16(v))) return CRANE_HIP_E_ALIGN;
        Seq& s = seqs_[id];
        const int64_t need = (len + P_ - 1) / P_;
        if (need > max_pps_ || len > 0x7fffffffLL) return CRANE_HIP_E_CAPACITY;
        // A page other sequences hold is not written: it is given up for another.
        int64_t kept = 0, back = 0;
        for (int32_t p : s.pages) {
            if (refs_[p] == 1 && kept < need) ++kept;
            else if (refs_[p] == 1) ++back;
        }
        if (need - kept > (int64_t)free_.size() + back) return CRANE_HIP_E_CAPACITY;
        std::vector<int32_t> pages;
        pages.reserve((size_t)need);
        for (int32_t p : s.pages)
            if (refs_[p] == 1 && (int64_t)pages.size() < need) pages.push_back(p);
        int64_t left = kept;
        for (size_t i = s.pages.size(); i-- > 0;) {  // from the last: free ids come back in order
            const int32_t p = s.pages[i];
            if (left > 0 && p == pages[left - 1]) --left;
            else drop(p);
        }
        while ((int64_t)pages.size() < need) pages.push_back(take());
        s.pages.swap(pages);
        s.len = len;
        if (len == 0) return CRANE_HIP_OK;
        const int rc = upload_one(s.pages, st);
        return rc ? rc : scatter(k, v, one_rows(), nullptr, 1, len, st);
    }

    // ---- shared pages: plan_* fill a plan and change nothing, commit_* apply it

    struct Fork {
        std::vector<Seq> children;
        Copies copies;
    };
    int plan_fork(int src, int64_t rows, int count, Fork* f) const {
        if (!live(src)) return CRANE_HIP_E_INVALID;
        const Seq& s = seqs_[src];
        const int64_t n = rows < 0 ? s.len : rows;
        if (n > s.len) return CRANE_HIP_E_INVALID;
        const int64_t full = n / P_, part = n % P_;
        if (count > max_seqs_ || (part && (int64_t)count > free_pages())) return CRANE_HIP_E_CAPACITY;
        f->children.resize((size_t)count);
        for (int c = 0; c < count; ++c) {
            Seq& child = f->children[c];
            child.live = true;
            child.len = n;
            child.pages.assign(s.pages.begin(), s.pages.begin() + full);
            if (part) {
                child.pages.push_back(free_[free_.size() - 1 - (size_t)c]);
                f->copies.add(s.pages[full], child.pages.back(), part);
            }
        }
        return CRANE_HIP_OK;
    }
    void commit_fork(Fork& f, const int* ids) {
        for (size_t c = 0; c < f.children.size(); ++c) {
            Seq& child = f.children[c];
            const int64_t full = child.len / P_;
            for (int64_t i = 0; i < full; ++i) hold(child.pages[i]);
            if (child.len % P_) take();  // the planned one
            seqs_[ids[c]] = std::move(child);
        }
    }

    struct Cut {
        int64_t rows = 0;
        bool copy = false;  // the last page is shared and becomes partial
        Copies copies;
    };
    int plan_truncate(int id, int64_t rows, Cut* c) const {
        if (!live(id) || in_batch(id) || rows < 0 || rows > seqs_[id].len) return CRANE_HIP_E_INVALID;
        const Seq& s = seqs_[id];
        const int64_t need = (rows + P_ - 1) / P_;
        c->rows = rows;
        c->copy = rows % P_ && refs_[s.pages[need - 1]] > 1;
        if (!c->copy) return CRANE_HIP_OK;
        // The page it takes: the list's last, or else the last page it gives back.
        int32_t page = free_.empty() ? -1 : free_.back();
        for (int64_t i = (int64_t)s.pages.size() - 1; i >= need; --i)
            if (refs_[s.pages[i]] == 1) page = s.pages[i];
        if (page < 0) return CRANE_HIP_E_CAPACITY;
        c->copies.add(s.pages[need - 1], page, rows % P_);
        return CRANE_HIP_OK;
    }
    void commit_truncate(int id, const Cut& c) {
        Seq& s = seqs_[id];
        const int64_t need = (c.rows + P_ - 1) / P_;
        while ((int64_t)s.pages.size() > need) {
            drop(s.pages.back());
            s.pages.pop_back();
        }
        if (c.copy) {
            drop(s.pages.back());
            s.pages.back() = take();
        }
        s.len = c.rows;
    }

    struct Move {
        std::vector<int32_t> to;    // every page's place afterwards
        std::vector<int32_t> free;  // the free list afterwards
        Copies copies;
    };
    int plan_compact(Move* m) const {
        const int64_t used = n_pages_ - free_pages();
        m->to.resize((size_t)n_pages_);
        m->free.reserve((size_t)n_pages_);
        int64_t hole = 0;
        for (int64_t p = 0; p < n_pages_; ++p) {
            m->to[p] = (int32_t)p;
            if (p < used || refs_[p] == 0) continue;
            while (refs_[hole] != 0) ++hole;  // as many free ids lie below `used` as held ones from it on
            m->to[p] = (int32_t)hole;
            m->copies.add((int32_t)p, (int32_t)hole, P_);
            ++hole;
        }
        for (int64_t p = n_pages_ - 1; p >= used; --p) m->free.push_back((int32_t)p);
        return CRANE_HIP_OK;
    }
    int commit_compact(Move& m, hipStream_t st) {
        for (size_t i = 0; i < m.copies.src.size(); ++i) {
            refs_[m.copies.dst[i]] = refs_[m.copies.src[i]];
            refs_[m.copies.src[i]] = 0;
        }
        free_.swap(m.free);
        TablePatch patch;
        patch.n = 0;
        int rc = CRANE_HIP_OK;
        for (int b = 0; b < B(); ++b) {
            const Seq& s = seqs_[batch_[b]];
            for (size_t i = 0; i < s.pages.size(); ++i) {
                if (m.to[s.pages[i]] == s.pages[i]) continue;
                patch.idx[patch.n] = (int32_t)((int64_t)b * max_pps_ + (int64_t)i);
                patch.val[patch.n] = m.to[s.pages[i]];
                if (++patch.n < kPatch) continue;
                rc = rc ? rc : launch_patch(d_table_, patch, st);
                patch.n = 0;
            }
        }
        for (Seq& s : seqs_)
            for (int32_t& p : s.pages) p = m.to[p];
        return rc || !patch.n ? rc : launch_patch(d_table_, patch, st);
    }

    // Attention of the batch's last S rows, shared pages read once per group.
    int64_t max_own() const {
        int64_t m = 0;
        for (int b = 0; b < B(); ++b) m = std::max(m, seqs_[batch_[b]].len - batch_shared_rows(b));
        return m;
    }
    int64_t mean_own() const {
        int64_t sum = 0;
        for (int b = 0; b < B(); ++b) sum += seqs_[batch_[b]].len - batch_shared_rows(b);
        return B() ? sum / B() : 0;
    }
    size_t shared_workspace(int Hq, int S) const {
        return crane_hip_attn_shared_workspace(batch_groups_.data(), n_groups_, max_len(), max_own(), mean_own(), B(),
                                               S, Hq, Hkv_, D_, dtype_);
    }
    int attention_shared(const void* q, int Hq, int S, float scale, int flags, void* ws, size_t ws_bytes, void* out,
                         hipStream_t st) const {
        if (S < 0) return CRANE_HIP_E_INVALID;
        if (batch_.empty() || S == 0) return CRANE_HIP_OK;
        for (int id : batch_)
            if (S > 1 && seqs_[id].len < S) return CRANE_HIP_E_INVALID;  // every sequence holds its S new rows
        if (max_len() == 0) return CRANE_HIP_E_INVALID;
        const int32_t *members = d_groups_ + 4 * n_groups_, *shared = members + n_members_;
        return crane_hip_attn_shared_paged(q, k_pool_, v_pool_, n_pages_, P_, d_table_, max_pps_, d_len_, max_len(),
                                           shared, d_groups_, members, batch_groups_.data(), n_groups_, max_own(),
                                           mean_own(), B(), S, Hq, Hkv_, D_, scale, flags, ws, ws_bytes, out, dtype_, st);
    }

    bool same_shape(const PagedKv& o) const {
        return Hkv_ == o.Hkv_ && D_ == o.D_ && dtype_ == o.dtype_ && P_ == o.P_ && n_pages_ == o.n_pages_;
    }
    int max_seqs() const { return max_seqs_; }
    void* k_pool() const { return k_pool_; }
    void* v_pool() const { return v_pool_; }
    int copy_into(std::vector<void*>& pools, const Copies& c, hipStream_t st) const {
        return crane_hip_copy_pages(pools.data(), (int)pools.size(), n_pages_, P_, Hkv_, D_, c.src.data(), c.dst.data(),
                                    c.rows.data(), (int)c.src.size(), dtype_, st);
    }

    void views(void** k, void** v, const int32_t** table, int64_t* stride, const int32_t** dlen) const {
        if (k) *k = k_pool_;
        if (v) *v = v_pool_;
        if (table) *table = d_table_;
        if (stride) *stride = max_pps_;
        if (dlen) *dlen = d_len_;
    }

  private:
    // A page's owners: take one for a first owner, add one, drop one.
    int32_t take() {
        const int32_t p = free_.back();
        free_.pop_back();
        refs_[p] = 1;
        return p;
    }
    void hold(int32_t p) {
        if (++refs_[p] == 2) ++shared_pages_;
    }
    void drop(int32_t p) {
        if (refs_[p] == 2) --shared_pages_;
        if (--refs_[p] == 0) free_.push_back(p);
    }
    int64_t batch_shared_rows(int b) const {
        return n_groups_ ? batch_groups_[(size_t)(4 * n_groups_ + n_members_ + b)] : 0;
    }

    static int upload(int32_t* dst, const std::vector<int32_t>& v, hipStream_t st) {
        return hip_rc(hipMemcpyAsync(dst, v.data(), sizeof(int32_t) * v.size(), hipMemcpyHostToDevice, st));
    }

    static int launch_patch(int32_t* table, const TablePatch& p, hipStream_t st) {
        hipLaunchKernelGGL(patch_table_kernel, dim3(1), dim3(kPatch), 0, st, table, p);
        return launch_status(hipGetLastError());
    }

    PagedRows one_rows() const { return PagedRows{d_one_, max_pps_, n_pages_, P_}; }

    // One sequence's page ids into the single-row table d_one_.
    int upload_one(const std::vector<int32_t>& pages, hipStream_t st) {
        std::vector<int32_t> row((size_t)max_pps_, -1);
        std::copy(pages.begin(), pages.end(), row.begin());
        int rc = hip_rc(hipMemcpyAsync(d_one_, row.data(), sizeof(int32_t) * row.size(), hipMemcpyHostToDevice, st));
        return rc ? rc : hip_rc(hipStreamSynchronize(st));  // `row` is a local staging buffer
    }

    int scatter(const void* k, const void* v, const PagedRows& rows, const int32_t* start, int B, int64_t S,
                hipStream_t st) {
        const int64_t n_chunks = (int64_t)B * Hkv_ * S * (int64_t)(row_bytes() / 16);
        if ((n_chunks + 255) / 256 > 0x7fffffffLL || S > 0x7fffffffLL) return CRANE_HIP_E_INVALID;
        hipLaunchKernelGGL(scatter_rows_kernel, dim3((unsigned)((n_chunks + 255) / 256)), dim3(256), 0, st,
                           (const uint8_t*)k, (const uint8_t*)v, (uint8_t*)k_pool_, (uint8_t*)v_pool_, rows, start, B,
                           Hkv_, (int)S, (int)row_bytes(), n_chunks);
        return launch_status(hipGetLastError());
    }

    void release() {
        for (void* p : {k_pool_, v_pool_, (void*)d_table_, (void*)d_len_, (void*)d_start_, (void*)d_one_,
                        (void*)d_groups_})
            if (p) (void)hipFree(p);
        k_pool_ = v_pool_ = nullptr;
        d_table_ = d_len_ = d_start_ = d_one_ = d_groups_ = nullptr;
    }

    int Hkv_, D_, dtype_;
    size_t es_;
    int P_;
    int64_t n_pages_;
    int max_seqs_, max_pps_;
    void* k_pool_ = nullptr;
    void* v_pool_ = nullptr;
    int32_t* d_table_ = nullptr;  // current batch: B rows of max_pps_ page ids
    int32_t* d_len_ = nullptr;    // current batch lengths
    int32_t* d_start_ = nullptr;  // prefill chunk starts
    int32_t* d_one_ = nullptr;    // one sequence's page ids (read_seq / write_seq)
    int32_t* d_groups_ = nullptr;  // current batch: groups, their members, shared rows (when there are groups)
    std::vector<int32_t> free_;
    std::vector<int32_t> refs_;   // owners of every page
    int64_t shared_pages_ = 0;    // pages of more than one owner
    std::vector<Seq> seqs_;
    std::vector<int> batch_;
    std::vector<int32_t> batch_groups_;  // what d_groups_ holds
    int n_groups_ = 0, n_members_ = 0;
};

}  // namespace crane

using crane::PagedKv;

struct crane_pkv {
    PagedKv impl;
    crane_pkv(int Hkv, int D, int dtype, int P, int64_t n_pages, int max_seqs, int max_pps)
        : impl(Hkv, D, dtype, P, n_pages, max_seqs, max_pps) {}
};

namespace {

// The caches of a call over several layers: distinct and non-null.
int check_caches(crane_pkv* const* caches, int n) {
    if (n < 0 || (n > 0 && !caches)) return CRANE_HIP_E_INVALID;
    std::vector<const crane_pkv*> seen(caches, caches + n);
    std::sort(seen.begin(), seen.end());
    if (n && (!seen[0] || std::adjacent_find(seen.begin(), seen.end()) != seen.end())) return CRANE_HIP_E_INVALID;
    return CRANE_HIP_OK;
}

// Every cache's planned copies, the pools of caches of one shape with the same copies
// in one launch.
template <class PLAN>
int copy_all(crane_pkv* const* caches, const std::vector<PLAN>& plans, hipStream_t st) {
    std::vector<char> done(plans.size(), 0);
    for (size_t i = 0; i < plans.size(); ++i) {
        if (done[i] || plans[i].copies.src.empty()) continue;
        const PagedKv& first = caches[i]->impl;
        std::vector<void*> pools;
        for (size_t j = i; j < plans.size(); ++j) {
            const PagedKv& c = caches[j]->impl;
            if (done[j] || !c.same_shape(first) || !(plans[j].copies == plans[i].copies)) continue;
            done[j] = 1;
            pools.push_back(c.k_pool());
            pools.push_back(c.v_pool());
        }
        const int rc = first.copy_into(pools, plans[i].copies, st);
        if (rc) return rc;
    }
    return CRANE_HIP_OK;
}

}  // namespace

extern "C" int crane_pkv_fork(crane_pkv* const* caches, int n, int seq_id, int64_t rows, int count, int* new_ids,
                              void* stream) {
    try {
        int rc = check_caches(caches, n);
        if (rc) return rc;
        if (count < 0 || rows < -1 || (count > 0 && !new_ids)) return CRANE_HIP_E_INVALID;
        if (n == 0 || count == 0) return CRANE_HIP_OK;
        std::vector<PagedKv::Fork> plans((size_t)n);
        for (int i = 0; i < n; ++i)
            if ((rc = caches[i]->impl.plan_fork(seq_id, rows, count, &plans[i]))) return rc;
        std::vector<int> ids;  // the lowest ids free in every cache
        for (int id = 0; id < caches[0]->impl.max_seqs() && (int)ids.size() < count; ++id) {
            bool open = true;
            for (int i = 0; i < n; ++i) open = open && id < caches[i]->impl.max_seqs() && !caches[i]->impl.live(id);
            if (open) ids.push_back(id);
        }
        if ((int)ids.size() < count) return CRANE_HIP_E_CAPACITY;
        if ((rc = copy_all(caches, plans, (hipStream_t)stream))) return rc;
        for (int i = 0; i < n; ++i) caches[i]->impl.commit_fork(plans[i], ids.data());
        std::copy(ids.begin(), ids.end(), new_ids);
        return CRANE_HIP_OK;
    } catch (...) {  // no memory
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" int crane_pkv_truncate(crane_pkv* const* caches, int n, int seq_id, int64_t rows, void* stream) {
    try {
        int rc = check_caches(caches, n);
        if (rc) return rc;
        std::vector<PagedKv::Cut> plans((size_t)n);
        for (int i = 0; i < n; ++i)
            if ((rc = caches[i]->impl.plan_truncate(seq_id, rows, &plans[i]))) return rc;
        if ((rc = copy_all(caches, plans, (hipStream_t)stream))) return rc;
        for (int i = 0; i < n; ++i) caches[i]->impl.commit_truncate(seq_id, plans[i]);
        return CRANE_HIP_OK;
    } catch (...) {
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" int crane_pkv_compact(crane_pkv* const* caches, int n, int64_t* moved, void* stream) {
    try {
        int rc = check_caches(caches, n);
        if (rc) return rc;
        std::vector<PagedKv::Move> plans((size_t)n);
        int64_t total = 0;
        for (int i = 0; i < n; ++i) {
            if ((rc = caches[i]->impl.plan_compact(&plans[i]))) return rc;
            total += (int64_t)plans[i].copies.src.size();
        }
        if ((rc = copy_all(caches, plans, (hipStream_t)stream))) return rc;
        for (int i = 0; i < n; ++i) {
            const int c = caches[i]->impl.commit_compact(plans[i], (hipStream_t)stream);
            rc = rc ? rc : c;
        }
        if (moved) *moved = total;
        return rc;
    } catch (...) {
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" size_t crane_pkv_shared_workspace(const crane_pkv* pkv, int Hq, int S) {
    return pkv ? pkv->impl.shared_workspace(Hq, S) : 0;
}

extern "C" int crane_pkv_attention_shared(const crane_pkv* pkv, const void* q, int Hq, int S, float scale, int flags,
                                          void* workspace, size_t ws_bytes, void* out, void* stream) {
    return pkv ? pkv->impl.attention_shared(q, Hq, S, scale, flags, workspace, ws_bytes, out, (hipStream_t)stream)
               : CRANE_HIP_E_INVALID;
}

extern "C" int crane_pkv_create(int Hkv, int D, int dtype, int page_rows, int64_t n_pages, int max_seqs,
                                int max_pages_per_seq, crane_pkv** out) {
    if (!out) return CRANE_HIP_E_INVALID;
    *out = nullptr;
    if (dtype != CRANE_HIP_F32 && dtype != CRANE_HIP_BF16) return CRANE_HIP_E_DTYPE;
    if (D != crane::kHeadDim) return CRANE_HIP_E_HEAD_DIM;
    if (Hkv <= 0 || Hkv > 65535 || max_seqs <= 0 || max_seqs > 65535 || max_pages_per_seq <= 0)
        return CRANE_HIP_E_INVALID;
    int32_t dummy = 0;  // the table pointer is not known yet; only the sizes are checked here
    const int rc = crane::check_paged(n_pages, page_rows, &dummy, max_pages_per_seq, Hkv);
    if (rc) return rc;
    crane_pkv* p = new (std::nothrow) crane_pkv(Hkv, D, dtype, page_rows, n_pages, max_seqs, max_pages_per_seq);
    if (!p) return CRANE_HIP_E_INVALID;
    const int irc = p->impl.init();
    if (irc) {
        delete p;
        return irc;
    }
    *out = p;
    return CRANE_HIP_OK;
}

extern "C" void crane_pkv_destroy(crane_pkv* pkv) { delete pkv; }

extern "C" int crane_pkv_seq_add(crane_pkv* pkv, int* seq_id) {
    if (!pkv || !seq_id) return CRANE_HIP_E_INVALID;
    return pkv->impl.seq_add(seq_id);
}

extern "C" int crane_pkv_seq_free(crane_pkv* pkv, int seq_id) {
    return pkv ? pkv->impl.seq_free(seq_id) : CRANE_HIP_E_INVALID;
}

extern "C" int64_t crane_pkv_seq_len(const crane_pkv* pkv, int seq_id) { return pkv ? pkv->impl.len(seq_id) : -1; }

extern "C" int64_t crane_pkv_free_pages(const crane_pkv* pkv) { return pkv ? pkv->impl.free_pages() : 0; }

extern "C" uint64_t crane_pkv_bytes(const crane_pkv* pkv) { return pkv ? pkv->impl.bytes() : 0; }

extern "C" int crane_pkv_set_batch(crane_pkv* pkv, const int* seq_ids, int B, void* stream) {
    try {
        return pkv ? pkv->impl.set_batch(seq_ids, B, (hipStream_t)stream) : CRANE_HIP_E_INVALID;
    } catch (...) {  // no memory
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" int crane_pkv_update(crane_pkv* pkv, const void* k, const void* v, int S, void* stream) {
    return pkv ? pkv->impl.update(k, v, S, (hipStream_t)stream) : CRANE_HIP_E_INVALID;
}

extern "C" int crane_pkv_append_qkv(crane_pkv* pkv, const void* qkv, int64_t qkv_row_stride, const void* q_norm_w,
                                    const void* k_norm_w, float eps, int order, const void* cos, const void* sin,
                                    int64_t cs_stride, int64_t table_rows, const int32_t* positions, void* q_out,
                                    int S, int Hq, void* stream) {
    if (!pkv) return CRANE_HIP_E_INVALID;
    return pkv->impl.append_qkv(qkv, qkv_row_stride, q_norm_w, k_norm_w, eps, order, cos, sin, cs_stride, table_rows,
                                positions, q_out, S, Hq, (hipStream_t)stream);
}

extern "C" int crane_pkv_decode(const crane_pkv* pkv, const void* q, int Hq, float scale, int score_mode,
                                void* workspace, size_t ws_bytes, void* out, void* stream) {
    return pkv ? pkv->impl.decode(q, Hq, scale, score_mode, workspace, ws_bytes, out, (hipStream_t)stream)
               : CRANE_HIP_E_INVALID;
}

extern "C" int crane_pkv_prefill(crane_pkv* pkv, const void* q, int Hq, int S, float scale, int flags, void* out,
                                 void* stream) {
    return pkv ? pkv->impl.prefill(q, Hq, S, scale, flags, out, (hipStream_t)stream) : CRANE_HIP_E_INVALID;
}

extern "C" int crane_pkv_read_seq(crane_pkv* pkv, int seq_id, void* k, void* v, void* stream) {
    try {
        return pkv ? pkv->impl.read_seq(seq_id, k, v, (hipStream_t)stream) : CRANE_HIP_E_INVALID;
    } catch (...) {  // no memory
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" int crane_pkv_write_seq(crane_pkv* pkv, int seq_id, const void* k, const void* v, int64_t len,
                                   void* stream) {
    try {
        return pkv ? pkv->impl.write_seq(seq_id, k, v, len, (hipStream_t)stream) : CRANE_HIP_E_INVALID;
    } catch (...) {  // no memory
        return CRANE_HIP_E_INVALID;
    }
}

extern "C" int crane_pkv_views(const crane_pkv* pkv, void** k_pool, void** v_pool, const int32_t** block_table,
                               int64_t* table_stride, const int32_t** dev_len) {
    if (!pkv) return CRANE_HIP_E_INVALID;
    pkv->impl.views(k_pool, v_pool, block_table, table_stride, dev_len);
    return CRANE_HIP_OK;
}
