// pages.hip -- copies of rows between pages of the K/V pools, and the grouping of
// sequences by the pages they share; the C ABI is crane_hip_copy_pages and
// crane_hip_group_prefixes in include/crane_shared.h.
//
// A page [Hkv, page_rows, D] of a pool is Hkv runs of page_rows rows, and a copy
// takes the first rows of each run.  The pairs and the pools' addresses go to the
// kernel as arguments: the lists are the host's (page lists live there), so nothing
// is uploaded and nothing waits.
#include <algorithm>
#include <vector>

#include "common.h"
#include "page_groups.h"
#include "../../include/crane_shared.h"

namespace crane {
namespace {

constexpr int kPools = 128;      // pools per launch: K and V of 64 layers
constexpr int kPairs = 128;      // pairs per launch
constexpr int kThreads = 256;
constexpr int kBlockBytes = 16 * kThreads;  // bytes of one head's run per workgroup

typedef unsigned int u32x4_v __attribute__((ext_vector_type(4)));

struct CopyArgs {
    uint8_t* pool[kPools];
    int32_t src[kPairs], dst[kPairs], rows[kPairs];
};

// One load and one store a thread.  Bound by HBM: the stores go past the caches, which
// leaves those to a source that is copied to several pages (72 pools, a page of 201 rows
// to 8 others, 267 MB in all: 36 us, 65 with plain stores; 97 pages to 97, 407 MB: 59 us
// for 76), and with 2, 4, 8 or 16 loads issued ahead of the stores the first of these
// takes 44 to 47 us, the second the same.
// grid: (heads x blocks of a run, pairs, pools)
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a, int blocks, int Hkv, int64_t run_bytes,
                                                              int row_bytes) {
    const int head = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const int64_t at = (int64_t)block * kBlockBytes + 16 * threadIdx.x;
    if (at >= (int64_t)a.rows[blockIdx.y] * row_bytes) return;
    uint8_t* pool = a.pool[blockIdx.z];
    const uint8_t* src = pool + ((int64_t)a.src[blockIdx.y] * Hkv + head) * run_bytes;
    uint8_t* dst = pool + ((int64_t)a.dst[blockIdx.y] * Hkv + head) * run_bytes;
    __builtin_nontemporal_store(*reinterpret_cast<const u32x4_v*>(src + at), reinterpret_cast<u32x4_v*>(dst + at));
}

// The lists sorted form a tree: a node is a run of them with `common` first pages in
// common, its kids the sub-runs with more.  A node opened as a group takes the lists
// below it that no deeper open node takes; each is then read as `common` pages fewer,
// but once:  saved = sum over lists of c(deepest open node above it) - sum over open
// nodes of c.  best() maximises that over the nodes to open, for every node and every
// possible open node above it (c = 0: none).  Nodes nested deeper than kDepth are left out,
// which bounds the recursion's stack and best()'s depth^2 sums.
class Grouping {
  public:
    explicit Grouping(const std::vector<PageList>& lists) : lists_(lists), order_(lists.size()) {
        for (size_t i = 0; i < order_.size(); ++i) order_[i] = (int32_t)i;
        std::sort(order_.begin(), order_.end(), [&](int32_t a, int32_t b) {
            const PageList &x = lists_[a], &y = lists_[b];
            const auto m = std::mismatch(x.ids, x.ids + std::min(x.n, y.n), y.ids);
            if (m.first != x.ids + std::min(x.n, y.n)) return *m.first < *m.second;
            return x.n != y.n ? x.n < y.n : a < b;
        });
    }
    PageGroups run() {
        PageGroups g;
        g.shared.assign(lists_.size(), 0);
        if (lists_.size() < 2) return g;
        Node root = build(0, order_.size(), 0, kDepth);
        std::vector<int64_t> above{0};
        best(root, above);
        std::vector<std::vector<int32_t>> open(1);
        std::vector<size_t> c{0};
        collect(root, 0, 1, open, c, {0});
        for (size_t i = 1; i < open.size(); ++i) {
            for (int32_t b : open[i]) {
                g.members.push_back(b);
                g.shared[b] = (int32_t)c[i];
            }
            g.start.push_back((int32_t)g.members.size());
        }
        return g;
    }

  private:
    static constexpr int kDepth = 512;
    struct Node {
        size_t lo, hi, common;
        std::vector<Node> kids;
        std::vector<char> open;  // by the open node above: whether to open this one
    };
    Node build(size_t lo, size_t hi, size_t common, int depth) {
        const PageList &a = lists_[order_[lo]], &b = lists_[order_[hi - 1]];
        // sorted: what the first and the last share, all share; an id below 0 names no page
        while (common < a.n && common < b.n && a.ids[common] == b.ids[common] && a.ids[common] >= 0) ++common;
        Node node{lo, hi, common, {}, {}};
        if (depth == 0) return node;
        for (size_t i = lo; i < hi;) {
            const PageList& p = lists_[order_[i]];
            size_t j = i + 1;
            if (p.n > common && p.ids[common] >= 0)
                while (j < hi && lists_[order_[j]].n > common && lists_[order_[j]].ids[common] == p.ids[common]) ++j;
            if (j - i > 1 && j - i < hi - lo) node.kids.push_back(build(i, j, common, depth - 1));
            i = j;
        }
        return node;
    }
    // What the lists below `node` add to the sum for every open node above (above[k]
    // = its c).
    std::vector<int64_t> best(Node& node, std::vector<int64_t>& above) {
        const int64_t c = (int64_t)node.common;
        int64_t singles = (int64_t)(node.hi - node.lo);
        const size_t n = above.size();
        above.push_back(c);
        std::vector<int64_t> kids(n + 1, 0);
        for (Node& kid : node.kids) {
            singles -= (int64_t)(kid.hi - kid.lo);
            const std::vector<int64_t> v = best(kid, above);
            for (size_t k = 0; k <= n; ++k) kids[k] += v[k];
        }
        above.pop_back();
        std::vector<int64_t> value(n);
        node.open.resize(n);
        const int64_t opened = kids[n] + (singles - 1) * c;
        for (size_t k = 0; k < n; ++k) {
            const int64_t closed = kids[k] + singles * above[k];
            node.open[k] = opened > closed;
            value[k] = std::max(opened, closed);
        }
        return value;
    }
    // The members of every open node; open[at[k]] is the group the k-th node above
    // stands for, open[0] the lists of no group.
    void collect(const Node& node, size_t k, size_t n, std::vector<std::vector<int32_t>>& open, std::vector<size_t>& c,
                 std::vector<size_t> at) {
        at.push_back(at[k]);
        if (node.open[k]) {
            at[n] = open.size();
            open.emplace_back();
            c.push_back(node.common);
        }
        const size_t below = node.open[k] ? n : k;
        size_t i = node.lo;
        for (const Node& kid : node.kids) {
            for (; i < kid.lo; ++i) open[at[below]].push_back(order_[i]);
            collect(kid, below, n + 1, open, c, at);
            i = kid.hi;
        }
        for (; i < node.hi; ++i) open[at[below]].push_back(order_[i]);
    }

    const std::vector<PageList>& lists_;
    std::vector<int32_t> order_;
};

}  // namespace

PageGroups group_pages(const std::vector<PageList>& lists) { return Grouping(lists).run(); }

}  // namespace crane

using namespace crane;

extern "C" int crane_hip_group_prefixes(const int32_t* table, int64_t stride, const int32_t* pages, int B,
                                        int32_t* shared_pages, int32_t* group_start, int32_t* group_seq,
                                        int* n_groups) {
    if (!n_groups || B < 0 || stride < 0) return CRANE_HIP_E_INVALID;
    *n_groups = 0;
    if (!group_start) return CRANE_HIP_E_INVALID;
    group_start[0] = 0;
    if (B == 0) return CRANE_HIP_OK;
    if (!pages || !shared_pages || !group_seq || (stride > 0 && !table)) return CRANE_HIP_E_INVALID;
    try {
        std::vector<PageList> lists((size_t)B);
        for (int b = 0; b < B; ++b) {
            if (pages[b] < 0 || pages[b] > stride) return CRANE_HIP_E_INVALID;
            lists[b] = {table + b * stride, (size_t)pages[b]};
        }
        const PageGroups g = group_pages(lists);
        std::copy(g.shared.begin(), g.shared.end(), shared_pages);
        std::copy(g.start.begin(), g.start.end(), group_start);
        std::copy(g.members.begin(), g.members.end(), group_seq);
        *n_groups = g.count();
    } catch (...) {  // no memory
        return CRANE_HIP_E_INVALID;
    }
    return CRANE_HIP_OK;
}

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
    if (blocks * Hkv > 0xffffffffLL / kThreads) return CRANE_HIP_E_INVALID;  // a grid's threads: 32 bits
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
            hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(blocks * Hkv), (unsigned)ni, (unsigned)np),
                               dim3(kThreads), 0, (hipStream_t)stream, a, (int)blocks, Hkv, run, row_bytes);
            rc = launch_status(hipGetLastError());
            if (rc) return rc;
        }
    }
    return CRANE_HIP_OK;
}
