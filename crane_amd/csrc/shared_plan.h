// shared_plan.h -- how a call of the attention over shared pages (shared.hip) is cut
// into workgroups: the forms and chunk sizes of both roles and the order of their
// items.  Nothing but arithmetic on sizes, so that it also compiles for the host alone.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace crane {
namespace {

constexpr int kAlign = 64;         // chunk bounds are multiples of it (whole steps of every form)
constexpr int kWaves = 4;
constexpr int kMaxChunk = 8192;    // rows per chunk: its pages' ids fit one lane each
constexpr int kMinChunk = 128;
constexpr int kCus = 256;
constexpr int64_t kMostThreads = 0xffffffffLL;  // of a grid
constexpr int kBlockRows = 128;    // query rows of a workgroup's block form

// A role's item x of `units` (segment, kv head, chunk) units with `blocks` row blocks
// each: ids that are equal mod 8 run on one XCD, which so gets the blocks of a unit,
// one after the other, and reads their keys through its own L2.  A segment's chunks are
// segs Hkv units apart: on 8 / gcd(8, segs Hkv) XCDs for each kv head, up to all 8.  Where
// that is a multiple of 8 they would stay on the XCDs of the heads, and the segments take
// turns (8 sequences at 2 kv heads, one of 30720 keys, the others of 7: 37 us for 19);
// with heads in eights every segment is on all XCDs anyway.  Where it is a multiple of 2 or
// 4 only, they do not: 2 sequences at 2 kv heads are on 4 XCDs each, 4 at one head on 2.
struct Item {
    int block, kvh, seg, chunk;
    bool ok;
    __host__ __device__ __forceinline__ Item(int x, int blocks, int Hkv, int segs, int chunks) {
        const int c = x / (8 * blocks), rem = x - c * 8 * blocks;
        block = rem >> 3;
        int unit = 8 * c + (rem & 7);
        ok = unit < segs * Hkv * chunks;
        kvh = unit % Hkv;
        unit /= Hkv;
        chunk = unit / segs;
        seg = unit - chunk * segs;
        if (Hkv % 8 != 0 && segs * Hkv % 8 == 0) seg = (seg + chunk) % segs;
    }
};

// A group's members as the device describes them, in the array whose entries the host's
// groups account for: never past those.  (More of them than the host's largest group are
// past the row blocks that are launched.)
struct Members {
    int first, n;
    __host__ __device__ __forceinline__ Members(int first_place, int count, int entries) {
        first = std::min(std::max(first_place, 0), entries);
        n = std::min(std::max(count, 0), entries - first);
    }
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a call is cut: whether sharing is used, and the forms (query rows per workgroup),
// row blocks and key chunks of both roles.
struct Plan {
    bool share;
    int max_group, max_shared;
    int members;  // entries of the members array the groups account for
    int shared_rows, own_rows;
    int64_t shared_tiles, own_tiles;
    int chunk;
    int64_t shared_splits, own_splits, shared_items, own_items;
    bool spread;  // one workgroup per CU
    bool fits;    // a grid; else no cut's workgroups do, and nothing but the groups' bounds is set
    size_t ml_off, total;  // of the workspace
};

// The sizes a plan is made for; groups (HOST): {first member's place, members, block
// table row, shared rows}.
struct Sizes {
    const int32_t* groups;
    int n_groups;
    int64_t max_kv, max_own, mean_own;
    int B, S, Hq, Hkv;
    bool bf16;
    int64_t R() const { return (int64_t)S * (Hq / Hkv); }  // query rows per (sequence, kv head)
    // the own role's most keys
    int64_t longest(const Plan& p) const { return p.share ? max_own : std::min(max_kv, max_own + p.max_shared); }
    int64_t rows() const { return (int64_t)B * Hq * S; }
    bool same(const Sizes& o) const {  // but for the groups' contents
        return n_groups == o.n_groups && max_kv == o.max_kv && max_own == o.max_own && mean_own == o.mean_own &&
               B == o.B && S == o.S && Hq == o.Hq && Hkv == o.Hkv && bf16 == o.bf16;
    }
};

// Microseconds for 128 keys of a workgroup that has a CU to itself, and of a CU kept busy
// by two, by the workgroup's query rows (f32: bound by v_mfma_f32_16x16x4_f32 either way;
// bf16 blocks: by their MFMAs and exponentials).
struct KeyCost {
    double alone, busy;
};
inline KeyCost key_cost(bool bf16, int rows) {
    if (!bf16) return rows == 16 ? KeyCost{2.2, 2.1} : KeyCost{3.7, 3.5};
    return rows == 16 ? KeyCost{1.1, 0.8} : rows == 32 ? KeyCost{1.0, 1.0} : KeyCost{2.2, 1.8};
}

// Up to 96 rows the 32-row form, whose waves each take keys of their own, is the faster
// (5 groups of 35 to 70 rows: 45 us in blocks of 128, 30 in 32s; 128 rows: 37 in either);
// a block reads its keys once for more rows.
inline int form_rows(int64_t rows, bool bf16) { return rows <= 16 ? 16 : !bf16 || rows <= 96 ? 32 : kBlockRows; }

// What a plan costs in microseconds: the CUs' work (all of it spread evenly, or a role's
// workgroups in turns of 256), the longest workgroup's, K and V from HBM at 5.5 TB/s and
// what is read again at 10, whichever is most (as a norm of high order, since near each
// other they add up); with more workgroups than CUs a part of the longest one as a tail;
// each workgroup's start and end, also of those that find nothing to do; the shared
// role's longer start; and what several chunks cost, the second kernel and the partial
// rows written and read (1 KiB each).
// The constants are a fit to 165 calls of random sizes, 28 cuts each, with the blocks' and
// the partial rows' costs held at what they measure: the cut it chooses takes 7% more than
// the best of the 28 on average, and 10% over 48 calls that took no part in the fit.
inline double plan_cost(const Sizes& z, Plan& p) {
    const KeyCost sc = key_cost(z.bf16, p.shared_rows), oc = key_cost(z.bf16, p.own_rows);
    double work, items = 0, once = 0, loads = 0, mean = std::max<double>(64, z.mean_own);
    double longest = std::min<double>(z.longest(p), p.chunk) * oc.alone / 128;
    auto rounds = [](double n) { return std::ceil(n / kCus); };
    const double per_chunk = 1.0 / p.chunk, per_block = 1.0 / p.shared_rows, R = z.R(), per_batch = 1.0 / z.B;
    for (int g = 0; g < z.n_groups; ++g) {
        const double members = z.groups[4 * g + 1], rows = z.groups[4 * g + 3];
        once += z.Hkv * rows;
        if (!p.share) {
            mean += members * rows * per_batch;
            continue;
        }
        const double tiles = z.Hkv * std::ceil(members * R * per_block);
        loads += tiles * rows;
        items += tiles * std::ceil(rows * per_chunk);
    }
    work = loads * sc.busy / 128;
    double even = 0;  // each role's workgroups in turns of 256 at their chunk's cost
    if (p.share) {
        const double keys = std::min(p.max_shared, p.chunk) / 128.0;
        longest = std::max(longest, keys * sc.alone);
        even = rounds(items) * keys * sc.busy;
    }
    const double own = (double)z.B * z.Hkv * p.own_tiles;
    once += (double)z.B * z.Hkv * z.mean_own;
    work += own * mean * oc.busy / 128;
    loads += own * mean;
    const double own_items = own * std::max(1.0, mean / p.chunk);
    items += own_items;
    even = std::max(even, rounds(own_items) * std::min<double>(mean, p.chunk) / 128 * oc.busy);
    work = std::max(work / kCus, even);
    p.spread = items <= 240 || p.shared_items + p.own_items <= kCus;
    const double memory = (once / 5.5e6 + std::max(0.0, loads - once) / 10e6) * (z.bf16 ? 512 : 1024);
    auto pow4 = [](double x) { return x * x * x * x; };
    double t = std::sqrt(std::sqrt(pow4(longest) + pow4(memory) + (items <= kCus ? 0 : pow4(work))));
    t += (items <= kCus ? 0 : 0.08 * longest) + 0.85 * p.share;
    t += 0.002 * items + 0.0032 * (p.shared_items + p.own_items);
    const double slots = p.shared_splits + p.own_splits;
    if (slots > 1) t += 1.1 + (slots > 32) * 1.0 + 2e-4 * z.rows() * slots;
    return t;
}

// Cuts the roles' keys into chunks; own chunk 0 starts on a multiple of kAlign, and is
// there without keys, too: its workgroups write the zeros of rows that see none.
inline void cut(const Sizes& z, int chunk, Plan* p) {
    p->chunk = chunk;
    p->shared_splits = p->share ? ceil_div(p->max_shared, chunk) : 0;
    p->own_splits = std::max<int64_t>(1, ceil_div(z.longest(*p) + (p->share ? kAlign : 0), chunk));
    p->shared_items = 8 * p->shared_tiles * ceil_div(z.n_groups * z.Hkv * p->shared_splits, 8);
    p->own_items = 8 * p->own_tiles * ceil_div((int64_t)z.B * z.Hkv * p->own_splits, 8);
}

// Chunk sizes tried, in units of 128 keys.
constexpr int kChunks[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 32, 48, 64};

inline Plan plan_for(const Sizes& z) {
    Plan p{}, best;
    for (int g = 0; g < z.n_groups; ++g) {
        p.max_group = std::max(p.max_group, (int)z.groups[4 * g + 1]);
        p.max_shared = std::max(p.max_shared, (int)z.groups[4 * g + 3]);
        p.members = std::max(p.members, (int)(z.groups[4 * g] + z.groups[4 * g + 1]));
    }
    best = p;
    const int64_t M = p.max_group * z.R();
    p.own_rows = form_rows(z.R(), z.bf16);
    p.own_tiles = ceil_div(z.R(), p.own_rows);
    double least = INFINITY;
    // Without sharing (a few short sequences do with one kernel, and one that fills whole
    // row blocks by itself may gain nothing) and with it.
    for (int share = 0; share < (M > 0 && p.max_shared > 0 ? 2 : 1); ++share) {
        p.share = share;
        p.shared_rows = share ? form_rows(M, z.bf16) : p.own_rows;
        p.shared_tiles = share ? ceil_div(M, p.shared_rows) : 0;
        for (int k : kChunks) {
            cut(z, kMinChunk * k, &p);
            p.fits = p.shared_items + p.own_items <= kMostThreads / (64 * kWaves);
            if (!p.fits) continue;
            const double t = plan_cost(z, p);
            if (!(t >= least)) {
                least = t;
                best = p;
            }
        }
    }
    return best;
}

}  // namespace
}  // namespace crane
