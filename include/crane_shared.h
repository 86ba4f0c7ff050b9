/*
 * crane_shared.h -- C ABI of the operators for sequences that share pages of a
 * paged KV cache (gfx950): attention in which the rows a group of sequences has
 * in common are read and multiplied once for the whole group, and copies of rows
 * between pages of a pool (a forked sequence's partial page, a compaction).
 *
 * Crane has no counterpart: every sequence holds its own K/V rows
 * (Attention.kv_cache, qwen3/modeling.rs:173-176), so n requests behind one
 * system prompt hold and read its rows n times.  crane_pkv.h has the manager
 * that shares pages and calls these launchers.  Conventions are those of
 * crane_hip.h: 0 or a CRANE_HIP_E_* status, arguments checked on the host before
 * anything is enqueued, nothing allocated or synchronised, everything ordered on
 * `stream`.
 */
#ifndef CRANE_SHARED_H
#define CRANE_SHARED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace crane_hip_attn_shared_paged needs for these sizes (the
 * arguments of the call); 0 where the call would be rejected or has nothing to
 * do. */
size_t crane_hip_attn_shared_workspace(const int32_t* groups_host, int n_groups, int64_t max_kv, int64_t max_own,
                                       int64_t mean_own, int B, int S, int Hq, int Hkv, int D, int dtype);

/* Attention of the last S rows of every sequence over its rows of the pools, the
 * rows shared by a group read once for the group.
 *
 * q        [B, Hq, S, D] (S = 1: a decode step's [B, Hq, D]); fewer than 2^26 rows
 * k_pool, v_pool, n_pages, page_rows, block_table, table_stride: as in
 *          crane_hip_attn_decode_paged; a page id outside [0, n_pages) reads as
 *          zero rows
 * kv_len   [B] int32, device: rows of every sequence, its S new ones included;
 *          query i sits at row kv_len[b] - S + i.  kv_len[b] <= max_kv
 * shared_rows [B] int32, device: sequence b shares its first shared_rows[b] rows
 *          (0: none) with every member of its group; any number, not only whole
 *          pages.  NULL when n_groups is 0
 * groups   [n_groups, 4] int32, device, 16-byte aligned: {s, n, b, r}: the group's
 *          members are the batch rows members[s .. s + n), it shares r rows, and they
 *          are read through row b of the block table (a member's).  A sequence with
 *          shared rows is in exactly one group, whose r is its shared_rows; other
 *          sequences are in none.  A description that breaks this gives unspecified
 *          results for the sequences concerned and stays in bounds
 * members  int32, device, B entries at most: as many as groups_host accounts for (the
 *          largest s + n of its groups); no entry past those is read
 * groups_host the same n_groups descriptions on the HOST, read before the call
 *          returns: they steer how the work is cut and bound what the device's may
 *          say (CRANE_HIP_E_INVALID for members or rows outside the batch)
 * max_own  host-side bound of kv_len[b] - shared_rows[b]; rows past it need not be
 *          attended.  max_own + a group's rows < 2^31 - 2^14
 * mean_own about what kv_len[b] - shared_rows[b] is on average: it steers how the
 *          work is cut, and whether the groups are used at all (their members' own
 *          table rows name the same rows), nothing else (negative counts as 0)
 * flags    CRANE_HIP_PREFILL_CAUSAL: query i sees rows [0, kv_len[b] - S + i];
 *          0: every query sees all kv_len[b] rows.  A query that sees none gets
 *          zeros.  Rows a query does not see have no influence on it, whatever
 *          they hold
 * workspace device scratch of at least crane_hip_attn_shared_workspace(...) bytes,
 *          16-byte aligned, any contents; calls that overlap in time must not
 *          share one.  May be NULL when that is 0
 * out      [B, S, Hq*D]
 *
 * CRANE_HIP_E_INVALID also where no cut of the work, into at least 128 and at most 8192
 * keys a workgroup, fits a grid of fewer than 2^24 workgroups (about 16 to 128 query rows
 * of a kv head each, every sequence counted with max_own keys).
 *
 * The scores, their softmax and all sums are f32 and only the probabilities (bf16
 * calls) are rounded before the product with V: candle's rounding of every score
 * to the model dtype, which crane_hip_attn_decode reproduces, is not part of this
 * call, so the two agree to that rounding and not bit for bit.  The order of the
 * sums follows the host-side bounds and the group sizes; two runs of one call
 * give the same bits. */
int crane_hip_attn_shared_paged(const void* q, const void* k_pool, const void* v_pool, int64_t n_pages, int page_rows,
                                const int32_t* block_table, int64_t table_stride, const int32_t* kv_len, int64_t max_kv,
                                const int32_t* shared_rows, const int32_t* groups, const int32_t* members,
                                const int32_t* groups_host, int n_groups, int64_t max_own, int64_t mean_own, int B,
                                int S, int Hq, int Hkv, int D, float scale, int flags, void* workspace,
                                size_t ws_bytes, void* out, int dtype, void* stream);

/* The groups of a batch whose sequences name the same first pages (host only, no
 * side effects): row b of `table` (HOST, `stride` ids a row) lists pages[b] page ids.
 * Writes shared_pages [B] (pages sequence b shares with its group; 0: in none),
 * group_start [B + 1] and group_seq [B] (as far as *n_groups groups need them).
 * Where sequences share more with some than with others, the grouping that reads
 * the fewest pages is taken (of those whose lists branch up to 512 times on the way
 * to a group's last shared page).  Ids below 0 are shared by none.  shared_pages times the
 * page's rows are crane_hip_attn_shared_paged's shared_rows where every shared page is
 * full of rows. */
int crane_hip_group_prefixes(const int32_t* table, int64_t stride, const int32_t* pages, int B, int32_t* shared_pages,
                             int32_t* group_start, int32_t* group_seq, int* n_groups);

/* Copy rows [0, rows[i]) of page src[i] to page dst[i] (all heads), i < n, in
 * every one of n_pools pools [n_pages, Hkv, page_rows, D] (the K and V pools of
 * one or of all layers).
 *
 * pools, src, dst, rows: HOST arrays, read before the call returns; rows may be
 *          NULL (whole pages).  pools[i] is device memory, 16-byte aligned, each
 *          a pool of its own
 * A page may be the source of several copies; a destination is named once and is
 * no copy's source (CRANE_HIP_E_INVALID otherwise).  Rows of dst[i] past rows[i]
 * keep what they hold. */
int crane_hip_copy_pages(void* const* pools, int n_pools, int64_t n_pages, int page_rows, int Hkv, int D,
                         const int32_t* src, const int32_t* dst, const int32_t* rows, int n, int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CRANE_SHARED_H */
