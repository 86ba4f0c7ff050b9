/*
 * crane_f8.h -- C ABI of the paged KV cache held in 8 bits (gfx950): the fused append
 * that quantises rows as it writes them, attention that reads the codes, and the way
 * back to values.
 *
 * Crane keeps K and V in the model dtype (Attention.kv_cache, qwen3/modeling.rs:173-176)
 * and has no counterpart: these operators stand beside the paged launchers of
 * crane_hip.h (append: qwen3/modeling.rs:382-423, 313-332; attention: :432-502).
 *
 * The cache.  K and V pools [n_pages, Hkv, page_rows, D] of one-byte codes (OCP e4m3,
 * torch.float8_e4m3fn) and, for each, a pool of scales [n_pages, Hkv, page_rows / 32] of
 * one byte (torch.float8_e8m0fnu): byte x stands for 2^(x - 127) and is the scale of 32
 * rows of a head, a block.  A value is its code times its block's scale, which bf16
 * holds exactly.  Scale bytes are 1 to 254 (the append writes 27 and more) and values finite,
 * below 2^128; others give unspecified values.  Rows are addressed as in the paged launchers: row j of sequence b
 * is row j % page_rows of page block_table[b * table_stride + j / page_rows].
 *
 * Conventions are those of crane_hip.h: 0 or a CRANE_HIP_E_* status, arguments checked on
 * the host before anything is enqueued, nothing allocated or synchronised, everything
 * ordered on `stream`.  dtype is that of q, of the rows and of the results
 * (CRANE_HIP_F32 or CRANE_HIP_BF16); device pointers are 16-byte aligned.
 */
#ifndef CRANE_F8_H
#define CRANE_F8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Cache rows that one scale byte covers. */
#define CRANE_F8_BLOCK_ROWS 32

/* The fused per-head QK-RMSNorm + RoPE of crane_hip_qknorm_rope_append_paged (its
 * arguments, but for the pools), k and v quantised into rows [cache_len[b], + S).
 *
 * The arithmetic is f32 throughout: q is rounded once, to dtype, and k and v once, to
 * their codes (crane_hip_qknorm_rope_append_paged rounds after every step, as candle's
 * ops do; the two agree to those roundings).  Of every block that rows land in:
 *   scale   the smallest 2^e >= 2^-100 with |x| <= 448 2^e for every finite x of the new
 *           rows; where the block holds rows of the sequence already, no smaller than
 *           its scale
 *   codes   x 2^-e rounded to nearest even, to 1.875 2^127 where that would be 2^128; a
 *           NaN or an infinity becomes a NaN.  Where the scale grew, the codes of the
 *           block's older rows are rounded to it (exactly, but for those that get
 *           subnormal)
 * A new row of q and k whose position is outside the tables is not written, and has no
 * part in the scale (of a block that begins with such rows alone it is 2^-100).  Nothing
 * else is written: rows behind cache_len[b] + S keep their codes.  A page that rows land in
 * must be in one row of the block table only. */
int crane_hip_qknorm_rope_append_paged_f8(const void* qkv, int64_t qkv_row_stride, const void* q_norm_w,
                                          const void* k_norm_w, float eps, int order, const void* cos,
                                          const void* sin, int64_t cs_stride, int64_t table_rows,
                                          const int32_t* positions, void* q_out, void* k_pool, void* v_pool,
                                          void* k_scale, void* v_scale, int64_t n_pages, int page_rows,
                                          const int32_t* block_table, int64_t table_stride,
                                          const int32_t* cache_len, int B, int S, int Hq, int Hkv, int D, int dtype,
                                          void* stream);

/* Bytes of workspace crane_hip_attn_paged_f8 needs for these sizes; 0 where it needs
 * none, the call would be rejected or has nothing to do. */
size_t crane_hip_attn_paged_f8_workspace(int64_t max_kv, int B, int S, int Hq, int Hkv, int D, int dtype);

/* Attention of the last S tokens of every sequence over its rows of the cache.
 *
 * q        [B, Hq, S, D] (S = 1: a decode step's [B, Hq, D])
 * kv_len   [B] int32, device: rows of every sequence, its S new ones included; query i
 *          sits at row kv_len[b] - S + i.  kv_len[b] <= max_kv (a longer sequence is
 *          taken as one of max_kv rows)
 * flags    CRANE_HIP_PREFILL_CAUSAL: query i sees rows [0, kv_len[b] - S + i]; 0: every
 *          query sees all kv_len[b] rows.  A query that sees none gets zeros.  Rows a
 *          query does not see have no influence on it, whatever they hold.  Rows of a
 *          page id outside [0, n_pages) count as zeros
 * scale    of the scores, positive, its product with log2 e finite
 * workspace device scratch of crane_hip_attn_paged_f8_workspace(...) bytes, 16-byte
 *          aligned, any contents; calls that overlap in time must not share one.  May be
 *          NULL when that is 0
 * out      [B, S, Hq*D]
 *
 * Scores, softmax and sums are f32 (sums of V's values up to 2^90 do not overflow: weights
 * are up to 2^16 before the division); bf16 calls round the probabilities before the
 * product with V, f32 calls split q and the probabilities into three bf16 parts, which
 * hold all of their bits.  The order of the sums follows the sizes: two runs of one call
 * give the same bits. */
int crane_hip_attn_paged_f8(const void* q, const void* k_pool, const void* v_pool, const void* k_scale,
                            const void* v_scale, int64_t n_pages, int page_rows, const int32_t* block_table,
                            int64_t table_stride, const int32_t* kv_len, int64_t max_kv, int B, int S, int Hq, int Hkv,
                            int D, float scale, int flags, void* workspace, size_t ws_bytes, void* out, int dtype,
                            void* stream);

/* Rows [0, kv_len[b]) of every sequence as values: k_out, v_out [B, Hkv, max_kv, D] in
 * dtype, zeros from kv_len[b] on and for rows of a page id outside [0, n_pages). */
int crane_hip_read_paged_f8(const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                            int64_t n_pages, int page_rows, const int32_t* block_table, int64_t table_stride,
                            const int32_t* kv_len, int64_t max_kv, int B, int Hkv, int D, void* k_out, void* v_out,
                            int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CRANE_F8_H */
