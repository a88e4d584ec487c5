/*
 * C ABI of the operators around a paged latent cache (MLA decode), for sm_100a: a new row written into its page, the
 * attention of one new token per sequence, and eviction by accumulated attention weight. They live in the same library as
 * the FP8 GEMM (libb200fp8mm.so), whose B200_FP8_MM_* return codes they use (0 = launched).
 *
 * The cache holds one row of dv + dr elements per token, shared by all query heads: the whole row is the key, its first dv
 * elements are the value, its last dr elements carry the rotary position. Slot j of sequence b is row
 * (block_table[b][j / page_size], j % page_size). Types: bf16 or fp16, the same for cache, rows, queries and outputs.
 *
 * Plain pointers and sizes; nothing is allocated; asynchronous on `stream`. Strides count elements. All indices that come
 * from device memory are checked there: a length below 0 counts as 0, one above the block table's capacity (pages_per_seq *
 * page_size) as the capacity; a page outside [0, pages) reads as rows of zeros and is never written.
 */
#ifndef B200_MLA_CACHE_H_
#define B200_MLA_CACHE_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { B200_MLA_CACHE_BF16 = 0, B200_MLA_CACHE_FP16 = 1 };

typedef struct {
  void* data;              /* 16-byte aligned                                                       */
  const int* block_table;  /* [batch][pages_per_seq], row pitch table_stride                        */
  const int* lens;         /* [batch]: rows each sequence holds                                     */
  int dtype;               /* B200_MLA_CACHE_*                                                      */
  int pages, page_size;
  int dv, dr;              /* dv: 128, 256, 384 or 512; dr: a multiple of 64; dv + dr at most 576   */
  int batch, pages_per_seq;
  long long page_stride, slot_stride;  /* multiples of 8, at least dv + dr                          */
  long long table_stride;
} b200_mla_cache;

/*
 * For every sequence: `row` [batch][dv + dr] goes to slot lens[b], its last dr elements rotated for position[b]; then
 * score[b][lens[b]] = 0 and slot_position[b][lens[b]] = position[b] (each may be NULL). A sequence whose lens[b] is negative
 * or at the capacity is left alone. If `q` is not NULL, the last dr elements of every q[b][h] ([batch][heads][dv + dr]) are
 * rotated for the same position into q_out (which may be q), the others copied.
 *   t < dr/2, a = position * theta^(-2t/dr):  y[t] = x[t] cos a - x[t+dr/2] sin a,  y[t+dr/2] = x[t+dr/2] cos a + x[t] sin a
 * in fp32 with the angle reduced in fp64, rounded once. lens is not changed. No two sequences may name the same page for their new
 * slots.
 */
int b200_mla_cache_append(const b200_mla_cache* cache, const void* row, long long row_stride, const int* position,
                          double theta, const void* q, long long q_sb, long long q_sh, void* q_out, long long qo_sb,
                          long long qo_sh, int heads, float* score, long long score_stride, int* slot_position,
                          long long slot_position_stride, void* stream);

/*
 * out[b][h] = sum_j p_j x_j[0..dv),  p = softmax_j(scale * q[b][h] . x_j),  j < lens[b];  lse[b][h] = log sum_j exp(.) (may be
 * NULL). A sequence without rows gets zeros and -inf, as does a head whose logits are all -inf. With score_out (else NULL):
 * score_out[b][j] = score[b][j] + sum_h p_j for j < lens[b]; slots behind are left as they were; score_out may be score. max_len:
 * lengths above it count as max_len (0: the capacity). q, out: [batch][heads][dv + dr] and [.. dv], last dimension contiguous; q
 * 16-byte aligned with strides that are multiples of 8. |scale| < 2^127. lse: contiguous. Sums, maxima and the joins of the splits are
 * fp32; the weights are rounded to the cache's type for the second product. Results do not depend on timing.
 * device_status: int[4] as for b200_fp8_mm (may be NULL).
 */
int b200_mla_cache_attend(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads, float scale,
                          void* out, long long out_sb, long long out_sh, float* lse, const float* score,
                          long long score_stride, float* score_out, long long score_out_stride, int max_len, void* workspace,
                          size_t workspace_bytes, int* device_status, void* stream);

/*
 * Self-test of the bounded waits (diagnostics): b200_mla_cache_attend with every wait inside the kernel limited to wait_limit_ns (1 ms ..
 * 100 ms), and with tile `skip_tile` of the first sequence left uncopied (a tile is 48 rows with up to 32 heads, else 64), so the waits
 * that depend on it run out. The kernel returns by itself; device_status (required) then reads
 * {B200_FP8_MM_DEV_WAIT_EXPIRED, wait, block, phase}, out is not valid, and the context stays usable. bf16 caches only. Workspace as without scores.
 */
int b200_mla_cache_attend_selftest_wait_expiry(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads,
                                               float scale, void* out, long long out_sb, long long out_sh, void* workspace,
                                               size_t workspace_bytes, unsigned long long wait_limit_ns, int skip_tile,
                                               int* device_status, void* stream);

/* Bytes that b200_mla_cache_attend needs (256-byte aligned, no particular contents). */
size_t b200_mla_cache_attend_workspace_bytes(int batch, int heads, int dv, int dr, int max_len, int with_score);

/*
 * Sequences with more than `budget` rows keep `budget` of them: those whose slot_position is above the sequence's largest
 * minus `recent`, then those of the largest score, the lower slot first among equals (NaN counts as the largest). A kept row
 * in a slot at or behind the budget moves to a slot before it that is given up, both in ascending order; its score and
 * position go along into score_out and position_out (slots below the new length are written; each may be its input), the
 * row in place inside the cache. lens_out[b] = min(lens[b], budget), and may be lens. Pages must not be shared with another
 * sequence below `budget`.
 */
int b200_mla_cache_evict(const b200_mla_cache* cache, const float* score, long long score_stride, const int* slot_position,
                         long long slot_position_stride, int budget, int recent, int* lens_out, float* score_out,
                         long long score_out_stride, int* position_out, long long position_out_stride, void* workspace,
                         size_t workspace_bytes, void* stream);

/* Bytes that b200_mla_cache_evict needs. */
size_t b200_mla_cache_evict_workspace_bytes(int batch, int capacity, int budget);

#ifdef __cplusplus
}
#endif
#endif /* B200_MLA_CACHE_H_ */
