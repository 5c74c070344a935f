/*
 * dejavu_b200_serving.h — C ABI of the kernels that serve requests of different lengths: a paged key/value cache, attention
 * over its pages and over packed prompts, sampling (libdejavu_b200_serving.so).
 *
 * Same conventions as dejavu_b200.h: raw device pointers, sizes, a CUDA stream as void*; work is only enqueued, never
 * allocated; DJV_OK or a negative DJV_ERR_* with a message in djv_last_error() (each library has its own). `dtype` is the
 * element type T of activations and caches: DJV_DTYPE_F16, DJV_DTYPE_BF16 or DJV_DTYPE_F32. Scores, softmax, sums and angles
 * are held in 32 bits or more.
 *
 * A paged cache is two pools of `pages` pages, K and V, of `page` tokens each: element (p, g, s, d) of a pool, page p, key/value
 * head g, token s of the page, dimension d, is at p * ld_page + g * ld_head + s * ld_slot + d (elements; the strides and the
 * pools' addresses are multiples of 16 bytes, so is a row of D elements). table (B, width) int32, rows ld_table apart: entry
 * (b, i) is the page of tokens i * page .. (i + 1) * page - 1 of sequence b. Entries behind a sequence's last token are not
 * read. Entries outside 0 .. pages - 1 that a kernel meets are counted (djv_paged_faults), their tokens are not stored and not
 * seen, and so it is with tokens behind the table's last column. Sequences may share pages that nobody writes to. Two rows of a
 * call that store into one slot of one page leave it with one or the other, or a mixture.
 *
 * pos points to B int64 on the device, so that a captured CUDA graph of a step stays valid.
 */
#ifndef DEJAVU_B200_SERVING_H
#define DEJAVU_B200_SERVING_H

#include "dejavu_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* New tokens enter a paged cache, rotated on the way. Rows cu[b] .. cu[b + 1] - 1 (cu: B + 1 int32, ascending) of q, k and v are the
 * tokens of sequence b from position pos[b] on; cu = NULL: one row per sequence, T = B. q (T, H, D), k and v (T, G, D): rows ldq,
 * ldk, ldv elements apart, heads hq, hk, hv apart, dimensions adjacent. Of every head of q and k the first 2 * half dimensions
 * are rotated in pairs, (i, i + half), or (2i, 2i + 1) if interleaved: angle = position * freqs[i], a product in 64 bits, cos and sin
 * times amp; half = 0: no rotation. q_out (T, H, D) and k_out (T, G, D) receive the rotated rows (NULL: not wanted; q_out = NULL: q is
 * not read). A row of no sequence, or at a position below 0, is not stored; its outputs are zeros. */
int djv_paged_append(int dtype, void *q_out, void *k_out, const void *q, long long ldq, long long hq, const void *k,
                     long long ldk, long long hk, const void *v, long long ldv, long long hv, void *k_pages, void *v_pages,
                     long long ld_page, long long ld_head, long long ld_slot, int pages, int page, const int32_t *table,
                     long long ld_table, int width, const long long *pos, const int32_t *cu, const float *freqs, float amp,
                     int half, int interleaved, int B, int T, int H, int G, int D, void *stream);

/* Attention of one new token per sequence over its cached tokens: out[b, h] = softmax(scale * q[b, h] . K) V over the tokens at
 * positions 0 .. pos[b] of sequence b, its own among them (appended before). pos[b] = -1, or no token that the table has a page
 * for: zeros. q (B, H, D), rows ldq and heads hq elements apart, and out (B, H, D), contiguous, start on multiples of 16 bytes, as
 * ldq and hq do; H % G == 0, D <= 256. Sums of splits of a long cache are joined in a fixed order: results repeat bit by bit.
 * scratch: djv_paged_attention_scratch_bytes bytes, 16-byte aligned, whose content does not matter; calls that may overlap on the
 * device have one each. */
size_t djv_paged_attention_scratch_bytes(int dtype, int B, int H, int G, int D, int page, int width);
int djv_paged_attention(int dtype, void *out, const void *q, long long ldq, long long hq, const void *k_pages, const void *v_pages,
                        long long ld_page, long long ld_head, long long ld_slot, int pages, int page, const int32_t *table,
                        long long ld_table, int width, const long long *pos, int B, int H, int G, int D, float scale, void *scratch,
                        size_t scratch_bytes, void *stream);

/* Table entries and positions that were refused since load (synchronises). */
unsigned djv_paged_faults(void);

/* Waits of the library's kernels on their own copies and products that ran out since load (0 in a healthy process; synchronises). */
unsigned djv_serving_timeouts(void);

/* Causal attention over whole prompts, packed: rows cu[b] .. cu[b + 1] - 1 (cu: B + 1 int32, ascending, within 0 .. T) of q (T, H, D), k
 * and v (T, G, D) are sequence b; row i sees rows j <= i of its sequence, whatever the others hold. Rows ldq, ldk, ldv elements
 * apart, heads hq, hk, hv apart, dimensions adjacent. H % G == 0, D <= 256. out (T, H, D), contiguous. Rows of no sequence:
 * zeros, or with keep_rest left as they are. The tensor cores take fp16 and bf16 where D, strides and addresses, out's among them, are
 * multiples of 16 bytes; all else goes to the CUDA cores, some 20 to 30 times slower. */
int djv_packed_attention(int dtype, void *out, const void *q, long long ldq, long long hq, const void *k, long long ldk, long long hk,
                         const void *v, long long ldv, long long hv, const int32_t *cu, int B, int T, int H, int G, int D, float scale,
                         int keep_rest, void *stream);
/* One token per row of logits (B, V), rows ld elements apart, from a given number u[b] in [0, 1) (fp32). Of the entries that are neither
 * -inf nor NaN, ordered by (logit descending, index ascending), with w_i = exp((x_i - max) / temperature), are kept
 *   the first top_k (0: all); of those the ones in front of which less than top_p of their sum lies, the first always (1 or more:
 *   all); of those the ones with w >= min_p.
 * token[b] (int64) is the lowest index at which the running sum of kept w, in index order, exceeds u[b] times their sum. A temperature
 * not above 0 takes the largest entry, equal ones the lowest index. A row without entries gets -1. Sums are as exact as 64 bits make them
 * wherever 32 could choose another token; entries more than 45 temperatures below the largest only count where they could (u below 1e-10).
 * Each setting is an array of B values on the device (float, int32, float, float) or, where that is NULL, the number beside it: of the
 * three real ones the bits of a double. */
int djv_sample(int dtype, long long *token, const void *logits, long long ld, const float *u, const float *temperature,
               long long temperature_bits, const int32_t *top_k, int top_k_all, const float *top_p, long long top_p_bits,
               const float *min_p, long long min_p_bits, int B, int V, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* DEJAVU_B200_SERVING_H */
