/* jq_kv_cache.h - what lies between the fused QKV linear and the o-projection of a decoder layer: rotary
 * positions, a paged key-value cache, attention of new tokens over it and eviction from it.
 *
 * A layer of a decode step, with the calls of jq_b200.h around these:
 *   jq_rms_norm_q8_1_device -> jq_mul_mat_q4_0_q8_1_device (q | k | v, fp32) -> jq_rope_kv_append_device
 *   -> jq_paged_attention_q8_1_device -> jq_mul_mat_q4_0_q8_1_device (o) -> ...
 * and, now and then, jq_kv_evict_device.
 *
 * The reference keeps fp32 keys and values of one sequence in one contiguous buffer per layer, casts all of it to fp16 for
 * every step and attends with a kernel per head group (src/cuda/kv_cache.cu:10,53, src/cuda/rope_neox_global_cache.cu:12,
 * src/cuda/fa/fa_double_buffer_kernel.cuh:103); it has one layout of rotary pairs, no pages, no batch and no eviction.
 *
 * As in jq_b200.h "device" entry points are asynchronous on the stream, allocate nothing, never synchronise and return a
 * jq_status with a message in jq_last_error().  Activations are fp32.  Everything they read may have been written by earlier
 * work on the stream.
 */
#ifndef JQ_KV_CACHE_H_
#define JQ_KV_CACHE_H_

#include <stddef.h>
#include <stdint.h>

#include "jq_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of a cache. */
typedef enum jq_kv_type {
    JQ_KV_F16 = 0,
    JQ_KV_BF16 = 1,
    JQ_KV_E4M3 = 2 /* 8-bit floating point, 4 exponent and 3 mantissa bits, no infinities */
} jq_kv_type;

/* The cache of one layer: a pool of pages that all sequences share, and a table that says which pages a sequence has.  Token
 * `i` of sequence `b` (counted within the cache: with eviction that is not its position in the text) lies in slot
 * i % page_size of page d_page_table[b * table_stride + i / page_size]; its `head_dim` elements of head `h` start at element
 * page * stride_page + slot * stride_slot + h * stride_head of d_k and of d_v, and are contiguous.  Any order of the three
 * strides will do.  A page belongs to one sequence (sequences that share the pages of a common start may read them).
 *
 * A page number outside [0, num_pages) is never followed: tokens there are neither written nor attended to, and
 * jq_device_fault() reports 4 if a kernel needed one.  Entries behind a sequence's last page are not looked at. */
typedef struct jq_kv_cache {
    void *d_k;                /* 16-byte aligned, as are all rows: strides in bytes are multiples of 16 */
    void *d_v;
    int type;                 /* jq_kv_type */
    int64_t num_pages;
    int64_t page_size;        /* tokens per page, any number */
    int64_t num_kv_heads;
    int64_t head_dim;         /* a multiple of 16, at most 256 */
    int64_t stride_page;      /* in elements, the same for keys and values */
    int64_t stride_slot;
    int64_t stride_head;
    float k_scale, v_scale;   /* a stored element stands for itself times this; 1 for plain 16-bit caches */
    const int32_t *d_page_table;
    int64_t num_seqs;         /* rows of the table */
    int64_t max_pages;        /* entries of a row */
    int64_t table_stride;     /* distance of two rows, in entries */
} jq_kv_cache;

/* ---- rotary positions ------------------------------------------------------------------------------ */

/* How the angles are stretched for contexts that are longer than the model was trained on. */
typedef enum jq_rope_scaling {
    JQ_ROPE_NONE = 0,
    JQ_ROPE_LINEAR = 1,     /* all angles divided by `factor` */
    JQ_ROPE_NTK = 2,        /* base * factor^(rotary_dim / (rotary_dim - 2)) in place of base */
    JQ_ROPE_YARN = 3,       /* pairs that turn less than once within original_length are divided by `factor`, those that turn 32
                               times and more are not, with a ramp over the pairs between; sine and cosine times 0.1 ln(factor) + 1 */
    JQ_ROPE_WAVELENGTH = 4  /* pairs with wavelengths over original_length are divided by `factor`, those under a quarter of it are
                               not, in between a blend that is linear in original_length / wavelength */
} jq_rope_scaling;

/* Host function.  Fills table_out with rotary_dim / 2 entries, one per pair: the turns per position as a 64-bit binary fraction,
 * rounded (pair i turns by base^(-2i / rotary_dim) radians per position before scaling).  A position times an entry, modulo 2^64,
 * is the exact fraction of a turn, so angles are as exact at position 2^31 as at position 1.  Copy the table to the device once.
 * *mscale_out receives the factor of sine and cosine (1 but for JQ_ROPE_YARN). */
int jq_rope_table(int64_t rotary_dim, double base, int scaling, double factor, int64_t original_length, uint64_t *table_out,
                  float *mscale_out);
/* The same from a model's own list of radians per position, finite numbers of any size and sign. */
int jq_rope_table_from(const double *radians, int64_t n_pairs, uint64_t *table_out);

/* Rotates the first rotary_dim elements (even, at most head_dim) of every head of every row by the row's position and copies the
 * others: x = d_x[row * x_stride_row + head * x_stride_head ...], out likewise.  A pair (a, b) becomes
 * (a cos - b sin, b cos + a sin) * mscale.  Pairs are elements i and i + rotary_dim / 2 (interleaved = 0) or 2i and 2i + 1
 * (interleaved = 1).  d_out may be d_x with the same strides, else the two must not overlap.  head_dim is even, at most 1024; rows and
 * heads may begin at any float (with 16-byte aligned ones it is faster).  The reference's rope_neox is interleaved = 0 with the whole head (src/cuda/rope_neox.cu:14). */
int jq_rope_device(void *stream, const float *d_x, float *d_out, const int32_t *d_positions, const uint64_t *d_table,
                   int64_t num_rows, int64_t num_heads, int64_t head_dim, int64_t rotary_dim, int64_t x_stride_row,
                   int64_t x_stride_head, int64_t out_stride_row, int64_t out_stride_head, int interleaved, float mscale);

/* The fused projection's output, row by row (d_qkv + row * qkv_stride: num_q_heads, then num_kv_heads of keys, then as many of values,
 * head_dim floats each): queries are rotated into d_q (row * q_stride_row + head * q_stride_head; may lie on the queries' own place),
 * keys are rotated and values copied into the cache, where row `r` becomes token d_index[r] of sequence d_seqs[r] (d_seqs NULL: of
 * sequence r).  Rows of a negative or too large sequence or index are padding: their queries are rotated, the cache is not touched.
 * No two rows may name the same token.  Values are divided by the cache's scale and rounded to nearest; what is beyond the type's
 * largest finite value becomes that value, NaN stays NaN.  d_qkv is 4-byte aligned at least; with 16-byte aligned rows it is faster. */
int jq_rope_kv_append_device(void *stream, const float *d_qkv, int64_t qkv_stride, float *d_q, int64_t q_stride_row,
                             int64_t q_stride_head, const int32_t *d_positions, const int32_t *d_index, const int32_t *d_seqs,
                             const uint64_t *d_table, int64_t rotary_dim, int64_t num_rows, int64_t num_q_heads,
                             const jq_kv_cache *cache, int interleaved, float mscale);

/* ---- attention ---------------------------------------------------------------------------------------- */

/* Bytes of workspace for jq_paged_attention_q8_1_device, whatever the lengths are; with `weights` for calls that accumulate weights
 * (4 bytes more for every row, query head and token that the page table has room for).
 * The size depends on the current device.  0 after an error. */
size_t jq_paged_attention_ws_bytes(int64_t num_rows, int64_t num_q_heads, const jq_kv_cache *cache, int weights);

/* Attention of one query token per row over the cache.  Row r (d_q + r * q_stride_row, heads q_stride_head apart, 16-byte aligned)
 * sees the first d_lens[r] tokens of sequence d_seqs[r] (NULL: of sequence r), with window > 0 only the last `window` of them.  Query
 * head h goes with key-value head h / (num_q_heads / num_kv_heads).
 *   out = sum_i p_i v_i, p = softmax(scale * q . k_i)
 * A row that sees nothing (length zero or less) gives zeros; a row whose sequence is outside [0, num_seqs) is padding and left as it
 * was in every output.  Lengths beyond max_pages * page_size count as that.  Elements of the cache that a row sees are finite, and with
 * JQ_KV_BF16 so are its logits and the sum of a column of its values in 32 bits; what
 * lies behind its length or before its window may be anything.  With JQ_KV_F16 and JQ_KV_E4M3 p_i is rounded to 2^-40 of the row's largest one
 * where that is more than 2^-23 of itself.  Several rows may see the same sequence (drafted tokens, a short
 * prompt: each with its own length).
 * d_out (fp32 [num_rows][num_q_heads * head_dim]) and d_xq (the Q8_1 blocks of that, for the o-projection, in `order` and `s_mode`;
 * head_dim % 32 == 0 and num_q_heads * head_dim % 128 == 0) are each optional, at least one is required.  The blocks are those that
 * jq_quantize_q8_1_device makes of d_out, bit for bit.
 * d_weights, unless NULL: fp32 [num_rows][num_kv_heads], weights_stride floats apart; to entry i < weights_len is added what this step's
 * query heads together gave to token i.  Entries that are not seen are left as they were.  d_seqs must then be NULL.
 * d_ws: jq_paged_attention_ws_bytes() bytes, 16-byte aligned, its first JQ_PAGED_ATTENTION_COUNTERS(num_rows, num_q_heads) bytes zero
 * before the first call.  One workspace serves calls of any sizes, caches and types one after the other, as long as it has the bytes of
 * each, and that many bytes of the call with the most rows and heads (4096 are enough for all) were zero before the first of them: what
 * counts lies in the same place in all, and every call leaves it zero again.  Calls that can overlap on the GPU (two streams, two graphs)
 * need workspaces of their own.
 * The result does not depend on the order in which blocks run.  num_rows * num_kv_heads * max_pages * page_size is at most 2^33
 * (with more than 16 query heads to a key head, or 8 of more than 128 elements, that over the passes it takes). */
#define JQ_PAGED_ATTENTION_COUNTERS(num_rows, num_q_heads) (4u * (size_t)(num_rows) * (size_t)(num_q_heads))
int jq_paged_attention_q8_1_device(void *stream, const float *d_q, int64_t q_stride_row, int64_t q_stride_head, int64_t num_rows,
                                   int64_t num_q_heads, const jq_kv_cache *cache, const int32_t *d_lens, const int32_t *d_seqs,
                                   float scale, int64_t window, float *d_out, void *d_xq, int order, int s_mode, float *d_weights,
                                   int64_t weights_stride, int64_t weights_len, void *d_ws, size_t ws_bytes);

/* ---- eviction ------------------------------------------------------------------------------------------- */

/* Cuts every sequence down to at most `keep` tokens, each key-value head by weights of its own (d_weights as above, one row of
 * weights_stride floats per sequence and head, max_len of them in use: d_lens[b] <= max_len, longer counts as max_len).
 * Of the d_lens[b] tokens the first `sinks` and the last `recent` stay (sinks + recent <= keep), then those of the largest weight, the
 * lower index first among equals (-0 equals 0; NaN counts as minus infinity).  They keep their order.  With n = min(d_lens[b], keep):
 *   d_kept[b][h][0 .. keep)  the tokens' indices before, ascending; -1 from n on
 *   d_new_lens[b]            n (may be d_lens itself)
 *   d_new_weights[b][h]      their weights, and zeros from n up to max_len (may be d_weights; new_weights_stride floats apart)
 * Keys and values move to tokens 0 .. n-1 of the pages in d_new_page_table (num_seqs rows, new_table_stride apart, new_max_pages
 * entries, keep <= new_max_pages * page_size), which are other pages of the same pool, each of one sequence (the cache's own table is
 * refused); the pages they come from may be shared.  With d_new_page_table NULL they move to the
 * front of the sequence's own pages, which no other sequence may have: of pages that sequences share for reading, a common start, move
 * them to new ones.  Tokens from n on are left as they were.  Rotated keys stay as they are: their positions do
 * not change.  max_len is at most jq_kv_evict_max_len() of the current device. */
int64_t jq_kv_evict_max_len(void);
int jq_kv_evict_device(void *stream, const jq_kv_cache *cache, const int32_t *d_lens, const float *d_weights, int64_t weights_stride,
                       int64_t max_len, int64_t keep, int64_t recent, int64_t sinks, const int32_t *d_new_page_table,
                       int64_t new_max_pages, int64_t new_table_stride, int32_t *d_kept, int32_t *d_new_lens,
                       float *d_new_weights, int64_t new_weights_stride);

#ifdef __cplusplus
}
#endif

#endif /* JQ_KV_CACHE_H_ */
