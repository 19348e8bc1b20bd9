/* consumer_int8_attention.h -- C ABI of the attention operators for MI355X (gfx950): what a
 * serving program runs between a layer's INT8 QKV projection and its output projection,
 * over a paged key/value cache of 4-bit values.
 *
 * Conventions are those of consumer_int8_amd.h: raw device pointers, int64 sizes, a
 * hipStream_t passed as `void*`, caller-owned buffers, no allocation, no synchronisation,
 * ci8_status codes with ci8_last_error() as the message, and every check before the first
 * HIP call. Descriptors are read during the call only. All calls can be captured into a
 * HIP graph. No reference counterpart: the reference's cache formats and kernels differ.
 *
 * The cache. A row is one head of one token: `dim` values in blocks of 32 channels. A value
 * is code * 2^(scale - 127): an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives;
 * sign in the top bit) times its block's power of two. Codes take dim/2 bytes (channel 2i in
 * the low half of byte i), scales dim/32 bytes; scale 255 makes the block NaN, and 253 and 254 may. Keys and values
 * each have
 *   codes  UINT8 [pages, heads, page_size, dim/2]   and
 *   scales UINT8 [pages, heads, page_size, dim/32],
 * contiguous inside a page, pages `*_page_stride` bytes apart. Slot s of the cache is row
 * s % page_size of page s / page_size.
 *
 * Quantizing a block with largest magnitude amax: scale 2^e with the smallest e for which
 * amax <= 7 * 2^e, held in -125 .. 125, codes the nearest of x / 2^e, ties to the even code (6
 * is the largest, so a value between 6 and 7 becomes 6). A block holding an infinity or a NaN
 * gets scale 255 and zero codes.
 */
#ifndef CONSUMER_INT8_ATTENTION_H
#define CONSUMER_INT8_ATTENTION_H

#include <stdint.h>

#include "consumer_int8_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* BF16 rows of heads: channel c of head h of token t is data[t * token_stride +
 * h * head_stride + c]. Strides in elements, multiples of 8; data 16-byte aligned. */
typedef struct ci8_heads {
  void* data;
  int64_t heads;
  int64_t token_stride;
  int64_t head_stride;
} ci8_heads;

/* RMS norm over a head: y = (x * (1 / sqrt(mean(x^2) + eps))) * weight, FP32, weight FP32
 * [dim] 16-byte aligned. Squares are summed in pairs of neighbours, then pairs of those and
 * so on, each operation rounded once. A NULL weight leaves the head as it is. */
typedef struct ci8_head_norm {
  const float* q_weight;
  const float* k_weight;
  double eps;
} ci8_head_norm;

/* Rotation of the first `rot` channels (16 <= rot <= dim, rot % 16 == 0; 0: none) by the
 * angles in `table` FP32 [rows, rot], 16-byte aligned: rot/2 cosines, then rot/2 sines. Pair i
 * is channels (i, i + rot/2), or (2i, 2i + 1) if interleaved != 0: (a, b) -> (a cos - b sin,
 * b cos + a sin), each product and sum rounded to FP32. positions INT64 [axes, tokens];
 * axis_of INT32 [rot/2] names each pair's axis and is needed where axes > 1. A position
 * outside [0, rows) or an axis outside [0, axes) gives NaN. */
typedef struct ci8_rotation {
  const float* table;
  int64_t rows;
  int64_t rot;
  const int64_t* positions;
  int64_t axes;
  const int32_t* axis_of;
  int64_t interleaved;
} ci8_rotation;

/* The cache above. Codes start on 16 bytes and scales on 8, and so do all their pages; each of
 * the four spans at most 32 GiB. */
typedef struct ci8_fp4_cache {
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  int64_t k_code_page_stride;
  int64_t k_scale_page_stride;
  int64_t v_code_page_stride;
  int64_t v_scale_page_stride;
  int64_t pages;
  int64_t heads;
  int64_t page_size; /* a power of two, 16..1024 */
} ci8_fp4_cache;

/* qk_norm_rope: norm, then rotation, of every query and key head in FP32; one rounding to
 * BF16. dim in {64, 128, 256}. q_out and k_out have their inputs' head counts; each may be
 * its input (the same descriptor), else outputs overlap nothing. tokens = 0 is a no-op. */
int ci8_qk_norm_rope(const ci8_heads* q, const ci8_heads* k, const ci8_heads* q_out,
                     const ci8_heads* k_out, const ci8_head_norm* norm,
                     const ci8_rotation* rotation, int64_t tokens, int64_t dim, void* stream);

/* append_fp4: keys, normed and rotated as above and not rounded on the way, and values are
 * quantized into the cache rows that slots INT64 [tokens] names; a slot outside the cache
 * (negative for a padding token) is skipped. Slots must differ: a row that several tokens
 * share may hold parts of each. Where q is not NULL the queries are normed and rotated into q_out as
 * ci8_qk_norm_rope does, in the same launch. */
int ci8_append_fp4(const ci8_heads* q, const ci8_heads* k, const ci8_heads* v,
                   const ci8_heads* q_out, const ci8_head_norm* norm,
                   const ci8_rotation* rotation, const int64_t* slots,
                   const ci8_fp4_cache* cache, int64_t tokens, int64_t dim, void* stream);

/* unpack_fp4: the rows that slots INT64 [count] names, as BF16 k and v [count, heads, dim]
 * (contiguous, 16-byte aligned), exactly; rows of slots outside the cache are zeros. */
int ci8_unpack_fp4(const ci8_fp4_cache* cache, const int64_t* slots, void* k, void* v,
                   int64_t count, int64_t dim, void* stream);

/* attention_fp4: causal attention of BF16 queries over the cache.
 * Sequence s has the tokens 0 .. context_lens[s]-1 in the cache; token j is row j % page_size
 * of page page_table[s, j / page_size] (INT32 [seqs, table_width]). Its queries are rows
 * q_starts[s] .. q_starts[s+1]-1 of q (q_starts INT32 [seqs+1], or NULL: row s alone), the
 * last of them at position context_lens[s]-1, and head h reads key head h / (q heads /
 * cache heads). A query at position p attends to tokens max(0, p - window + 1) .. p (window
 * 0: all up to p) by softmax(scale * q.k); out BF16 [tokens, q heads, dim] contiguous, lse
 * FP32 [tokens, q heads] (may be NULL) the natural logarithm of the sum of exp(scale * q.k).
 * A query that attends to nothing gives zeros and -inf; what a query does not attend to,
 * NaN or not, does not reach it. Table entries outside the cache are
 * tokens that nobody attends to; lengths are clamped to 0 .. table_width * page_size and
 * q_starts to 0 .. tokens; sequences of more than max_q queries are computed up to max_q;
 * rows of q in no sequence are not written. Products are BF16 x BF16 with FP32 sums, the
 * statistics FP32, the weights rounded to BF16 before they meet the values.
 * workspace: FP32 [65536, dim + 2], 16-byte aligned, any content, one a stream.
 * q heads a multiple of the cache's heads; scale finite; max_q >= 1; window >= 0;
 * table_width * page_size at most 2^26 - 4096. */
int ci8_attention_fp4(const ci8_heads* q, const ci8_fp4_cache* cache,
                      const int32_t* page_table, int64_t table_width,
                      const int32_t* context_lens, const int32_t* q_starts, int64_t seqs,
                      int64_t tokens, int64_t dim, void* workspace, void* out, float* lse,
                      double scale, int64_t max_q, int64_t window, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CONSUMER_INT8_ATTENTION_H */
