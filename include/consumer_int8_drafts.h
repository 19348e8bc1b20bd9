/* consumer_int8_drafts.h -- C ABI of the operators of speculative decoding for MI355X (gfx950):
 * attention of a tree of drafted tokens over the 4-bit cache of consumer_int8_attention.h, the
 * probabilities that a vocabulary's logits stand for, which drafted tokens stand by them, and the
 * accepted rows' way to consecutive rows of the cache.
 *
 * Conventions are those of consumer_int8_attention.h: raw device pointers, int64 sizes, a
 * hipStream_t passed as `void*`, caller-owned buffers, no allocation, no synchronisation, every
 * check before the first HIP call, no reference counterpart. All calls can be captured into a HIP
 * graph.
 *
 * A tree. The rows of sequence s are q_starts[s] .. q_starts[s+1]-1 (INT32 [seqs+1]), at most 64 of
 * them drafted at once. parents INT32 [rows] names each row's parent by its number in the
 * sequence; a parent comes before its child, and any number outside [0, own number) is none: such a
 * row hangs on the context alone. Row 0 is the last token that is certain, and the root of what is
 * verified. The depth of a row is how many ancestors it has.
 */
#ifndef CONSUMER_INT8_DRAFTS_H
#define CONSUMER_INT8_DRAFTS_H

#include <stdint.h>

#include "consumer_int8_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* attention_fp4_tree: ci8_attention_fp4 for trees. All rows of sequence s are in the cache, row i of n
 * as token context_lens[s] - n + i; its position is context_lens[s] - n + its depth. It attends to the
 * tokens before the tree whose position its window reaches, to its ancestors that the window
 * reaches, and to itself. max_q is at most 64. Blocks of 64 rows (max_q times the query heads of a
 * key head; 32 rows at dim 256) times (table_width * page_size / 32 + 41) stay under 2^24. All else is as
 * ci8_attention_fp4 says. */
int ci8_attention_fp4_tree(const ci8_heads* q, const ci8_fp4_cache* cache,
                           const int32_t* page_table, int64_t table_width,
                           const int32_t* context_lens, const int32_t* q_starts,
                           const int32_t* parents, int64_t seqs, int64_t tokens, int64_t dim,
                           void* workspace, void* out, float* lse, double scale, int64_t max_q,
                           int64_t window, void* stream);

/* move_fp4: in each sequence of n rows, for i = 0 .. n-1 in order, cache row slots[rows[i]] is copied
 * to slots[i] where i < rows[i] < n, keys and values of all heads; rows INT32 [tokens] are numbers in
 * the sequence, slots INT64 [tokens] cache rows, no two alike. Other numbers move nothing, and
 * neither do slots outside the cache. With rows the path of ci8_verify_drafts, the accepted
 * tokens' keys and values end up in the sequence's first slots. */
int ci8_move_fp4(const ci8_fp4_cache* cache, const int32_t* rows, const int64_t* slots,
                 const int32_t* q_starts, int64_t seqs, int64_t tokens, int64_t dim, void* stream);

/* Bytes of the workspace of the next two, 16-byte aligned, any content, one a stream. */
#define CI8_SAMPLING_WORKSPACE_BYTES (1 << 20)

/* token_probs: p = softmax(logits / temperature) of each row, FP32. logits BF16 (logit_bits 16) or FP32
 * (32) [tokens, vocab], rows logit_stride values apart; temperature FP32 [tokens], NULL for 1
 * everywhere; probs FP32 [tokens, vocab], rows prob_stride apart. Temperature 0 gives 1 at the first of
 * the largest logits and 0 elsewhere. A row of -inf alone gives zeros; a row with a NaN gives NaN
 * everywhere, and so do one with +inf at a temperature above 0 and a negative or NaN temperature.
 * probs may be FP32 logits themselves (the same rows); else they overlap nothing. vocab is 1 .. 2^24. */
int ci8_token_probs(const void* logits, int64_t logit_bits, int64_t logit_stride,
                    const float* temperature, float* probs, int64_t prob_stride, int64_t tokens,
                    int64_t vocab, void* workspace, void* stream);

/* verify_drafts: which drafted tokens stand, so that what is returned is distributed as if drawn
 * from the target alone, and the token that follows them.
 *
 * target FP32 [tokens, vocab] (rows target_stride apart): in row r what follows the token of row r.
 * draft, the same for the drafter, or NULL; ids INT64 [tokens] the rows' tokens; parents INT32
 * [tokens], or NULL where each row's parent is the row before it; uniforms FP32 [tokens] in [0, 1).
 *
 * From row c = 0 on, its children (rows whose parent is c) are tried in order; the first that
 * stands is the next c. With p the target's and q the drafter's row c:
 *   with draft, children drawn independently from q: w = max(p - a q, 0), a = 0, S = 1 at first; child
 *     x with number u stands if u q(x) S < w(x); if not, a grows by S and S becomes the sum of the
 *     new w (so w / S is max(w / S - q, 0), made to sum to 1, of the w before);
 *   without, children are certain choices: w = p, S = 1; child x stands if u S < w(x); if not, S
 *     loses w(x) and w(x) becomes 0.
 * Children drawn without replacement are neither: what is returned would not be so distributed.
 * Where none stands, or c has no child, the next token is the first whose running sum of w passes u
 * times the sum of w, with u the number of the sequence's row 0; where w is zero everywhere, p takes
 * its place; where p is, too, the next token is -1. In 64 bits throughout.
 *
 * path INT32 [tokens]: in sequence s the numbers of the accepted rows (0 first), then -1; accepted
 * INT32 [seqs] how many, row 0 counted; next INT64 [seqs]. A sequence without rows gives 0 and -1.
 * Values of target and draft that are not positive and finite count as 0, tokens outside the
 * vocabulary never stand, numbers outside [0, 1) count as the nearest inside and NaN as 0. Rows past
 * the 64th of a sequence are not tried (-1). Rows in no sequence are not written. seqs at most 16384, vocab
 * 1 .. 2^24. */
int ci8_verify_drafts(const float* target, int64_t target_stride, const float* draft,
                      int64_t draft_stride, const int64_t* ids, const int32_t* parents,
                      const int32_t* q_starts, const float* uniforms, int64_t seqs, int64_t tokens,
                      int64_t vocab, void* workspace, int32_t* path, int32_t* accepted,
                      int64_t* next, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CONSUMER_INT8_DRAFTS_H */
