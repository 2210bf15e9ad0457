/* Verification of drafted tokens against the target's probabilities, from given random numbers (no counterpart in the
 * reference's C header): the step behind a verify batch.
 *
 * Request r was fed n = query_start_loc[r + 1] - query_start_loc[r] tokens: its last token and n - 1 drafted ones.  Row i of its
 * rows of target_probs is the target's distribution of the token behind row i, the same row of draft_probs the one that the
 * drafted token (tokens[row + 1]) was drawn from; draft_probs NULL: drafted tokens count as certain (probability one).
 *   draft i + 1 is accepted  <=>  accept_uniforms[row i] * q(x) < p(x), and all drafts before it are
 *   the last token is drawn behind the accepted ones from max(p - q, 0) where a draft was refused (from p where that is zero
 *   everywhere), from p where no draft is left: the lowest x whose running sum exceeds sample_uniforms[r] * total
 * so that the tokens are distributed as the target's own.  Probabilities are fp32 and need not be normalised for the draw; entries
 * that are negative, infinite or NaN count as zero there.  Comparisons and sums are in 64 bits: tokens are those of exact
 * arithmetic but for numbers within 2^-40 of a border.  A row of a request that is decoded greedily is one-hot.
 * A drafted token outside [0, vocab_size) ends the drafts: behind it the token is drawn from p (padding of captured steps). */
#ifndef WARP34_DRAFTS_H
#define WARP34_DRAFTS_H

#include "warp34_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 56 bytes; the pointers are DEVICE pointers */
typedef struct {
    const int32_t* query_start_loc;   /* [num_reqs + 1] */
    const int32_t* tokens;            /* [total_tokens] the tokens that were fed */
    const uint8_t* valid_req_mask;    /* [num_reqs] or NULL; zero: nothing of the request is read or written */
    int64_t        target_row_stride; /* elements between rows, at least vocab_size */
    int64_t        draft_row_stride;
    int32_t        num_reqs;
    int32_t        total_tokens;
    int32_t        max_q_len;         /* host's bound on n, 0: not known; nothing depends on it as yet */
    int32_t        vocab_size;
} warp34_draft_batch;

#if defined(__cplusplus)
static_assert(sizeof(warp34_draft_batch) == 56, "warp34_draft_batch ABI size");
#else
_Static_assert(sizeof(warp34_draft_batch) == 56, "warp34_draft_batch ABI size");
#endif

/* out_tokens [total_tokens]: rows of a request hold the accepted drafts, then the token drawn, then -1 (the drawn one is -1 as well
 * where the row of p has no positive entry).  emitted_counts [num_reqs]: accepted drafts and one, which is also the number of fed
 * tokens whose cache rows and states stay (state_tokens of warp34_linear_attention_*); 0 for a request without rows.
 * accept_uniforms: fp32 [total_tokens], sample_uniforms: fp32 [num_reqs], in [0, 1).  out_tokens and
 * emitted_counts overlap no input.
 * Scratch (16-byte aligned, warp34_verify_drafts_scratch_bytes): the vocabulary is summed by many workgroups; without it by one for
 * each request, with the same tokens but for those within the rounding of a 64-bit sum of a border.
 * hipErrorInvalidValue: a missing pointer, vocab_size < 1, strides below vocab_size, more than 2^20 requests; num_reqs <= 0 or
 * total_tokens <= 0 return 0 without a launch, nothing is written.  Two calls that may run at once need a workspace each. */
int warp34_verify_drafts(const warp34_exec* ex, const warp34_draft_batch* batch, const float* target_probs,
                         const float* draft_probs, const float* accept_uniforms, const float* sample_uniforms,
                         int32_t* out_tokens, int32_t* emitted_counts);
size_t warp34_verify_drafts_scratch_bytes(int num_reqs, int vocab_size);

#ifdef __cplusplus
}
#endif
#endif /* WARP34_DRAFTS_H */
