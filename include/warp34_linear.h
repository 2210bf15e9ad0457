/* Linear attention over per-request states (no counterpart in the reference's C header).
 *
 * A layer of this kind keeps, for each request and value head, one matrix S [k_head_dim][v_head_dim] in fp32 in place of a cache.
 * For the tokens of request r, value head h and its key head h / (num_v_heads / num_k_heads):
 *   S = exp(log_decay[t][h]) * S + k_t v_t^T          out_t = scale * S^T q_t
 * states are kept in slots (state_base + slot * slot_stride_bytes, [num_v_heads][k_head_dim][v_head_dim]): the request starts from
 * slot state_in_slots[r] and what it leaves goes to slot state_out_slots[r].  The step descriptor of the host side carries both,
 * and has_initial_state.
 *
 * One entry serves prompts, single tokens and drafted tokens.  max_q_len, the host's bound on a request's tokens (0: not known,
 * total_tokens), chooses the kernel for the whole batch: up to 4 tokens (8 where num_reqs * num_v_heads * v_head_dim is above 32 768) one token after the
 * other, all in fp32, each off by 2^-22 of its terms' size at most; beyond, chunks of 64 tokens, of the exactness given below, cut by it into parts.  A bound that is wrong
 * costs time, or that exactness, and nothing else. */
#ifndef WARP34_LINEAR_H
#define WARP34_LINEAR_H

#include "warp34_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 32 bytes */
typedef struct {
    uint64_t state_base;        /* device address of fp32 states, 16-byte aligned */
    uint64_t slot_stride_bytes; /* at least 4 * num_v_heads * k_head_dim * v_head_dim, a multiple of 16 */
    int32_t  num_k_heads;       /* heads of q and k; divides num_v_heads */
    int32_t  num_v_heads;       /* heads of v, log_decay, out and the states */
    int32_t  k_head_dim;        /* 64 or 128 */
    int32_t  v_head_dim;        /* 64 or 128 */
} warp34_linear_state_layout;

/* 88 bytes.  Every pointer is a DEVICE pointer; all but query_start_loc may be NULL. */
typedef struct {
    const int32_t* query_start_loc;   /* [num_reqs + 1] */
    const int32_t* state_in_slots;    /* [num_reqs]; negative, or no array: the request starts from zeros */
    const int32_t* has_initial_state; /* [num_reqs]; zero: the request starts from zeros whatever its slot */
    const int32_t* state_out_slots;   /* [num_reqs]; negative, or no array: no state is written */
    const int32_t* state_tokens;      /* [num_reqs] the state written is the one behind that many of the request's tokens
                                         (clamped to 0 ... their number); no array: behind all of them */
    const uint8_t* valid_req_mask;    /* [num_reqs]; zero: nothing of the request is read or written */
    int32_t        num_reqs;
    int32_t        total_tokens;
    int32_t        max_q_len;
    float          scale;
    int32_t        q_row_stride;      /* elements between tokens: of q, k, v, out (multiples of 8, at least heads * dim, at most 2^23) */
    int32_t        k_row_stride;
    int32_t        v_row_stride;
    int32_t        out_row_stride;
    int32_t        decay_row_stride;  /* elements between tokens of log_decay; 0: one row of decays for all tokens */
    int32_t        reserved;
} warp34_linear_attention_batch;

#if defined(__cplusplus)
static_assert(sizeof(warp34_linear_state_layout) == 32, "warp34_linear_state_layout ABI size");
static_assert(sizeof(warp34_linear_attention_batch) == 88, "warp34_linear_attention_batch ABI size");
#else
_Static_assert(sizeof(warp34_linear_state_layout) == 32, "warp34_linear_state_layout ABI size");
_Static_assert(sizeof(warp34_linear_attention_batch) == 88, "warp34_linear_attention_batch ABI size");
#endif

/* q, k: [total_tokens, num_k_heads, k_head_dim], v, out: [total_tokens, num_v_heads, v_head_dim], 16 bits (fp16 for _f16, bf16 for
 * _bf16), rows as far apart as the strides say (packed projections are read in place); q, k, v and out 16-byte aligned.
 * log_decay: fp32 [total_tokens, num_v_heads], at most zero; minus infinity forgets what was before the token; NULL: no decay.
 * out may be NULL: only the states move on (the accepted part of a drafted step, say: state_tokens may be what
 * warp34_verify_drafts has written).  A request without tokens copies its state from slot to slot; the same slot may be the input
 * of several requests.  A request's output slot may be its own input slot; apart from that no output slot may be another request's
 * input or output.  Rows of no request are left as they were.  The rows and the states that a request reads must be finite, for its
 * outputs those behind state_tokens too; masked requests and rows behind the last one may hold anything, and for the states what is
 * behind state_tokens.
 * Exactness, in parts of the terms' size (of a state: faded |S| + sum of weighted |k| |v|^T; of an output: scale |q|^T times that): a prompt's products take
 * 16-bit operands in parts, which leave states, fp32 throughout, within 2^-20 for each 64 tokens that still count, and outputs within 2^-15 (bf16) or 2^-19 (fp16)
 * beside their state's error and their own rounding; where terms cancel, that shows.  fp16 adds, of each of its operands, 2^-50 of the largest value of
 * a column weighted at its chunk's end, state of a column, or weight of a row; weights below 2^-126 count as zero.  What is summed up (q . k, S^T q, k v^T) has to stay
 * below 2^100 in size.
 * Scratch (16-byte aligned, of warp34_linear_attention_scratch_bytes): prompts are cut into parts that run at once; with less, into
 * fewer, without any a request's heads run side by side and its tokens one part after another.  The order of summation depends on
 * max_q_len, num_reqs, total_tokens, the layout, the request's lengths, the scratch, and on which of out and state_tokens are there, and
 * on nothing else: the same call gives the same bits.  Two calls that may run at once need a workspace each.
 * hipErrorInvalidValue: a missing ex, layout, batch, query_start_loc, q, k or v, counts (more than 2^20 heads) or strides out of
 * range, a missing state_base where slots are named, a decay stride that is neither 0 nor at least num_v_heads, a scale that is not
 * finite; hipErrorNotSupported: other head dimensions, alignments.
 * No requests or no tokens bound (num_reqs <= 0, total_tokens < 0) return 0 without a launch. */
int warp34_linear_attention_f16(const warp34_exec* ex, const warp34_linear_state_layout* layout,
                                const warp34_linear_attention_batch* batch, const void* q, const void* k, const void* v,
                                const float* log_decay, void* out);
int warp34_linear_attention_bf16(const warp34_exec* ex, const warp34_linear_state_layout* layout,
                                 const warp34_linear_attention_batch* batch, const void* q, const void* k, const void* v,
                                 const float* log_decay, void* out);
/* Bytes of scratch that such a call can make use of; 0 where it needs none. */
size_t warp34_linear_attention_scratch_bytes(const warp34_linear_state_layout* layout, int num_reqs, int total_tokens, int max_q_len);

#ifdef __cplusplus
}
#endif
#endif /* WARP34_LINEAR_H */
