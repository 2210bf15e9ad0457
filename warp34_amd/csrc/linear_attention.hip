// Entry points of linear attention: checks, and the choice of the kernel.
#include <cmath>

#include "attn_launch.h"
#include "linear_attention.h"

namespace w34 {

template <typename T, int DK, int DV>
static int linear_launch(const warp34_exec* ex, const warp34_linear_attention_batch* b, const LinearArgs& a) {
    if (!grid_fits((long long)a.num_reqs * a.v_heads, 2 * DV)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((linear_step_kernel<T, DK, DV>), dim3((unsigned)a.num_reqs * (unsigned)a.v_heads), dim3(2 * DV), 0, (hipStream_t)ex->stream, a);
    return (int)hipGetLastError();
}

template <typename T>
static int linear_entry(const warp34_exec* ex, const warp34_linear_state_layout* y, const warp34_linear_attention_batch* b, const void* q, const void* k,
                        const void* v, const float* log_decay, void* out) {
    if (!ex || !y || !b || !q || !k || !v || !b->query_start_loc) return (int)hipErrorInvalidValue;
    if (y->num_k_heads <= 0 || y->num_v_heads <= 0 || y->num_v_heads % y->num_k_heads != 0 || !std::isfinite(b->scale)) return (int)hipErrorInvalidValue;
    if (y->num_v_heads > (1 << 20)) return (int)hipErrorInvalidValue;
    if ((y->k_head_dim != 64 && y->k_head_dim != 128) || (y->v_head_dim != 64 && y->v_head_dim != 128)) return (int)hipErrorNotSupported;
    const int k_row = y->num_k_heads * y->k_head_dim, v_row = y->num_v_heads * y->v_head_dim;
    if (b->q_row_stride < k_row || b->k_row_stride < k_row || b->v_row_stride < v_row || (out && b->out_row_stride < v_row) ||
        (log_decay && b->decay_row_stride != 0 && b->decay_row_stride < y->num_v_heads))
        return (int)hipErrorInvalidValue;
    const bool states = b->state_in_slots != nullptr || b->state_out_slots != nullptr;
    if (states && (!y->state_base || y->slot_stride_bytes < 4ull * (uint64_t)v_row * (uint64_t)y->k_head_dim)) return (int)hipErrorInvalidValue;
    if (((b->q_row_stride | b->k_row_stride | b->v_row_stride) & 7) != 0 || (out && (b->out_row_stride & 7) != 0) ||
        (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15u) != 0 || ((uintptr_t)log_decay & 3u) != 0 ||
        (states && ((y->state_base | y->slot_stride_bytes) & 15u) != 0))
        return (int)hipErrorNotSupported;
    if (b->num_reqs <= 0 || b->total_tokens < 0 || (!out && !b->state_out_slots)) return 0;
    const LinearArgs a{b->query_start_loc, b->state_in_slots, b->has_initial_state, b->state_out_slots, b->state_tokens, b->valid_req_mask,
                       (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, log_decay, (uint16_t*)out, y->state_base, y->slot_stride_bytes,
                       b->num_reqs, b->total_tokens, y->num_k_heads, y->num_v_heads, y->num_v_heads / y->num_k_heads,
                       b->q_row_stride, b->k_row_stride, b->v_row_stride, b->out_row_stride, b->decay_row_stride, b->scale};
    if (y->k_head_dim == 128) return y->v_head_dim == 128 ? linear_launch<T, 128, 128>(ex, b, a) : linear_launch<T, 128, 64>(ex, b, a);
    return y->v_head_dim == 128 ? linear_launch<T, 64, 128>(ex, b, a) : linear_launch<T, 64, 64>(ex, b, a);
}

}  // namespace w34

using namespace w34;

extern "C" size_t warp34_linear_attention_scratch_bytes(const warp34_linear_state_layout* layout, int num_reqs, int total_tokens, int max_q_len) {
    (void)layout, (void)num_reqs, (void)total_tokens, (void)max_q_len;
    return 0;
}
extern "C" int warp34_linear_attention_f16(const warp34_exec* ex, const warp34_linear_state_layout* layout, const warp34_linear_attention_batch* batch,
                                           const void* q, const void* k, const void* v, const float* log_decay, void* out) {
    return linear_entry<F16>(ex, layout, batch, q, k, v, log_decay, out);
}
extern "C" int warp34_linear_attention_bf16(const warp34_exec* ex, const warp34_linear_state_layout* layout, const warp34_linear_attention_batch* batch,
                                            const void* q, const void* k, const void* v, const float* log_decay, void* out) {
    return linear_entry<BF16>(ex, layout, batch, q, k, v, log_decay, out);
}
