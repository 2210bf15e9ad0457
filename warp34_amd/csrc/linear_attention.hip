// Entry points of linear attention: checks, and the choice of the kernel.
#include <cmath>

#include "attn_launch.h"
#include "linear_chunk.h"

namespace w34 {

constexpr int kLinearPlaces = 256;  // of workgroups of eight waves, a unit each; of four waves there is room for more, and half as many count as one
constexpr int kLinearMostStride = 1 << 23;  // elements: a chunk's rows are within 2^31 bytes
// Up to so many parts of a request are joined by the kernel of the rows, each part reading what those before it add; more by a launch of their own:
// 6 parts 21.2 -> 17.8 us, 8 parts of 32 heads 116.5 -> 112.0, 16 parts of 4 heads 20.9 -> 24.0 and of 16 heads 70.1 -> 69.5.
constexpr int kLinearJoined = 8;

static long long linear_most(int total_tokens, int max_q_len) { return max_q_len > 0 && max_q_len < total_tokens ? max_q_len : total_tokens; }

// Whether a batch goes by the recurrent kernel, whose time grows with a request's tokens, or by chunks, of which it is one up to 64 tokens and whose
// workgroups have a unit each: up to 4 tokens where one round of those holds the batch, up to 8 where there are more.  us recurrent / by chunks, of
// 32 heads of 128 x 128: 8 requests of 4 tokens 12.1 / 12.3, of 8 16.0 / 12.4; 16 of 8 21.8 / 22.5, of 10 24.5 / 22.6; 32 of 4 34.6 / 46.0, of 8
// 43.6 / 46.6, of 12 53.1 / 47.8; of 64 x 64: 8 of 4 5.8 / 6.0, 16 of 5 8.7 / 8.5, 32 of 8 14.9 / 14.2.
static bool linear_steps(const warp34_linear_state_layout* y, int num_reqs, int total_tokens, int max_q_len) {
    return linear_most(total_tokens, max_q_len) <= ((long long)num_reqs * y->num_v_heads * y->v_head_dim <= 256 * 128 ? 4 : 8);
}

// How a batch is cut up.
struct LinearShape {
    int length;       // tokens of a part, 0: requests are walked from end to end
    long long parts;  // at most
    bool joined;      // by the rows' kernel
    size_t bytes;     // of scratch
};

// A request walked from end to end takes a chunk's time for each of its chunks, however few the workgroups are; parts make two or three launches and
// half as much work again, in rounds of as many workgroups as there are places.  How long they are, and whether there are any, goes by these times, in
// us, of
//   a walk   3.5 + 3.4 a chunk of the longest request, up to 4.1 where all places are taken, and as much longer as there are more workgroups
//   parts    6 a chunk of a part and a round, 12 and 12 more for each round behind the first + 0.5 a part of the longest request, or 5 + 0.25 where a
//            launch joins them.
// Measured, 32 heads of 128 x 128 walked and in parts: 333 tokens 24.5 / 19.4, twice 25.7 / 25.4; 500 31.7 / 22.1, three times 34.6 / 38.7; 1 024 59 / 30,
// four times 65.6 / 66.9; 8 192 447 / 103; 4 x 4 096 247 / 211, 5 x 4 096 263 / 389.
static LinearShape linear_shape(const warp34_linear_state_layout* y, int num_reqs, int total_tokens, int max_q_len, bool kept, bool rows, size_t scratch) {
    const long long most = (linear_most(total_tokens, max_q_len) + kLinearChunk - 1) / kLinearChunk, total = total_tokens / kLinearChunk + 1;  // in chunks
    const long long heads = y->num_v_heads, size = (long long)y->k_head_dim * y->v_head_dim, places = kLinearPlaces * (128 / y->v_head_dim);
    const double full = (double)num_reqs * heads / places;
    LinearShape s{0, 0, false, 0};
    double best = 3.5 + most * (3.4 + 0.7 * min(full, 1.0)) * max(full, 1.0);
    for (long long chunks = 1; chunks < most; chunks += 1 + chunks / 32) {
        const long long cuts = (most + chunks - 1) / chunks, length = chunks * kLinearChunk;
        if ((cuts - 1) * heads >= 2 * places) continue;
        // those there will be, about, and those there are room for: ceil(n / length) <= (n - 1) / length + 1 over the requests, of which those
        // without tokens have one too, and one more for a cut behind the kept tokens
        const long long about = min(num_reqs * cuts, total / chunks + (num_reqs + 1) / 2);
        const long long parts = (total_tokens - 1) / length + num_reqs + (kept ? min(num_reqs, total_tokens) : 0);
        const bool joined = rows && cuts + kept <= kLinearJoined;
        const size_t bytes = ((size_t)parts * heads * 4 + 15) / 16 * 16 + (size_t)(parts + (joined ? num_reqs : 0)) * heads * size * 4;
        const double time = (12.0 + 6.0 * chunks) * ((about * heads + places - 1) / places) + (joined ? 0.5 * cuts : 5.0 + 0.25 * cuts);
        if (time >= best || bytes > scratch || !grid_fits(parts * heads * (size / 1024), 256)) continue;
        best = time;
        s.length = (int)length, s.parts = parts, s.joined = joined, s.bytes = bytes;
    }
    return s;
}

static LinearLength linear_length(int tokens) {
    int s = 31;
    while (tokens > 1ll << (s - 31)) ++s;
    return tokens > 0 ? LinearLength{tokens, (uint32_t)(((1ull << s) + (uint64_t)tokens - 1) / (uint64_t)tokens), s - 32} : LinearLength{0, 0, 0};
}

template <typename T, int DK, int DV>
static int linear_chunk_launch(const warp34_exec* ex, const LinearArgs& a, const LinearShape& shape) {
    const long long columns = (long long)a.v_heads;
    const hipStream_t stream = (hipStream_t)ex->stream;
    LinearParts p{nullptr, nullptr, nullptr, linear_length(shape.length), (int)shape.parts};
    if (shape.length == 0) {
        if (!grid_fits(a.num_reqs * columns, 4 * DV)) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL((linear_chunk_kernel<T, DK, DV, kLinearWalk>), dim3((unsigned)(a.num_reqs * columns)), dim3(4 * DV), 0, stream, a, p);
        return (int)hipGetLastError();
    }
    const long long scans = (long long)a.num_reqs * a.v_heads * (DK * DV / 1024);
    if (!grid_fits(shape.parts * columns, 4 * DV) || !grid_fits(scans, 256)) return (int)hipErrorInvalidValue;
    p.states = (float*)(uintptr_t)ex->scratch_ptr;
    const long long slot = (long long)a.v_heads * (DK * DV);
    if (shape.joined) p.starts = p.states + shape.parts * slot;
    p.fades = p.states + (shape.parts + (shape.joined ? a.num_reqs : 0)) * slot;
    const dim3 grid((unsigned)(shape.parts * columns));
    hipLaunchKernelGGL((linear_chunk_kernel<T, DK, DV, kLinearSums>), grid, dim3(4 * DV), 0, stream, a, p);
    int rc = (int)hipGetLastError();
    if (rc) return rc;
    if (!shape.joined) {
        hipLaunchKernelGGL(linear_scan_kernel, dim3((unsigned)scans), dim3(256), 0, stream, a, p, DK);
        rc = (int)hipGetLastError();
        if (rc || a.out == nullptr) return rc;
    }
    hipLaunchKernelGGL((linear_chunk_kernel<T, DK, DV, kLinearRows>), grid, dim3(4 * DV), 0, stream, a, p);
    return (int)hipGetLastError();
}

template <typename T, int DK, int DV>
static int linear_launch(const warp34_exec* ex, const warp34_linear_state_layout* y, const warp34_linear_attention_batch* b, const LinearArgs& a) {
    if (linear_steps(y, b->num_reqs, b->total_tokens, b->max_q_len)) {
        if (!grid_fits((long long)a.num_reqs * a.v_heads, 2 * DV)) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL((linear_step_kernel<T, DK, DV>), dim3((unsigned)a.num_reqs * (unsigned)a.v_heads), dim3(2 * DV), 0, (hipStream_t)ex->stream, a);
        return (int)hipGetLastError();
    }
    const bool usable = ex->scratch_ptr != 0 && (ex->scratch_ptr & 15u) == 0;
    const LinearShape shape = linear_shape(y, b->num_reqs, b->total_tokens, b->max_q_len, b->state_tokens != nullptr, a.out != nullptr, usable ? ex->scratch_size : 0);
    return linear_chunk_launch<T, DK, DV>(ex, a, shape);
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
    if (b->q_row_stride > kLinearMostStride || b->k_row_stride > kLinearMostStride || b->v_row_stride > kLinearMostStride ||
        (out && b->out_row_stride > kLinearMostStride))
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
                       b->num_reqs, b->total_tokens, y->num_v_heads, y->v_head_dim, y->num_v_heads / y->num_k_heads,
                       b->q_row_stride, b->k_row_stride, b->v_row_stride, b->out_row_stride, b->decay_row_stride, b->scale};
    if (y->k_head_dim == 128) return y->v_head_dim == 128 ? linear_launch<T, 128, 128>(ex, y, b, a) : linear_launch<T, 128, 64>(ex, y, b, a);
    return y->v_head_dim == 128 ? linear_launch<T, 64, 128>(ex, y, b, a) : linear_launch<T, 64, 64>(ex, y, b, a);
}

}  // namespace w34

using namespace w34;

extern "C" size_t warp34_linear_attention_scratch_bytes(const warp34_linear_state_layout* layout, int num_reqs, int total_tokens, int max_q_len) {
    if (!layout || num_reqs <= 0 || total_tokens <= 0 || layout->num_v_heads <= 0 || layout->num_v_heads > (1 << 20) ||
        (layout->k_head_dim != 64 && layout->k_head_dim != 128) || (layout->v_head_dim != 64 && layout->v_head_dim != 128))
        return 0;
    if (linear_steps(layout, num_reqs, total_tokens, max_q_len)) return 0;
    size_t bytes = 0;  // of the calls that such a batch may come in
    for (int way = 0; way < 4; ++way) bytes = max(bytes, linear_shape(layout, num_reqs, total_tokens, max_q_len, way & 1, way & 2, ~(size_t)0).bytes);
    return bytes;
}
extern "C" int warp34_linear_attention_f16(const warp34_exec* ex, const warp34_linear_state_layout* layout, const warp34_linear_attention_batch* batch,
                                           const void* q, const void* k, const void* v, const float* log_decay, void* out) {
    return linear_entry<F16>(ex, layout, batch, q, k, v, log_decay, out);
}
extern "C" int warp34_linear_attention_bf16(const warp34_exec* ex, const warp34_linear_state_layout* layout, const warp34_linear_attention_batch* batch,
                                            const void* q, const void* k, const void* v, const float* log_decay, void* out) {
    return linear_entry<BF16>(ex, layout, batch, q, k, v, log_decay, out);
}
