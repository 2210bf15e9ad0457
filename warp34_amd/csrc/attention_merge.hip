// Joins attention results over disjoint key sets by the logarithms of their sums:
//
//   lse = ln sum_p exp(lse_p)        out = sum_p exp(lse_p - lse) out_p
//
// in 32 bits, rounded once.  A part whose lse is minus infinity saw no key: what its row holds does not matter.  One pass: the sums
// are kept relative to a running maximum.  Bound: HBM, every part read once: two parts of 131 072 fp16 rows of 256 in 36.7 us (5.5 TB/s, as a large copy),
// eight of 32 768 in 30.6; eight of 512 in 3.8, a launch.
#include "attn_lanes.h"
#include "attn_launch.h"

namespace w34 {

// A thread takes eight elements of a row, head_dim / 8 threads a row.  Parts go by in groups of kMergeGroup, whose loads travel
// together (2 / 4 / 8: two parts of 131 072 rows 37.0 / 36.7 / 40.0 us, eight of 32 768 30.5 / 30.6 / 32.3).
constexpr int kMergeGroup = 4;

template <typename T>
__global__ __launch_bounds__(256) void attention_merge_kernel(const uint16_t* parts, const float* lse_parts, int num_parts, int64_t part_stride,
                                                              int64_t lse_part_stride, uint16_t* out, float* lse_out, int64_t num_rows, int head_dim,
                                                              int rows_per_block) {
    const int pieces = head_dim >> 3;
    const int r = small_div((int)threadIdx.x, pieces), e = ((int)threadIdx.x - r * pieces) * 8;
    const int64_t row = (int64_t)blockIdx.x * rows_per_block + r;
    if (r >= rows_per_block || row >= num_rows) return;
    const uint16_t* src = parts + row * head_dim + e;
    const float* lse_src = lse_parts + row;
    float m = -INFINITY, sum = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    for (int p0 = 0; p0 < num_parts; p0 += kMergeGroup) {
        float l[kMergeGroup];
        uint4 w[kMergeGroup];
#pragma unroll
        for (int g = 0; g < kMergeGroup; ++g) {
            const int p = min(p0 + g, num_parts - 1);
            l[g] = lse_src[p * lse_part_stride];
            w[g] = *reinterpret_cast<const uint4*>(src + p * part_stride);
            if (p0 + g >= num_parts) l[g] = -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int g = 0; g < kMergeGroup; ++g) top = fmaxf(top, l[g] * kLog2e);
        if (top > m) {  // (false as well where nothing has been seen so far)
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
            sum *= alpha;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] *= alpha;
            m = top;
        }
#pragma unroll
        for (int g = 0; g < kMergeGroup; ++g) {
            if (l[g] == -INFINITY) continue;
            const float weight = __builtin_amdgcn_exp2f(__builtin_fmaf(l[g], kLog2e, -m));
            sum += weight;
            const uint32_t x[4] = {w[g].x, w[g].y, w[g].z, w[g].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                acc[2 * k] = __builtin_fmaf(weight, T::to_f32((uint16_t)x[k]), acc[2 * k]);
                acc[2 * k + 1] = __builtin_fmaf(weight, T::to_f32((uint16_t)(x[k] >> 16)), acc[2 * k + 1]);
            }
        }
    }
    const float inv = m == -INFINITY && sum == 0.f ? 0.f : 1.0f / sum;
    uint4 w;
    uint32_t* x = &w.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (uint32_t)T::from_f32(acc[2 * k] * inv) | (uint32_t)T::from_f32(acc[2 * k + 1] * inv) << 16;
    *reinterpret_cast<uint4*>(out + row * head_dim + e) = w;
    if (lse_out != nullptr && e == 0) lse_out[row] = (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

template <typename T>
static int attention_merge_entry(const warp34_exec* ex, const void* parts, const float* lse_parts, int num_parts, int64_t part_stride,
                                 int64_t lse_part_stride, void* out, float* lse_out, int64_t num_rows, int head_dim) {
    if (!ex || !parts || !lse_parts || !out || num_parts <= 0 || head_dim <= 0) return (int)hipErrorInvalidValue;
    if (num_rows <= 0) return 0;
    if ((head_dim & 7) != 0 || head_dim > 2048 || ((((uintptr_t)parts) | ((uintptr_t)out)) & 15u) != 0 || (part_stride & 7) != 0)
        return (int)hipErrorNotSupported;
    const int rows_per_block = 256 / (head_dim >> 3);
    if (num_rows > (int64_t)0x7FFFFFFF * rows_per_block || !grid_fits((num_rows + rows_per_block - 1) / rows_per_block, 256)) return (int)hipErrorInvalidValue;
    if (num_parts > 1 && (part_stride < num_rows * head_dim || lse_part_stride < num_rows)) return (int)hipErrorInvalidValue;
    const int64_t blocks = (num_rows + rows_per_block - 1) / rows_per_block;
    hipLaunchKernelGGL((attention_merge_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)ex->stream, (const uint16_t*)parts, lse_parts,
                       num_parts, part_stride, lse_part_stride, (uint16_t*)out, lse_out, num_rows, head_dim, rows_per_block);
    return (int)hipGetLastError();
}

}  // namespace w34

using namespace w34;

extern "C" int warp34_attention_merge_f16(const warp34_exec* ex, const void* parts, const float* lse_parts, int num_parts, int64_t part_stride,
                                          int64_t lse_part_stride, void* out, float* lse_out, int64_t num_rows, int head_dim) {
    return attention_merge_entry<F16>(ex, parts, lse_parts, num_parts, part_stride, lse_part_stride, out, lse_out, num_rows, head_dim);
}
extern "C" int warp34_attention_merge_bf16(const warp34_exec* ex, const void* parts, const float* lse_parts, int num_parts, int64_t part_stride,
                                           int64_t lse_part_stride, void* out, float* lse_out, int64_t num_rows, int head_dim) {
    return attention_merge_entry<BF16>(ex, parts, lse_parts, num_parts, part_stride, lse_part_stride, out, lse_out, num_rows, head_dim);
}
