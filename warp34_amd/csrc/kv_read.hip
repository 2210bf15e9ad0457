// Reading a paged cache back: the K and V rows of given slots, decoded to 16-bit rows, the other half of the append (kv_write.hip).
//
//   plain rows    x[e] = code(e) * d(block of e)                      (16-bit rows: the element itself)
//   rotated rows  x[e] = sign(e) / 16 * sum_f (-1)^popcount(e & f) code(f) d(block of f)
//
// computed in 32 bits and rounded once.  A row's bytes are read once and 2 x head_dim bytes written once.  Rotated rows are bound by vector
// issue and HBM together: 32 768 TQ4 rows of two kv heads, K and V, into BF16 in 18 to 19 us (84.5 MB, 4.5 to 4.7 TB/s; 62 vector instructions a row;
// at 91 of them 22 us, with rows apart and a branch each 24); 333 Q8_0 rows 3.7 us, a launch.  Rows stored as they are: 60 000 of four kv heads, K and V, BF16
// 92 us (5.4 TB/s, as a large copy), Q8_0 97 (3.9), FP8 88 (4.2).
#include "attn_lanes.h"
#include "attn_launch.h"
#include "kv_encode.h"
#include "wht_products.h"

namespace w34 {

// One slab (K or V) and where its rows go; base 0: not wanted.
struct ReadSide {
    uint64_t base, page_stride, head_stride, token_stride;
    uint16_t* out;
    int64_t row_stride;  // elements
    int format;
};
struct ReadParams {
    ReadSide side[2];
    const int32_t* slots;
    int rows, head_dim, block_size;
    uint32_t block_magic;
};

__device__ __forceinline__ int slot_page(int slot, const ReadParams& P) {
    int page = (int)__umulhi((uint32_t)slot, P.block_magic);  // the quotient or one less
    return page + ((slot - page * P.block_size >= P.block_size) ? 1 : 0);
}
__device__ __forceinline__ const slab_byte* row_address(const ReadSide& S, const ReadParams& P, int slot, int head) {
    const int page = slot_page(slot, P);
    return slab_at(S.base) + (uint64_t)(uint32_t)page * S.page_stride + (uint64_t)(uint32_t)head * S.head_stride +
           (uint64_t)(uint32_t)(slot - page * P.block_size) * S.token_stride;
}
// Lane l of a wave holds centroid l % 16; a code's low four bits pick one from the wave, all of whose lanes take part.
__device__ __forceinline__ float lane_centroid() {
    const int n = lane_id() & 15;
    float c = kCentroids[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) c = n == i ? kCentroids[i] : c;
    return c;
}
__device__ __forceinline__ float centroid_of(float mine, uint32_t code) {
    return __int_as_float(__builtin_amdgcn_ds_bpermute((int)(code & 15u) << 2, __float_as_int(mine)));
}
template <typename TOut>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    return (uint32_t)TOut::from_f32(a) | (uint32_t)TOut::from_f32(b) << 16;
}

// Rows stored as they are: a thread takes eight elements of one row, head_dim / 8 threads a row.  blockIdx.y: the kv head,
// blockIdx.z: K or V.  (No thread leaves before the end: the table of the centroids is spread over the lanes of a wave.)
template <typename TOut>
__global__ __launch_bounds__(256) void kv_read_plain_kernel(const ReadParams P, int first_side, int rows_per_block) {
    const ReadSide& S = P.side[first_side + (int)blockIdx.z];
    const int head = (int)blockIdx.y;
    const int pieces = P.head_dim >> 3;
    const int r = small_div((int)threadIdx.x, pieces), e = ((int)threadIdx.x - r * pieces) * 8;
    const int64_t row = (int64_t)blockIdx.x * rows_per_block + r;
    const int slot = r < rows_per_block && row < P.rows ? P.slots[row] : -1;
    const bool live = slot >= 0;  // else: row untouched
    const slab_byte* src = row_address(S, P, live ? slot : 0, head);
    uint4 w = {0u, 0u, 0u, 0u};
    if (S.format == WARP34_KV_FORMAT_FP16 || S.format == WARP34_KV_FORMAT_BF16) {
        if (live) w = __builtin_bit_cast(uint4, load_as<u4>(src + 2 * e));
        if (S.format != TOut::kStorageFormat) {
            uint32_t* x = &w.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint16_t lo = (uint16_t)x[k], hi = (uint16_t)(x[k] >> 16);
                x[k] = S.format == WARP34_KV_FORMAT_FP16 ? pack_out<TOut>(F16::to_f32(lo), F16::to_f32(hi))
                                                         : pack_out<TOut>(BF16::to_f32(lo), BF16::to_f32(hi));
            }
        }
    } else {
        float v[8], d = 0.f;
        if (S.format == WARP34_KV_FORMAT_TQ4) {  // blocks of 66 bytes: fp16 scale, 128 codes of four bits
            uint32_t word = 0u;
            if (live) {
                const slab_byte* block = src + 66 * (e >> 7);
                const slab_byte* codes = block + 2 + ((e & 127) >> 1);
                word = (uint32_t)load_as<uint16_t>(codes) | (uint32_t)load_as<uint16_t>(codes + 2) << 16;
                d = F16::to_f32(load_as<uint16_t>(block));
            }
            const float mine = lane_centroid();
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = centroid_of(mine, word >> (4 * k));
        } else {
            uint32_t codes[2] = {0u, 0u};
            const bool fp8 = S.format == WARP34_KV_FORMAT_FP8_E4M3;
            if (live) {  // Q8_0: blocks of 68 bytes
                const slab_byte* block = fp8 ? src : src + 68 * (e >> 6);
                const slab_byte* at = fp8 ? src + e : block + 4 + (e & 63);
                codes[0] = load_as<uint32_t>(at), codes[1] = load_as<uint32_t>(at + 4);
                d = load_as<float>(fp8 ? src + 256 + 4 * (e >> 7) : block);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t c = codes[k];
                if (fp8) {
                    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
                    v[4 * k] = a[0], v[4 * k + 1] = a[1], v[4 * k + 2] = b[0], v[4 * k + 3] = b[1];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * k + i] = (float)(int8_t)(c >> (8 * i));
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= d;
        w = uint4{pack_out<TOut>(v[0], v[1]), pack_out<TOut>(v[2], v[3]), pack_out<TOut>(v[4], v[5]), pack_out<TOut>(v[6], v[7])};
    }
    if (live) *reinterpret_cast<uint4*>(S.out + row * S.row_stride + (int64_t)head * P.head_dim + e) = w;
}

// Rotated rows of 256 elements, kReadRows rows a wave, by the two products of wht_products.h.
// Memory wants wider pieces than four elements a lane: of four rows at a time lane (n, b) loads X[n] of row b, and the pieces change
// places by swaps of 16 and of 32 lanes; two rows' results change places so that a lane stores eight elements in a run.  (For that the
// columns of Z are out of order, in groups of four: 0, 8, 4, 12.)
// X is the bare codes, of which eight bits are one part and centroids have two in a table; the scales
// multiply Z, whose rows 4 b .. 4 b + 3 lie in one block: relative to a power of two above the row's largest scale, so that the parts
// stay inside fp16's range whatever the scales.
// us at 4 / 8 / 16 rows a wave: 200 TQ4 rows 3.3 / 3.9 / 5.7, 2 000 3.7 / 4.4 / 6.1, 32 768 18.7 / 18.7 / 19.0.
constexpr int kReadRows = 4;
typedef u2v u2_at2 __attribute__((aligned(2)));
typedef u4 u4_at4 __attribute__((aligned(4)));

// Both parts of each centroid times kLutGain.
struct CentroidParts {
    uint32_t of[16];
};
constexpr CentroidParts make_centroid_parts() {
    CentroidParts t{};
    for (int c = 0; c < 16; ++c) {
        const _Float16 hi = (_Float16)(kLutGain * kCentroids[c]);
        t.of[c] = (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(kLutGain * kCentroids[c] - (float)hi)) << 16;
    }
    return t;
}
__device__ __constant__ constexpr CentroidParts kCentroidParts = make_centroid_parts();
template <typename TOut>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (TOut::kStorageFormat == WARP34_KV_FORMAT_BF16) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf2));
    } else {
        return pack_h2(a, b);
    }
}

// (two waves a SIMD at least: with the whole register file the products' results would go through the accumulation registers)
template <typename TOut, int FORMAT>
__global__ __launch_bounds__(256, 2) void kv_read_rotated_kernel(const ReadParams P, int first_side) {
    const ReadSide& S = P.side[first_side + (int)blockIdx.z];
    const int head = (int)blockIdx.y;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n = lane & 15, b = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * kReadRows;

    constexpr int kGroups = kReadRows / 4;
    constexpr bool kTq4 = FORMAT == WARP34_KV_FORMAT_TQ4;
    uint32_t code[kGroups][4], scale[kGroups];  // X[n] of row b, the scale of block n % 2 or n % 4 of it
    unsigned long long live[kGroups];
    const uint32_t mine = kTq4 ? kCentroidParts.of[n] : 0u;
    const int to_e = 16 * n + 8 * (b & 1);  // the elements this lane stores, of row b >> 1 of two
    const uint32_t signs = kSignMask[to_e >> 5] >> (to_e & 31);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int64_t row = row0 + 4 * g + b;
        const int slot = row < P.rows ? P.slots[row] : -1;
        live[g] = __ballot(slot >= 0);
        scale[g] = 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) code[g][k] = 0u;
        if (slot >= 0) {
            const slab_byte* src = row_address(S, P, slot, head);
            if constexpr (kTq4) {
                const u2v w = load_as<u2_at2>(src + 66 * (n >> 3) + 2 + 8 * (n & 7));
                code[g][0] = w[0], code[g][1] = w[1];
                scale[g] = load_as<uint16_t>(src + 66 * (n & 1));
            } else {
                const bool fp8 = FORMAT == WARP34_KV_FORMAT_FP8_E4M3;
                const u4 w = load_as<u4_at4>(src + (fp8 ? 16 * n : 68 * (n >> 2) + 4 + 16 * (n & 3)));
#pragma unroll
                for (int k = 0; k < 4; ++k) code[g][k] = w[k];
                scale[g] = load_as<uint32_t>(src + (fp8 ? 256 + 4 * (n & 1) : 68 * (n & 3)));
            }
        }
    }
    const h8 had = hadamard_column(n, b);
    const h8 had_cols = hadamard_column((n & 3) + ((n & 4) << 1) + ((n & 8) >> 1), b);  // of the column of Z where lane n is
    u4 flip;  // the signs, as bits of the row's 16-bit numbers
#pragma unroll
    for (int k = 0; k < 4; ++k) flip[k] = (signs << (15 - 2 * k) & 0x8000u) | (signs << (30 - 2 * k) & 0x80000000u);
    const int scale_from = 4 * (FORMAT == WARP34_KV_FORMAT_Q8_0 ? b : b >> 1);  // the lane (times four) that has the scale of Z's rows 4 b .. 4 b + 3
    uint16_t* to = S.out + (row0 + (b >> 1)) * S.row_stride + (int64_t)head * 256 + to_e;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        // four rows: row k's piece b in this lane
        uint32_t piece[4];
        if constexpr (kTq4) {
            const auto p = __builtin_amdgcn_permlane32_swap(code[g][0], code[g][1], false, false);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const auto q = __builtin_amdgcn_permlane16_swap(p[k], p[k], false, false);
                piece[2 * k] = q[0] >> (16 * (b & 1)), piece[2 * k + 1] = q[1] >> (16 * (b & 1));
            }
        } else {
            const auto p = __builtin_amdgcn_permlane32_swap(code[g][0], code[g][2], false, false);
            const auto q = __builtin_amdgcn_permlane32_swap(code[g][1], code[g][3], false, false);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const auto r = __builtin_amdgcn_permlane16_swap(p[k], q[k], false, false);
                piece[2 * k] = r[0], piece[2 * k + 1] = r[1];
            }
        }
        // the scales of row b relative to a power of two above the largest
        const float d = kTq4 ? F16::to_f32((uint16_t)scale[g]) * kLutInvGain : __uint_as_float(scale[g]);
        float top = fmaxf(fabsf(d), fabsf(lane_xor<1>(d, lane)));
        if constexpr (FORMAT == WARP34_KV_FORMAT_Q8_0) top = fmaxf(top, lane_xor<2>(top, lane));
        const int above = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
        const float relative = __builtin_amdgcn_ldexpf(d, -above);
        uint2 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // (rows that are not wanted too, as zeros: no branch keeps one row waiting for another)
            const uint32_t c = piece[k];
            const float share = __int_as_float(__builtin_amdgcn_ds_bpermute(64 * k + scale_from, __float_as_int(relative)));
            const int up = __builtin_amdgcn_readlane(above, 16 * k);
            u4 x = {0u, 0u, 0u, 0u};
            if constexpr (kTq4) {
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = (uint32_t)__builtin_amdgcn_ds_bpermute((int)((i == 0 ? c << 2 : c >> (4 * i - 2)) & 60u), (int)mine);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x05040100u);
                    x[2 + i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302u);
                }
            } else if constexpr (FORMAT == WARP34_KV_FORMAT_FP8_E4M3) {
                x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false));
                x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true));
            } else {  // 0x6400 | (q + 128) is 1152 + q in fp16
                const uint32_t u = c ^ 0x80808080u;
                const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
                x[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
                x[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
            }
            const f4 none = {0.f, 0.f, 0.f, 0.f};
            const f4 z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), had_cols, none, 0, 0, 0);
            float zs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                zs[i] = z[i] * share;
                asm("" : "+v"(zs[i]));  // both parts are taken from the product rounded to 32 bits
            }
            const f4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(two_parts(zs), had, none, 0, 0, 0);
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_ldexpf(y[i], up - 4);
            w[k] = uint2{pack_pair<TOut>(v[0], v[1]), pack_pair<TOut>(v[2], v[3])};
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {  // rows k (lanes 0 .. 31) and k + 1
            const auto x = __builtin_amdgcn_permlane32_swap(w[k].x, w[k + 1].x, false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[k].y, w[k + 1].y, false, false);
            if ((live[g] >> (16 * (k + (b >> 1)))) & 1ull) *reinterpret_cast<u4*>(to + (4 * g + k) * S.row_stride) = u4{x[0], y[0], x[1], y[1]} ^ flip;
        }
    }
}

static bool rotated_rows(int format, int transform, int head_dim) {
    return transform == WARP34_KV_TRANSFORM_RADEMACHER_WHT256 && head_dim == 256 && (format == WARP34_KV_FORMAT_TQ4 || is_8bit_format(format));
}

// 16-bit rows are loaded 16 bytes at a time, the parts of the others by what their elements are aligned to
static bool rows_aligned_for_read(int format, uint64_t strides_and_base) {
    const unsigned mask = format == WARP34_KV_FORMAT_TQ4 ? 1u : is_8bit_format(format) ? 3u : 15u;
    return (strides_and_base & mask) == 0;
}

template <typename TOut>
static int kv_read_entry(const warp34_exec* ex, const warp34_kv_layer_layout* l, const int32_t* slots, int num_rows, void* k_out, void* v_out,
                         int k_row_stride, int v_row_stride) {
    if (!ex || !l || (!k_out && !v_out)) return (int)hipErrorInvalidValue;
    if (num_rows <= 0 || l->local_kv_heads <= 0) return 0;
    if (!slots || l->block_size <= 0 || l->head_dim <= 0 || l->head_dim > 256 || l->local_kv_heads > 65535) return (int)hipErrorInvalidValue;
    const int64_t min_stride = (int64_t)l->local_kv_heads * l->head_dim;
    ReadParams P{};
    P.slots = slots;
    P.rows = num_rows;
    P.head_dim = l->head_dim;
    P.block_size = l->block_size;
    P.block_magic = block_magic_for(l->block_size);
    P.side[0] = ReadSide{l->k_base, l->k_page_stride_bytes, l->k_head_stride_bytes, l->k_token_stride_bytes, (uint16_t*)k_out, k_row_stride, l->k_format};
    P.side[1] = ReadSide{l->v_base, l->v_page_stride_bytes, l->v_head_stride_bytes, l->v_token_stride_bytes, (uint16_t*)v_out, v_row_stride, l->v_format};
    const int transforms[2] = {l->k_transform, l->v_transform};
    for (const ReadSide& S : P.side) {
        if (!S.out) continue;
        if (!S.base || S.row_stride < min_stride) return (int)hipErrorInvalidValue;
        if (!format_supported_for_write(S.format, transforms[&S - P.side], l->head_dim) || (l->head_dim & 7) != 0 ||
            !rows_aligned_for_read(S.format, S.base | S.page_stride | S.head_stride | S.token_stride) || (((uintptr_t)S.out) & 15u) != 0 ||
            (S.row_stride & 7) != 0) {
            return (int)hipErrorNotSupported;
        }
    }
    const bool rotated[2] = {rotated_rows(l->k_format, l->k_transform, l->head_dim), rotated_rows(l->v_format, l->v_transform, l->head_dim)};
    const int rows_per_block = 256 / (l->head_dim >> 3);
    const auto blocks = [&](int per_block) { return (unsigned)(((int64_t)num_rows + per_block - 1) / per_block); };
    for (int side = 0; side < 2; ++side)
        if (P.side[side].out && !grid_fits(blocks(rotated[side] ? 4 * kReadRows : rows_per_block), 256)) return (int)hipErrorInvalidValue;
    const unsigned heads = (unsigned)l->local_kv_heads;
    const auto launch = [&](int first, int sides) {
        hipStream_t stream = (hipStream_t)ex->stream;
        if (!rotated[first]) {
            hipLaunchKernelGGL((kv_read_plain_kernel<TOut>), dim3(blocks(rows_per_block), heads, (unsigned)sides), dim3(256), 0, stream, P, first,
                               rows_per_block);
            return;
        }
        const dim3 grid(blocks(4 * kReadRows), heads, (unsigned)sides);
        if (P.side[first].format == WARP34_KV_FORMAT_TQ4) {
            hipLaunchKernelGGL((kv_read_rotated_kernel<TOut, WARP34_KV_FORMAT_TQ4>), grid, dim3(256), 0, stream, P, first);
        } else if (P.side[first].format == WARP34_KV_FORMAT_FP8_E4M3) {
            hipLaunchKernelGGL((kv_read_rotated_kernel<TOut, WARP34_KV_FORMAT_FP8_E4M3>), grid, dim3(256), 0, stream, P, first);
        } else {
            hipLaunchKernelGGL((kv_read_rotated_kernel<TOut, WARP34_KV_FORMAT_Q8_0>), grid, dim3(256), 0, stream, P, first);
        }
    };
    const bool together = k_out && v_out && rotated[0] == rotated[1] && (!rotated[0] || l->k_format == l->v_format);
    if (together) {
        launch(0, 2);
    } else {
        if (k_out) launch(0, 1);
        if (v_out) launch(1, 1);
    }
    return (int)hipGetLastError();
}

}  // namespace w34

using namespace w34;

extern "C" int warp34_kv_cache_read_f16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const int32_t* slot_mapping, int num_rows,
                                        void* k_out, void* v_out, int k_row_stride, int v_row_stride) {
    return kv_read_entry<F16>(ex, layout, slot_mapping, num_rows, k_out, v_out, k_row_stride, v_row_stride);
}
extern "C" int warp34_kv_cache_read_bf16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const int32_t* slot_mapping, int num_rows,
                                         void* k_out, void* v_out, int k_row_stride, int v_row_stride) {
    return kv_read_entry<BF16>(ex, layout, slot_mapping, num_rows, k_out, v_out, k_row_stride, v_row_stride);
}
