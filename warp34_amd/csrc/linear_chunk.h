// Linear attention of prompts: tokens go by in chunks of 64.  With G the running sum of g (log2 domain) inside a chunk,
//
//   O_i = 2^G_i S^T q_i + sum_{j <= i} (q_i . k_j) 2^(G_i - G_j) v_j          S' = 2^G_end S + sum_j k_j (2^(G_end - G_j) v_j)^T
//
// Workgroup = 32 NW columns of a value head, a wave 32 of them with their part of the state in registers; 32x32x16 MFMAs:
//   P^T = K Q^T        one 32x32 tile a wave (three of them: a chunk's second half of keys is not seen by its first half of queries),
//                      weighted, and laid into LDS as the operands of the product below
//   O^T = S^T Q^T      the state's registers are the operand as they stand: lane (n, b) has column n for rows (i & 3) + 8 (i >> 2) + 4 b,
//                      eight of them are 16 channels of which q is read in the same order
//   O^T += V^T P^T     v through transposing reads (ds_read_b64_tr_b16: lane l of 16 gets column l of four rows of 16 values)
//   S += K^T V'        k and v through transposing reads, v weighted in registers
// Weights are exponentials of differences of G, which is summed in 64 bits and held as two 32-bit numbers: where all but the last
// tokens have faded away, the sums are large and the differences small.
// Operands of 16 bits are rounded states, weights and weighted values.  P and S have two parts (16 bits of bf16, 22 of fp16), so that outputs
// show their own rounding only; v' has three for bf16 where the state itself comes out (24 bits), two for fp16.  fp16 has little range:
// v' and S are scaled by powers of two of a wave, P by one of a row, to put the largest at 2^14; what is lost are bits 2^-39 below it.
#pragma once

#include <type_traits>

#include "linear_attention.h"

namespace w34 {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4v lds_s4;

constexpr int kLinearChunk = 64;
constexpr float kLeastDecay = -200.f;  // e^-200 times any fp32 number is zero in 32 bits: smaller ones, minus infinity among them, change nothing

// A prompt cut into parts of `length` tokens, which run at once, and once more behind the tokens that its state keeps.
struct LinearParts {
    float* states;  // [part][value head][k_head_dim * v_head_dim] in the order of the registers: what a part adds, then what it starts from
    float* fades;   // [part][value head] 2^(sum of the part's g)
    int log_length;
    int most;  // parts that there is room for
};

__device__ __forceinline__ int linear_parts_of(int n, int kept, int log_length) {
    const int whole = (n + (1 << log_length) - 1) >> log_length;
    return whole + (kept > 0 && kept < n && (kept & ((1 << log_length) - 1)) != 0 ? 1 : 0);
}
__device__ __forceinline__ void linear_part_range(int n, int kept, int log_length, int part, int& begin, int& end) {
    const int length = 1 << log_length, cut = kept >> log_length;
    const bool extra = kept > 0 && kept < n && (kept & (length - 1)) != 0;
    const int p = extra && part > cut ? part - 1 : part;
    begin = p << log_length, end = min(begin + length, n);
    if (extra && part == cut) end = kept;
    if (extra && part == cut + 1) begin = kept;
}
__device__ __forceinline__ int linear_request_parts(const LinearArgs& a, int req, int log_length) {
    if (req >= a.num_reqs || (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0)) return 0;
    const int lo = max(0, a.query_start_loc[req]), n = max(0, min(a.query_start_loc[req + 1], a.total_tokens) - lo);
    return linear_parts_of(n, a.state_tokens == nullptr ? n : min(max(a.state_tokens[req], 0), n), log_length);
}
// Request and number within it of a part; false behind the last one.  A wave looks at 64 requests at a time.
__device__ __forceinline__ bool linear_find_part(const LinearArgs& a, int log_length, int index, int& req, int& part) {
    const int lane = lane_id();
    for (int base = 0; base < a.num_reqs; base += 64) {
        const int mine = linear_request_parts(a, base + lane, log_length);
        int run = mine;
#pragma unroll
        for (int by = 1; by < 64; by *= 2) {
            const int o = __shfl_up(run, by, 64);
            if (lane >= by) run += o;
        }
        const int total = __shfl(run, 63, 64);
        if (index < total) {
            const int owner = __builtin_ctzll(__ballot(index < run));
            req = __builtin_amdgcn_readfirstlane(base + owner);
            part = __builtin_amdgcn_readfirstlane(index - __shfl(run - mine, owner, 64));
            return true;
        }
        index -= total;
    }
    return false;
}
// Number of the first part of a request.
__device__ __forceinline__ int linear_first_part(const LinearArgs& a, int log_length, int req) {
    int count = 0;
    for (int base = 0; base < req; base += 64) count += base + lane_id() < req ? linear_request_parts(a, base + lane_id(), log_length) : 0;
#pragma unroll
    for (int by = 32; by; by /= 2) count += __shfl_xor(count, by, 64);
    return __builtin_amdgcn_readfirstlane(count);
}

template <typename T>
__device__ __forceinline__ f16v linear_mfma(u4 a, u4 b, f16v c) {
    if constexpr (T::kStorageFormat == WARP34_KV_FORMAT_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}
// Two numbers as PARTS pairs of 16 bits whose sums they are.
template <typename T, int PARTS>
__device__ __forceinline__ void linear_split(float x, float y, uint32_t (&w)[PARTS]) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if constexpr (T::kStorageFormat == WARP34_KV_FORMAT_BF16) {
            w[p] = (uint32_t)T::from_f32(x) | (uint32_t)T::from_f32(y) << 16;
            x -= __uint_as_float(w[p] << 16);
            y -= __uint_as_float(w[p] & 0xFFFF0000u);
        } else {
            w[p] = pack_h2(x, y);
            x -= half_lo_to_f32(w[p]);
            y -= half_hi_to_f32(w[p]);
        }
    }
}
// The e for which 2^e puts `top` at 2^14, at most 100: 2^e and 2^-e are numbers.  0 for zero, and for what is not finite.
__device__ __forceinline__ int scale_exponent(float top) {
    const int e = (int)(__float_as_uint(top) >> 23 & 255u);
    return e == 0 || e == 255 ? 0 : min(141 - e, 100);
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int by = 32; by; by /= 2) x = fmaxf(x, __shfl_xor(x, by, 64));
    return x;
}

// Where 16 bytes of a row are: operand reads of 16 rows and the four rows of a transposing read touch all banks.
template <int PIECES>
__device__ __forceinline__ uint32_t linear_piece(int row, int piece) {
    static_assert(PIECES == 8 || PIECES == 16, "rows of 128 or 256 bytes");
    const int x = PIECES == 16 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
    return (uint32_t)(row * PIECES * 16 + (piece ^ x) * 16);
}

enum { kLinearWalk, kLinearSums, kLinearRows };  // a whole request; what a part adds to the state; a part's rows

template <int DK, int NW>
struct LinearLds {
    static constexpr int kQ = 0, kK = kLinearChunk * DK * 2, kV = 2 * kK, kP = kV + kLinearChunk * NW * 64;
    static constexpr int kG = kP + 3 * 4096;       // [64] G as two numbers
    static constexpr int kW = kG + 64 * 8;         // [64] 2^(G_end - G_j)
    static constexpr int kFade = kW + 64 * 4;      // 2^G_end
    static constexpr int kRow = kFade + 16;        // [3][32] what P's rows are to be multiplied by (fp16)
    static constexpr int kBytes = kRow + 3 * 32 * 4;
};

template <typename T, int DK, int NW, int MODE>
__global__ __launch_bounds__(64 * NW, 2) void linear_chunk_kernel(const LinearArgs a, const LinearParts p) {
    typedef LinearLds<DK, NW> L;
    constexpr bool kBf16 = T::kStorageFormat == WARP34_KV_FORMAT_BF16;
    constexpr int kThreads = 64 * NW, KP = DK / 8, VP = 4 * NW, KT = DK / 32;  // pieces of 16 bytes a row, tiles of 32 channels
    constexpr int kLoads = kLinearChunk * KP / kThreads;
    constexpr int kParts = !kBf16 ? 2 : MODE == kLinearRows ? 2 : 3;  // of weighted values
    __shared__ __attribute__((aligned(16))) uint8_t smem[L::kBytes];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n32 = lane & 31, b = lane >> 5;
    const int slices = a.v_dim / (32 * NW), columns = a.v_heads * slices;
    int at = (int)(blockIdx.x % (uint32_t)columns), group = (int)(blockIdx.x / (uint32_t)columns);
    // workgroups go round the eight dies: value heads of the same keys on the same one
    if (a.v_heads % 8 == 0) at = (at % 8) * (columns / 8) + at / 8;
    const int head = at / slices, slice = at - head * slices, kh = head / a.group;
    int req = group, part = 0;
    if (MODE == kLinearWalk) {
        if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    } else {
        if (!linear_find_part(a, p.log_length, group, req, part)) return;
    }
    const LinearRequest r = linear_request(a, req, head, DK * a.v_dim);
    const int col0 = slice * 32 * NW, my_col = col0 + 32 * wave + n32;

    int begin = 0, stop = r.n;
    if (MODE != kLinearWalk) linear_part_range(r.n, r.kept, p.log_length, part, begin, stop);
    else if (a.out == nullptr) stop = r.kept;

    f16v s[KT];
#pragma unroll
    for (int d = 0; d < KT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[d][i] = 0.f;
    int unit = 0;  // s holds the state times 2^unit (fp16)
    // this wave's share of a part's state in scratch
    float* const mine = MODE == kLinearWalk ? nullptr
                                            : p.states + ((int64_t)group * a.v_heads + head) * (DK * a.v_dim) + (int64_t)(slice * NW + wave) * (32 * DK) + lane * 4;
    if (MODE == kLinearWalk && r.in != nullptr) {
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[d][i] = r.in[(32 * d + (i & 3) + 8 * (i >> 2) + 4 * b) * a.v_dim + my_col];
    }
    if (MODE == kLinearRows) {
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int ig = 0; ig < 4; ++ig) {
                const f4 x = *reinterpret_cast<const f4*>(mine + (d * 4 + ig) * 256);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[d][4 * ig + i] = x[i];
            }
    }
    const auto put_state = [&]() {
        const float by = power_of_two(-unit);
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.out[(32 * d + (i & 3) + 8 * (i >> 2) + 4 * b) * a.v_dim + my_col] = kBf16 ? s[d][i] : s[d][i] * by;
    };
    if (MODE == kLinearWalk && r.kept == 0 && r.out != nullptr) put_state();

    // a chunk on its way: rows behind its last token are zeros, whatever is there
    const bool with_q = MODE != kLinearSums && a.out != nullptr;
    uint4 qx[kLoads], kx[kLoads], vx[4];
    float gx = 0.f;
    int chunk_end = begin;
    const auto chunk_stop = [&](int t) { return min(t + kLinearChunk, MODE == kLinearWalk && t < r.kept ? r.kept : stop); };
    const auto fetch = [&](int t, int end) {
        const int last = end - 1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int x = tid + i * kThreads, row = x / KP, piece = x % KP;
            const int64_t tok = r.lo + min(t + row, last);
            kx[i] = *reinterpret_cast<const uint4*>(a.k + tok * a.k_stride + kh * DK + piece * 8);
            if (with_q) qx[i] = *reinterpret_cast<const uint4*>(a.q + tok * a.q_stride + kh * DK + piece * 8);
            if (t + row > last) kx[i] = qx[i] = uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = tid + i * kThreads, row = x / VP, piece = x % VP;
            const int64_t tok = r.lo + min(t + row, last);
            vx[i] = *reinterpret_cast<const uint4*>(a.v + tok * a.v_stride + head * a.v_dim + col0 + piece * 8);
            if (t + row > last) vx[i] = uint4{0, 0, 0, 0};
        }
        gx = 0.f;
        if (a.g != nullptr && wave == NW - 1 && t + lane <= last) gx = a.g[(int64_t)(r.lo + t + lane) * a.g_stride + head];
    };
    const auto at_lds = [&](uint32_t offset) { return smem + offset; };
    const auto put = [&]() {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int x = tid + i * kThreads;
            *reinterpret_cast<uint4*>(at_lds(L::kK + linear_piece<KP>(x / KP, x % KP))) = kx[i];
            if (with_q) *reinterpret_cast<uint4*>(at_lds(L::kQ + linear_piece<KP>(x / KP, x % KP))) = qx[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = tid + i * kThreads;
            *reinterpret_cast<uint4*>(at_lds(L::kV + linear_piece<VP>(x / VP, x % VP))) = vx[i];
        }
        if (wave == NW - 1) {
            double run = (double)(gx < kLeastDecay ? kLeastDecay : gx) * 1.4426950408889634;
#pragma unroll
            for (int by = 1; by < 64; by *= 2) {
                const double o = __shfl_up(run, by, 64);
                if (lane >= by) run += o;
            }
            const double all = __shfl(run, 63, 64);
            const float hi = (float)run;
            *reinterpret_cast<float2*>(at_lds(L::kG + lane * 8)) = make_float2(hi, (float)(run - hi));
            *reinterpret_cast<float*>(at_lds(L::kW + lane * 4)) = __builtin_amdgcn_exp2f((float)(all - run));
            if (lane == 0) *reinterpret_cast<float2*>(at_lds(L::kFade)) = make_float2(__builtin_amdgcn_exp2f((float)all), (float)all);
        }
    };
    const auto operand = [&](uint32_t offset) { return *reinterpret_cast<const u4*>(at_lds(offset)); };
    // rows 16 step + 4 b + 0 .. 3 and the same + 8, columns 8 first_piece + n32
    const auto transposed = [&](uint32_t base, auto pieces, int first_piece, int step) -> u4 {
        constexpr int PIECES = decltype(pieces)::value;
        const int j = lane & 15, row = 16 * step + 4 * b + (j >> 2), piece = first_piece + 2 * (lane >> 4 & 1) + (j >> 1 & 1);
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem + base + 8u * (uint32_t)(j & 1);
        const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)(lds + linear_piece<PIECES>(row, piece))));
        const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)(lds + linear_piece<PIECES>(row + 8, piece))));
        const u2v u = __builtin_bit_cast(u2v, x), w = __builtin_bit_cast(u2v, y);
        return u4{u[0], u[1], w[0], w[1]};
    };

    // Tile 0: queries 0 .. 31 over keys 0 .. 31, 1: queries 32 .. 63 over keys 0 .. 31, 2: over keys 32 .. 63.
    const auto weights = [&](int tile) {
        const int kt = tile == 2 ? 1 : 0, qt = tile == 0 ? 0 : 1;
        f16v x;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
        for (int step = 0; step < DK / 16; ++step)
            x = linear_mfma<T>(operand(L::kK + linear_piece<KP>(32 * kt + n32, 2 * step + b)), operand(L::kQ + linear_piece<KP>(32 * qt + n32, 2 * step + b)), x);
        const float2 gi = *reinterpret_cast<const float2*>(at_lds(L::kG + (32 * qt + n32) * 8));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = (i & 3) + 8 * (i >> 2) + 4 * b;
            const float2 gj = *reinterpret_cast<const float2*>(at_lds(L::kG + (32 * kt + key) * 8));
            const float w = x[i] * __builtin_amdgcn_exp2f((gi.x - gj.x) + (gi.y - gj.y));
            x[i] = tile == 1 || key <= n32 ? w : 0.f;
        }
        if constexpr (!kBf16) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
            const int e = scale_exponent(top);
            const float by = power_of_two(e);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= by;
            if (b == 0) *reinterpret_cast<float*>(at_lds(L::kRow + (tile * 32 + n32) * 4)) = power_of_two(-e);
        }
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            u4 hi, lo;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t w[2];
                linear_split<T, 2>(x[8 * step + 2 * k], x[8 * step + 2 * k + 1], w);
                hi[k] = w[0], lo[k] = w[1];
            }
            *reinterpret_cast<u4*>(at_lds(L::kP + tile * 4096 + step * 1024 + lane * 16)) = hi;
            *reinterpret_cast<u4*>(at_lds(L::kP + tile * 4096 + 2048 + step * 1024 + lane * 16)) = lo;
        }
    };

    float part_sum = 0.f;  // of g, for the scan over parts
    if (begin < stop) fetch(begin, chunk_end = chunk_stop(begin));
    for (int t = begin; t < stop;) {
        const int end = chunk_end, length = end - t;
        __syncthreads();
        put();
        __syncthreads();
        if (end < stop) fetch(end, chunk_end = chunk_stop(end));
        const bool two = length > 32;
        f16v o[2];
        if (with_q) {
            if (NW == 4) {
                if (wave == 0 || (wave < 3 && two)) weights(wave);
            } else if (wave == 0) {
                weights(0);
                if (two) weights(1);
            } else if (two) {
                weights(2);
            }
            // the state's part of the rows
            int e = 0;
            if constexpr (!kBf16) {
                float top = 0.f;
#pragma unroll
                for (int d = 0; d < KT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[d][i]));
                e = scale_exponent(wave_max(top));
            }
            const float by = power_of_two(e);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[q][i] = 0.f;
#pragma unroll
            for (int step = 0; step < DK / 16; ++step) {
                u4 part_of[2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = 8 * (step & 1) + 2 * k;
                    uint32_t w[2];
                    float x = s[step >> 1][i], y = s[step >> 1][i + 1];
                    if (!kBf16) x *= by, y *= by;
                    linear_split<T, 2>(x, y, w);
                    part_of[0][k] = w[0], part_of[1][k] = w[1];
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (q == 1 && !two) continue;
                    const u2v x = *reinterpret_cast<const u2v*>(at_lds(L::kQ + linear_piece<KP>(32 * q + n32, 2 * step) + 8 * b));
                    const u2v y = *reinterpret_cast<const u2v*>(at_lds(L::kQ + linear_piece<KP>(32 * q + n32, 2 * step + 1) + 8 * b));
                    const u4 qo = {x[0], x[1], y[0], y[1]};
                    o[q] = linear_mfma<T>(part_of[0], qo, o[q]);
                    o[q] = linear_mfma<T>(part_of[1], qo, o[q]);
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float2 gi = *reinterpret_cast<const float2*>(at_lds(L::kG + (32 * q + n32) * 8));
                const float f = __builtin_amdgcn_exp2f(gi.x + gi.y) * (kBf16 ? 1.f : power_of_two(-e - unit));
#pragma unroll
                for (int i = 0; i < 16; ++i) o[q][i] *= f;
            }
        }
        u4 v[4];
#pragma unroll
        for (int step = 0; step < 4; ++step) v[step] = transposed(L::kV, std::integral_constant<int, VP>{}, 4 * wave, step);
        if (with_q) {
            __syncthreads();
#pragma unroll
            for (int tile = 0; tile < 3; ++tile) {
                if (tile > 0 && !two) continue;
                const int kt = tile == 2 ? 1 : 0, qt = tile == 0 ? 0 : 1;
                if constexpr (kBf16) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[qt] = linear_mfma<T>(v[2 * kt + (x & 1)], operand(L::kP + tile * 4096 + x * 1024 + lane * 16), o[qt]);
                } else {
                    f16v sum;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum = linear_mfma<T>(v[2 * kt + (x & 1)], operand(L::kP + tile * 4096 + x * 1024 + lane * 16), sum);
                    const float f = *reinterpret_cast<const float*>(at_lds(L::kRow + (tile * 32 + n32) * 4));
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[qt][i] = __builtin_fmaf(sum[i], f, o[qt][i]);
                }
            }
            // lanes n32 and n32 + 32 have one row's columns in turns of four: exchanged, each has eight in a row
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = t + 32 * q + n32;
                uint16_t* to = a.out + (int64_t)(r.lo + row) * a.out_stride + head * a.v_dim + col0 + 32 * wave + 8 * b;
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = (uint32_t)T::from_f32(o[q][2 * k] * a.scale) | (uint32_t)T::from_f32(o[q][2 * k + 1] * a.scale) << 16;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const auto x = __builtin_amdgcn_permlane32_swap(w[4 * k], w[4 * k + 2], false, false);
                    const auto y = __builtin_amdgcn_permlane32_swap(w[4 * k + 1], w[4 * k + 3], false, false);
                    if (row < end) *reinterpret_cast<u4*>(to + 16 * k) = u4{x[0], y[0], x[1], y[1]};
                }
            }
        }
        // the state moves on
        const float2 fade = *reinterpret_cast<const float2*>(at_lds(L::kFade));
        if (MODE == kLinearSums) part_sum += fade.y;
        if (MODE != kLinearRows || end < stop) {
            int next = unit;
            if constexpr (!kBf16) {
                uint32_t top = 0;
#pragma unroll
                for (int step = 0; step < 4; ++step)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = max_u16x2(top, v[step][k] & 0x7FFF7FFFu);
                const float largest = wave_max(fmaxf(half_lo_to_f32(top), half_hi_to_f32(top)));
                if (largest > 0.f && largest < INFINITY) next = scale_exponent(largest);
            }
            const float by = kBf16 ? fade.x : fade.x * power_of_two(next - unit), values = power_of_two(next);
            unit = next;
#pragma unroll
            for (int d = 0; d < KT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[d][i] *= by;
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                if (16 * step >= length) continue;
                u4 x[kParts];
                const f4 w0 = *reinterpret_cast<const f4*>(at_lds(L::kW + (16 * step + 4 * b) * 4)), w1 = *reinterpret_cast<const f4*>(at_lds(L::kW + (16 * step + 8 + 4 * b) * 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f4 w = k < 2 ? w0 : w1;
                    float y = T::to_f32((uint16_t)v[step][k]) * w[2 * (k & 1)], z = T::to_f32((uint16_t)(v[step][k] >> 16)) * w[2 * (k & 1) + 1];
                    if (!kBf16) y *= values, z *= values;
                    uint32_t parts[kParts];
                    linear_split<T, kParts>(y, z, parts);
#pragma unroll
                    for (int q = 0; q < kParts; ++q) x[q][k] = parts[q];
                }
#pragma unroll
                for (int d = 0; d < KT; ++d) {
                    const u4 k = transposed(L::kK, std::integral_constant<int, KP>{}, 4 * d, step);
#pragma unroll
                    for (int q = 0; q < kParts; ++q) s[d] = linear_mfma<T>(k, x[q], s[d]);
                }
            }
        }
        t = end;
        if (MODE == kLinearWalk && t == r.kept && r.out != nullptr) put_state();
    }
    if (MODE == kLinearSums) {
        const float by = power_of_two(-unit);
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int ig = 0; ig < 4; ++ig) {
                f4 x;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = kBf16 ? s[d][4 * ig + i] : s[d][4 * ig + i] * by;
                *reinterpret_cast<f4*>(mine + (d * 4 + ig) * 256) = x;
            }
        if (tid == 0 && slice == 0) p.fades[(int64_t)group * a.v_heads + head] = __builtin_amdgcn_exp2f(part_sum);
    }
}

// The states that the parts start from, and the one that is kept: S = fade_p S + U_p over a request's parts.  A thread has four elements of a
// head's state, in the order of the registers of the kernel above.
__global__ __launch_bounds__(256) void linear_scan_kernel(const LinearArgs a, const LinearParts p, int k_dim) {
    const int size = k_dim * a.v_dim, blocks = size / 1024;
    const int block = (int)(blockIdx.x % (uint32_t)blocks), at = (int)(blockIdx.x / (uint32_t)blocks);
    const int head = at % a.v_heads, req = at / a.v_heads;
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const LinearRequest r = linear_request(a, req, head, size);
    const int first = linear_first_part(a, p.log_length, req), parts = linear_parts_of(r.n, r.kept, p.log_length);
    const int x = block * 256 + (int)threadIdx.x;  // [32 columns][32 channels][4 x 8 channels][lane]
    const int lane = x & 63, ig = x >> 6 & 3, tiles = k_dim / 32, d = (x >> 8) % tiles, w = (x >> 8) / tiles;
    const int row = 32 * d + 8 * ig + 4 * (lane >> 5), col = 32 * w + (lane & 31);
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (r.in != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = r.in[(row + i) * a.v_dim + col];
    }
    const auto keep = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.out[(row + i) * a.v_dim + col] = s[i];
    };
    if (r.kept == 0 && r.out != nullptr) keep();
    float* slot = p.states + ((int64_t)first * a.v_heads + head) * size + (int64_t)x * 4;
    for (int part = 0; part < parts && first + part < p.most; ++part, slot += (int64_t)a.v_heads * size) {
        const f4 u = *reinterpret_cast<const f4*>(slot);
        const float fade = p.fades[(int64_t)(first + part) * a.v_heads + head];
        *reinterpret_cast<f4*>(slot) = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(fade, s[i], u[i]);
        int begin, end;
        linear_part_range(r.n, r.kept, p.log_length, part, begin, end);
        if (end == r.kept && r.out != nullptr) keep();
    }
}

}  // namespace w34
