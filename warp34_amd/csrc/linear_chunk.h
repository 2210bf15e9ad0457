// Linear attention of prompts: tokens go by in chunks of 64.  With G the running sum of g (log2 domain) inside a chunk,
//
//   O_i = 2^G_i S^T q_i + sum_{j <= i} (q_i . k_j) 2^(G_i - G_j) v_j          S' = 2^G_end S + sum_j k_j (2^(G_end - G_j) v_j)^T
//
// Workgroup = the columns of a value head, a wave 32 of them with their part of the state in registers; 32x32x16 MFMAs:
//   P^T = K Q^T        one 32x32 tile a wave (three of them: a chunk's second half of keys is not seen by its first half of queries),
//                      weighted, and laid into LDS as the operands of the product below
//   O^T = S^T Q^T      the state's registers are the operand as they stand: lane (n, b) has column n for channels 16 (i >> 3) + 8 b + (i & 7)
//   O^T += V^T P^T     v through transposing reads (ds_read_b64_tr_b16: lane l of 16 gets column l of four rows of 16 values)
//   S += K^T V'        k and v through transposing reads, v weighted in registers
// Weights are exponentials of differences of G, which is summed in 64 bits and held as two 32-bit numbers: where all but the last
// tokens have faded away, the sums are large and the differences small.
// Operands of 16 bits are rounded states, weights and weighted values.  P and S have two parts (16 bits of bf16, 22 of fp16), so that outputs
// show their own rounding only; v' has three for bf16 where the state itself comes out (24 bits), two for fp16.  fp16 has little range:
// v' and S are scaled by powers of two of a wave, P by one of a row, to put the largest at 2^14; what is lost are bits 2^-39 below it.
#pragma once

#include "linear_attention.h"
#include "wave_sums.h"

namespace w34 {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4v lds_s4;

constexpr int kLinearChunk = 64;
constexpr float kLeastHold = 1.f / 65536;  // a state's registers take their factor up when it falls below this
constexpr double kNearFades = 100.0;       // log2 of what 32 tokens may fade by to be weighted by two factors
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
        const int total = __builtin_amdgcn_readlane(run, 63);
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
template <typename T>
__device__ __forceinline__ uint32_t linear_pack(float x, float y) {
    if constexpr (T::kStorageFormat == WARP34_KV_FORMAT_BF16) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, bf2));
    } else {
        return pack_h2(x, y);
    }
}
// Two numbers as PARTS pairs of 16 bits whose sums they are.  (What a pair of bf16 leaves of its numbers is also a dot product with (-1, 0) and
// (0, -1), half as many instructions, but v_dot2_f32_bf16 issues every 16 cycles: a chunk of rows took 7 % longer.)
template <typename T, int PARTS>
__device__ __forceinline__ void linear_split(float x, float y, uint32_t (&w)[PARTS]) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        w[p] = linear_pack<T>(x, y);
        if (p + 1 == PARTS) break;
        if constexpr (T::kStorageFormat == WARP34_KV_FORMAT_BF16) {
            x -= __uint_as_float(w[p] << 16);
            y -= __uint_as_float(w[p] & 0xFFFF0000u);
        } else {  // as in split_weights(): one mixed-precision fma each
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(x) : "v"(x), "v"(w[p]));
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(y) : "v"(y), "v"(w[p]));
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

// Rows in LDS are 16 bytes longer than they need to be, and of 16 rows the place of one is its number with the two pairs of bits exchanged: an
// operand read of 16 rows touches all banks, and so do the four rows of a transposing read, 64 bytes apart with two columns of 32 each.
constexpr int linear_row(int bytes) { return bytes + 16; }
__device__ __forceinline__ int linear_place(int row) { return (row & ~15) | (row & 3) << 2 | (row >> 2 & 3); }

// `rows` rows of `width` 16-bit elements from `base` on: loads behind the last row give zeros, stores there are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t linear_rows(const uint16_t* base, int rows, int stride, int width) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 2 * ((rows - 1) * stride + width), 0x00020000);
}

enum { kLinearWalk, kLinearSums, kLinearRows };  // a whole request; what a part adds to the state; a part's rows

template <int DK, int NW>
struct LinearLds {
    static constexpr int kKRow = linear_row(DK * 2), kVRow = linear_row(NW * 64);
    static constexpr int kQ = 0, kK = kLinearChunk * kKRow, kV = 2 * kK, kP = kV + kLinearChunk * kVRow;
    static constexpr int kRow = kP + 3 * 4096;     // [3][32] what P's rows are to be multiplied by (fp16)
    static constexpr int kTables = kRow + 3 * 32 * 4;
    // of a chunk and of the next one, [64] each: G as two numbers, what v, the state's part of a row and P are multiplied by
    static constexpr int kG = 0, kW = 64 * 8, kState = kW + 256, kAcross = kState + 256, kUp = kAcross + 256, kDown = kUp + 256, kChunk = kDown + 256;
    static constexpr int kTableBytes = kChunk + 16;
    static constexpr int kBytes = kTables + 2 * kTableBytes;
};

template <typename T, int DK, int NW, int MODE>
__global__ __launch_bounds__(64 * NW, NW == 4 || DK == 64 ? 2 : 1) void linear_chunk_kernel(const LinearArgs a, const LinearParts p) {
    typedef LinearLds<DK, NW> L;
    constexpr bool kBf16 = T::kStorageFormat == WARP34_KV_FORMAT_BF16;
    constexpr int DV = 32 * NW, kThreads = 64 * NW, KP = DK / 8, VP = 4 * NW, KT = DK / 32;  // pieces of 16 bytes a row, tiles of 32 channels
    constexpr int kLoads = kLinearChunk * KP / kThreads;
    constexpr int kParts = !kBf16 ? 2 : MODE == kLinearRows ? 2 : 3;  // of weighted values
    __shared__ __attribute__((aligned(16))) uint8_t smem[L::kBytes];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n32 = lane & 31, b = lane >> 5;
    const int group = (int)(blockIdx.x / (uint32_t)a.v_heads);
    int head = (int)(blockIdx.x - (uint32_t)group * (uint32_t)a.v_heads);
    // workgroups go round the eight dies: value heads of the same keys on the same one
    if (a.v_heads % 8 == 0) head = (head % 8) * (a.v_heads / 8) + head / 8;
    const int kh = head / a.group;
    int req = group, part = 0;
    if (MODE == kLinearWalk) {
        if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    } else {
        if (!linear_find_part(a, p.log_length, group, req, part)) return;
    }
    LinearRequest r = linear_request(a, req, head, DK * DV);
    r.lo = __builtin_amdgcn_readfirstlane(r.lo), r.n = __builtin_amdgcn_readfirstlane(r.n), r.kept = __builtin_amdgcn_readfirstlane(r.kept);
    const int state_at = 8 * b * DV + 32 * wave + n32;  // element of the state that is this lane's first

    int begin = 0, stop = r.n;
    if (MODE != kLinearWalk) linear_part_range(r.n, r.kept, p.log_length, part, begin, stop);
    else if (a.out == nullptr) stop = r.kept;
    begin = __builtin_amdgcn_readfirstlane(begin), stop = __builtin_amdgcn_readfirstlane(stop);

    f16v s[KT];
#pragma unroll
    for (int d = 0; d < KT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[d][i] = 0.f;
    int unit = 0;  // s holds the state times 2^unit (fp16), or over `hold` (bf16)
    float hold = 1.f;
    // this wave's share of a part's state in scratch
    float* const mine = MODE == kLinearWalk ? nullptr
                                            : p.states + ((int64_t)group * a.v_heads + head) * (DK * DV) + wave * (32 * DK) + lane * 4;
    if (MODE == kLinearWalk && r.in != nullptr) {
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[d][i] = r.in[state_at + (32 * d + 16 * (i >> 3) + (i & 7)) * DV];
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
#pragma unroll
    for (int d = 0; d < KT; ++d) asm volatile("" : "+v"(s[d]));
    const auto put_state = [&]() {
        const float by = kBf16 ? hold : power_of_two(-unit);
        int first = state_at;
        asm volatile("" : "+v"(first));  // addresses are worked out here, not kept in registers through the chunks
        linear_float* const to = r.out + first;
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) to[(32 * d + 16 * (i >> 3) + (i & 7)) * DV] = s[d][i] * by;
    };
    if (MODE == kLinearWalk && r.kept == 0 && r.out != nullptr) put_state();

    // a chunk on its way
    const bool with_q = MODE == kLinearRows || (MODE == kLinearWalk && a.out != nullptr);
    u4 qx[kLoads], kx[kLoads], vx[4];
    float gx = 0.f;
    int chunk_end = begin;
    const auto chunk_stop = [&](int t) { return min(t + kLinearChunk, MODE == kLinearWalk && t < r.kept ? r.kept : stop); };
    const int k_row = tid / KP, k_piece = tid % KP, v_row = tid / VP, v_piece = tid % VP;  // its first 16 bytes; the others are rows further down
    const auto fetch = [&](int t, int end) {
        const int rows = end - t;
        const int64_t tok = r.lo + t;
        const auto k = linear_rows(a.k + tok * a.k_stride + kh * DK, rows, a.k_stride, DK), v = linear_rows(a.v + tok * a.v_stride + head * DV, rows, a.v_stride, DV);
        const auto q = linear_rows(a.q + tok * a.q_stride + kh * DK, rows, a.q_stride, DK);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) kx[i] = __builtin_amdgcn_raw_buffer_load_b128(k, 2 * a.k_stride * (k_row + i * (kThreads / KP)) + 16 * k_piece, 0, 0);
        if (with_q) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) qx[i] = __builtin_amdgcn_raw_buffer_load_b128(q, 2 * a.q_stride * (k_row + i * (kThreads / KP)) + 16 * k_piece, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) vx[i] = __builtin_amdgcn_raw_buffer_load_b128(v, 2 * a.v_stride * (v_row + i * (kThreads / VP)) + 16 * v_piece, 0, 0);
    };
    const auto fetch_decays = [&](int t, int end) {
        gx = 0.f;
        if (a.g != nullptr && t + lane < end) gx = a.g[(int64_t)(r.lo + t + lane) * a.g_stride + head];
    };
    const auto put = [&]() {
        uint8_t* const kt = smem + L::kK + linear_place(k_row) * L::kKRow + k_piece * 16;
        uint8_t* const vt = smem + L::kV + linear_place(v_row) * L::kVRow + v_piece * 16;
        // a thread's further rows are whole sixteens away, or eights (two places)
        constexpr auto further = [](int rows) { return (rows & ~15) + (rows & 8 ? 2 : 0); };
        static_assert(kThreads / KP % 8 == 0 && kThreads / VP % 16 == 0, "rows of a pass");
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            *reinterpret_cast<u4*>(kt + further(i * (kThreads / KP)) * L::kKRow) = kx[i];
            if (with_q) *reinterpret_cast<u4*>(kt + (L::kQ - L::kK) + further(i * (kThreads / KP)) * L::kKRow) = qx[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<u4*>(vt + i * (kThreads / VP) * L::kVRow) = vx[i];
    };
    // The last wave's: the tables of a chunk, before which the state is its registers times `held`.  Their g is fetched a chunk before that.
    uint8_t* tables = smem + L::kTables;  // of the present chunk, and of the next one
    uint8_t* next_tables = tables + L::kTableBytes;
    const auto put_tables = [&](uint8_t* to, float held) {
        const double run = wave_run((double)(gx < kLeastDecay ? kLeastDecay : gx) * 1.4426950408889634);
        const double all = lane_value(run, 63), half = lane_value(run, 31), start = lane_value(run, 0), middle = lane_value(run, 32);
        const float hi = (float)run, fade = __builtin_amdgcn_exp2f((float)all), next = fade * held;
        const bool again = !kBf16 || next < kLeastHold;  // the registers take the factor up
        const auto put = [&](int at, float x) { *reinterpret_cast<float*>(to + at + lane * 4) = x; };
        *reinterpret_cast<float2*>(to + L::kG + lane * 8) = make_float2(hi, (float)(run - hi));
        put(L::kW, __builtin_amdgcn_exp2f((float)(all - run)) * (again ? 1.f : 1.f / next));
        if constexpr (MODE != kLinearSums) {
            const double centre = lane < 32 ? 0.5 * (start + half) : 0.5 * (middle + all);
            put(L::kState, __builtin_amdgcn_exp2f((float)run) * (held * a.scale));
            put(L::kAcross, __builtin_amdgcn_exp2f((float)(lane < 32 ? half - run : run - half)));
            put(L::kUp, __builtin_amdgcn_exp2f((float)(run - centre)));
            put(L::kDown, __builtin_amdgcn_exp2f((float)(centre - run)));
        }
        const float near = start - half < kNearFades && middle - all < kNearFades ? 1.f : 0.f;
        if (lane == 0) *reinterpret_cast<f4*>(to + L::kChunk) = f4{next, again ? 1.f : 0.f, (float)all, near};
    };
    const uint8_t* const row_at = smem + linear_place(n32) * L::kKRow + 16 * b;  // channels 8 b .. + 7 of 16 of row n32
    const auto k_operand = [&](int kt, int step) { return *reinterpret_cast<const u4*>(row_at + L::kK + 32 * kt * L::kKRow + 32 * step); };
    const auto q_operand = [&](int qt, int step) { return *reinterpret_cast<const u4*>(row_at + L::kQ + 32 * qt * L::kKRow + 32 * step); };
    uint8_t* const p_at = smem + L::kP + lane * 16;
    // transposed: rows 16 step + 4 b + 0 .. 3 and the same + 8, a column a lane of 32.  Of 16 channels of k the second four and the third change
    // places, so that eight registers of a lane's state are eight channels in a row, 8 b .. + 7 of 16, as q and k are read above.
    const int j16 = lane & 15, tr_place = 4 * (j16 >> 2) + b, tr_byte = 32 * (lane >> 4 & 1);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const uint32_t kt_at = lds0 + (uint32_t)(L::kK + tr_place * L::kKRow + tr_byte + 16 * (j16 & 1) + 4 * (j16 & 2));
    const uint32_t vt_at = lds0 + (uint32_t)(L::kV + tr_place * L::kVRow + 64 * wave + tr_byte + 8 * (j16 & 3));
    const auto transposed = [&](uint32_t at, int row_bytes) -> u4 {
        const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)at));
        const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)(at + 2u * (uint32_t)row_bytes)));
        const u2v u = __builtin_bit_cast(u2v, x), w = __builtin_bit_cast(u2v, y);
        return u4{u[0], u[1], w[0], w[1]};
    };

    // Tile 0: queries 0 .. 31 over keys 0 .. 31, 1: queries 32 .. 63 over keys 0 .. 31, 2: over keys 32 .. 63.
    const auto weights = [&](int tile, bool near) {
        const int kt = tile == 2 ? 1 : 0, qt = tile == 0 ? 0 : 1;
        f16v x = {};
#pragma unroll
        for (int step = 0; step < DK / 16; ++step)
            x = linear_mfma<T>(k_operand(kt, step), q_operand(qt, step), x);
        // 2^(G_i - G_j) as a product: by way of G at the border between the halves, or at the middle of the half where it fades by little there
        if (tile == 1 || near) {
            const float row = *reinterpret_cast<const float*>(tables + (tile == 1 ? L::kAcross : L::kUp) + (32 * qt + n32) * 4) * a.scale;
            const uint8_t* const columns = tables + (tile == 1 ? L::kAcross : L::kDown) + (32 * kt + 4 * b) * 4;
#pragma unroll
            for (int ig = 0; ig < 4; ++ig) {
                const f4 w = *reinterpret_cast<const f4*>(columns + 32 * ig);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = x[4 * ig + i] * row * w[i];
                    x[4 * ig + i] = tile == 1 || i + 8 * ig + 4 * b <= n32 ? y : 0.f;
                }
            }
        } else {
            const float2 gi = *reinterpret_cast<const float2*>(tables + L::kG + (32 * qt + n32) * 8);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = (i & 3) + 8 * (i >> 2) + 4 * b;
                const float2 gj = *reinterpret_cast<const float2*>(tables + L::kG + (32 * kt + key) * 8);
                const float y = x[i] * __builtin_amdgcn_exp2f((gi.x - gj.x) + (gi.y - gj.y)) * a.scale;
                x[i] = key <= n32 ? y : 0.f;
            }
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
            if (b == 0) *reinterpret_cast<float*>(smem + L::kRow + (tile * 32 + n32) * 4) = power_of_two(-e);
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
            *reinterpret_cast<u4*>(p_at + tile * 4096 + step * 1024) = hi;
            *reinterpret_cast<u4*>(p_at + tile * 4096 + 2048 + step * 1024) = lo;
        }
    };

    float part_sum = 0.f;  // of g, for the scan over parts
    if (begin < stop) {
        fetch(begin, chunk_end = chunk_stop(begin));
        if (wave == NW - 1) {
            fetch_decays(begin, chunk_end);
            put_tables(tables, 1.f);
            if (chunk_end < stop) fetch_decays(chunk_end, chunk_stop(chunk_end));
        }
    }
    // A chunk's rows go out when the next chunk's v takes their place, each thread's 16 bytes by itself: whole rows side by side.
    u4 ox[4];
    const auto take_rows = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) ox[i] = *reinterpret_cast<const u4*>(smem + L::kV + (linear_place(v_row) + i * (kThreads / VP)) * L::kVRow + v_piece * 16);
    };
    const auto store_rows = [&](int from, int to) {
        const auto rows = linear_rows(a.out + (int64_t)(r.lo + from) * a.out_stride + head * DV, to - from, a.out_stride, DV);
#pragma unroll
        for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b128(ox[i], rows, 2 * a.out_stride * (v_row + i * (kThreads / VP)) + 16 * v_piece, 0, 0);
    };
    int before = begin;  // where the chunk before the present one begins
    for (int t = begin; t < stop;) {
        const int end = chunk_end;
        if (with_q && t > begin) take_rows();
        put();
        __syncthreads();
        if (with_q && t > begin) store_rows(before, t);
        before = t;
        const f4 chunk = *reinterpret_cast<const f4*>(tables + L::kChunk);
        if (end < stop) fetch(end, chunk_end = chunk_stop(end));
        if (wave == NW - 1 && end < stop) {  // while the other waves weight P
            const bool again = chunk[1] != 0.f;
            put_tables(next_tables, again ? 1.f : chunk[0]);
            if (chunk_end < stop) fetch_decays(chunk_end, chunk_stop(chunk_end));
        }
        f16v o[2] = {};
        if (with_q) {
            if (NW == 4 ? wave < 3 : wave == 1) weights(NW == 4 ? wave : 2, chunk[3] != 0.f);
            if (NW == 2 && wave == 0) weights(0, chunk[3] != 0.f), weights(1, true);
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
                    const u4 qo = q_operand(q, step);
                    o[q] = linear_mfma<T>(part_of[0], qo, o[q]);
                    o[q] = linear_mfma<T>(part_of[1], qo, o[q]);
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float f = *reinterpret_cast<const float*>(tables + L::kState + (32 * q + n32) * 4) * (kBf16 ? 1.f : power_of_two(-e - unit));
#pragma unroll
                for (int i = 0; i < 16; ++i) o[q][i] *= f;
            }
        }
        u4 v[4];
#pragma unroll
        for (int step = 0; step < 4; ++step) v[step] = transposed(vt_at + 16 * step * L::kVRow, L::kVRow);
        if (with_q) {
            __syncthreads();
#pragma unroll
            for (int tile = 0; tile < 3; ++tile) {
                const int kt = tile == 2 ? 1 : 0, qt = tile == 0 ? 0 : 1;
                if constexpr (kBf16) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[qt] = linear_mfma<T>(v[2 * kt + (x & 1)], *reinterpret_cast<const u4*>(p_at + tile * 4096 + x * 1024), o[qt]);
                } else {
                    f16v sum = {};
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum = linear_mfma<T>(v[2 * kt + (x & 1)], *reinterpret_cast<const u4*>(p_at + tile * 4096 + x * 1024), sum);
                    const float f = *reinterpret_cast<const float*>(smem + L::kRow + (tile * 32 + n32) * 4);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[qt][i] = __builtin_fmaf(sum[i], f, o[qt][i]);
                }
            }
            // to where v was, whose operands are in registers: lane (n32, b) has columns 8 k + 4 b .. + 3 of row n32
            uint8_t* const to = smem + L::kV + linear_place(n32) * L::kVRow + 64 * wave + 8 * b;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<u2v*>(to + 32 * q * L::kVRow + 16 * k) = u2v{linear_pack<T>(o[q][4 * k], o[q][4 * k + 1]), linear_pack<T>(o[q][4 * k + 2], o[q][4 * k + 3])};
        }
        // the state moves on
        const bool again = chunk[1] != 0.f;
        if (MODE == kLinearSums) part_sum += chunk[2];
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
            const float by = kBf16 ? chunk[0] : chunk[0] * power_of_two(next - unit), values = power_of_two(next);
            unit = next;
            hold = again ? 1.f : chunk[0];
            if (__builtin_amdgcn_readfirstlane(again)) {
#pragma unroll
                for (int d = 0; d < KT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[d][i] *= by;
            }
            // values are weighted, and keys asked for, a step ahead of their products
            const auto weigh = [&](int step, u4 (&x)[kParts]) {
                const f4 w0 = *reinterpret_cast<const f4*>(tables + L::kW + (16 * step + 4 * b) * 4), w1 = *reinterpret_cast<const f4*>(tables + L::kW + (16 * step + 8 + 4 * b) * 4);
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
            };
            u4 x[2][kParts], k[2][KT];
            weigh(0, x[0]);
#pragma unroll
            for (int d = 0; d < KT; ++d) k[0][d] = transposed(kt_at + 64 * d, L::kKRow);
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                __builtin_amdgcn_sched_barrier(0);
                if (step < 3) {
#pragma unroll
                    for (int d = 0; d < KT; ++d) k[(step + 1) & 1][d] = transposed(kt_at + 16 * (step + 1) * L::kKRow + 64 * d, L::kKRow);
                    weigh(step + 1, x[(step + 1) & 1]);
                }
#pragma unroll
                for (int q = 0; q < kParts; ++q)
#pragma unroll
                    for (int d = 0; d < KT; ++d) s[d] = linear_mfma<T>(k[step & 1][d], x[step & 1][q], s[d]);
                if (step < 3) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * KT + 2, 0);
#pragma unroll
                    for (int i = 0; i < kParts * KT; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 20 / KT, 0);
                    }
                }
            }
        }
        t = end;
        {
            uint8_t* const x = tables;
            tables = next_tables, next_tables = x;
        }
        __syncthreads();
        if (MODE == kLinearWalk && t == r.kept && r.out != nullptr) put_state();
    }
    if (with_q && begin < stop) {
        take_rows();
        store_rows(before, stop);
    }
    if (MODE == kLinearSums) {
        const float by = kBf16 ? hold : power_of_two(-unit);
#pragma unroll
        for (int d = 0; d < KT; ++d)
#pragma unroll
            for (int ig = 0; ig < 4; ++ig) {
                f4 x;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = s[d][4 * ig + i] * by;
                *reinterpret_cast<f4*>(mine + (d * 4 + ig) * 256) = x;
            }
        if (tid == 0) p.fades[(int64_t)group * a.v_heads + head] = __builtin_amdgcn_exp2f(part_sum);
    }
}

constexpr int kScanAhead = 4;

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
    const int row = 32 * d + 16 * (ig >> 1) + 8 * (lane >> 5) + 4 * (ig & 1), col = 32 * w + (lane & 31);
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
    const int64_t step = (int64_t)a.v_heads * size;
    const int count = min(parts, p.most - first);
    // what four parts add travels while the four before them are gone through
    f4 u[kScanAhead];
    float fade[kScanAhead];
    const auto fetch = [&](int i, int part) {
        if (part < count) u[i] = *reinterpret_cast<const f4*>(slot + part * step), fade[i] = p.fades[(int64_t)(first + part) * a.v_heads + head];
    };
#pragma unroll
    for (int i = 0; i < kScanAhead; ++i) fetch(i, i);
    for (int part0 = 0; part0 < count; part0 += kScanAhead) {
#pragma unroll
        for (int k = 0; k < kScanAhead; ++k) {
            const int part = part0 + k;
            if (part >= count) break;
            const f4 add = u[k];
            const float by = fade[k];
            fetch(k, part + kScanAhead);
            *reinterpret_cast<f4*>(slot + part * step) = s;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(by, s[i], add[i]);
            int begin, end;
            linear_part_range(r.n, r.kept, p.log_length, part, begin, end);
            if (end == r.kept && r.out != nullptr) keep();
        }
    }
}

}  // namespace w34
