// Linear attention of prompts: tokens go by in chunks of 64.  With G the running sum of g (log2 domain) inside a chunk,
//
//   O_i = 2^G_i S^T q_i + sum_{j <= i} (q_i . k_j) 2^(G_i - G_j) v_j          S' = 2^G_end S + sum_j k_j (2^(G_end - G_j) v_j)^T
//
// Workgroup = the columns of a value head, a wave 16 of them with their part of the state in registers; 16x16x32 MFMAs:
//   P^T = K Q^T        in tiles of 16 x 16, a pair of them a wave, weighted, and laid into LDS as the operands of the product below
//   O^T = S^T Q^T      the state's registers are the operand as they stand: lane (n, g) has column n for channels 16 m + 4 g + i; q is laid into
//                      LDS in the order of two such tiles, and k is read in it
//   O^T += V^T P^T     v through transposing reads (ds_read_b64_tr_b16: lane l of 16 gets column l of four rows of 16 values)
//   S += K^T V'        k and v through transposing reads, v weighted in registers
// Weights are exponentials of differences of G, which is summed in 64 bits and held as two 32-bit numbers: where all but the last
// tokens have faded away, the sums are large and the differences small.
// Operands of 16 bits are rounded states, weights and weighted values.  P and S have two parts (16 bits of bf16, 22 of fp16), so that outputs
// show their own rounding (8 and 11 bits) as long as their terms do not cancel by as much as lies between; v' has three for bf16 where the
// state itself comes out (24 bits), two for fp16.  fp16 has little range: weighted values and S are scaled by a power of two of their
// column, P by one of its row, to put the largest at 2^14, and what the first part leaves is held times 2^11 and has sums of its own.
// So 22 bits stay of what is up to 2^28 below the largest, and bits 2^-50 below it are lost.
//
// Bound: instruction issue.  A wave's chunk is 98 products of 16 cycles and 477 vector instructions of four, the two waves of a SIMD take 6 950 of the
// 8 600 cycles that a chunk of a full batch lasts: splits and products of a wave wait for each other, and the clock falls to 1.8 .. 2.0 GHz.  8 x 4 096 tokens of 32
// heads of 128 x 128 walked in 270 .. 280 us (3.5 a chunk, 250 TFLOP/s, 3.1 TB/s), 8 192 tokens in parts in 103, 333 tokens of 16 heads in 19.
// Tile: a wave has 16 columns so that eight waves hold a state of 128 x 128 in 32 registers each and share one copy of k and q.  Four waves of 32
// columns with 32x32x16 products took 301 us, two workgroups of four waves of 16 columns, each with a copy, 3 to 40 % longer.  A chunk laid
// into LDS beside the one at work, for two barriers instead of three, took 9 % longer.
#pragma once

#include "linear_attention.h"
#include "wave_sums.h"

namespace w34 {

typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4v lds_s4;

constexpr int kLinearChunk = 64;
constexpr float kLeastHold = 1.f / 65536;  // a state's registers take their factor up when it falls below this
constexpr double kNearFades = 100.0;       // log2 of what 32 tokens may fade by to be weighted by two factors
constexpr float kLeastDecay = -200.f;  // e^-200 times any fp32 number is zero in 32 bits: smaller ones, minus infinity among them, change nothing

// Tokens of a part, a multiple of 64, and how many of them are in a number below 2^31: n / tokens = n * ceil(2^s / tokens) >> s for s = 31 + log2 of
// the tokens, rounded up.
struct LinearLength {
    int tokens;
    uint32_t factor;
    int shift;  // s - 32
    __device__ __forceinline__ int in(int n) const { return (int)(__umulhi((uint32_t)n, factor) >> shift); }
};
// A prompt cut into parts, which run at once, and once more behind the tokens that its state keeps.
struct LinearParts {
    float* states;  // [part][value head][k_head_dim * v_head_dim] in the order of the registers: what a part adds, then what it starts from
    float* fades;   // [part][value head] 2^(sum of the part's g)
    float* starts;  // [request][value head] as in states, where the rows' kernel joins the parts by itself: what the requests start from; else nullptr
    LinearLength length;
    int most;  // parts that there is room for
};

__device__ __forceinline__ int linear_parts_of(int n, int kept, const LinearLength& length) {
    const int whole = n <= 0 ? 1 : length.in(n - 1) + 1;  // a request without tokens has a part for its state
    return whole + (kept > 0 && kept < n && kept != length.in(kept) * length.tokens ? 1 : 0);
}
__device__ __forceinline__ void linear_part_range(int n, int kept, const LinearLength& length, int part, int& begin, int& end) {
    const int cut = length.in(kept);
    const bool extra = kept > 0 && kept < n && kept != cut * length.tokens;
    const int p = extra && part > cut ? part - 1 : part;
    begin = p * length.tokens, end = n - begin < length.tokens ? n : begin + length.tokens;
    if (extra && part == cut) end = kept;
    if (extra && part == cut + 1) begin = kept;
}
__device__ __forceinline__ int linear_request_parts(const LinearArgs& a, int req, const LinearLength& length) {
    if (req >= a.num_reqs || (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0)) return 0;
    const int lo = max(0, a.query_start_loc[req]), n = max(0, min(a.query_start_loc[req + 1], a.total_tokens) - lo);
    return linear_parts_of(n, a.state_tokens == nullptr ? n : min(max(a.state_tokens[req], 0), n), length);
}
// Request and number within it of a part; false behind the last one.  A wave looks at 64 requests at a time.
__device__ __forceinline__ bool linear_find_part(const LinearArgs& a, const LinearLength& length, int index, int& req, int& part) {
    const int lane = lane_id();
    for (int base = 0; base < a.num_reqs; base += 64) {
        const int mine = linear_request_parts(a, base + lane, length);
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
__device__ __forceinline__ int linear_first_part(const LinearArgs& a, const LinearLength& length, int req) {
    int count = 0;
    for (int base = 0; base < req; base += 64) count += base + lane_id() < req ? linear_request_parts(a, base + lane_id(), length) : 0;
#pragma unroll
    for (int by = 32; by; by /= 2) count += __shfl_xor(count, by, 64);
    return __builtin_amdgcn_readfirstlane(count);
}

template <typename T>
__device__ __forceinline__ f4 linear_mfma(u4 a, u4 b, f4 c) {
    if constexpr (T::kStorageFormat == WARP34_KV_FORMAT_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
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
constexpr float kRestUp = 2048.f, kRestDown = 1.f / 2048.f;  // the second part of fp16 is held times that
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
            x *= kRestUp, y *= kRestUp;
        }
    }
}
// The e for which 2^e puts `top` at 2^14, at most 126: 2^e and 2^-e are numbers.  0 for zero, and for what is not finite.
__device__ __forceinline__ int scale_exponent(float top) {
    const int e = (int)(__float_as_uint(top) >> 23 & 255u);
    return e == 0 || e == 255 ? 0 : min(141 - e, 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// Where 16 bytes of a row are in LDS, as the number they are found under in it: rows of PIECES = 8 or 16.  A wave's 16-byte reads go by lanes 0 .. 3,
// 12 .. 15 and 20 .. 27, then 4 .. 11, 16 .. 19 and 28 .. 31 (and the same of its second half): pieces g and g + 1 of rows {0 .. 3, 12 .. 15} and {4 .. 11}
// must differ, which they do where rows 12 .. 15 have the other halves of the pairs that rows 0 .. 3 have.  A transposing read takes 32 bytes of eight
// rows at a time: there the pairs must differ.  Cycles a read without and with a conflict: 4 and 8, transposing 2 and 4.
template <int PIECES>
__device__ __forceinline__ int linear_turn(int row) {
    constexpr int kHalf = PIECES / 2;
    const int x = PIECES == 16 ? row & 15 : row >> 1 & 7, low = x & (kHalf - 1);
    return x < kHalf ? 2 * low : 2 * (low ^ (kHalf / 2)) + 1;
}
template <int PIECES>
__device__ __forceinline__ uint32_t linear_place(int row, int piece) {
    return (uint32_t)(row * PIECES * 16 + (piece ^ linear_turn<PIECES>(row)) * 16);
}

// `rows` rows of `width` 16-bit elements from `base` on: loads behind the last row give zeros, stores there are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t linear_rows(const uint16_t* base, int rows, int stride, int width) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 2 * ((rows - 1) * stride + width), 0x00020000);
}

enum { kLinearWalk, kLinearSums, kLinearRows };  // a whole request; what a part adds to the state; a part's rows

template <int DK, int DV>
struct LinearLds {
    static constexpr int kKRow = DK * 2, kVRow = DV * 2;
    static constexpr int kQ = 0, kK = kLinearChunk * kKRow, kV = 2 * kK, kP = kV + kLinearChunk * kVRow;
    static constexpr int kRow = kP + 6 * 2048;     // [6][16] what P's rows are to be multiplied by (fp16)
    static constexpr int kTables = kRow + 6 * 16 * 4;
    // of a chunk and of the next one, [64] each: G as two numbers, what v, the state's part of a row and P are multiplied by
    static constexpr int kG = 0, kW = 64 * 8, kState = kW + 256, kAcross = kState + 256, kUp = kAcross + 256, kDown = kUp + 256, kChunk = kDown + 256;
    static constexpr int kTableBytes = kChunk + 16;
    static constexpr int kBytes = kTables + 2 * kTableBytes;
};

template <typename T, int DK, int DV, int MODE>
__global__ __launch_bounds__(4 * DV, 2) void linear_chunk_kernel(const LinearArgs a, const LinearParts p) {
    typedef LinearLds<DK, DV> L;
    constexpr bool kBf16 = T::kStorageFormat == WARP34_KV_FORMAT_BF16;
    constexpr int NW = DV / 16, kThreads = 64 * NW, KP = DK / 8, VP = DV / 8, KM = DK / 16;  // pieces of 16 bytes a row, tiles of 16 channels
    constexpr int kLoads = kLinearChunk * KP / kThreads, kVLoads = kLinearChunk * VP / kThreads;
    constexpr int kParts = !kBf16 ? 2 : MODE == kLinearRows ? 2 : 3;  // of weighted values
    __shared__ __attribute__((aligned(16))) uint8_t smem[L::kBytes];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int group = (int)(blockIdx.x / (uint32_t)a.v_heads);
    int head = (int)(blockIdx.x - (uint32_t)group * (uint32_t)a.v_heads);
    // workgroups go round the eight dies: value heads of the same keys on the same one
    if (a.v_heads % 8 == 0) head = (head % 8) * (a.v_heads / 8) + head / 8;
    const int kh = head / a.group;
    int req = group, part = 0;
    if (MODE == kLinearWalk) {
        if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    } else {
        if (!linear_find_part(a, p.length, group, req, part)) return;
    }
    LinearRequest r = linear_request(a, req, head, DK * DV);
    r.lo = __builtin_amdgcn_readfirstlane(r.lo), r.n = __builtin_amdgcn_readfirstlane(r.n), r.kept = __builtin_amdgcn_readfirstlane(r.kept);
    const int state_at = 4 * g4 * DV + 16 * wave + n16;  // element of the state that is this lane's first

    int begin = 0, stop = r.n;
    if (MODE != kLinearWalk) linear_part_range(r.n, r.kept, p.length, part, begin, stop);
    else if (a.out == nullptr) stop = r.kept;
    begin = __builtin_amdgcn_readfirstlane(begin), stop = __builtin_amdgcn_readfirstlane(stop);

    f4 s[KM];
#pragma unroll
    for (int m = 0; m < KM; ++m) s[m] = f4{0.f, 0.f, 0.f, 0.f};
    float hold = 1.f;  // s holds the state over it (bf16; fp16: 1)
    // this wave's share of a part's state in scratch, and of the one that its request starts from
    const auto share = [&](float* states, int i) { return states + ((int64_t)i * a.v_heads + head) * (DK * DV) + wave * (16 * DK) + lane * 4; };
    float* const mine = MODE == kLinearWalk ? nullptr : share(p.states, group);
    const bool joins = MODE != kLinearWalk && p.starts != nullptr;
    if ((MODE == kLinearWalk || (MODE == kLinearSums && joins && part == 0)) && r.in != nullptr) {
#pragma unroll
        for (int m = 0; m < KM; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][i] = r.in[state_at + (16 * m + i) * DV];
    }
    if (MODE == kLinearSums && joins && part == 0 && r.in != nullptr) {
        float* const to = share(p.starts, req);
#pragma unroll
        for (int m = 0; m < KM; ++m) *reinterpret_cast<f4*>(to + m * 256) = s[m], s[m] = f4{0.f, 0.f, 0.f, 0.f};
    }
    if (MODE == kLinearRows && !joins) {
#pragma unroll
        for (int m = 0; m < KM; ++m) s[m] = *reinterpret_cast<const f4*>(mine + m * 256);
    }
    if (MODE == kLinearRows && joins) {  // as linear_scan_kernel() does
        if (r.in != nullptr) {
            const float* const from = share(p.starts, req);
#pragma unroll
            for (int m = 0; m < KM; ++m) s[m] = *reinterpret_cast<const f4*>(from + m * 256);
        }
        for (int i = 0; i < part; ++i) {
            const float* const from = share(p.states, group - part + i);
            const float fade = p.fades[(int64_t)(group - part + i) * a.v_heads + head];
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const f4 u = *reinterpret_cast<const f4*>(from + m * 256);
#pragma unroll
                for (int c = 0; c < 4; ++c) s[m][c] = __builtin_fmaf(fade, s[m][c], u[c]);
            }
        }
    }
    // The loads end here: pending in front of the loop, they would be waited for in it, and with them the chunk that is on its way there.
#pragma unroll
    for (int m = 0; m < KM; ++m) asm volatile("" : "+v"(s[m]));
    const auto put_state = [&]() {
        const float by = hold;
        int first = state_at;
        asm volatile("" : "+v"(first));  // addresses are worked out here, not kept in registers through the chunks
        linear_float* const to = r.out + first;
#pragma unroll
        for (int m = 0; m < KM; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[(16 * m + i) * DV] = s[m][i] * by;
    };
    if ((MODE == kLinearWalk || (MODE == kLinearRows && joins && part == 0)) && r.kept == 0 && r.out != nullptr) put_state();

    if (MODE == kLinearRows && joins && r.kept > 0 && stop == r.kept && r.out != nullptr) {  // the state behind the part
        const float fade = p.fades[(int64_t)group * a.v_heads + head];
#pragma unroll
        for (int m = 0; m < KM; ++m) {
            const f4 u = *reinterpret_cast<const f4*>(mine + m * 256);
#pragma unroll
            for (int i = 0; i < 4; ++i) r.out[state_at + (16 * m + i) * DV] = __builtin_fmaf(fade, s[m][i], u[i]);
        }
    }

    // a chunk on its way
    const bool with_q = MODE == kLinearRows || (MODE == kLinearWalk && a.out != nullptr);
    u4 qx[kLoads], kx[kLoads], vx[kVLoads];
    float gx = 0.f;
    int chunk_end = begin;
    const auto chunk_stop = [&](int t) { return min(t + kLinearChunk, MODE == kLinearWalk && t < r.kept ? r.kept : stop); };
    const int k_row = tid / KP, k_piece = tid % KP, v_row = tid / VP, v_piece = tid % VP;  // its first 16 bytes; the others are rows further down
    static_assert(kThreads / KP % 16 == 0 && kThreads / VP % 16 == 0, "whole sixteens of rows further down");
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
        for (int i = 0; i < kVLoads; ++i) vx[i] = __builtin_amdgcn_raw_buffer_load_b128(v, 2 * a.v_stride * (v_row + i * (kThreads / VP)) + 16 * v_piece, 0, 0);
    };
    const auto fetch_decays = [&](int t, int end) {
        gx = 0.f;
        if (a.g != nullptr && t + lane < end) gx = a.g[(int64_t)(r.lo + t + lane) * a.g_stride + head];
    };
    // k and v as they are; of 32 channels of q, fours 0 and 4, 1 and 5, 2 and 6, 3 and 7 side by side
    uint8_t* const k_to = smem + L::kK + linear_place<KP>(k_row, k_piece);
    uint8_t* const v_to = smem + L::kV + linear_place<VP>(v_row, v_piece);
    uint8_t* const q_to = smem + L::kQ + linear_place<KP>(k_row, (k_piece & ~3) | (2 * k_piece & 3)) + 8 * (k_piece >> 1 & 1);
    uint8_t* const q_to2 = smem + L::kQ + linear_place<KP>(k_row, (k_piece & ~3) | (2 * k_piece & 3) | 1) + 8 * (k_piece >> 1 & 1);
    const auto put = [&]() {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            *reinterpret_cast<u4*>(k_to + i * (kThreads / KP) * L::kKRow) = kx[i];
            if (with_q) {
                *reinterpret_cast<u2v*>(q_to + i * (kThreads / KP) * L::kKRow) = u2v{qx[i][0], qx[i][1]};
                *reinterpret_cast<u2v*>(q_to2 + i * (kThreads / KP) * L::kKRow) = u2v{qx[i][2], qx[i][3]};
            }
        }
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) *reinterpret_cast<u4*>(v_to + i * (kThreads / VP) * L::kVRow) = vx[i];
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
            put(L::kState, __builtin_amdgcn_exp2f((float)run) * held);
            put(L::kAcross, __builtin_amdgcn_exp2f((float)(lane < 32 ? half - run : run - half)));
            put(L::kUp, __builtin_amdgcn_exp2f((float)(run - centre)));
            put(L::kDown, __builtin_amdgcn_exp2f((float)(centre - run)));
        }
        const float near = start - half < kNearFades && middle - all < kNearFades ? 1.f : 0.f;
        if (lane == 0) *reinterpret_cast<f4*>(to + L::kChunk) = f4{next, again ? 1.f : 0.f, (float)all, near};
    };
    // of row n16 of sixteen channels 4 g .. + 3 and 16 + 4 g .. + 3 of 32
    const uint32_t q_at = linear_place<KP>(n16, g4), k_at = linear_place<KP>(n16, g4 >> 1) + 8 * (g4 & 1);
    const auto q_operand = [&](int sixteen, int step) { return *reinterpret_cast<const u4*>(smem + L::kQ + 16 * sixteen * L::kKRow + (q_at ^ (64u * step))); };
    const auto k_operand = [&](int sixteen, int step) {
        const uint8_t* const at = smem + L::kK + 16 * sixteen * L::kKRow;
        const u2v x = *reinterpret_cast<const u2v*>(at + (k_at ^ (64u * step))), y = *reinterpret_cast<const u2v*>(at + (k_at ^ (64u * step + 32u)));
        return u4{x[0], x[1], y[0], y[1]};
    };
    // transposed: rows 4 g .. + 3 and 16 + 4 g .. + 3 of 32, a column a lane of 16
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const int tr_row = 4 * g4 + (n16 >> 2);
    const uint32_t kt_at = linear_place<KP>(tr_row, n16 >> 1 & 1) + 8 * (n16 & 1);
    const uint32_t vt_at = lds0 + L::kV + linear_place<VP>(tr_row, 2 * wave + (n16 >> 1 & 1)) + 8 * (n16 & 1);
    const auto transposed = [&](uint32_t at, int row_bytes) -> u4 {
        const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)at));
        const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)(at + 16u * (uint32_t)row_bytes)));
        const u2v u = __builtin_bit_cast(u2v, x), w = __builtin_bit_cast(u2v, y);
        return u4{u[0], u[1], w[0], w[1]};
    };

    // P: pair 0, 1: queries 0 .. 15, 16 .. 31 over keys 0 .. 31; 2, 3: queries 32 .. 47, 48 .. 63 over these; 4, 5: over keys 32 .. 63.
    // A tile has keys 4 g .. + 3 of 16 in lane (query, g): two are an operand of 32 keys in the order of the transposing reads.
    const auto weights = [&](int pair, bool near) {
        const int query = pair < 4 ? pair : pair - 2, keys = pair < 4 ? 0 : 2;  // in sixteens
        const bool across = pair == 2 || pair == 3;
        f4 x[2] = {};
#pragma unroll
        for (int step = 0; step < DK / 32; ++step) {
            const u4 q = q_operand(query, step);
#pragma unroll
            for (int k = 0; k < 2; ++k) x[k] = linear_mfma<T>(k_operand(keys + k, step), q, x[k]);
        }
        // 2^(G_i - G_j) as a product: by way of G at the border between the halves, or at the middle of the half where it fades by little there.
        // The factors, up to 2^50, are multiplied by each other first: q . k times one of them need not be a number.
        const int i0 = 16 * query + n16, j0 = 16 * keys + 4 * g4;
        if (across || near) {
            const float row = *reinterpret_cast<const float*>(tables + (across ? L::kAcross : L::kUp) + i0 * 4);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f4 w = *reinterpret_cast<const f4*>(tables + (across ? L::kAcross : L::kDown) + (j0 + 16 * k) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] = j0 + 16 * k + i <= i0 ? x[k][i] * (row * w[i]) : 0.f;
            }
        } else {
            const float2 gi = *reinterpret_cast<const float2*>(tables + L::kG + i0 * 8);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 gj = *reinterpret_cast<const float2*>(tables + L::kG + (j0 + 16 * k + i) * 8);
                    const float y = x[k][i] * __builtin_amdgcn_exp2f((gi.x - gj.x) + (gi.y - gj.y));
                    x[k][i] = j0 + 16 * k + i <= i0 ? y : 0.f;
                }
        }
        if constexpr (!kBf16) {
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[k][i]));
            const int e = scale_exponent(max_over_rows(top));
            const float by = power_of_two(e);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] *= by;
            if (g4 == 0) *reinterpret_cast<float*>(smem + L::kRow + (pair * 16 + n16) * 4) = power_of_two(-e);
        }
        u4 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t w[2];
            linear_split<T, 2>(x[k >> 1][2 * (k & 1)], x[k >> 1][2 * (k & 1) + 1], w);
            hi[k] = w[0], lo[k] = w[1];
        }
        *reinterpret_cast<u4*>(smem + L::kP + pair * 2048 + lane * 16) = hi;
        *reinterpret_cast<u4*>(smem + L::kP + pair * 2048 + 1024 + lane * 16) = lo;
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
    u4 ox[kVLoads];
    const auto take_rows = [&]() {
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) ox[i] = *reinterpret_cast<const u4*>(v_to + i * (kThreads / VP) * L::kVRow);
    };
    const auto store_rows = [&](int from, int to) {
        const auto rows = linear_rows(a.out + (int64_t)(r.lo + from) * a.out_stride + head * DV, to - from, a.out_stride, DV);
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) __builtin_amdgcn_raw_buffer_store_b128(ox[i], rows, 2 * a.out_stride * (v_row + i * (kThreads / VP)) + 16 * v_piece, 0, 0);
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
        const bool again = __builtin_amdgcn_readfirstlane(chunk[1] != 0.f);
        if (wave == NW - 1 && end < stop) {  // while the other waves weight P
            put_tables(next_tables, again ? 1.f : chunk[0]);
            if (chunk_end < stop) fetch_decays(chunk_end, chunk_stop(chunk_end));
        }
        f4 o[4] = {};
        if (with_q) {
            const bool near = __builtin_amdgcn_readfirstlane(chunk[3] != 0.f);
            if (NW == 8) {
                if (wave < 6) weights(wave, near);
            } else if (wave < 3) {
                weights(2 * wave, near);
                weights(2 * wave + 1, near);
            }
            // the state's part of the rows
            float by = 1.f;
            f4 down = {1.f, 1.f, 1.f, 1.f}, low[4] = {};  // fp16: the rest's sums
            if constexpr (!kBf16) {
                float top = 0.f;
#pragma unroll
                for (int m = 0; m < KM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(s[m][i]));
                const int e = scale_exponent(max_over_rows(top));  // of the lane's column; the product has columns 4 g .. + 3
                by = power_of_two(e);
#pragma unroll
                for (int i = 0; i < 4; ++i) down[i] = __shfl(power_of_two(-e), 4 * g4 + i, 64);
            }
            u4 part_of[2][2], qo[2][4];
            const auto operands = [&](int step) {
#pragma unroll
                for (int q = 0; q < 4; ++q) qo[step & 1][q] = q_operand(q, step);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t w[2];
                    float x = s[2 * step + (k >> 1)][2 * (k & 1)], y = s[2 * step + (k >> 1)][2 * (k & 1) + 1];
                    if (!kBf16) x *= by, y *= by;
                    linear_split<T, 2>(x, y, w);
                    part_of[step & 1][0][k] = w[0], part_of[step & 1][1][k] = w[1];
                }
            };
            operands(0);
#pragma unroll
            for (int step = 0; step < DK / 32; ++step) {
                if (step + 1 < DK / 32) operands(step + 1);
                // a product's result is an operand of another one 32 cycles after its start at the earliest, twice the time of its own: sums take turns
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f4& to = !kBf16 && x ? low[q] : o[q];
                        to = linear_mfma<T>(part_of[step & 1][x], qo[step & 1][q], to);
                    }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float f = *reinterpret_cast<const float*>(tables + L::kState + (16 * q + n16) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!kBf16) o[q][i] = __builtin_fmaf(low[q][i], kRestDown, o[q][i]) * down[i];
                    o[q][i] *= f;
                }
            }
        }
        u4 v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) v[u] = transposed(vt_at + 32 * u * L::kVRow, L::kVRow);
        if (with_q) {
            __syncthreads();
            f4 rest[4] = {};
#pragma unroll
            for (int pair = 0; pair < 6; ++pair) {
                const int q = pair < 4 ? pair : pair - 2, u = pair < 4 ? 0 : 1;
                const u4 hi = *reinterpret_cast<const u4*>(smem + L::kP + pair * 2048 + lane * 16), lo = *reinterpret_cast<const u4*>(smem + L::kP + pair * 2048 + 1024 + lane * 16);
                if constexpr (kBf16) {
                    o[q] = linear_mfma<T>(v[u], hi, o[q]);
                    rest[q] = linear_mfma<T>(v[u], lo, rest[q]);
                } else {
                    const f4 sum = linear_mfma<T>(v[u], hi, f4{}), low = linear_mfma<T>(v[u], lo, f4{});
                    const float f = *reinterpret_cast<const float*>(smem + L::kRow + (pair * 16 + n16) * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[q][i] = __builtin_fmaf(__builtin_fmaf(low[i], kRestDown, sum[i]), f, o[q][i]);
                }
            }
            // to where v was, whose operands are in registers: lane (n, g) has columns 4 g .. + 3 of row n
            uint8_t* const to = smem + L::kV + linear_place<VP>(n16, 2 * wave + (g4 >> 1)) + 8 * (g4 & 1);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[q][i] = (o[q][i] + rest[q][i]) * a.scale;
                *reinterpret_cast<u2v*>(to + 16 * q * L::kVRow) = u2v{linear_pack<T>(o[q][0], o[q][1]), linear_pack<T>(o[q][2], o[q][3])};
            }
        }
        // the state moves on
        if (MODE == kLinearSums) part_sum += chunk[2];
        if (MODE != kLinearRows || end < stop) {
            hold = again ? 1.f : chunk[0];
            float y[2][8], values = 1.f;  // weighted values
            const auto weigh = [&](int u) {
                const f4 w0 = *reinterpret_cast<const f4*>(tables + L::kW + (32 * u + 4 * g4) * 4), w1 = *reinterpret_cast<const f4*>(tables + L::kW + (32 * u + 16 + 4 * g4) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f4 w = i < 2 ? w0 : w1;
                    y[u][2 * i] = T::to_f32((uint16_t)v[u][i]) * w[2 * (i & 1)], y[u][2 * i + 1] = T::to_f32((uint16_t)(v[u][i] >> 16)) * w[2 * (i & 1) + 1];
                }
            };
            u4 x[2][kParts], k[2][KM];
            const auto operands = [&](int u) {
#pragma unroll
                for (int m = 0; m < KM; ++m) k[u][m] = transposed(lds0 + L::kK + 32 * u * L::kKRow + (kt_at ^ (32u * m)), L::kKRow);
                if (kBf16) weigh(u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t parts[kParts];
                    linear_split<T, kParts>(kBf16 ? y[u][2 * i] : y[u][2 * i] * values, kBf16 ? y[u][2 * i + 1] : y[u][2 * i + 1] * values, parts);
#pragma unroll
                    for (int q = 0; q < kParts; ++q) x[u][q][i] = parts[q];
                }
            };
            if constexpr (kBf16) {
                if (again) {
#pragma unroll
                    for (int m = 0; m < KM; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[m][i] *= chunk[0];
                }
                operands(0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (u == 0) operands(1);
#pragma unroll
                    for (int q = 0; q < kParts; ++q)
#pragma unroll
                        for (int m = 0; m < KM; ++m) s[m] = linear_mfma<T>(k[u][m], x[u][q], s[m]);
                }
            } else {
                weigh(0), weigh(1);
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fabsf(y[0][i]), fabsf(y[1][i])));
                const int e = scale_exponent(max_over_rows(top));  // of the lane's column, which is that of its part of the state
                values = power_of_two(e);
                const float down = power_of_two(-e);
                operands(0), operands(1);
#pragma unroll
                for (int m = 0; m < KM; ++m) {
                    f4 sum = linear_mfma<T>(k[0][m], x[0][0], f4{}), low = linear_mfma<T>(k[0][m], x[0][1], f4{});
                    sum = linear_mfma<T>(k[1][m], x[1][0], sum), low = linear_mfma<T>(k[1][m], x[1][1], low);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[m][i] = __builtin_fmaf(__builtin_fmaf(low[i], kRestDown, sum[i]), down, chunk[0] * s[m][i]);
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
#pragma unroll
        for (int m = 0; m < KM; ++m) *reinterpret_cast<f4*>(mine + m * 256) = s[m] * hold;
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
    const int first = linear_first_part(a, p.length, req), parts = linear_parts_of(r.n, r.kept, p.length);
    const int x = block * 256 + (int)threadIdx.x;  // [16 columns][16 channels][lane]
    const int lane = x & 63, tiles = k_dim / 16, m = (x >> 6) % tiles, w = (x >> 6) / tiles;
    const int row = 16 * m + 4 * (lane >> 4), col = 16 * w + (lane & 15);
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
            linear_part_range(r.n, r.kept, p.length, part, begin, end);
            if (end == r.kept && r.out != nullptr) keep();
        }
    }
}

}  // namespace w34
