// Scored paged attention of few query columns for each kv head: one new token, or the tokens of a verify step; over 16-bit and 8-bit rows.
//
// Workgroup = one chunk of one tile's keys x one kv head, eight waves; a wave takes every eighth half unit (16 keys) of the chunk:
//   S^T = K Q^T      16x16x32 MFMAs, A = 16 key rows (lane (n, b): row n), B = query columns; lane (n, b) gets the scores of keys
//                    4 b .. 4 b + 3 for column n, so that the softmax state of a column is a scalar of four lanes
//   O^T += V^T P^T   A = channels x keys, B = the weights where they stand: each weight has a high and a low 16-bit part in the two
//                    halves of a product of 32 keys, over the same values: 22 bits of it, down to 2^-24 (block scales ride on the weights
//                    of quantised rows, so that small values come to that end first: 1e-6 has an error of 3e-3 to 1e-2 into bf16 outputs)
// Rows go from the pages to registers as they are stored; key loads of the next half unit travel during the softmax and the value
// product, value loads during the next scores.  Only the scales of quantised rows go through LDS.
// At the end the waves' states are joined through LDS, and the chunks' by scored_join_kernel.
//
// Bound: HBM over many keys (32 requests of 1k to 64k keys: FP16 411 us = 5.3 TB/s, FP8 223 = 4.8, Q8_0 235 = 4.7; a large copy of the
// card 5.1, reads alone 6.0), round trips over few: one request on 700 FP16 keys 10.7 us, of which kernel 7.4 (arguments and lengths 1.5,
// first rows 1.5, a half unit 1.7, join of the waves 2) and the join's launch 3.  16 windows of 4 096 BF16 keys, head_dim 128: 25.9 us, kernel 20, of
// which 9 to 12 stream.  Q8_0 verify steps of 5 x 4 tokens on 3k to 21k keys 34.5 us: 17 for eight half units a wave, 400 vector
// instructions each, tiles of 16 columns twice over the rows.  (Tiles of 32 columns: 34.0 there, 29.6 for 32.4 over FP8, but 24.9 for 17.6 where
// 4 requests look at 4 000 keys: not kept.  Waves in step by a barrier every step: no gain.)
#pragma once

#include "scored_attn.h"

namespace w34 {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef u4 u4_at4 __attribute__((aligned(4)));
typedef u2v u2_at4 __attribute__((aligned(4)));

constexpr int kScoredWaves = 8;

template <bool IS_BF16>
__device__ __forceinline__ f4 mfma_rows(u4 a, u4 b, f4 c) {
    if constexpr (IS_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}
__device__ __forceinline__ uint32_t pack_bf2(float x, float y) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, bf2));
}

// ---- what the decode kernels share ----

// The tile, the chunk and the keys of a workgroup, in half units [begin, end); false: nothing to do.  PAIRS: chunks of whole pairs of half
// units.  counts: room for the batch's tiles in LDS, free again afterwards.
struct DecodeStart {
    ScoredWork work;
    ScoredTile t;
    int begin, end;
};
template <bool PAIRS>
__device__ __forceinline__ bool decode_start(const ScoredParams& P, uint8_t* counts, int tid, int lane, int kv_sub, DecodeStart& s) {
    s.work = ScoredWork{(int)blockIdx.x, 0, 1, 0};
    if (P.target > 0 && P.entries <= 64) {  // lane e: entry e, all a wave has to know
        ScoredTile mine = {0, 0, 0, 0, 0};
        if (lane < P.entries) mine = scored_tile(P, lane);
        const int halves = lane < P.entries ? tile_halves_guess(P, mine) : -1;
        const auto count = [&](int) { return halves; };
        const int per = chunk_length(P, lane, count);
        s.work = find_work(P, per, (int)blockIdx.x, lane, count);
        if (s.work.entry < 0) return false;
        const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s.work.entry); };
        s.t = ScoredTile{of(mine.req), of(mine.tok0), of(mine.tokens), of(mine.pos0), of(mine.seq_after)};
    } else {
        if (P.target > 0) {
            int* halves = reinterpret_cast<int*>(counts);
            for (int e = tid; e < P.entries; e += kScoredWaves * 64) halves[e] = tile_halves_guess(P, scored_tile(P, e));
            __syncthreads();
            const auto count = [&](int e) { return halves[e]; };
            const int per = chunk_length(P, lane, count);
            s.work = find_work(P, per, (int)blockIdx.x, lane, count);
            if (s.work.entry < 0) return false;
            __syncthreads();
        }
        s.t = scored_tile(P, s.work.entry);
        if (s.t.tokens <= 0) return false;
    }
    int key_first, key_last;
    tile_keys(P, s.t, lane, key_first, key_last);
    if (s.work.chunk == 0 && kv_sub == 0 && tid == 0 && P.target > 0) {
        P.table[2 * s.work.entry] = s.work.first_record;
        P.table[2 * s.work.entry + 1] = s.work.chunks;
    }
    const int halves = tile_halves(key_first, key_last);
    int per = fast_div(halves + s.work.chunks - 1, s.work.chunks);
    if (PAIRS) per = (per + 1) & ~1;
    s.begin = (key_first >> 4) + s.work.chunk * per;
    s.end = key_first > key_last ? s.begin : max(s.begin, min(s.begin + per, (key_last >> 4) + 1));
    return true;
}

// The largest / least number of each 16 lanes, in all of them.
template <typename F>
__device__ __forceinline__ int row_reduce(int v, F&& f) {
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
    return f(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // row_mirror
}
// Whether any of the 16 lanes of the lane's row has it.
__device__ __forceinline__ bool any_of_row(bool mine, int b) { return ((uint32_t)(__ballot(mine) >> (16 * b)) & 0xFFFFu) != 0u; }

// A lane's column: its token's keys [lo, hi], position and slope; of the tile: the keys that every live column sees, the live columns.
struct DecodeColumn {
    int tok, head, pos, lo, hi;
    bool ok;
    int all_from, all_to;  // uniform
    uint32_t live;
    float slope2;
};
__device__ __forceinline__ DecodeColumn decode_column(const ScoredParams& P, const ScoredTile& t, int head0, int col) {
    const warp34_attention_batch& B = P.B;
    DecodeColumn c;
    const int mine = column_token(col, P);
    c.tok = min(t.tok0 + mine, B.total_tokens - 1);
    c.ok = mine < t.tokens && (B.valid_token_mask == nullptr || B.valid_token_mask[c.tok] != 0);
    c.head = min(head0 + (col - mine * P.q_group), P.num_q_heads - 1);
    c.pos = t.pos0 + mine;
    c.lo = 0, c.hi = -1;
    if (c.ok) token_keys(P, c.tok, c.pos, t.seq_after, c.lo, c.hi);
    c.all_from = __builtin_amdgcn_readfirstlane(row_reduce(c.ok ? c.lo : 0, [](int a, int b) { return max(a, b); }));
    c.all_to = __builtin_amdgcn_readfirstlane(row_reduce(c.ok ? c.hi : 0x7fffffff, [](int a, int b) { return min(a, b); }));
    c.live = (uint32_t)(__ballot(c.ok) & 0xFFFFull);
    c.slope2 = P.slopes != nullptr && c.ok ? P.slopes[c.head] * kLog2e : 0.f;
    return c;
}

// Query columns of quantised rows: a wave brings every eighth of COLS columns to LDS, rotated where the keys are, in two fp16 parts (the
// second is zero where nothing is rotated: 11 bits are all there are).  They are relative to a power of two, so that the largest element
// is 2^12 to 2^13: fp16 holds a query whatever its size, and the second parts of its smaller elements are still normal numbers.
constexpr int kQueryTop = 13;
template <typename TQ, int COLS, int STRIDE>
struct QueryColumns {
    uint2 raw[COLS / kScoredWaves];
    __device__ __forceinline__ void load(const ScoredParams& P, const ScoredTile& t, int head0, int wave, int lane) {
#pragma unroll
        for (int k = 0; k < COLS / kScoredWaves; ++k) {
            const int c = wave + kScoredWaves * k, ct = column_token(c, P);
            const int tok = min(t.tok0 + ct, P.B.total_tokens - 1), head = min(head0 + c - ct * P.q_group, P.num_q_heads - 1);
            raw[k] = *reinterpret_cast<const uint2*>(P.q + ((size_t)tok * P.num_q_heads + (size_t)head) * 256 + 4 * lane);
        }
    }
    // Waits for them: in front of the loads of rows, which may be none, so that nobody would know how many to leave on their way.
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int k = 0; k < COLS / kScoredWaves; ++k) asm volatile("" : "+v"(raw[k].x), "+v"(raw[k].y));
    }
    __device__ __forceinline__ void bring(const ScoredParams& P, uint32_t live, int wave, int lane, uint16_t* high, uint16_t* low, float* scales) const;
};
template <typename TQ, int COLS, int STRIDE>
__device__ __forceinline__ void QueryColumns<TQ, COLS, STRIDE>::bring(const ScoredParams& P, uint32_t live, int wave, int lane, uint16_t* high,
                                                                      uint16_t* low, float* scales) const {
#pragma unroll
    for (int k8 = 0; k8 < COLS / kScoredWaves; ++k8) {
        const int c = wave + kScoredWaves * k8;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if ((live >> c) & 1u) {
            const uint32_t x = raw[k8].x ^ P.q_flip, y = raw[k8].y ^ P.q_flip;
            v[0] = TQ::to_f32((uint16_t)x), v[1] = TQ::to_f32((uint16_t)(x >> 16));
            v[2] = TQ::to_f32((uint16_t)y), v[3] = TQ::to_f32((uint16_t)(y >> 16));
        }
        if (P.rot_q) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = apply_sign(v[k], 4 * lane + k);
            wht256_wave(v, lane);
        }
        const float top = wave_top(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
        const int e = top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_ldexpf(v[k], kQueryTop - e);
        uint32_t h0, h1, l0, l1;
        split_weights(v[0], v[1], h0, l0);
        split_weights(v[2], v[3], h1, l1);
        *reinterpret_cast<uint2*>(high + c * STRIDE + 4 * lane) = uint2{h0, h1};
        *reinterpret_cast<uint2*>(low + c * STRIDE + 4 * lane) = uint2{l0, l1};
        if (lane == 0) scales[c] = __builtin_amdgcn_ldexpf(1.0f, e - kQueryTop);
    }
}

// The pages of a tile's keys: 64 entries of its block table in the lanes of a wave.
struct PageWalk {
    const slab_byte* k_slab;
    const slab_byte* v_slab;
    const int32_t* blocks;
    int slot_base, pages;
    __device__ __forceinline__ void fetch(const ScoredParams& P, int slot, int lane) {
        slot_base = slot;
        pages = slot + lane < P.B.max_blocks_per_req ? blocks[slot + lane] : 0;
    }
    __device__ __forceinline__ void start(const ScoredParams& P, const ScoredTile& t, int kv_head, int half, int lane) {
        k_slab = slab_at(P.L.k_base) + (uint64_t)(uint32_t)kv_head * P.L.k_head_stride_bytes;
        v_slab = slab_at(P.L.v_base) + (uint64_t)(uint32_t)kv_head * P.L.v_head_stride_bytes;
        blocks = P.B.block_tables + (size_t)t.req * P.B.max_blocks_per_req;
        fetch(P, page_slot(half * 16, P), lane);
    }
    // rows of a half unit; half units in order: none from a page in front of the last one's, whose entries may be gone
    __device__ __forceinline__ void locate(const ScoredParams& P, int half, int row_bytes, int lane, const slab_byte*& k_rows, const slab_byte*& v_rows) {
        const int pos = half * 16, slot = page_slot(pos, P);
        if (slot - slot_base >= 64) {  // uniform
            fetch(P, slot, lane);
            asm volatile("" : "+v"(pages));  // (the wait stands here and not behind the branch, for whatever is on its way)
        }
        const uint32_t page = (uint32_t)max(__builtin_amdgcn_readlane(pages, slot - slot_base), 0);
        const uint32_t in_page = (uint32_t)(pos - slot * P.L.block_size) * (uint32_t)row_bytes;
        k_rows = k_slab + (uint64_t)page * P.L.k_page_stride_bytes + in_page;
        v_rows = v_slab + (uint64_t)page * P.L.v_page_stride_bytes + in_page;
    }
};

// The waves' states of COLS columns joined and the columns finished.  Every wave has its sums in its region [column][HD + 8] of `regions`,
// slot 16 k + 4 b + i for row 4 b + i of MFMA k = g J + j (channel 16 J g + J row + j), and its (m, l) in ml[wave][16]; wave c joins
// columns c and c + 8, through its own `reorder` of HD floats.  A barrier lies before the call.
template <typename TQ, int HD, int J, int COLS>
__device__ __forceinline__ void join_waves(const ScoredParams& P, const DecodeStart& s, int kv_sub, int head0, uint32_t live, int wave, int lane,
                                           const uint8_t* regions, int region_bytes, const float* ml, float* reorder, float value_scale) {
    constexpr int kColStride = HD + 8;
    const int at = (4 * lane) & (HD - 1);
    const int k = at >> 4, g = k / J, j = k % J, row = at & 15;
#pragma unroll 1
    for (int c = wave; c < COLS; c += kScoredWaves) {
        if (!((live >> c) & 1u)) continue;
        f2 state[kScoredWaves];
        f4 part[kScoredWaves];
#pragma unroll
        for (int w = 0; w < kScoredWaves; ++w) {
            state[w] = *reinterpret_cast<const f2*>(ml + (w * 16 + c) * 2);
            part[w] = *reinterpret_cast<const f4*>(regions + w * region_bytes + (c * kColStride + at) * 4);
        }
        float m = kNegBig, l = 0.f;
#pragma unroll
        for (int w = 0; w < kScoredWaves; ++w) m = fmaxf(m, state[w][0]);
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kScoredWaves; ++w) {
            const float weight = __builtin_amdgcn_exp2f(state[w][0] - m);
            l += weight * state[w][1];
            acc += part[w] * weight;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) reorder[16 * J * g + J * (row + i) + j] = acc[i];
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        const f4 sum = *reinterpret_cast<const f4*>(reorder + at);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        if (s.work.chunks > 1) {
            const size_t record = ((size_t)(s.work.first_record + s.work.chunk) * gridDim.y + kv_sub) * COLS + c;
            if (4 * lane < HD) *reinterpret_cast<f4*>(P.part_acc + record * HD + 4 * lane) = sum;
            if (lane == 0) *reinterpret_cast<f2*>(P.part_ml + 2 * record) = f2{m, l};
        } else {
            float v[4] = {sum[0], sum[1], sum[2], sum[3]};
            const int ct = column_token(c, P);
            finish_row<TQ, HD>(P, s.t.tok0 + ct, head0 + c - ct * P.q_group, lane, v, m, l, value_scale);
        }
    }
}

// What a storage format is made of.  SCALES: block scales of a row.  Key operand m, lane b: elements element(m, b) .. + 7.  Values:
// GROUPS groups of 16 J channels, one block scale each (quantised rows); MFMA j of group g has channel 16 J g + J r + j in row r.
template <int KVF, int HD>
struct ScoredRows {
    static constexpr bool kTq4 = KVF == WARP34_KV_FORMAT_TQ4, kFp8 = KVF == WARP34_KV_FORMAT_FP8_E4M3, kQ8 = KVF == WARP34_KV_FORMAT_Q8_0;
    static constexpr bool k16 = !kTq4 && !kFp8 && !kQ8;
    static constexpr int kRowBytes = kTq4 ? 132 : kFp8 ? 264 : kQ8 ? 272 : 2 * HD;
    static constexpr int kOps = HD / 32;                      // key operands of a row
    static constexpr int kScales = k16 ? 0 : kQ8 ? 4 : 2;
    static constexpr int kGroups = kQ8 ? 4 : HD / 128, kJ = kQ8 ? 4 : 8;
    static constexpr int kKeyRegs = k16 ? kOps : 4;  // of 16 bytes
    // what the values in the operands are to be multiplied by: TQ4 look-ups hold kLutGain times the centroid (in the end), 8-bit codes
    // come as code / 256 (E4M3) or code / 128, which keeps the low part of a weight, times that gain, out of fp16's subnormal range
    static constexpr float kValueGain = kFp8 ? 256.0f : kQ8 ? 128.0f : 1.0f;
    static constexpr float kOutScale = kTq4 ? kLutInvGain : 1.0f;
    __device__ static constexpr int element(int m, int b) {
        return k16 ? 32 * m + 8 * b : 64 * (m >> 1) + 16 * b + 8 * (m & 1);
    }
};

// LDS: [query columns], over which the counts of the tiles lie at the start and the waves' regions at the end; [a finished column of each
// wave][(m, l) of the waves][scales of the waves]
template <int KVF, int HD>
struct ScoredLds {
    using R = ScoredRows<KVF, HD>;
    static constexpr int kColStride = HD + 8;  // floats of a column in a region
    static constexpr int kRegion = 16 * kColStride * 4;
    static constexpr int kQStride = HD + 8;    // 16-bit elements
    static constexpr int kQ = 0, kQLow = kQ + 16 * kQStride * 2, kQScale = kQLow + 16 * kQStride * 2;
    static constexpr int kReorder = kScoredWaves * kRegion;
    static constexpr int kMl = kReorder + kScoredWaves * HD * 4;
    static constexpr int kScale = kMl + kScoredWaves * 16 * 8;
    static constexpr int kBytes = kScale + (R::k16 ? 0 : kScoredWaves * 2 * 4 * 16 * 4);
    static_assert(kBytes <= 160 * 1024 && kMaxSplitEntries * 4 <= kReorder && kQScale + 64 <= kReorder, "decode LDS budget");
};

template <typename TQ, int KVF, int HD, bool CAP>
__global__ __launch_bounds__(kScoredWaves * 64, 1) void scored_decode_kernel(const ScoredParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    using R = ScoredRows<KVF, HD>;
    using M = ScoredLds<KVF, HD>;
    constexpr bool IS_BF16 = R::k16 && TQ::kStorageFormat == WARP34_KV_FORMAT_BF16;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, b = lane >> 4;
    const int kv_sub = (int)blockIdx.y;
    const int kv_head = P.q_subgroups == 1 ? kv_sub : fast_div(kv_sub, P.q_subgroups);
    const int head0 = kv_head * P.gqa + (kv_sub - kv_head * P.q_subgroups) * P.q_group;

    DecodeStart s0;
    if (!decode_start<false>(P, smem, tid, lane, kv_sub, s0)) return;
    const int end = s0.end;
    PageWalk walk;
    walk.start(P, s0.t, kv_head, s0.begin, lane);
    const DecodeColumn col = decode_column(P, s0.t, head0, n);
    if (col.live == 0u) return;
    const bool sloped = P.slopes != nullptr;

    // ---- what comes from memory first: the queries, then the rows of this wave's first half unit ----
    u4 q_high[R::kOps], q_low[R::kOps];
    QueryColumns<TQ, 16, M::kQStride> columns;
    if constexpr (R::k16) {
        const uint16_t* src = P.q + ((size_t)col.tok * P.num_q_heads + (size_t)col.head) * HD;
#pragma unroll
        for (int m = 0; m < R::kOps; ++m) q_high[m] = *reinterpret_cast<const u4*>(src + R::element(m, b));
    } else {
        columns.load(P, s0.t, head0, wave, lane);
    }
    const slab_byte* k_rows;
    const slab_byte* v_rows;
    const auto locate = [&](int half) { walk.locate(P, half, R::kRowBytes, lane, k_rows, v_rows); };
    u4 kr[R::kKeyRegs];
    uint32_t k_scale = 0, v_scale = 0;   // Q8_0: of row n, block b
    u2v k_scales = {0u, 0u}, v_scales = {0u, 0u};  // FP8: both of row n
    u4 vr16[R::k16 ? R::kGroups : 1][4];
    u2v vr8[R::kFp8 ? 2 : 1][4];
    uint32_t vr4[R::kQ8 ? 4 : 1][4];
    const auto load_keys = [&]() {
        const slab_byte* row = k_rows + (uint32_t)(n * R::kRowBytes);
        if constexpr (R::k16) {
#pragma unroll
            for (int m = 0; m < R::kOps; ++m) kr[m] = load_as<u4>(row + 64 * m + 16 * b);
        } else if constexpr (R::kFp8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) kr[c] = load_as<u4_at4>(row + 64 * c + 16 * b);
            k_scales = load_as<u2_at4>(row + 256);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) kr[c] = load_as<u4_at4>(row + 68 * c + 4 + 16 * b);
            k_scale = load_as<uint32_t>(row + 68 * b);
        }
    };
    const auto load_values = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const slab_byte* row = v_rows + (uint32_t)((4 * b + i) * R::kRowBytes);
            if constexpr (R::k16) {
#pragma unroll
                for (int g = 0; g < R::kGroups; ++g) vr16[g][i] = load_as<u4>(row + 256 * g + 16 * n);
            } else if constexpr (R::kFp8) {
#pragma unroll
                for (int g = 0; g < 2; ++g) vr8[g][i] = load_as<u2_at4>(row + 128 * g + 8 * n);
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) vr4[g][i] = load_as<uint32_t>(row + 68 * g + 4 + 4 * n);
            }
        }
        const slab_byte* row = v_rows + (uint32_t)(n * R::kRowBytes);
        if constexpr (R::kFp8) v_scales = load_as<u2_at4>(row + 256);
        if constexpr (R::kQ8) v_scale = load_as<uint32_t>(row + 68 * b);
    };
    int half = s0.begin + wave;
    if constexpr (!R::k16) columns.arrived();
    if (half < end) {
        locate(half);
        load_keys();
        load_values();
    }

    // ---- query operands ----
    float cs = score_factor(P, 1.0f), cc = P.cap_arg;
    uint16_t* qh = reinterpret_cast<uint16_t*>(smem + M::kQ);
    uint16_t* ql = reinterpret_cast<uint16_t*>(smem + M::kQLow);
    if constexpr (R::k16) {
#pragma unroll
        for (int m = 0; m < R::kOps; ++m) {
            q_high[m] ^= P.q_flip;
            if (!col.ok) q_high[m] = u4{0u, 0u, 0u, 0u};
        }
    } else {
        float* qs = reinterpret_cast<float*>(smem + M::kQScale);
        columns.bring(P, col.live, wave, lane, qh, ql, qs);
        __syncthreads();
#pragma unroll
        for (int m = 0; m < R::kOps; ++m) {
            q_high[m] = *reinterpret_cast<const u4*>(qh + n * M::kQStride + R::element(m, b));
            q_low[m] = *reinterpret_cast<const u4*>(ql + n * M::kQStride + R::element(m, b));
        }
        cs = score_factor(P, qs[n]);
        cc = cap_factor(P, qs[n]);
    }
    const bool two_parts = !R::k16 && P.rot_q != 0;

    // Block scales are loaded a row a lane and used four rows a lane: an exchange through 256 bytes of LDS for each kind.
    float* scale_area = reinterpret_cast<float*>(smem + M::kScale + wave * (2 * 4 * 16 * 4));
    const auto exchange = [&](float* area, uint32_t one, u2v two) {
        if constexpr (R::kFp8) {
            if (b < 2) area[16 * b + n] = __uint_as_float(b == 0 ? two[0] : two[1]);
        } else if constexpr (R::kQ8) {
            area[16 * b + n] = __uint_as_float(one);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };

    f4 o[R::kGroups * R::kJ];
#pragma unroll
    for (int k = 0; k < R::kGroups * R::kJ; ++k) o[k] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNegBig, l_run = 0.f;

    while (half < end) {
        const int next = half + kScoredWaves;
        const bool more = next < end;
        const int pos = half * 16 + 4 * b;  // of this lane's first key

        // ---- scores ----
        f4 s = {0.f, 0.f, 0.f, 0.f};
        if constexpr (R::k16) {
#pragma unroll
            for (int m = 0; m < R::kOps; ++m) s = mfma_rows<IS_BF16>(kr[m], q_high[m], s);
        } else {
            exchange(scale_area, k_scale, k_scales);
            constexpr int kPerBlock = 8 / R::kScales;
#pragma unroll
            for (int blk = 0; blk < R::kScales; ++blk) {
                f4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int mm = 0; mm < kPerBlock; ++mm) {
                    const int m = blk * kPerBlock + mm;
                    u4 a;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint32_t word = kr[m >> 1][2 * (m & 1) + w];
                        uint32_t x, y;
                        if constexpr (R::kFp8) {
                            x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false));
                            y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true));
                        } else {  // 0x6400 | (q + 128) is 1152 + q in fp16
                            const uint32_t u = word ^ 0x80808080u;
                            const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
                            x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
                            y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
                        }
                        a[2 * w] = x;
                        a[2 * w + 1] = y;
                    }
                    part = mfma_rows<false>(a, q_high[m], part);
                    if (two_parts) part = mfma_rows<false>(a, q_low[m], part);
                }
                const f4 d = *reinterpret_cast<const f4*>(scale_area + 16 * blk + 4 * b);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(d[i], part[i], s[i]);
            }
        }
        if (more) {
            locate(next);
            load_keys();
        }

        // ---- terms, masks, softmax ----
        const bool masked = !(half * 16 >= col.all_from && half * 16 + 15 <= col.all_to);  // uniform
        ScoreMap map = map_scores<CAP, true, 4>(s, cs, cc, P);
        float x[4] = {s[0], s[1], s[2], s[3]}, p[4];
        if (sloped) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(-col.slope2, fabsf((float)(col.pos - (pos + i))), __builtin_fmaf(x[i], map.ca, map.cb));
            map = ScoreMap{1.0f, 0.f};
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pos + i >= col.lo && pos + i <= col.hi ? x[i] : -INFINITY;
        }
        const float top = max_over_rows(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        const float m_new = fmaxf(m_run, __builtin_fmaf(top, map.ca, map.cb));
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], map.ca, map.cb - m_new));
            sum += p[i];
        }
        l_run = l_run * alpha + sum;
        if (__ballot(alpha != 1.0f) != 0ull) {
#pragma unroll
            for (int k = 0; k < R::kGroups * R::kJ; ++k) o[k] *= alpha;
        }

        // ---- values ----
        // rows that no live column sees count as zeros: they may hold anything
        bool row_ok[4] = {true, true, true, true};
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) row_ok[i] = any_of_row(pos + i >= col.lo && pos + i <= col.hi, b);
        }
        u4 w;
        if constexpr (R::k16) {
            if constexpr (IS_BF16) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    w[k] = pack_bf2(p[2 * k], p[2 * k + 1]);
                    w[2 + k] = pack_bf2(p[2 * k] - __uint_as_float(w[k] << 16), p[2 * k + 1] - __uint_as_float(w[k] & 0xFFFF0000u));
                }
            } else {
                uint32_t h0, h1, l0, l1;
                split_weights(p[0], p[1], h0, l0);
                split_weights(p[2], p[3], h1, l1);
                w = u4{h0, h1, l0, l1};
            }
        } else {
            exchange(scale_area + 64, v_scale, v_scales);
        }
#pragma unroll
        for (int g = 0; g < R::kGroups; ++g) {
            if constexpr (!R::k16) {
                const f4 d = *reinterpret_cast<const f4*>(scale_area + 64 + 16 * g + 4 * b);
                float pd[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pd[i] = mul_legacy(p[i] * R::kValueGain, row_ok[i] ? d[i] : 0.f);
                uint32_t h0, h1, l0, l1;
                split_weights(pd[0], pd[1], h0, l0);
                split_weights(pd[2], pd[3], h1, l1);
                w = u4{h0, h1, l0, l1};
            }
            if constexpr (R::k16) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) vr16[g][i][k] = row_ok[i] ? vr16[g][i][k] : 0u;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                    const uint32_t v01 = __builtin_amdgcn_perm(vr16[g][1][j >> 1], vr16[g][0][j >> 1], sel);
                    const uint32_t v23 = __builtin_amdgcn_perm(vr16[g][3][j >> 1], vr16[g][2][j >> 1], sel);
                    o[g * 8 + j] = mfma_rows<IS_BF16>(u4{v01, v23, v01, v23}, w, o[g * 8 + j]);
                }
            } else {
                constexpr int kWords = R::kFp8 ? 2 : 1;
#pragma unroll
                for (int x4 = 0; x4 < kWords; ++x4) {
                    uint32_t c[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (R::kFp8) c[i] = row_ok[i] ? vr8[g][i][x4] : 0u;
                        else c[i] = row_ok[i] ? vr4[g][i] : 0u;
                    }
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {  // two channels: bytes {t0, t1} of one, {t0, t1} of the other
                        const uint32_t sel = jj ? 0x07030602u : 0x05010400u;
                        const uint32_t c01 = __builtin_amdgcn_perm(c[1], c[0], sel), c23 = __builtin_amdgcn_perm(c[3], c[2], sel);
                        uint32_t v01[2], v23[2];
                        if constexpr (R::kFp8) {
                            v01[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c01, 0.00390625f, false));
                            v01[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c01, 0.00390625f, true));
                            v23[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c23, 0.00390625f, false));
                            v23[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c23, 0.00390625f, true));
                        } else {  // 0x4800 | (q + 128) is 9 + q / 128 in fp16
                            const uint32_t u01 = c01 ^ 0x80808080u, u23 = c23 ^ 0x80808080u;
                            const h2 bias = {(_Float16)9.0f, (_Float16)9.0f};
                            const auto wide = [&](uint32_t u, uint32_t s2) {
                                return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x48484848u, u, s2)) - bias);
                            };
                            v01[0] = wide(u01, 0x04010400u), v01[1] = wide(u01, 0x04030402u);
                            v23[0] = wide(u23, 0x04010400u), v23[1] = wide(u23, 0x04030402u);
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            f4& acc = o[g * R::kJ + 4 * x4 + 2 * jj + k];
                            acc = mfma_rows<false>(u4{v01[k], v23[k], v01[k], v23[k]}, w, acc);
                        }
                    }
                }
            }
        }
        if (more) load_values();
        half = next;
    }
    l_run = sum_over_rows(l_run);

    // ---- the waves' states joined ----
    float* ml = reinterpret_cast<float*>(smem + M::kMl);
    if constexpr (!R::k16) __syncthreads();  // the query columns are not read any more
    float* region = reinterpret_cast<float*>(smem + wave * M::kRegion);
    if (col.ok) {
#pragma unroll
        for (int k = 0; k < R::kGroups * R::kJ; ++k) *reinterpret_cast<f4*>(region + n * M::kColStride + 16 * k + 4 * b) = o[k];
        if (b == 0) *reinterpret_cast<f2*>(ml + (wave * 16 + n) * 2) = f2{m_run, l_run};
    }
    __syncthreads();
    join_waves<TQ, HD, R::kJ, 16>(P, s0, kv_sub, head0, col.live, wave, lane, smem, M::kRegion, ml, reinterpret_cast<float*>(smem + M::kReorder + wave * HD * 4),
                                  1.0f);
}

}  // namespace w34
