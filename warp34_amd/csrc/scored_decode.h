// Scored paged attention of few query columns for each kv head: one new token, or the tokens of a verify step.
//
// Workgroup = one chunk of one tile's keys x one kv head, eight waves; a wave takes every eighth half unit (16 keys) of the chunk:
//   S^T = K Q^T      16x16x32 MFMAs, A = 16 key rows (lane (n, b): row n), B = query columns; lane (n, b) gets the scores of keys
//                    4 b .. 4 b + 3 for column n, so that the softmax state of a column is a scalar of four lanes
//   O^T += V^T P^T   A = channels x keys, B = the weights where they stand: each weight has a high and a low 16-bit part in the two
//                    halves of a product of 32 keys, over the same values, so it loses nothing
// Rows go from the pages to registers as they are stored; key loads of the next half unit travel during the softmax and the value
// product, value loads during the next scores.  Only the scales of quantised rows and the TQ4 look-ups go through LDS.
// At the end the waves' states are joined through LDS, and the chunks' by scored_join_kernel.
#pragma once

#include "scored_attn.h"

namespace w34 {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef u4 u4_at4 __attribute__((aligned(4)));
typedef u4 u4_at2 __attribute__((aligned(2)));
typedef uint32_t u1_at2 __attribute__((aligned(2)));
typedef u2v u2_at4 __attribute__((aligned(4)));

constexpr int kScoredWaves = 8;

// TQ4 keys: the look-ups' fp16 numbers are up to 9.4e-5 from the centroids, which would be 1e-4 of a score and 2e-5 of a row's lse where a
// few keys carry it.  So the keys have a table of their own behind the other, entries of eight bytes: the pair of the first table and the
// pair of what is missing, 32 copies (a read of eight bytes goes by 32 lanes at a time).
constexpr int kKeyTable = 65536;
__host__ __device__ constexpr uint32_t centroid_rest_of(int code) {
    return __builtin_bit_cast(uint16_t, (_Float16)(kLutGain * kCentroids[code] - (float)(_Float16)(kLutGain * kCentroids[code])));
}
__device__ __forceinline__ uint32_t centroid_rest(uint32_t code) {
    uint32_t r = centroid_rest_of(0);
#pragma unroll
    for (int c = 1; c < 16; ++c) r = code == (uint32_t)c ? centroid_rest_of(c) : r;
    return r;
}
__device__ __forceinline__ void build_key_table(uint8_t* smem, int tid, int wave) {  // by 512 threads, as build_pair_table
    const uint32_t code = (uint32_t)tid >> 4 & 15u, lo = centroid_bits(code), lo_rest = centroid_rest(code);
    const bool odd = (wave >> 2) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t v = lo | (odd ? centroid_bits_of(2 * i + 1) << 16 : centroid_bits_of(2 * i) << 16);
        const uint32_t w = lo_rest | (odd ? centroid_rest_of(2 * i + 1) << 16 : centroid_rest_of(2 * i) << 16);
        *reinterpret_cast<u4*>(smem + kKeyTable + (tid + 512 * i) * 16) = u4{v, w, v, w};
    }
}
typedef __attribute__((address_space(3))) const u2v lds_cu2;
// lane_bits: (lane % 32) * 8 | 0x100, whose second byte is the table's place
__device__ __forceinline__ u2v key_read(uint32_t code_word, uint32_t lane_bits, int byte) {
    return *reinterpret_cast<lds_cu2*>((uintptr_t)__builtin_amdgcn_perm(code_word, lane_bits, 0x0c010400u + ((uint32_t)byte << 8)));
}

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
    static constexpr int kKeyRegs = kTq4 ? 2 : k16 ? kOps : 4;  // of 16 bytes
    // what the values in the operands are to be multiplied by: TQ4 look-ups hold kLutGain times the centroid, 8-bit codes come as
    // code / 256 (E4M3) or code / 128, which keeps the low part of a weight, times that gain, out of fp16's subnormal range
    static constexpr float kValueGain = kFp8 ? 256.0f : kQ8 ? 128.0f : 1.0f;
    static constexpr float kOutScale = kTq4 ? kLutInvGain : 1.0f;
    __device__ static constexpr int element(int m, int b) {
        return kTq4 ? 128 * (m >> 2) + 32 * b + 8 * (m & 3) : k16 ? 32 * m + 8 * b : 64 * (m >> 1) + 16 * b + 8 * (m & 1);
    }
};

// LDS: [TQ4 tables][query columns], over which the counts of the tiles lie at the start and the waves' regions and the joined columns at
// the end; [(m, l) of the waves][scales of the waves]
template <int KVF, int HD>
struct ScoredLds {
    using R = ScoredRows<KVF, HD>;
    static constexpr int kColStride = HD + 8;                     // floats of a column in a region
    static constexpr int kRegion = 16 * kColStride * 4;
    static constexpr int kTable = R::kTq4 ? 2 * kKeyTable : 0;
    static constexpr int kQStride = HD + 8;                       // 16-bit elements
    static constexpr int kQ = kTable, kQLow = kQ + 16 * kQStride * 2, kQScale = kQLow + 16 * kQStride * 2;
    static constexpr int kJoined = kScoredWaves * kRegion;
    static constexpr int kLoopEnd = kQScale + 64;
    static constexpr int kMl = kJoined + kRegion > kLoopEnd ? kJoined + kRegion : kLoopEnd;
    static constexpr int kScale = kMl + kScoredWaves * 16 * 8;
    static constexpr int kBytes = kScale + kScoredWaves * 2 * 4 * 16 * 4;
    static_assert(kBytes <= 160 * 1024 && kMaxSplitEntries * 4 <= kJoined, "decode LDS budget");
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
    const warp34_kv_layer_layout& L = P.L;
    const warp34_attention_batch& B = P.B;
    const int kv_sub = (int)blockIdx.y;
    const int kv_head = P.q_subgroups == 1 ? kv_sub : fast_div(kv_sub, P.q_subgroups);
    const int head0 = kv_head * P.gqa + (kv_sub - kv_head * P.q_subgroups) * P.q_group;

    // ---- what this workgroup works on ----
    ScoredWork work = {(int)blockIdx.x, 0, 1, 0};
    ScoredTile t;
    if (P.target > 0 && P.entries <= 64) {  // lane e: entry e, all a wave has to know
        ScoredTile mine = {0, 0, 0, 0, 0};
        if (lane < P.entries) mine = scored_tile(P, lane);
        const int halves = lane < P.entries ? tile_halves_guess(P, mine) : -1;
        const auto count = [&](int) { return halves; };
        const int per = chunk_length(P, lane, count);
        work = find_work(P, per, (int)blockIdx.x, lane, count);
        if (work.entry < 0) return;
        const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, work.entry); };
        t = ScoredTile{of(mine.req), of(mine.tok0), of(mine.tokens), of(mine.pos0), of(mine.seq_after)};
    } else {
        if (P.target > 0) {
            int* halves = reinterpret_cast<int*>(smem);
            for (int e = tid; e < P.entries; e += kScoredWaves * 64) halves[e] = tile_halves_guess(P, scored_tile(P, e));
            __syncthreads();
            const auto count = [&](int e) { return halves[e]; };
            const int per = chunk_length(P, lane, count);
            work = find_work(P, per, (int)blockIdx.x, lane, count);
            if (work.entry < 0) return;
            __syncthreads();  // the counts lie where the tables come
        }
        t = scored_tile(P, work.entry);
        if (t.tokens <= 0) return;
    }
    int key_first, key_last;
    tile_keys(P, t, lane, key_first, key_last);
    if (work.chunk == 0 && kv_sub == 0 && tid == 0 && P.target > 0) {
        P.table[2 * work.entry] = work.first_record;
        P.table[2 * work.entry + 1] = work.chunks;
    }
    const int all_halves = tile_halves(key_first, key_last);
    const int per = fast_div(all_halves + work.chunks - 1, work.chunks);
    const int begin = (key_first >> 4) + work.chunk * per;
    const int end = key_first > key_last ? begin : max(begin, min(begin + per, (key_last >> 4) + 1));

    // ---- this lane's column ----
    const int my_t = column_token(n, P);
    const int my_tok = min(t.tok0 + my_t, B.total_tokens - 1);
    const bool col_ok = my_t < t.tokens && (B.valid_token_mask == nullptr || B.valid_token_mask[my_tok] != 0);
    const int my_head = head0 + (n - my_t * P.q_group);
    const int my_pos = t.pos0 + my_t;
    int lo = 0, hi = -1;
    if (col_ok) token_keys(P, my_tok, my_pos, t.seq_after, lo, hi);
    int all_from = col_ok ? lo : 0, all_to = col_ok ? hi : 0x7fffffff;  // keys that every live column sees
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        all_from = max(all_from, __shfl_xor(all_from, d, 64));
        all_to = min(all_to, __shfl_xor(all_to, d, 64));
    }
    all_from = __builtin_amdgcn_readfirstlane(all_from);
    all_to = __builtin_amdgcn_readfirstlane(all_to);
    const uint32_t live = (uint32_t)(__ballot(col_ok) & 0xFFFFull);
    if (live == 0u) return;
    const float slope2 = P.slopes != nullptr && col_ok ? P.slopes[my_head] * kLog2e : 0.f;
    const bool sloped = P.slopes != nullptr;

    // ---- TQ4 table, query operands ----
    if constexpr (R::kTq4) {
        build_pair_table(smem, tid, wave);
        build_key_table(smem, tid, wave);
    }
    u4 q_high[R::kOps], q_low[R::kOps];
    float cs = P.scale2, cc = P.cap_arg;
    if constexpr (R::k16) {
        const uint16_t* src = P.q + ((size_t)my_tok * P.num_q_heads + (size_t)min(my_head, P.num_q_heads - 1)) * HD;
#pragma unroll
        for (int m = 0; m < R::kOps; ++m) {
            q_high[m] = *reinterpret_cast<const u4*>(src + R::element(m, b)) ^ P.q_flip;
            if (!col_ok) q_high[m] = u4{0u, 0u, 0u, 0u};
        }
    } else {
        // A wave brings two columns: rotated where the keys are, relative to a power of two above their largest element so that
        // fp16 holds them whatever their size, in two parts (the second is zero where nothing is rotated: 11 bits are all there are).
        uint16_t* qh = reinterpret_cast<uint16_t*>(smem + M::kQ);
        uint16_t* ql = reinterpret_cast<uint16_t*>(smem + M::kQLow);
        float* qs = reinterpret_cast<float*>(smem + M::kQScale);
#pragma unroll
        for (int c = wave; c < 16; c += kScoredWaves) {
            const int ct = column_token(c, P);
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if ((live >> c) & 1u) {
                const uint16_t* src = P.q + ((size_t)(t.tok0 + ct) * P.num_q_heads + (size_t)(head0 + c - ct * P.q_group)) * HD + 4 * lane;
                uint2 raw = *reinterpret_cast<const uint2*>(src);
                raw.x ^= P.q_flip, raw.y ^= P.q_flip;
                v[0] = TQ::to_f32((uint16_t)raw.x), v[1] = TQ::to_f32((uint16_t)(raw.x >> 16));
                v[2] = TQ::to_f32((uint16_t)raw.y), v[3] = TQ::to_f32((uint16_t)(raw.y >> 16));
            }
            if (P.rot_q) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = apply_sign(v[k], 4 * lane + k);
                wht256_wave(v, lane);
            }
            float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
            top = wave_top(top);
            const int e = top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_ldexpf(v[k], -e);
            uint32_t h0, h1, l0, l1;
            split_weights(v[0], v[1], h0, l0);
            split_weights(v[2], v[3], h1, l1);
            *reinterpret_cast<uint2*>(qh + c * M::kQStride + 4 * lane) = uint2{h0, h1};
            *reinterpret_cast<uint2*>(ql + c * M::kQStride + 4 * lane) = uint2{l0, l1};
            if (lane == 0) qs[c] = __builtin_amdgcn_ldexpf(1.0f, e);
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < R::kOps; ++m) {
            q_high[m] = *reinterpret_cast<const u4*>(qh + n * M::kQStride + R::element(m, b));
            q_low[m] = *reinterpret_cast<const u4*>(ql + n * M::kQStride + R::element(m, b));
        }
        const float mine = qs[n] * R::kOutScale;
        cs *= mine;
        cc *= mine;
    }
    const bool two_parts = !R::k16 && P.rot_q != 0;

    // ---- rows ----
    const slab_byte* k_slab = slab_at(L.k_base) + (uint64_t)(uint32_t)kv_head * L.k_head_stride_bytes;
    const slab_byte* v_slab = slab_at(L.v_base) + (uint64_t)(uint32_t)kv_head * L.v_head_stride_bytes;
    const int32_t* blocks = B.block_tables + (size_t)t.req * B.max_blocks_per_req;
    int slot_base = page_slot(begin * 16, P);
    int pages = slot_base + lane < B.max_blocks_per_req ? blocks[slot_base + lane] : 0;  // 64 entries of the block table
    const slab_byte* k_rows;
    const slab_byte* v_rows;
    const auto locate = [&](int half) {
        const int pos = half * 16, slot = page_slot(pos, P);
        if (slot - slot_base >= 64) {  // uniform
            slot_base = slot;
            pages = slot_base + lane < B.max_blocks_per_req ? blocks[slot_base + lane] : 0;
        }
        const uint32_t page = (uint32_t)max(__builtin_amdgcn_readlane(pages, slot - slot_base), 0);
        const uint32_t in_page = (uint32_t)(pos - slot * L.block_size) * (uint32_t)R::kRowBytes;
        k_rows = k_slab + (uint64_t)page * L.k_page_stride_bytes + in_page;
        v_rows = v_slab + (uint64_t)page * L.v_page_stride_bytes + in_page;
    };
    u4 kr[R::kKeyRegs];
    uint32_t k_scale = 0, v_scale = 0;   // TQ4: of row n, block b & 1; Q8_0: of row n, block b
    u2v k_scales = {0u, 0u}, v_scales = {0u, 0u};  // FP8: both of row n
    u4 vr16[R::k16 ? R::kGroups : 1][4];
    u2v vr8[R::kFp8 ? 2 : 1][4];
    uint32_t vr4[R::kQ8 ? 4 : R::kTq4 ? 2 : 1][4];
    const auto load_keys = [&]() {
        const slab_byte* row = k_rows + (uint32_t)(n * R::kRowBytes);
        if constexpr (R::k16) {
#pragma unroll
            for (int m = 0; m < R::kOps; ++m) kr[m] = load_as<u4>(row + 64 * m + 16 * b);
        } else if constexpr (R::kTq4) {
#pragma unroll
            for (int h = 0; h < 2; ++h) kr[h] = load_as<u4_at2>(row + 66 * h + 2 + 16 * b);
            k_scale = load_as<uint16_t>(row + 66 * (b & 1));
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
            } else if constexpr (R::kTq4) {
#pragma unroll
                for (int g = 0; g < 2; ++g) vr4[g][i] = load_as<u1_at2>(row + 66 * g + 2 + 4 * n);
            } else if constexpr (R::kFp8) {
#pragma unroll
                for (int g = 0; g < 2; ++g) vr8[g][i] = load_as<u2_at4>(row + 128 * g + 8 * n);
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) vr4[g][i] = load_as<uint32_t>(row + 68 * g + 4 + 4 * n);
            }
        }
        const slab_byte* row = v_rows + (uint32_t)(n * R::kRowBytes);
        if constexpr (R::kTq4) v_scale = load_as<uint16_t>(row + 66 * (b & 1));
        if constexpr (R::kFp8) v_scales = load_as<u2_at4>(row + 256);
        if constexpr (R::kQ8) v_scale = load_as<uint32_t>(row + 68 * b);
    };
    // Block scales are loaded a row a lane and used four rows a lane: an exchange through 256 bytes of LDS for each kind.
    float* scale_area = reinterpret_cast<float*>(smem + M::kScale + wave * (2 * 4 * 16 * 4));
    const auto exchange = [&](float* area, uint32_t one, u2v two) {
        if constexpr (R::kTq4) {
            if (b < 2) area[16 * b + n] = F16::to_f32((uint16_t)one);
        } else if constexpr (R::kFp8) {
            if (b < 2) area[16 * b + n] = __uint_as_float(b == 0 ? two[0] : two[1]);
        } else if constexpr (R::kQ8) {
            area[16 * b + n] = __uint_as_float(one);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };
    const uint32_t lut_lane = (uint32_t)lane << 2, key_lane = ((uint32_t)lane & 31u) << 3 | 0x100u;

    f4 o[R::kGroups * R::kJ];
#pragma unroll
    for (int k = 0; k < R::kGroups * R::kJ; ++k) o[k] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNegBig, l_run = 0.f;

    int half = begin + wave;
    if (half < end) {
        locate(half);
        load_keys();
        load_values();
    }
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
                    u4 a, rest;
                    if constexpr (R::kTq4) {
                        const uint32_t word = kr[m >> 2][m & 3];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const u2v pair = key_read(word, key_lane, k);
                            a[k] = pair[0];
                            rest[k] = pair[1];
                        }
                    } else {
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
                    }
                    part = mfma_rows<false>(a, q_high[m], part);
                    if constexpr (R::kTq4) part = mfma_rows<false>(rest, q_high[m], part);
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
        const bool masked = !(half * 16 >= all_from && half * 16 + 15 <= all_to);  // uniform
        ScoreMap map = map_scores<CAP, 4>(s, cs, cc, P);
        float x[4] = {s[0], s[1], s[2], s[3]}, p[4];
        if (sloped) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(-slope2, fabsf((float)(my_pos - (pos + i))), __builtin_fmaf(x[i], map.ca, map.cb));
            map = ScoreMap{1.0f, 0.f};
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pos + i >= lo && pos + i <= hi ? x[i] : -INFINITY;
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
        // rows that no token of the tile sees count as zeros: a page's rest may hold anything
        bool row_ok[4] = {true, true, true, true};
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) row_ok[i] = pos + i >= key_first && pos + i <= key_last;
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
            if constexpr (R::kTq4) {
                uint32_t even[2], odd[2];  // of tokens 0, 1 and of 2, 3: a byte = code of the first | code of the second << 4
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    const uint32_t wa = vr4[g][2 * t2], wb = vr4[g][2 * t2 + 1];
                    even[t2] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    odd[t2] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sel = 0x0c0c0400u + ((uint32_t)(j >> 1) << 8);
                    const uint32_t v01 = lut_read((j & 1) ? odd[0] : even[0], lut_lane, sel);
                    const uint32_t v23 = lut_read((j & 1) ? odd[1] : even[1], lut_lane, sel);
                    o[g * 8 + j] = mfma_rows<false>(u4{v01, v23, v01, v23}, w, o[g * 8 + j]);
                }
            } else if constexpr (R::k16) {
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

    // ---- the waves' states joined: regions of 16 columns, a column in the order of the accumulators ----
    float* ml = reinterpret_cast<float*>(smem + M::kMl);
    __syncthreads();  // table and query columns are not read any more
    float* region = reinterpret_cast<float*>(smem + wave * M::kRegion);
#pragma unroll
    for (int k = 0; k < R::kGroups * R::kJ; ++k) *reinterpret_cast<f4*>(region + n * M::kColStride + 16 * k + 4 * b) = o[k];
    if (b == 0) *reinterpret_cast<f2*>(ml + (wave * 16 + n) * 2) = f2{m_run, l_run};
    __syncthreads();
    float* joined = reinterpret_cast<float*>(smem + M::kJoined);
    constexpr int kPieces = HD / 4;                       // of four floats
    constexpr int kStep = kScoredWaves * 64 / 16;         // threads of a column
    const int col = tid / kStep;
    float m_col = kNegBig;
#pragma unroll
    for (int w = 0; w < kScoredWaves; ++w) m_col = fmaxf(m_col, ml[(w * 16 + col) * 2]);
    float weight[kScoredWaves], l_col = 0.f;
#pragma unroll
    for (int w = 0; w < kScoredWaves; ++w) {
        weight[w] = __builtin_amdgcn_exp2f(ml[(w * 16 + col) * 2] - m_col);
        l_col += weight[w] * ml[(w * 16 + col) * 2 + 1];
    }
#pragma unroll
    for (int piece = tid % kStep; piece < kPieces; piece += kStep) {
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kScoredWaves; ++w)
            acc += *reinterpret_cast<const f4*>(smem + w * M::kRegion + (col * M::kColStride + 4 * piece) * 4) * weight[w];
        const int k = piece >> 2, g = k / R::kJ, j = k % R::kJ, r = 4 * (piece & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) joined[col * M::kColStride + 16 * R::kJ * g + R::kJ * (r + i) + j] = acc[i];
    }
    __syncthreads();
    if (tid % kStep == 0) {
        ml[col * 2] = m_col;  // (wave 0's states: read by everybody before the barrier)
        ml[col * 2 + 1] = l_col;
    }
    __syncthreads();
    const int kv_subs = (int)gridDim.y;
    for (int c = wave; c < 16; c += kScoredWaves) {
        if (!((live >> c) & 1u)) continue;
        const f4 acc = *reinterpret_cast<const f4*>(joined + c * M::kColStride + ((4 * lane) & (HD - 1)));
        const float m_c = ml[2 * c], l_c = ml[2 * c + 1];
        if (work.chunks > 1) {
            const size_t record = ((size_t)(work.first_record + work.chunk) * kv_subs + kv_sub) * 16 + c;
            if (4 * lane < HD) *reinterpret_cast<f4*>(P.part_acc + record * HD + 4 * lane) = acc;
            if (lane == 0) *reinterpret_cast<f2*>(P.part_ml + 2 * record) = f2{m_c, l_c};
        } else {
            float v[4] = {acc[0], acc[1], acc[2], acc[3]};
            const int ct = column_token(c, P);
            finish_row<TQ, HD>(P, t.tok0 + ct, head0 + c - ct * P.q_group, lane, v, m_c, l_c, R::kOutScale);
        }
    }
}

}  // namespace w34
