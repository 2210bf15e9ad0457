// Scored paged attention of up to eight query columns over TQ4 rows.
//
// The work of a wave is 32 keys (a unit) at a time.  What would be products with half of their columns empty carries second parts:
//   S^T = K Q^T      columns 0..7 of B are the high parts of the eight queries, 8..15 their low parts, and a look-up gives the high and
//                    the low part of two centroids: one product of 16 keys x 16 channels is all four products of parts.  A score is the
//                    sum of columns n and n + 8.
//   O^T += V^T P^T   columns 0..7 are the high parts of the weights of 32 keys, 8..15 the low parts, both over the same values.
// Operands are the look-ups as they come: a byte of a row is two codes, its table entry the pair of fp16 numbers.
//
// (As the 16-column kernel with the parts in products of their own, 16 keys at a time: 300 vector instructions and 40 products for what
// takes 170 and 24 here, 209 us for 32 requests of 1k to 64k keys.)  Now 147 to 156 us, 3.9 to 4.1 TB/s: vector work 53 % of the SIMD cycles, products
// 18 %, look-ups 40 % of the LDS cycles and a wave waits a third; waves a barrier apart at most 165 to 203 us, so what overlaps is waves out of
// step.  One request of 131 072 keys, capped, 29.2 us: 12.5 stream 69 MB at 5.5 TB/s, 5.6 pass before (lengths 1.6, pages and first rows 3.6), the waves' join
// takes 3, the join's launch 5 to 6.
#pragma once

#include "scored_decode.h"

namespace w34 {

typedef u4 u4_at2 __attribute__((aligned(2)));
typedef uint32_t u1_at2 __attribute__((aligned(2)));

constexpr int kTq4Cols = 8;

// The table: entries of eight bytes, the pair of fp16 numbers of a byte's two codes and the pair of what they are short of the centroids;
// 32 copies (a read goes by 32 lanes at a time).  The fp16 numbers are up to 9.4e-5 from the centroids, which would be 1e-4 of a score and
// 2e-5 of a row's lse where a few keys carry it: keys take both, values the first alone.
// What centroids are multiplied by: with kLutGain alone the second parts of small ones would be below fp16's smallest normal number.
constexpr float kTableGain = 4096.0f * kLutGain, kTableInvGain = kLutInvGain / 4096.0f;
struct TwoPartPairs {
    u2v of[256];
};
constexpr TwoPartPairs make_two_part_pairs() {
    TwoPartPairs t{};
    for (int e = 0; e < 256; ++e) {
        uint32_t v = 0, w = 0;
        for (int k = 0; k < 2; ++k) {
            const float c = kTableGain * kCentroids[e >> (4 * k) & 15];
            const _Float16 hi = (_Float16)c;
            v |= (uint32_t)__builtin_bit_cast(uint16_t, hi) << (16 * k);
            w |= (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(c - (float)hi)) << (16 * k);
        }
        t.of[e] = u2v{v, w};
    }
    return t;
}
__device__ __constant__ constexpr TwoPartPairs kTwoPartPairs = make_two_part_pairs();
// By 512 threads, 16 bytes at tid + 512 i of the table: entries (tid >> 4) + 32 i, which travel while the batch is planned.
struct TableEntries {
    u2v of[8];
    __device__ __forceinline__ void load(int tid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) of[i] = kTwoPartPairs.of[(tid >> 4) + 32 * i];
    }
    __device__ __forceinline__ void store(uint8_t* smem, int tid) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<u4*>(smem + (tid + 512 * i) * 16) = u4{of[i][0], of[i][1], of[i][0], of[i][1]};
    }
};
typedef __attribute__((address_space(3))) const u2v lds_cu2;
// table_lane: the place of the lane's copy, (lane % 32) * 8; the table lies at 0
__device__ __forceinline__ u2v key_read(uint32_t code_word, uint32_t table_lane, int byte) {
    return *reinterpret_cast<lds_cu2*>((uintptr_t)__builtin_amdgcn_perm(code_word, table_lane, 0x0c0c0400u + ((uint32_t)byte << 8)));
}

// fp16(w), or what that leaves of w where low is 1, of two weights
__device__ __forceinline__ uint32_t weight_part(float a, float b, float low) {
    const uint32_t high = pack_h2(a, b);
    float r0, r1;
    asm("v_fma_mix_f32 %0, -%2, %3, %1 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(a), "v"(high), "v"(low));
    asm("v_fma_mix_f32 %0, -%2, %3, %1 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(b), "v"(high), "v"(low));
    return pack_h2(r0, r1);
}

// LDS: [table][query columns], over which the counts of the tiles lie at the start and the waves' regions at the end; [a
// finished column of each wave][(m, l) of the waves][scales of the waves]
struct Tq4Lds {
    static constexpr int kColStride = 256 + 8, kRegion = kTq4Cols * kColStride * 4;
    static constexpr int kQStride = 256 + 8;
    static constexpr int kQ = 65536, kQLow = kQ + kTq4Cols * kQStride * 2, kQScale = kQLow + kTq4Cols * kQStride * 2;
    static constexpr int kLoopEnd = kQScale + 64, kReorder = kLoopEnd > kScoredWaves * kRegion ? kLoopEnd : kScoredWaves * kRegion;
    static constexpr int kMl = kReorder + kScoredWaves * 256 * 4;
    static constexpr int kScale = kMl + kScoredWaves * 16 * 8;
    static constexpr int kBytes = kScale + kScoredWaves * 2 * 64 * 4;
    static_assert(kBytes <= 160 * 1024 && kMaxSplitEntries * 4 <= kQ, "decode LDS budget");
};

template <typename TQ, bool CAP>
__global__ __launch_bounds__(kScoredWaves * 64, 1) void scored_decode_tq4_kernel(const ScoredParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    using M = Tq4Lds;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, b = lane >> 4;
    const int kv_sub = (int)blockIdx.y;
    const int kv_head = P.q_subgroups == 1 ? kv_sub : fast_div(kv_sub, P.q_subgroups);
    const int head0 = kv_head * P.gqa + (kv_sub - kv_head * P.q_subgroups) * P.q_group;

    TableEntries entries;
    entries.load(tid);
    DecodeStart s0;
    if (!decode_start<true>(P, smem, tid, lane, kv_sub, s0)) return;
    const int end = s0.end;
    PageWalk walk;
    walk.start(P, s0.t, kv_head, s0.begin, lane);

    // ---- rows of a unit: half units `half` and `half + 1` (the same again where the tile ends before it: its keys are hidden) ----
    u4 kr[2][2];              // [half][block]: row n, codes 32 b .. 32 b + 31 of the block
    uint32_t vr[2][2][4];     // [half][block][i]: row 4 b + i, codes 8 n .. 8 n + 7 of the block
    uint32_t k_scale, v_scale;  // half b >> 1, row n, block b & 1
    const slab_byte* k_rows[2];
    const slab_byte* v_rows[2];
    const auto locate = [&](int half) {
        walk.locate(P, half, 132, lane, k_rows[0], v_rows[0]);
        walk.locate(P, half + 1 < end ? half + 1 : half, 132, lane, k_rows[1], v_rows[1]);
    };
    const auto load_keys = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) kr[h][blk] = load_as<u4_at2>(k_rows[h] + (uint32_t)(n * 132 + 16 * b + 66 * blk + 2));
        k_scale = load_as<uint16_t>((b < 2 ? k_rows[0] : k_rows[1]) + (uint32_t)(n * 132 + 66 * (b & 1)));
    };
    const auto load_values = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) vr[h][blk][i] = load_as<u1_at2>(v_rows[h] + (uint32_t)(b * 528 + 4 * n + 132 * i + 66 * blk + 2));
        v_scale = load_as<uint16_t>((b < 2 ? v_rows[0] : v_rows[1]) + (uint32_t)(n * 132 + 66 * (b & 1)));
    };
    QueryColumns<TQ, kTq4Cols, M::kQStride> columns;
    columns.load(P, s0.t, head0, wave, lane);

    const DecodeColumn col = decode_column(P, s0.t, head0, n & 7);
    const uint32_t live = col.live & 0xFFu;
    if (live == 0u) return;
    const bool sloped = P.slopes != nullptr;

    // ---- table, first loads, query operands ----
    entries.store(smem, tid);
    int half = s0.begin + 2 * wave;
    columns.arrived();
    if (half < end) {
        locate(half);
        load_keys();
        load_values();
    }
    uint16_t* qh = reinterpret_cast<uint16_t*>(smem + M::kQ);
    uint16_t* ql = reinterpret_cast<uint16_t*>(smem + M::kQLow);
    float* qs = reinterpret_cast<float*>(smem + M::kQScale);
    columns.bring(P, live, wave, lane, qh, ql, qs);
    __syncthreads();
    u4 q[16];  // [block][word of the row][half of the word]
#pragma unroll
    for (int m = 0; m < 8; ++m) {
        const u4 w = *reinterpret_cast<const u4*>((n < 8 ? qh : ql) + (n & 7) * M::kQStride + 128 * (m >> 2) + 32 * b + 8 * (m & 3));
        q[2 * m] = u4{w[0], w[0], w[1], w[1]};
        q[2 * m + 1] = u4{w[2], w[2], w[3], w[3]};
    }
    const float cs = score_factor(P, qs[n & 7] * kTableInvGain), cc = cap_factor(P, qs[n & 7] * kTableInvGain);
    const float low_part = n < 8 ? 0.f : 1.f;
    const uint32_t table_lane = ((uint32_t)lane & 31u) << 3;

    // Scales are loaded a row a lane and used four rows a lane: an exchange through LDS, [half][block][16 rows].
    float* k_area = reinterpret_cast<float*>(smem + M::kScale + wave * (2 * 64 * 4));
    float* v_area = k_area + 64;
    const auto exchange = [&](float* area, uint32_t d) {
        area[16 * b + n] = F16::to_f32((uint16_t)d);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };

    f4 o[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNegBig, l_run = 0.f;

    while (half < end) {
        const int next = half + 2 * kScoredWaves;
        const bool more = next < end;
        const int pos = half * 16 + 4 * b;  // of this lane's first key; the second half unit's are 16 further

        // ---- scores ----
        exchange(k_area, k_scale);
        f4 part[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) part[h][blk] = f4{0.f, 0.f, 0.f, 0.f};
        // (look-ups a step ahead of the products: the compiler on its own waits for each, to save registers)
        u4 a[2][4];
        const auto key_operands = [&](int m, int w, u4 (&to)[4]) {
#pragma unroll
            for (int hb = 0; hb < 4; ++hb) {
                const u2v x = key_read(kr[hb >> 1][hb & 1][m], table_lane, 2 * w), y = key_read(kr[hb >> 1][hb & 1][m], table_lane, 2 * w + 1);
                to[hb] = u4{x[0], x[1], y[0], y[1]};
            }
        };
        key_operands(0, 0, a[0]);
#pragma unroll
        for (int mw = 0; mw < 8; ++mw) {
            __builtin_amdgcn_sched_barrier(0);
            if (mw < 7) key_operands((mw + 1) >> 1, (mw + 1) & 1, a[(mw + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int hb = 0; hb < 4; ++hb) part[hb >> 1][hb & 1] = mfma_rows<false>(a[mw & 1][hb], q[8 * (hb & 1) + mw], part[hb >> 1][hb & 1]);
        }
        f4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f4 d0 = *reinterpret_cast<const f4*>(k_area + 32 * h + 4 * b), d1 = *reinterpret_cast<const f4*>(k_area + 32 * h + 16 + 4 * b);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float mine = __builtin_fmaf(d1[i], part[h][1][i], d0[i] * part[h][0][i]);
                s[h][i] = mine + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(mine), 0x128, 0xF, 0xF, false));  // row_ror:8
            }
        }
        // (behind the last unit the rows stay where they are and are loaded again: a load under a condition would be waited for at once.  The walk
        // cannot be asked for them a second time: the page of the first half unit may lie in front of the entries that it holds by then)
        if (more) locate(next);
        load_keys();

        // ---- terms, masks, softmax ----
        const bool masked = !(half * 16 >= col.all_from && half * 16 + 31 <= col.all_to);  // uniform
        float x[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]}, p[8];
        ScoreMap map = map_scores<CAP, true, 8>(x, cs, cc, P);
        const auto at = [&](int i) { return pos + (i & 3) + 16 * (i >> 2); };
        if (sloped) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(-col.slope2, fabsf((float)(col.pos - at(i))), __builtin_fmaf(x[i], map.ca, map.cb));
            map = ScoreMap{1.0f, 0.f};
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = at(i) >= col.lo && at(i) <= col.hi ? x[i] : -INFINITY;
        }
        const float top = max_over_rows(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))));
        const float m_new = fmaxf(m_run, __builtin_fmaf(top, map.ca, map.cb));
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], map.ca, map.cb - m_new));
            sum += p[i];
        }
        l_run = l_run * alpha + sum;
        if (__ballot(alpha != 1.0f) != 0ull) {
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] *= alpha;
        }

        // ---- values ----
        exchange(v_area, v_scale);
        uint32_t codes[2][2][2][2];  // [block][of even, of odd channels][half][pair of rows]: a byte = code of the first row | code of the second << 4
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    const uint32_t wa = vr[h][blk][2 * t2], wb = vr[h][blk][2 * t2 + 1];
                    codes[blk][0][h][t2] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    codes[blk][1][h][t2] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                }
        load_values();
        u4 w[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f4 d = *reinterpret_cast<const f4*>(v_area + 32 * h + 16 * blk + 4 * b);
                if (masked) {  // rows that no live column sees count as zeros: they may hold anything
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = any_of_row(at(4 * h + i) >= col.lo && at(4 * h + i) <= col.hi, b) ? d[i] : 0.f;
                }
                float pd[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pd[i] = mul_legacy(p[4 * h + i], d[i]);
                w[blk][2 * h] = weight_part(pd[0], pd[1], low_part);
                w[blk][2 * h + 1] = weight_part(pd[2], pd[3], low_part);
            }
        }
        u4 v[2][2];
        const auto value_operands = [&](int j2, u4 (&to)[2]) {  // of products 2 j2 and 2 j2 + 1
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t sel = 0x0c0c0400u + ((uint32_t)(j2 & 3) << 8);
#pragma unroll
                for (int x = 0; x < 4; ++x) to[k][x] = lut_read(codes[j2 >> 2][k][x >> 1][x & 1], table_lane, sel);
            }
        };
        value_operands(0, v[0]);
#pragma unroll
        for (int j2 = 0; j2 < 8; ++j2) {
            __builtin_amdgcn_sched_barrier(0);
            if (j2 < 7) value_operands(j2 + 1, v[(j2 + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; ++k) o[2 * j2 + k] = mfma_rows<false>(v[j2 & 1][k], w[j2 >> 2], o[2 * j2 + k]);
        }
        half = next;
    }
    l_run = sum_over_rows(l_run);

    // ---- the waves' states joined ----
    __syncthreads();  // tables and query columns are not read any more
    float* ml = reinterpret_cast<float*>(smem + M::kMl);
    float* region = reinterpret_cast<float*>(smem + wave * M::kRegion);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        f4 sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = o[k][i] + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(o[k][i]), 0x128, 0xF, 0xF, false));
        if (n < 8 && col.ok) *reinterpret_cast<f4*>(region + n * M::kColStride + 16 * k + 4 * b) = sum;
    }
    if (n < 8 && b == 0) *reinterpret_cast<f2*>(ml + (wave * 16 + n) * 2) = f2{m_run, l_run};
    __syncthreads();
    join_waves<TQ, 256, 8, kTq4Cols>(P, s0, kv_sub, head0, live, wave, lane, smem, M::kRegion, ml, reinterpret_cast<float*>(smem + M::kReorder + wave * 1024),
                                     kTableInvGain);
}

}  // namespace w34
