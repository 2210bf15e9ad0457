// Scored paged attention of many query columns for each kv head: chunks of prompts.
//
// Workgroup = 256 query columns (tokens x the q heads of a kv head) x a range of keys, eight waves of 32 columns each.  The workgroup
// walks the keys in units of 32, one barrier a unit; between two barriers
//   the rows of a later unit travel from the pages to LDS (LDS-direct loads: no register holds them),
//   every wave multiplies:  S^T = K Q^T and O^T += V^T P^T in 32x32x16 MFMAs, and
//   quantised rows of the next unit are widened into the 16-bit tiles that the products read, between the products of values.
// A lane (n, b) has the scores of column n for the keys (i & 3) + 8 (i >> 2) + 4 b, i = 0 .. 15: eight of them are, where they stand, a
// B operand of the value product over 16 keys, whose A operand comes out of row-major LDS by the transposing reads
// (ds_read_b64_tr_b16: lane l of 16 gets column l of four rows of 16 values).  So both tiles are row-major and nothing is shuffled.
//   key tile    row r, 16-byte piece p at p ^ (r & 15): the operand reads of 16 rows touch all banks
//   value tile  row r, piece p at p ^ 4 (r & 3): the four rows of a transposing read touch all banks
//
// Why this shape: 128 sums and 64 query registers a lane are what two waves a SIMD have room for, and each operand read from LDS serves 32
// columns.  4 requests of 2 048 tokens on 16 384 keys, 16 + 2 heads, capped: BF16 2.36 to 2.42 ms (980 TFLOP/s; a large matrix product of the
// library 1 390), FP8 2.85 to 3.04, TQ4 3.03 (770), Q8_0 3.25.  What bounds it is a wave's own chain: of 6 400 cycles a TQ4 unit the products of a SIMD's
// two waves take 2 050, vector work 54 % of the cycles (a cap's exponential and reciprocal, the weights' exponentials and the widening most of
// it), LDS 34 %, and a wave waits 39 %.  Left out for timing: cap and exponentials -7 %, widening -14 %, operand reads -15 %, all three -36 %;
// the rows' pages made no difference.  Two sums side by side for the scores need 16 registers more than there are (packed documents 107 ->
// 119 us); operands three products ahead the same (TQ4 3.31 ms).  Values a unit later in half of the waves: -5 %; widening between
// products: FP8 -7 %, Q8_0 -9 %, TQ4 -1.5 %.
#pragma once

#include "scored_decode.h"
#include "wht_products.h"

namespace w34 {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4;
typedef __attribute__((address_space(3))) const f4 lds_f4c;

typedef u4 u4_at8 __attribute__((aligned(8)));

constexpr int kChunkWaves = 8;
constexpr int kChunkCols = 32 * kChunkWaves;
constexpr int kChunkUnit = 32;
// A column's maximum is raised only by scores that exceed it by more than this (log2 domain): a weight may be up to 2^8, which costs
// none of its bits, and the multiplication of 128 sums a lane is spared in nearly all units.  us with slack / without: packed documents
// 108 / 114, 9 requests of 300 to 900 BF16 tokens 471 / 488, 4 x 2 048 on 16 384 TQ4 keys 3 078 / 3 136.
constexpr float kChunkSlack = 8.0f;

constexpr int kKeysAhead = 2, kValuesAhead = 2;  // operands are read from LDS so many products before their own

template <bool IS_BF16>
__device__ __forceinline__ f16v mfma_tile(u4 a, u4 b, f16v c) {
    if constexpr (IS_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}
// 16 bytes a lane to LDS: lane l's from base + voffset + IMM to lds + IMM + 16 l
template <int IMM>
__device__ __forceinline__ void load_to_lds(uint32_t voffset, const uint8_t* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3" : : "v"(voffset), "s"(base), "s"(lds), "n"(IMM) : "memory");
}
// The value again where it is asked for: what follows from it is worked out anew in every unit and not kept in registers.
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ const uint8_t* uniform_pointer(const uint8_t* p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32));
    return reinterpret_cast<const uint8_t*>((uintptr_t)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ void chunk_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory"); }
__device__ __forceinline__ u4 lds_u4(uint32_t at) { return *reinterpret_cast<__attribute__((address_space(3))) const u4*>((uintptr_t)at); }
__device__ __forceinline__ uint32_t lds_u1(uint32_t at) { return *reinterpret_cast<lds_cu32*>((uintptr_t)at); }
__device__ __forceinline__ u2v lds_u2(uint32_t at) { return *reinterpret_cast<__attribute__((address_space(3))) const u2v*>((uintptr_t)at); }
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) { return *reinterpret_cast<__attribute__((address_space(3))) const uint16_t*>((uintptr_t)at); }
__device__ __forceinline__ f4 lds_f4(uint32_t at) { return *reinterpret_cast<lds_f4c*>((uintptr_t)at); }
__device__ __forceinline__ void lds_put(uint32_t at, u4 v) { *reinterpret_cast<__attribute__((address_space(3))) u4*>((uintptr_t)at) = v; }

template <int KVF, int HD>
struct ChunkLds {
    using R = ScoredRows<KVF, HD>;
    static constexpr int kRow = 2 * HD;                       // of a tile
    static constexpr int kTile = kChunkUnit * kRow;           // keys or values
    static constexpr int kTable = R::kTq4 ? 256 * 128 : 0;
    static constexpr int kTiles = kTable;                     // two units of keys
    static constexpr int kValues = kTiles + 2 * kTile;        // three units of values
    static constexpr int kRun = 16 * R::kRowBytes;            // of a page
    static constexpr int kRawUnit = R::k16 ? 0 : (4 * kRun + 16);
    static constexpr int kRaw = kTiles + 5 * kTile;           // two units of {keys 0-15, 16-31, values 0-15, 16-31} as stored
    static constexpr int kScale = kRaw + 2 * kRawUnit;        // two units of key scales [4][32]
    static constexpr int kLoop = kScale + (R::k16 ? 0 : 2 * 4 * 32 * 4);
    // before the loop: tile counts of the batch; eight query columns of each wave at a time.  After it: eight columns of sums.
    static constexpr int kColStride = HD + 8;
    static constexpr int kCounts = kTiles + kChunkWaves * 8 * kColStride * 4;
    static constexpr int kQScale = kCounts + kMaxSplitEntries * 4;
    static constexpr int kHist = kQScale + kChunkCols * 4;
    static constexpr int kEnds = kHist + 64 * 4;
    static constexpr int kRanges = kLoop > kEnds ? kLoop : kEnds;  // first and last key of each token, where a tile has gaps
    static constexpr int kBytes = kRanges + kChunkCols * 8;
    static_assert(kBytes <= 160 * 1024 && kRun % 16 == 0, "chunk LDS budget");
};

// TQ4: the pair table (a byte's two codes, as fp16) in 32 copies.
__device__ __forceinline__ void build_narrow_table(uint8_t* smem, int tid, int wave) {  // by 512 threads: 16 bytes at tid + 512 i, entries (tid >> 3) + 64 i
    const uint32_t lo = centroid_bits((uint32_t)tid >> 3 & 15u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = lo | centroid_bits((uint32_t)(wave >> 1) + 4u * i) << 16;
        *reinterpret_cast<u4*>(smem + (tid + 512 * i) * 16) = u4{v, v, v, v};
    }
}

// Roundings, beside those of the inputs' types: rotated queries and TQ4 keys are one fp16 part (the keys' block scales multiply the
// scores in 32 bits); quantised values are fp16(scale * code), TQ4 ones from the fp16 table; weights are one operand of the values'
// type.  (Weights that carry the block scales would spare the values' rounding and need two parts, half as many products again: a
// block-wide error of a weight is gathered in one channel by the rotation back.)  l adds up the weights before that rounding: lse keeps its
// 32 bits, and a row's average has the roundings of its weights.  2-norm of the error: rotated rows 4.5e-4, un-rotated 8-bit rows 2.8e-4 into fp16
// outputs, whose own rounding is 2.1e-4; 1.8e-3 and 1.7e-3 of 1.7e-3 into bf16 ones, 2.1e-3 of 1.6e-3 over BF16 rows (packed documents).  Of TQ4's
// the queries are 2.8e-4, values 2.1e-4, weights 1.2e-4, and second parts of queries would be 64 registers more.  Values below 2^-14 have fp16's
// absolute steps: of decoded values of 1e-5 / 1e-6 the error into bf16 outputs is 1.9e-3 / 7.3e-3.
// Over quantised rows 13 to 24 words a lane lie in scratch memory (16-bit rows none); a version that puts sums there has ten times as many.
template <typename TQ, int KVF, int HD, bool CAP>
__global__ __launch_bounds__(kChunkWaves * 64, 1) void scored_chunk_kernel(const ScoredParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    using R = ScoredRows<KVF, HD>;
    using M = ChunkLds<KVF, HD>;
    constexpr bool IS_BF16 = R::k16 && TQ::kStorageFormat == WARP34_KV_FORMAT_BF16;
    constexpr int kSteps = HD / 16, kDims = HD / 32;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, b = lane >> 5;
    const warp34_kv_layer_layout& L = P.L;
    const warp34_attention_batch& B = P.B;
    // the kv heads of a slot start together
    const int started = (int)(blockIdx.x + gridDim.x * blockIdx.y), kv_subs = (int)gridDim.y;
    const int slot = kv_subs == 1 ? started : fast_div(started, kv_subs), kv_sub = started - slot * kv_subs;
    const int kv_head = P.q_subgroups == 1 ? kv_sub : fast_div(kv_sub, P.q_subgroups);
    const int head0 = kv_head * P.gqa + (kv_sub - kv_head * P.q_subgroups) * P.q_group;

    // ---- what this workgroup works on ----
    ScoredWork work = {slot, 0, 1, 0};
    if (P.target > 0) {
        int* halves = reinterpret_cast<int*>(smem + M::kCounts);
        int* hist = reinterpret_cast<int*>(smem + M::kHist);
        if (tid < 64) hist[tid] = 0;
        for (int e = tid; e < P.entries; e += kChunkWaves * 64) halves[e] = tile_halves_guess(P, scored_tile(P, e));
        __syncthreads();
        const auto count = [&](int e) { return halves[e]; };
        const int per = chunk_length(P, lane, count);
        work = find_work_by_length(P, per, slot, tid, kChunkWaves * 64, lane, hist, count);
        if (work.entry < 0) return;
        if (work.chunk == 0 && kv_sub == 0 && tid == 0) {
            P.table[2 * work.entry] = work.first_record;
            P.table[2 * work.entry + 1] = work.chunks;
        }
    } else {
        work.entry = (int)gridDim.x - 1 - slot;  // the tiles with most keys first
    }
    const ScoredTile t = scored_tile(P, work.entry);
    if (t.tokens <= 0) return;
    int key_first, key_last;
    bool gaps;  // rows in between may be seen by no token
    tile_keys<true>(P, t, lane, key_first, key_last, &gaps);
    const int all_halves = tile_halves(key_first, key_last);
    const int per = (fast_div(all_halves + work.chunks - 1, work.chunks) + 1) & ~1;  // whole units
    const int begin = ((key_first >> 4) + work.chunk * per) * 16;  // keys
    const int end = key_first > key_last ? begin : max(begin, min(begin + per * 16, key_last + 1));
    const int units = (end - begin + kChunkUnit - 1) / kChunkUnit;

    // ---- this lane's column ----
    const int col = 32 * wave + n;
    const int my_t = column_token(col, P);
    const int my_tok = min(t.tok0 + my_t, B.total_tokens - 1);
    const bool col_ok = my_t < t.tokens && (B.valid_token_mask == nullptr || B.valid_token_mask[my_tok] != 0);
    const int my_head = min(head0 + (col - my_t * P.q_group), P.num_q_heads - 1);
    const int my_pos = t.pos0 + my_t;
    int lo = 0, hi = -1;
    if (col_ok) token_keys(P, my_tok, my_pos, t.seq_after, lo, hi);
    // keys that every live column of the wave sees, and that any sees
    const auto least = [](int x, int y) { return min(x, y); };
    const auto most = [](int x, int y) { return max(x, y); };
    const auto over_columns = [&](int v, auto&& f) {  // (rows of 16 lanes, then rows 0 and 1)
        v = row_reduce(v, f);
        return f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
    };
    const int all_from = over_columns(col_ok ? lo : 0, most), all_to = over_columns(col_ok ? hi : 0x7fffffff, least);
    const int any_from = over_columns(lo <= hi ? lo : 0x7fffffff, least), any_to = over_columns(lo <= hi ? hi : -1, most);
    const uint32_t live = (uint32_t)__ballot(col_ok);
    const bool sloped = P.slopes != nullptr;
    const float slope2 = sloped && col_ok ? P.slopes[my_head] * kLog2e : 0.f;

    // ---- loader: waves 2 i and 2 i + 1 bring half each of run i (keys 0-15, 16-31, values 0-15, 16-31) ----
    const int run = wave >> 1, part = wave & 1;
    const bool loads_v = run >= 2;
    const uint8_t* slab = reinterpret_cast<const uint8_t*>((uintptr_t)(loads_v ? L.v_base : L.k_base)) +
                          (uint64_t)(uint32_t)kv_head * (loads_v ? L.v_head_stride_bytes : L.k_head_stride_bytes);
    const uint64_t page_stride = loads_v ? L.v_page_stride_bytes : L.k_page_stride_bytes;
    const int32_t* blocks = B.block_tables + (size_t)t.req * B.max_blocks_per_req;
    int slot_base = page_slot(begin, P);
    int pages = slot_base + lane < B.max_blocks_per_req ? blocks[slot_base + lane] : 0;
    constexpr int kShare = M::kRun / 2;
    const auto issue = [&](int u, uint32_t values) {
        const int pos = begin + u * kChunkUnit + 16 * (run & 1);
        uint64_t off = 0;
        if (pos <= key_last) {  // (a run behind the keys: rows of page 0, which nobody sees)
            const int slot = page_slot(pos, P);
            if (slot - slot_base >= 64) {
                slot_base = slot;
                pages = slot_base + lane < B.max_blocks_per_req ? blocks[slot_base + lane] : 0;
            }
            const uint32_t page = (uint32_t)max(__builtin_amdgcn_readlane(pages, slot - slot_base), 0);
            off = (uint64_t)page * page_stride + (uint32_t)(pos - slot * L.block_size) * (uint32_t)R::kRowBytes;
        }
        const uint8_t* src = uniform_pointer(slab + off + part * kShare);
        if constexpr (R::k16) {
            // rows 8 part + ..: the piece that belongs to a lane's place
            constexpr int kPieces = M::kRow / 16, kRows = 64 / kPieces;  // of a row, of an instruction
            const uint32_t dst = (loads_v ? values : (uint32_t)(M::kTiles + (u & 1) * M::kTile)) + (uint32_t)((run & 1) * M::kRun + part * kShare);
            const int at_lane = here(lane), r = at_lane / kPieces, p = at_lane % kPieces;
            const auto one = [&](auto imm) {
                constexpr int i = decltype(imm)::value;
                const int row = 8 * part + i * kRows + r;
                const uint32_t v = (uint32_t)(r * M::kRow + 16 * (p ^ (loads_v ? 4 * (row & 3) : (row & 15))));
                load_to_lds<1024 * i>(v, src, dst);
            };
            one(std::integral_constant<int, 0>{});
            one(std::integral_constant<int, 1>{});
            if constexpr (kShare > 2048) {
                one(std::integral_constant<int, 2>{});
                one(std::integral_constant<int, 3>{});
            }
        } else {
            const uint32_t dst = (uint32_t)(M::kRaw + (u & 1) * M::kRawUnit + run * M::kRun + part * kShare), v = 16u * (uint32_t)here(lane);
            load_to_lds<0>(v, src, dst);
            if constexpr (kShare >= 2048) load_to_lds<1024>(v, src, dst);
            constexpr int kRest = kShare % 1024;
            if (v < (uint32_t)kRest) load_to_lds<kShare - kRest>(v, src, dst);
        }
    };
    // (a run's place is none of what the queries' columns go through)
    uint32_t v_last = (uint32_t)(M::kValues + 2 * M::kTile), v_now = (uint32_t)M::kValues, v_next = (uint32_t)(M::kValues + M::kTile);
    if (units > 0) issue(0, v_now);
    if (!R::k16 && units > 1) issue(1, 0u);

    // where the rotations of queries and of results have a lane's four elements, their signs as bits of 16-bit numbers, and the matrix
    const auto rotation = [&](int& piece, uint2& piece_flip, u4& had) {
        const int at_lane = here(lane), r = at_lane & 15, c = at_lane >> 4;
        piece = 16 * r + 4 * c;
        const uint32_t signs = kSignMask[piece >> 5] >> (piece & 31);
        piece_flip = uint2{(signs << 15 & 0x8000u) | (signs << 30 & 0x80000000u), (signs << 13 & 0x8000u) | (signs << 28 & 0x80000000u)};
        had = __builtin_bit_cast(u4, hadamard_column(r, c));
    };

    // ---- table and query operands: lane (n, b) holds Q[column n][16 m + 8 b .. + 7] ----
    if constexpr (R::kTq4) build_narrow_table(smem, tid, wave);
    u4 q[kSteps];
    float cs = score_factor(P, 1.0f), cc = P.cap_arg;
    if constexpr (R::k16) {
        const uint16_t* src = P.q + ((size_t)my_tok * P.num_q_heads + (size_t)my_head) * HD + 8 * b;
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
            q[m] = *reinterpret_cast<const u4*>(src + 16 * m) ^ P.q_flip;
            if (!col_ok) q[m] = u4{0u, 0u, 0u, 0u};
        }
    } else if (!P.rot_q) {
        // as given, relative to a power of two above the column's largest element: fp16 holds its 11 bits whatever its size
        const uint16_t* src = P.q + ((size_t)my_tok * P.num_q_heads + (size_t)my_head) * HD + 8 * b;
        float top = 0.f;
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
            q[m] = *reinterpret_cast<const u4*>(src + 16 * m) ^ P.q_flip;
            if (!col_ok) q[m] = u4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int m = 0; m < kSteps; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = q[m][k];
                top = fmaxf(top, fmaxf(fabsf(TQ::to_f32((uint16_t)w)), fabsf(TQ::to_f32((uint16_t)(w >> 16)))));
            }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        const int e = top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
#pragma unroll
        for (int m = 0; m < kSteps; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = q[m][k];
                q[m][k] = pack_h2(__builtin_amdgcn_ldexpf(TQ::to_f32((uint16_t)w), -e), __builtin_amdgcn_ldexpf(TQ::to_f32((uint16_t)(w >> 16)), -e));
            }
        const float mine = __builtin_amdgcn_ldexpf(R::kOutScale, e);
        cs = score_factor(P, mine);
        cc = cap_factor(P, mine);
    } else {
        // Rotated by two products a column (wht_products.h; in vector instructions, as the results' rotation back, 8 requests of 400 to 600 TQ4
        // tokens in windows of 64 took 98.9 instead of 81.5 us), eight columns of the wave at a time through LDS, their loads together and those of
        // the next eight ahead.  Elements go in relative to a power of two above the column's largest, as fp16 holds them.
        int piece;
        uint2 piece_flip;
        u4 had;
        rotation(piece, piece_flip, had);
        uint16_t* area = reinterpret_cast<uint16_t*>(smem + M::kTiles + wave * 8 * M::kColStride * 4);
        float* scales = reinterpret_cast<float*>(smem + M::kQScale) + 32 * wave;
        uint2 raw[8];
        const auto load_columns = [&](int g) {
#pragma unroll
            for (int c8 = 0; c8 < 8; ++c8) {
                const int c = 8 * g + c8, ct = column_token(32 * wave + c, P);
                raw[c8] = uint2{0u, 0u};
                if ((live >> c) & 1u)
                    raw[c8] = *reinterpret_cast<const uint2*>(P.q + ((size_t)(t.tok0 + ct) * P.num_q_heads + (size_t)(head0 + 32 * wave + c - ct * P.q_group)) * HD + piece);
            }
        };
        load_columns(0);
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
            uint2 now[8];
#pragma unroll
            for (int c8 = 0; c8 < 8; ++c8) now[c8] = uint2{raw[c8].x ^ P.q_flip ^ piece_flip.x, raw[c8].y ^ P.q_flip ^ piece_flip.y};
            if (g < 3) load_columns(g + 1);
#pragma unroll
            for (int c8 = 0; c8 < 8; ++c8) {
                const uint32_t two = max_u16x2(now[c8].x & 0x7FFF7FFFu, now[c8].y & 0x7FFF7FFFu);
                const float top = TQ::to_f32((uint16_t)wave_largest((int)max(two & 0xFFFFu, two >> 16)));
                const int e = top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
                const auto in = [&](uint32_t w) {
                    return pack_h2(__builtin_amdgcn_ldexpf(TQ::to_f32((uint16_t)w), -e), __builtin_amdgcn_ldexpf(TQ::to_f32((uint16_t)(w >> 16)), -e));
                };
                const f4 none = {0.f, 0.f, 0.f, 0.f};
                const f4 z = mfma_rows<false>(u4{in(now[c8].x), in(now[c8].y), 0u, 0u}, had, none);
                const float zs[4] = {z[0], z[1], z[2], z[3]};
                const f4 y = mfma_rows<false>(__builtin_bit_cast(u4, two_parts(zs)), had, none);
                *reinterpret_cast<uint2*>(area + c8 * M::kColStride + piece) = uint2{pack_h2(y[0], y[1]), pack_h2(y[2], y[3])};
                if (lane == 0) scales[8 * g + c8] = __builtin_amdgcn_ldexpf(R::kOutScale, e - 4);
            }
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            __builtin_amdgcn_wave_barrier();
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            if ((n >> 3) == g) {
#pragma unroll
                for (int m = 0; m < kSteps; ++m) q[m] = *reinterpret_cast<const u4*>(area + (n & 7) * M::kColStride + 16 * m + 8 * b);
            }
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            __builtin_amdgcn_wave_barrier();
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
        }
        cs = score_factor(P, scales[n]);
        cc = cap_factor(P, scales[n]);
    }
    if (gaps && tid < t.tokens) {
        int from = 0, to = -1;
        if (B.valid_token_mask == nullptr || B.valid_token_mask[t.tok0 + tid] != 0) token_keys(P, t.tok0 + tid, t.pos0 + tid, t.seq_after, from, to);
        *reinterpret_cast<u2v*>(smem + M::kRanges + 8 * tid) = u2v{(uint32_t)from, (uint32_t)to};
    }
    __syncthreads();  // the areas become tiles

    // ---- raw rows of unit u -> its tiles and scales ----
    // A thread takes pieces c and c + 16 (8 elements each) of a key row and of a value row.  Each piece in steps, which stand between
    // the products of values: what a step reads from LDS the next one uses.
    struct Widening {
        uint32_t row, codes, keys, values, scale;  // places in LDS
        uint32_t raw[2], d, scale_raw;
        u4 w;
        bool seen;
    };
    const auto widen_start = [&](int u, uint32_t values, Widening& x) {
        const int at_tid = here(tid), r = at_tid >> 4, c = at_tid & 15;
        const uint32_t raw = (uint32_t)(M::kRaw + (u & 1) * M::kRawUnit);
        const int row_pos = begin + u * kChunkUnit + r;
        x.seen = row_pos >= key_first && row_pos <= key_last;
        x.row = raw + (uint32_t)(r * R::kRowBytes) + (R::kQ8 ? 68u * (uint32_t)(c >> 3) : 0u);
        x.codes = R::kTq4 ? x.row + 4u * (uint32_t)c : R::kFp8 ? x.row + 8u * (uint32_t)c : x.row + 4u + 8u * (uint32_t)(c & 7);
        x.keys = (uint32_t)(M::kTiles + (u & 1) * M::kTile + r * M::kRow + 16 * (c ^ (r & 15)));
        x.values = values + (uint32_t)(r * M::kRow + 16 * (c ^ 4 * (r & 3)));
        // key scales: [block][row], by the first threads
        x.scale = (uint32_t)(M::kScale + (u & 1) * 512 + 4 * at_tid);
        if (at_tid < R::kScales * 32) {
            const uint32_t from = raw + (uint32_t)((at_tid & 31) * R::kRowBytes), blk = (uint32_t)at_tid / 32u;
            x.scale_raw = R::kTq4 ? lds_u16(from + 66u * blk) : lds_u1(R::kFp8 ? from + 256u + 4u * blk : from + 68u * blk);
        }
    };
    const auto widen_scales = [&](Widening& x) {
        if (here(tid) < R::kScales * 32)
            *reinterpret_cast<__attribute__((address_space(3))) float*>((uintptr_t)x.scale) = R::kTq4 ? F16::to_f32((uint16_t)x.scale_raw) : __uint_as_float(x.scale_raw);
    };
    const auto widen_load = [&](int piece, Widening& x) {  // piece: 2 (values) + the half of the row
        const int side = piece >> 1, h = piece & 1;
        const uint32_t from = x.codes + (uint32_t)(side * 2 * M::kRun), row = x.row + (uint32_t)(side * 2 * M::kRun);
        if constexpr (R::kTq4) {
            // (reads of four bytes must be aligned, the codes of the first half start at byte 2)
            x.raw[0] = lds_u1(from + (h ? 68u : 0u));
            if (h == 0) x.raw[1] = lds_u1(from + 4u);
            if (side == 1) x.d = lds_u16(row + (h ? 66u : 0u));
        } else if constexpr (R::kFp8) {
            const u2v two = lds_u2(from + 128u * (uint32_t)h);
            x.raw[0] = two[0], x.raw[1] = two[1];
            if (side == 1) x.d = lds_u1(row + 256u + 4u * (uint32_t)h);
        } else {
            x.raw[0] = lds_u1(from + 136u * (uint32_t)h), x.raw[1] = lds_u1(from + 136u * (uint32_t)h + 4u);
            if (side == 1) x.d = lds_u1(row + 136u * (uint32_t)h);
        }
    };
    const auto widen_look_up = [&](int piece, Widening& x) {
        if constexpr (R::kTq4) {
            const uint32_t codes = (piece & 1) ? x.raw[0] : __builtin_amdgcn_alignbit(x.raw[1], x.raw[0], 16);
            const uint32_t copy = ((uint32_t)here(tid) & 31u) << 2;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t pair = lds_u1(((k == 0 ? codes << 7 : codes >> (8 * k - 7)) & 0x7F80u) | copy);
                x.w[k] = pair;
            }
        }
    };
    const auto widen_store = [&](int piece, Widening& x) {
        const int side = piece >> 1, h = piece & 1;
        if constexpr (R::kTq4) {
            if (side == 1) {
                const uint32_t d16 = x.seen ? x.d : 0u;
                const h2 d = __builtin_bit_cast(h2, d16 | d16 << 16);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t pair = x.w[k];  // (a scalar in between: a bit cast of a vector's element reads its first one)
                    x.w[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, pair) * d);
                }
            }
        } else {
            const float d = x.seen ? __uint_as_float(x.d) : 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t code = x.raw[k], lo2, hi2;
                if (side == 1) {
                    code = x.seen ? code : 0u;
                    float f[4];
                    if constexpr (R::kFp8) {
                        const f2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)code, false), s = __builtin_amdgcn_cvt_pk_f32_fp8((int)code, true);
                        f[0] = p[0], f[1] = p[1], f[2] = s[0], f[3] = s[1];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(code >> (8 * i));
                    }
                    lo2 = pack_h2(f[0] * d, f[1] * d);
                    hi2 = pack_h2(f[2] * d, f[3] * d);
                } else if constexpr (R::kFp8) {
                    lo2 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(code, 1.0f, false));
                    hi2 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(code, 1.0f, true));
                } else {  // 0x6400 | (q + 128) is 1152 + q in fp16
                    const uint32_t u8 = code ^ 0x80808080u;
                    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
                    lo2 = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u8, 0x04010400u)) - bias);
                    hi2 = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u8, 0x04030402u)) - bias);
                }
                x.w[2 * k] = lo2;
                x.w[2 * k + 1] = hi2;
            }
        }
        lds_put((side ? x.values : x.keys) + 256u * (uint32_t)h, x.w);
    };
    const auto widen = [&](int u, uint32_t values) {
        Widening x;
        widen_start(u, values, x);
        widen_scales(x);
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) {
            widen_load(piece, x);
            widen_look_up(piece, x);
            widen_store(piece, x);
        }
    };

    f16v o[kDims];
#pragma unroll
    for (int k = 0; k < kDims; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[k][i] = 0.f;
    float m_run = kNegBig, l_run = 0.f;

    u4 w[2];               // the weights of the wave's last scored unit
    bool weighted = false;  // it has some (uniform)
    const auto score = [&](int u) {
        const int at_lane = here(lane), n = at_lane & 31, b = at_lane >> 5;
        const int u0 = begin + u * kChunkUnit;
        weighted = u0 <= any_to && u0 + kChunkUnit - 1 >= any_from;  // uniform
        if (!weighted) return;
        const uint32_t tiles = (uint32_t)(M::kTiles + (u & 1) * M::kTile);
        const uint32_t scale = (uint32_t)(M::kScale + (u & 1) * 512);
        // ---- scores ----
        f16v s;
        {
            const uint32_t row = tiles + (uint32_t)(n * M::kRow), swap = 16u * (uint32_t)(b ^ (n & 15));
            constexpr int kBlocks = R::k16 ? 1 : R::kScales, kPer = kSteps / kBlocks;
            // operands are read kKeysAhead products before their own (the compiler would read each right before it, to save registers)
            const auto k_operand = [&](int m) { return lds_u4(row + (swap ^ (uint32_t)(32 * (m & 7))) + 256u * (m >> 3)); };
            u4 a[kKeysAhead + 1];
#pragma unroll
            for (int m = 0; m < kKeysAhead; ++m) a[m] = k_operand(m);
#pragma unroll
            for (int blk = 0; blk < kBlocks; ++blk) {
                f16v part_s;
#pragma unroll
                for (int i = 0; i < 16; ++i) part_s[i] = 0.f;
#pragma unroll
                for (int mm = 0; mm < kPer; ++mm) {
                    const int m = blk * kPer + mm;
                    __builtin_amdgcn_sched_barrier(0);
                    if (m + kKeysAhead < kSteps) a[(m + kKeysAhead) % (kKeysAhead + 1)] = k_operand(m + kKeysAhead);
                    __builtin_amdgcn_sched_barrier(0);
                    part_s = mfma_tile<IS_BF16>(a[m % (kKeysAhead + 1)], q[m], part_s);
                }
                if constexpr (R::k16) {
                    s = part_s;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f4 d = lds_f4(scale + (uint32_t)(128 * blk + 32 * k + 16 * b));
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[4 * k + i] = blk == 0 ? d[i] * part_s[4 * k + i] : __builtin_fmaf(d[i], part_s[4 * k + i], s[4 * k + i]);
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- terms, masks, softmax ----
        const bool masked = !(u0 >= all_from && u0 + kChunkUnit - 1 <= all_to);  // uniform
        ScoreMap map = map_scores<CAP, false, 16>(s, cs, cc, P);
        if (sloped) {
            const float at = (float)(my_pos - u0 - 4 * b);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_fmaf(-slope2, fabsf(at - (float)((i & 3) + 8 * (i >> 2))), __builtin_fmaf(s[i], map.ca, map.cb));
            map = ScoreMap{1.0f, 0.f};
        }
        if (masked) {
            const int from = lo - u0 - 4 * b, to = hi - u0 - 4 * b;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int k = (i & 3) + 8 * (i >> 2);
                s[i] = k >= from && k <= to ? s[i] : -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        top = __builtin_fmaf(top, map.ca, map.cb);
        if (__ballot(top > m_run + kChunkSlack) != 0ull) {
            const float m_new = top > m_run + kChunkSlack ? top : m_run;
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int k = 0; k < kDims; ++k) o[k] *= alpha;
        }
        const float less = map.cb - m_run;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], map.ca, less));
            sum += s[i];
        }
        l_run += sum;
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k >> 2][k & 3] = IS_BF16 ? pack_bf2(s[2 * k], s[2 * k + 1]) : pack_h2(s[2 * k], s[2 * k + 1]);
    };
    // The values of a unit, and between their products the widening of another one.
    const auto add_values = [&](uint32_t values, auto widening, int widen_unit, uint32_t widen_to) {
        constexpr bool kWidens = decltype(widening)::value;
        if (!weighted) {
            if constexpr (kWidens) widen(widen_unit, widen_to);
            return;
        }
        // lane l reads row (l & 15) >> 2 of four, 8 bytes at 8 (l & 3) of the 32 of its 16 channels
        const int at_lane = here(lane), j = at_lane & 15;
        const uint32_t v_at = values + (uint32_t)((4 * (at_lane >> 5) + (j >> 2)) * M::kRow) + 64u * (uint32_t)(j >> 2) + 32u * (uint32_t)(at_lane >> 4 & 1) + 8u * (uint32_t)(j & 3);
        const auto v_operand = [&](int dt, int step) -> u4 {
            const uint32_t at = (v_at ^ (64u * (uint32_t)(dt & 3))) + 256u * (uint32_t)(dt >> 2) + (uint32_t)(step * 16 * M::kRow);
            const s4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)at));
            const s4v c = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>((uintptr_t)(at + 8u * M::kRow)));
            const u2v x = __builtin_bit_cast(u2v, a), y = __builtin_bit_cast(u2v, c);
            return u4{x[0], x[1], y[0], y[1]};
        };
        Widening x;
        if constexpr (kWidens) widen_start(widen_unit, widen_to, x);
        u4 a[kValuesAhead + 1];
#pragma unroll
        for (int i = 0; i < kValuesAhead; ++i) a[i] = v_operand(i >> 1, i & 1);
#pragma unroll
        for (int i = 0; i < 2 * kDims; ++i) {
            const int next = i + kValuesAhead, piece = i >> 2;
            __builtin_amdgcn_sched_barrier(0);
            if (next < 2 * kDims) a[next % (kValuesAhead + 1)] = v_operand(next >> 1, next & 1);
            if constexpr (kWidens) {
                if ((i & 3) == 0) widen_load(piece, x);
                if ((i & 3) == 1) widen_look_up(piece, x);
                if ((i & 3) == 3) widen_store(piece, x);
                if (i == 2) widen_scales(x);
            }
            __builtin_amdgcn_sched_barrier(0);
            o[i >> 1] = mfma_tile<IS_BF16>(a[i % (kValuesAhead + 1)], w[i & 1], o[i >> 1]);
        }
    };
    // Value rows that no token of the tile sees count as zeros: they may hold anything.  Quantised ones in front of the first key and behind
    // the last come as zeros out of the widening.  Where there are gaps 16 lanes share a row, and look at the tokens' ranges in turn.
    const auto clear_unseen = [&](int u, uint32_t values) {
        const int u0 = begin + u * kChunkUnit;
        if (!gaps && (!R::k16 || (u0 >= key_first && u0 + kChunkUnit - 1 <= key_last))) return;  // uniform
        constexpr int kPieces = M::kTile / 16;
        static_assert(kPieces % (kChunkWaves * 64) == 0 && (M::kRow / 16) % 16 == 0, "all lanes take part, 16 to a row");
        for (int p = here(tid); p < kPieces; p += kChunkWaves * 64) {
            const int pos = u0 + p / (M::kRow / 16);
            bool seen = pos >= key_first && pos <= key_last;
            if (gaps) {
                int some = 0;
                for (int k = p & 15; k < t.tokens; k += 16) {
                    const u2v range = lds_u2((uint32_t)(M::kRanges + 8 * k));
                    some |= pos >= (int)range[0] && pos <= (int)range[1] ? 1 : 0;
                }
                seen = row_reduce(some, [](int x, int y) { return x | y; }) != 0;
            }
            if (!seen) lds_put(values + (uint32_t)(16 * p), u4{0u, 0u, 0u, 0u});
        }
        chunk_barrier();
    };

    // Waves w and w + 4 share a SIMD.  The second of them multiplies the values of a unit in the next interval, before its scores, so that
    // the products of one run beside the other's vector work: widen, scores, softmax, values | values, widen, scores, softmax.  Values stay
    // for two intervals: three tiles of them.
    const bool late = wave >= 4;
    if constexpr (!R::k16) {
        chunk_barrier();
        if (units > 0) widen(0, v_now);
    }
    for (int u = 0; u < units; ++u) {
        chunk_barrier();  // unit u's tiles are whole, the next one's rows have landed; nobody reads what is overwritten below
        if constexpr (R::k16) {
            if (u + 1 < units) issue(u + 1, v_next);
        } else {
            if (u + 2 < units) issue(u + 2, 0u);
        }
        clear_unseen(u, v_now);
        __builtin_amdgcn_sched_barrier(0);
        // (behind the last unit: old rows, to tiles that nobody reads)
        if (late) add_values(v_last, std::integral_constant<bool, !R::k16>{}, u + 1, v_next);
        __builtin_amdgcn_sched_barrier(0);
        score(u);
        __builtin_amdgcn_sched_barrier(0);
        if (!late) add_values(v_now, std::integral_constant<bool, !R::k16>{}, u + 1, v_next);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t free = v_last;
        v_last = v_now, v_now = v_next, v_next = free;
    }
    if (late && units > 0) add_values(v_last, std::false_type{}, 0, 0u);
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
        l_run = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    chunk_barrier();

    // ---- rows out ----
    if (work.chunks > 1 || HD != 256 || !P.rot_out) {  // as they stand: a lane has pairs of four channels of its column
        if (!col_ok) return;
        if (work.chunks > 1) {
            const size_t record = ((size_t)(work.first_record + work.chunk) * kv_subs + kv_sub) * kChunkCols + col;
            float* to = P.part_acc + record * HD + 4 * b;
#pragma unroll
            for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<f4*>(to + 32 * dt + 8 * k) = f4{o[dt][4 * k], o[dt][4 * k + 1], o[dt][4 * k + 2], o[dt][4 * k + 3]};
            if (b == 0) *reinterpret_cast<f2*>(P.part_ml + 2 * record) = f2{m_run, l_run};
        } else {
            const size_t row = (size_t)my_tok * P.num_q_heads + (size_t)my_head;
            const bool some = l_run > 0.f || l_run != l_run;
            const float inv = some ? R::kOutScale / l_run : 0.f;  // (a row without keys: zeros)
            uint16_t* to = P.out + row * HD + 8 * b;
            const auto pack = [&](float x, float y) { return TQ::kStorageFormat == WARP34_KV_FORMAT_BF16 ? pack_bf2(x * inv, y * inv) : pack_h2(x * inv, y * inv); };
#pragma unroll
            for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
                for (int k = 0; k < 4; k += 2) {  // the half wave with b = 0 takes channels 0 .. 7 of 16, the other one 8 .. 15
                    const auto x = __builtin_amdgcn_permlane32_swap(pack(o[dt][4 * k], o[dt][4 * k + 1]), pack(o[dt][4 * k + 4], o[dt][4 * k + 5]), false, false);
                    const auto y = __builtin_amdgcn_permlane32_swap(pack(o[dt][4 * k + 2], o[dt][4 * k + 3]), pack(o[dt][4 * k + 6], o[dt][4 * k + 7]), false, false);
                    *reinterpret_cast<u4_at8*>(to + 32 * dt + 8 * k) = u4{x[0], y[0], x[1], y[1]};
                }
            if (P.lse != nullptr && b == 0) P.lse[row] = some ? (m_run + __builtin_amdgcn_logf(l_run)) * 0.6931471805599453f : -INFINITY;
        }
        return;
    }
    // rotated back by two products a column, eight columns of a wave at a time through LDS
    int piece;
    uint2 piece_flip;
    u4 had;
    rotation(piece, piece_flip, had);
    float* area = reinterpret_cast<float*>(smem + M::kTiles + wave * 8 * M::kColStride * 4);
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        if ((n >> 3) == g) {
#pragma unroll
            for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<f4*>(area + (n & 7) * M::kColStride + 32 * dt + 8 * k + 4 * b) = f4{o[dt][4 * k], o[dt][4 * k + 1], o[dt][4 * k + 2], o[dt][4 * k + 3]};
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll 4
        for (int c8 = 0; c8 < 8; ++c8) {
            const int c = 8 * g + c8;
            if (!((live >> c) & 1u)) continue;
            const f4 acc = *reinterpret_cast<const f4*>(area + c8 * M::kColStride + piece);
            const float m_c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m_run), c));
            const float l_c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l_run), c));
            const int ct = column_token(32 * wave + c, P);
            const size_t row = (size_t)(t.tok0 + ct) * P.num_q_heads + (size_t)(head0 + 32 * wave + c - ct * P.q_group);
            const bool some = l_c > 0.f || l_c != l_c;
            const float inv = some ? R::kOutScale / l_c : 0.f;  // (a row without keys: zeros)
            float v[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
#pragma unroll
            for (int k = 0; k < 4; ++k) asm("" : "+v"(v[k]));  // both parts are taken from the product rounded to 32 bits
            const f4 none = {0.f, 0.f, 0.f, 0.f};
            const f4 z = mfma_rows<false>(__builtin_bit_cast(u4, two_parts(v)), had, none);
            float zs[4] = {z[0] * 0.0625f, z[1] * 0.0625f, z[2] * 0.0625f, z[3] * 0.0625f};
#pragma unroll
            for (int k = 0; k < 4; ++k) asm("" : "+v"(zs[k]));
            const f4 y = mfma_rows<false>(__builtin_bit_cast(u4, two_parts(zs)), had, none);
            const auto pack = [](float x0, float x1) { return TQ::kStorageFormat == WARP34_KV_FORMAT_BF16 ? pack_bf2(x0, x1) : pack_h2(x0, x1); };
            *reinterpret_cast<uint2*>(P.out + row * HD + piece) = uint2{pack(y[0], y[1]) ^ piece_flip.x, pack(y[2], y[3]) ^ piece_flip.y};
            if (P.lse != nullptr && lane == 0) P.lse[row] = some ? (m_c + __builtin_amdgcn_logf(l_c)) * 0.6931471805599453f : -INFINITY;
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_wave_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    }
}

}  // namespace w34
