// Scored paged attention, what its kernels share: the arguments, a query token's keys, the score terms, the cut of a batch into tiles
// and chunks, and the end of a row.
//
//   x(t, k)   = sm_scale q_t . k_k,  capped: cap tanh(x / cap),  then less slope[h] |position of t - k|
//   keys of t = [max(0, window's first, document_starts[t]), min(max(causal or all, prefix_ends[t] - 1), last of the sequence)]
//   out       = sum_k 2^(x log2e - m) v_k / l,  lse = ln 2 (m + log2 l)
//
// Every kernel works with x log2e.
#pragma once

#include "attn_lanes.h"

namespace w34 {

struct ScoredParams {
    warp34_kv_layer_layout L;
    warp34_attention_batch B;
    const uint16_t* q;
    uint16_t* out;
    const float* slopes;
    const int32_t* document_starts;
    const int32_t* prefix_ends;
    float* lse;
    float scale2;     // |sm_scale| log2e
    uint32_t q_flip;  // sm_scale < 0: the sign bits of a pair of query elements
    float cap2;       // cap log2e; 0: no cap
    float cap_arg;    // 2 |sm_scale| log2e / cap: exp2 of it times q.k is exp(2 x / cap)
    int wide_cap;     // the cap is so large that tanh of a small argument needs its series (kWideCap)
    int num_q_heads, gqa, q_group, q_subgroups;
    int tok_tile;     // query tokens of a tile
    int tiles;        // tiles of a request (a bound)
    int entries;      // requests x tiles: tiles of the batch, some of them empty
    int target;       // slots for chunks, for each kv head; 0: no split, a workgroup for each entry
    int round;        // slots for each kv head that fill the chip
    int full_rounds;  // the cut looks for full rounds of chunks; 0: no more chunks than target
    int records;      // partial records the scratch holds, for each kv head
    int min_halves;   // shortest chunk
    float* part_acc;  // [record][kv_sub][column][head_dim]
    float* part_ml;   // [record][kv_sub][column]{m, l}
    int32_t* table;   // [entry]{first record, chunks}
    uint32_t block_magic, q_group_magic;
    int rot_q, rot_out;
};

// tanh(u) = 1 - 2 / (exp(2 u) + 1) is off by some 2^-23 whatever u, which the cap multiplies: 6e-6 of a score at a cap of 50, 6e-5 at
// this one.  Where few keys make a row that shows in its lse: the decode kernels take small arguments through the series, and so does
// the chunk kernel, whose queries are rounded to more than that, beyond this cap.
constexpr float kWideCap = 512.0f;
// Larger caps count as this one: no score comes near it (kNegBig is none), and twice the cap and its reciprocal, which the scales of queries
// multiply, stay numbers of 32 bits.
constexpr float kLargestCap = 1.0e30f;

// Scores s (q . k times what the column's scale is in) become y with x = y ca + cb in the log2 domain, ca >= 0, so that the largest y is
// the largest x and exp2's argument x - m is one fma.  No cap: y = s, x = y cs.  Cap without the series: y = -1 / (exp(2 x / cap) + 1),
// x = cap2 + 2 cap2 y.  cs > 0 and cc: the column's scale times scale2 / cap_arg.
// The series stands for |u| < 1/4, where what follows its last term is below 2^-26 of it.
struct ScoreMap {
    float ca, cb;
};
// cs.  Not 0, where the scale is or where it leaves 32 bits together with a small query's: hidden keys have scores of minus infinity, which
// would become NaN.  (1e-37 of a score is nothing beside the others.)
__device__ __forceinline__ float score_factor(const ScoredParams& P, float column_scale) {
    const float f = P.scale2 * column_scale;
    return f < 1.0e-37f ? 1.0e-37f : f;
}
// cc.  Finite, however small the cap and large the query: a score of 0 stays 0.
__device__ __forceinline__ float cap_factor(const ScoredParams& P, float column_scale) { return fminf(P.cap_arg * column_scale, 3.0e38f); }
template <bool CAP, bool SERIES, int N, typename V>
__device__ __forceinline__ ScoreMap map_scores(V& s, float cs, float cc, const ScoredParams& P) {
    if constexpr (!CAP) {
        return ScoreMap{cs, 0.f};
    } else if (!SERIES && !P.wide_cap) {  // (uniform, and outside the loop)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[i] * cc));
        return ScoreMap{2.0f * P.cap2, P.cap2};
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = s[i] * cc, u = a * (0.5f / kLog2e), uu = u * u;
            const float x = __builtin_fmaf(2.0f * P.cap2, __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(a)), P.cap2);
            float series = __builtin_fmaf(uu, 62.0f / 2835.0f, -17.0f / 315.0f);
            series = __builtin_fmaf(uu, series, 2.0f / 15.0f);
            series = __builtin_fmaf(uu, series, -1.0f / 3.0f);
            series = P.cap2 * u * __builtin_fmaf(uu, series, 1.0f);
            s[i] = fabsf(u) < 0.25f ? series : x;
        }
        return ScoreMap{1.0f, 0.f};
    }
}

__device__ __forceinline__ int page_slot(int pos, const ScoredParams& P) {
    int q = (int)__umulhi((uint32_t)pos, P.block_magic);  // the quotient or one less
    return q + ((pos - q * P.L.block_size >= P.L.block_size) ? 1 : 0);
}
__device__ __forceinline__ int column_token(int col, const ScoredParams& P) { return (int)(((uint32_t)col * P.q_group_magic) >> 16); }

// Keys of a token: lo > hi where it has none.
__device__ __forceinline__ void token_keys(const ScoredParams& P, int tok, int pos, int seq_after, int& lo, int& hi) {
    const warp34_attention_batch& B = P.B;
    hi = B.mask_mode == WARP34_ATTN_MASK_NONCAUSAL_WINDOW ? seq_after - 1 : pos;
    if (P.prefix_ends != nullptr) hi = max(hi, max(P.prefix_ends[tok], 0) - 1);
    hi = min(hi, seq_after - 1);
    lo = B.sliding_window > 0 ? max(0, pos - B.sliding_window + 1) : 0;
    if (P.document_starts != nullptr) lo = max(lo, P.document_starts[tok]);
}

// A tile: some query tokens of one request.  tokens 0: there is nothing to do.
struct ScoredTile {
    int req, tok0, tokens;
    int pos0, seq_after;  // position of its first token
};
__device__ __forceinline__ ScoredTile scored_tile(const ScoredParams& P, int entry) {
    const warp34_attention_batch& B = P.B;
    const int req = P.tiles == 1 ? entry : fast_div(entry, P.tiles);
    const int first = (entry - req * P.tiles) * P.tok_tile;
    const int lo = B.query_start_loc[req], hi = B.query_start_loc[req + 1], seq = B.seq_lens_after[req];
    const int ctx = B.context_lens_before != nullptr ? B.context_lens_before[req] : seq - (hi - lo);
    const bool valid = B.valid_req_mask == nullptr || B.valid_req_mask[req] != 0;
    const int tokens = min(min(hi - lo - first, P.tok_tile), B.total_tokens - lo - first);
    return ScoredTile{req, lo + first, valid && lo >= 0 ? max(tokens, 0) : 0, ctx + first, seq};
}
// Sums and largest numbers of a wave by lane shifts inside the vector unit (an exchange through LDS takes a hundred cycles a step).
template <int CTRL, int ROWS>
__device__ __forceinline__ int shifted_in(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xF, false); }
template <typename F>
__device__ __forceinline__ int wave_scan(int v, int none, F&& f) {  // inclusive; none: what changes nothing
    v = f(v, shifted_in<0x111, 0xF>(none, v));  // row_shr:1, 2, 4, 8
    v = f(v, shifted_in<0x112, 0xF>(none, v));
    v = f(v, shifted_in<0x114, 0xF>(none, v));
    v = f(v, shifted_in<0x118, 0xF>(none, v));
    v = f(v, shifted_in<0x142, 0xA>(none, v));  // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
    return f(v, shifted_in<0x143, 0xC>(none, v));
}
__device__ __forceinline__ int wave_prefix(int v) {
    return wave_scan(v, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); }
__device__ __forceinline__ int wave_largest(int v) {
    return __builtin_amdgcn_readlane(wave_scan(v, (int)0x80000000, [](int a, int b) { return max(a, b); }), 63);
}
__device__ __forceinline__ int wave_least(int v) {
    return __builtin_amdgcn_readlane(wave_scan(v, 0x7fffffff, [](int a, int b) { return min(a, b); }), 63);
}
// The largest of a wave's numbers >= 0, in all lanes.
__device__ __forceinline__ float wave_top(float v) {
    return __int_as_float(wave_largest(__float_as_int(v)));
}

// The largest of a wave's numbers, none of them NaN, and their sum.
__device__ __forceinline__ float wave_most(float v) {
    const auto f = [](int a, int b) { return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); };
    return __int_as_float(__builtin_amdgcn_readlane(wave_scan(__float_as_int(v), __float_as_int(-INFINITY), f), 63));
}
__device__ __forceinline__ float wave_total(float v) {
    const auto f = [](int a, int b) { return __float_as_int(__int_as_float(a) + __int_as_float(b)); };
    return __int_as_float(__builtin_amdgcn_readlane(wave_scan(__float_as_int(v), 0, f), 63));
}

// First and last key that any live token of a tile sees; first > last where none does.  (The append writes no rows of masked tokens: what
// lies there is not to count as a row of the tile.)  A lane a token.  GAPS: *gaps is false where every key in between is seen too, as far as
// the tokens in their order tell: each one's keys touch the span of those before it.
template <bool GAPS = false>
__device__ __forceinline__ void tile_keys(const ScoredParams& P, const ScoredTile& t, int lane, int& first, int& last, bool* gaps = nullptr) {
    const uint8_t* token_mask = P.B.valid_token_mask;
    int lo, hi;
    if constexpr (GAPS) *gaps = false;
    if (P.document_starts == nullptr && P.prefix_ends == nullptr && token_mask == nullptr) {  // the first token's window, the last one's reach
        token_keys(P, t.tok0, t.pos0, t.seq_after, first, hi);
        token_keys(P, t.tok0, t.pos0 + t.tokens - 1, t.seq_after, lo, last);
    } else {
        const auto least = [](int a, int b) { return min(a, b); };
        const auto most = [](int a, int b) { return max(a, b); };
        first = 0x7fffffff;
        last = -1;
        for (int base = 0; base < t.tokens; base += 64) {
            const int k = base + lane;
            int from = 0x7fffffff, to = -1;
            if (k < t.tokens && (token_mask == nullptr || token_mask[t.tok0 + k] != 0)) {
                token_keys(P, t.tok0 + k, t.pos0 + k, t.seq_after, lo, hi);
                if (lo <= hi) from = lo, to = hi;
            }
            const int from_upto = wave_scan(from, 0x7fffffff, least), to_upto = wave_scan(to, -1, most);
            if constexpr (GAPS) {
                int from_before = __shfl_up(from_upto, 1, 64), to_before = __shfl_up(to_upto, 1, 64);
                from_before = min(lane > 0 ? from_before : 0x7fffffff, first);
                to_before = max(lane > 0 ? to_before : -1, last);
                if (__ballot(from <= to && to_before >= 0 && (from > to_before + 1 || to < from_before - 1)) != 0ull) *gaps = true;
            }
            first = min(first, __builtin_amdgcn_readlane(from_upto, 63));
            last = max(last, __builtin_amdgcn_readlane(to_upto, 63));
        }
    }
    first = __builtin_amdgcn_readfirstlane(first);
    last = __builtin_amdgcn_readfirstlane(last);
}
// The half units of a tile as the cut of a batch counts them: by its first and last token.  (Tokens between them may see others; then the
// tile's chunks are longer or shorter, and no less right.)
__device__ __forceinline__ int tile_halves_guess(const ScoredParams& P, const ScoredTile& t) {
    if (t.tokens <= 0) return -1;
    int lo0, hi0, lo1, hi1;
    token_keys(P, t.tok0, t.pos0, t.seq_after, lo0, hi0);
    token_keys(P, t.tok0 + t.tokens - 1, t.pos0 + t.tokens - 1, t.seq_after, lo1, hi1);
    const int first = min(lo0, lo1), last = max(hi0, hi1);
    return first <= last ? (last >> 4) - (first >> 4) + 1 : 0;
}
// Half units: 16 keys from a multiple of 16 on, which lie in one page.
__device__ __forceinline__ int tile_halves(int first, int last) { return first <= last ? (last >> 4) - (first >> 4) + 1 : 0; }

// The cut of a batch.  All tiles have chunks of up to `per` half units, a tile's chunks are of one length, and a live tile has one at
// least.  Tiles with several chunks have a record for each: no more than the scratch holds.  P.full_rounds == 0: the shortest `per` that
// needs no more than P.target chunks.  Otherwise, where the tiles make a round of workgroups by themselves, only what is longer than an even
// share by more than a chunk costs is cut; where they do not, the chunks make one full round, or two where one would be a chunk's
// cost longer than an even share (a chunk more than a round takes a round of its own).  us a call, cutting all to even shares / so: 9 requests
// of 300 to 900 BF16 tokens on 1 000 to 9 000 keys 391 / 412, packed documents (tiles of 1 to 43 units) 123 / 109; chunks of 1 / 256 of the keys
// always / so: 600 tokens on 5 000 FP8 keys 148 / 106, 6 requests of 100 to 500 TQ4 tokens 172 / 136, prefix over FP8 331 / 334.
// count(e): the half units of entry e, -1 for tiles without tokens.
// Entries of a batch that is cut.  us a call, up to 2 048 / up to 512: one request of 60 000 keys among 600 of 100 94 / 620, among 1 800 306 / 765;
// 600 requests of 16 to 4 000 keys, which need no cut, 467 / 456.
constexpr int kMaxSplitEntries = 2048;
constexpr int kChunkCost = 32;          // what a workgroup takes beside its keys, in half units
__device__ __forceinline__ int chunks_of(int halves, int per) { return halves < 0 ? 0 : max(1, fast_div(halves + per - 1, per)); }
template <typename Count>
__device__ __forceinline__ int chunk_length(const ScoredParams& P, int lane, Count&& count) {
    int total = 0, live = 0;
    for (int e = lane; e < P.entries; e += 64) {
        const int h = count(e);
        total += max(h, 0);
        live += h >= 0 ? 1 : 0;
    }
    total = wave_sum(total);
    live = wave_sum(live);
    const auto fits = [&](int per, int limit) {
        int n = 0, several = 0;
        for (int e = lane; e < P.entries; e += 64) {
            const int c = chunks_of(count(e), per);
            n += c;
            several += c > 1 ? c : 0;
        }
        return wave_sum(n) <= limit && wave_sum(several) <= P.records;
    };
    int limit = P.target, per;
    if (P.full_rounds == 0) {
        per = (total + limit - 1) / limit;
    } else {
        const int even = (total + P.round - 1) / P.round;  // what a CU has of it
        if (live >= P.round) {
            per = even + kChunkCost;
        } else if (fits(even + kChunkCost, min(P.target, P.round))) {
            limit = min(P.target, P.round);
            per = even;
        } else {
            limit = min(P.target, 2 * P.round);
            per = (even + 1) / 2;
        }
    }
    per = max(per, P.min_halves);
    if (P.entries == 1 ? chunks_of(total, per) <= P.records : fits(per, limit)) return per;
    // sum of ceil(h / per) <= total / per + live, so this many halves a chunk are enough for any number of slots above live
    int low = per, high = max(per + 1, (total + max(limit - live, 1) - 1) / max(limit - live, 1));
    while (high < 1 << 27 && !fits(high, limit)) {  // (a tile has no more half units than that)
        low = high;
        high *= 2;
    }
    while (high - low > max(1, low >> 5)) {
        const int mid = (low + high) >> 1;
        if (fits(mid, limit)) high = mid;
        else low = mid;
    }
    return high;
}
// The tile and chunk of a slot, and the record of the tile's first chunk; entry -1: the slot stays empty.
struct ScoredWork {
    int entry, chunk, chunks, first_record;
};
template <typename Count>
__device__ __forceinline__ ScoredWork find_work(const ScoredParams& P, int per, int slot, int lane, Count&& count) {
    int before = 0, records = 0;
    for (int base = 0; base < P.entries; base += 64) {
        const int mine = base + lane < P.entries ? chunks_of(count(base + lane), per) : 0, split = mine > 1 ? mine : 0;
        const int upto = before + wave_prefix(mine), records_upto = records + wave_prefix(split);
        const unsigned long long hit = __ballot(slot < upto);
        if (hit != 0ull) {
            const int l = (int)__builtin_ctzll(hit);
            const int n = __builtin_amdgcn_readlane(mine, l), end = __builtin_amdgcn_readlane(upto, l);
            return ScoredWork{base + l, slot - (end - n), n, __builtin_amdgcn_readlane(records_upto, l) - n};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        records = __builtin_amdgcn_readlane(records_upto, 63);
    }
    return ScoredWork{-1, 0, 0, 0};
}

// The same with the longest chunks first: workgroups start in the order of their slots, so what starts last is short, and the batch ends
// at once on all CUs.  64 classes of length; hist: in LDS, zeros at first.  For all threads of a workgroup (threads: their number).
__device__ __forceinline__ int length_class(int halves, int chunks, float classes_per_half) {
    return 63 - min(63, (int)((float)fast_div(halves + chunks - 1, chunks) * classes_per_half));
}
template <typename Count>
__device__ __forceinline__ ScoredWork find_work_by_length(const ScoredParams& P, int per, int slot, int tid, int threads, int lane, int* hist, Count&& count) {
    const float scale = 64.0f / (float)(per + 1);
    for (int e = tid; e < P.entries; e += threads) {
        const int h = count(e), c = chunks_of(h, per);
        if (c > 0) atomicAdd(&hist[length_class(h, c, scale)], c);
    }
    __syncthreads();
    const int chunks = hist[lane], chunks_upto = wave_prefix(chunks);
    const unsigned long long classes = __ballot(slot < chunks_upto);
    if (classes == 0ull) return ScoredWork{-1, 0, 0, 0};
    const int cls = (int)__builtin_ctzll(classes);
    const int rest = slot - (__builtin_amdgcn_readlane(chunks_upto, cls) - __builtin_amdgcn_readlane(chunks, cls));
    int before = 0, records = 0;
    for (int base = 0; base < P.entries; base += 64) {
        const int h = base + lane < P.entries ? count(base + lane) : -1, c = chunks_of(h, per);
        const int mine = c > 0 && length_class(h, c, scale) == cls ? c : 0, split = c > 1 ? c : 0;
        const int upto = before + wave_prefix(mine), records_upto = records + wave_prefix(split);
        const unsigned long long hit = __ballot(rest < upto);
        if (hit != 0ull) {
            const int l = (int)__builtin_ctzll(hit);
            const int n = __builtin_amdgcn_readlane(mine, l), end = __builtin_amdgcn_readlane(upto, l);
            return ScoredWork{base + l, rest - (end - n), n, __builtin_amdgcn_readlane(records_upto, l) - n};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        records = __builtin_amdgcn_readlane(records_upto, 63);
    }
    return ScoredWork{-1, 0, 0, 0};
}

// The end of a row: lane l holds channels 4 l .. 4 l + 3 of the sum, un-normalised; value_scale: what the sums have to be multiplied by.
template <typename TQ, int HD>
__device__ __forceinline__ void finish_row(const ScoredParams& P, int tok, int head, int lane, float (&v)[4], float m, float l, float value_scale) {
    const size_t row = (size_t)tok * P.num_q_heads + (size_t)head;
    const float inv = l > 0.f || l != l ? value_scale / l : 0.f;  // (a row without keys: zeros)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= inv;
    if (HD == 256 && P.rot_out) {
        wht256_wave(v, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = apply_sign(v[k], 4 * lane + k);
    }
    if (4 * lane < HD) {
        const uint32_t a = (uint32_t)TQ::from_f32(v[0]) | (uint32_t)TQ::from_f32(v[1]) << 16;
        const uint32_t b = (uint32_t)TQ::from_f32(v[2]) | (uint32_t)TQ::from_f32(v[3]) << 16;
        *reinterpret_cast<uint2*>(P.out + row * HD + 4 * lane) = uint2{a, b};
    }
    if (P.lse != nullptr && lane == 0) P.lse[row] = l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// Joins the chunks of rows.  SPREAD: a workgroup of eight waves for each column of each tile, wave w adds up chunks w, w + 8, ... (one
// request and kv head has up to 256 chunks, 512 at head_dim 128).  Otherwise a wave a column, kJoinCols columns a workgroup: many tiles, of which few have several chunks (a
// workgroup for each of the 131 072 columns of 256 tiles and two kv heads took 190 us to find that, one for eight columns 24 us).
constexpr int kJoinCols = 64;
template <typename TQ, int HD, bool SPREAD>
__global__ __launch_bounds__(512) void scored_join_kernel(const ScoredParams P, int columns, float value_scale) {
    __shared__ __align__(16) float sums[SPREAD ? 8 : 1][SPREAD ? HD : 4];
    const int entry = (int)blockIdx.x, kv_sub = (int)blockIdx.y;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const ScoredTile t = scored_tile(P, entry);
    if (t.tokens <= 0) return;
    const int first = P.table[2 * entry], chunks = P.table[2 * entry + 1];
    if (chunks <= 1) return;
    const int kv_subs = P.L.local_kv_heads * P.q_subgroups;
    const int end_col = SPREAD ? (int)blockIdx.z + 1 : kJoinCols * ((int)blockIdx.z + 1);
    for (int col = SPREAD ? (int)blockIdx.z : kJoinCols * (int)blockIdx.z + wave; col < end_col; col += 8) {
        const int mine = column_token(col, P);
        if (mine >= t.tokens) return;
        const int tok = t.tok0 + mine;
        if (P.B.valid_token_mask != nullptr && P.B.valid_token_mask[tok] == 0) continue;
        const auto record = [&](int c) { return ((size_t)(first + c) * kv_subs + kv_sub) * columns + col; };
        const int at = (4 * lane) & (HD - 1);
        constexpr int kStep = SPREAD ? 8 : 1, kBatch = 8;  // chunks from one to the next of a wave; loads that travel together
        static_assert(64 % (kStep * kBatch) == 0, "what is loaded is added up before the weights of the next 64 chunks");
        const int own = SPREAD ? wave : 0;
        f4 part[kBatch];
        const auto load = [&](int from) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                if (from + kStep * k < chunks) part[k] = *reinterpret_cast<const f4*>(P.part_acc + record(from + kStep * k) * HD + at);
        };
        const auto states = [&](int base) {
            return base + lane < chunks ? *reinterpret_cast<const f2*>(P.part_ml + 2 * record(base + lane)) : f2{kNegBig, 0.f};
        };
        f2 ml = states(0);
        load(own);  // (before their weights are known)
        float m = ml[0];
        for (int base = 64; base < chunks; base += 64) m = fmaxf(m, states(base)[0]);
        m = wave_most(m);
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
        for (int base = 0; base < chunks; base += 64) {
            if (base > 0) ml = states(base);
            const float w = __builtin_amdgcn_exp2f(ml[0] - m);
            l += ml[1] * w;
            const int end = min(64, chunks - base);
            for (int from = own; from < end; from += kBatch * kStep) {
                if (base + from > own) load(base + from);
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (from + kStep * k < end) acc += part[k] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), from + kStep * k));
            }
        }
        l = wave_total(l);
        float v[4] = {acc[0], acc[1], acc[2], acc[3]};
        if constexpr (SPREAD) {
            if (4 * lane < HD) *reinterpret_cast<f4*>(&sums[wave][at]) = acc;
            __syncthreads();
            if (wave != 0) return;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const f4 s = *reinterpret_cast<const f4*>(&sums[w][at]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += s[k];
            }
        }
        const int head = (kv_sub / P.q_subgroups) * P.gqa + (kv_sub % P.q_subgroups) * P.q_group + (col - mine * P.q_group);
        finish_row<TQ, HD>(P, tok, head, lane, v, m, l, value_scale);
    }
}

}  // namespace w34
