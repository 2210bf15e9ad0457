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
    float scale2;     // |sm_scale| log2e, not 0 (hidden keys have scores of minus infinity)
    uint32_t q_flip;  // sm_scale < 0: the sign bits of a pair of query elements
    float cap2;       // cap log2e; 0: no cap
    float cap_arg;    // 2 |sm_scale| log2e / cap: exp2 of it times q.k is exp(2 x / cap)
    int wide_cap;     // the cap is so large that tanh of a small argument needs its series (kWideCap)
    int num_q_heads, gqa, q_group, q_subgroups;
    int tok_tile;     // query tokens of a tile
    int tiles;        // tiles of a request (a bound)
    int entries;      // requests x tiles: tiles of the batch, some of them empty
    int target;       // slots for chunks, for each kv head; 0: no split, a workgroup for each entry
    int min_halves;   // shortest chunk
    float* part_acc;  // [slot][kv_sub][column][head_dim]
    float* part_ml;   // [slot][kv_sub][column]{m, l}
    int32_t* table;   // [entry]{first slot, chunks}
    uint32_t block_magic, q_group_magic;
    int rot_q, rot_out;
};

// tanh(u) = 1 - 2 / (exp(2 u) + 1) is off by some 2^-23 whatever u, which the cap multiplies: 6e-5 at this cap, beyond it small
// arguments go through the series.
constexpr float kWideCap = 512.0f;

// Scores s (q . k times what the column's scale is in) become y with x = y ca + cb in the log2 domain, ca >= 0, so that the largest y is
// the largest x and exp2's argument x - m is one fma.  No cap: y = s, x = y cs.  Cap: y = -1 / (exp(2 x / cap) + 1), x = cap2 + 2 cap2 y.
// cs >= 0 and cc: the column's scale times scale2 / cap_arg.  (The choice stands outside the loop: one uniform branch.)
struct ScoreMap {
    float ca, cb;
};
template <bool CAP, int N, typename V>
__device__ __forceinline__ ScoreMap map_scores(V& s, float cs, float cc, const ScoredParams& P) {
    if constexpr (!CAP) {
        return ScoreMap{cs, 0.f};
    } else if (!P.wide_cap) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[i] * cc));
        return ScoreMap{2.0f * P.cap2, P.cap2};
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = s[i] * cc, u = a * (0.5f / kLog2e), uu = u * u;
            const float x = __builtin_fmaf(2.0f * P.cap2, __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(a)), P.cap2);
            const float series = __builtin_fmaf(uu, __builtin_fmaf(uu, __builtin_fmaf(uu, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
            s[i] = fabsf(u) < 0.1f ? s[i] * cs * series : x;
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
// First and last key that any token of a tile sees; first > last where none does.
__device__ __forceinline__ void tile_keys(const ScoredParams& P, const ScoredTile& t, int& first, int& last) {
    if (P.document_starts == nullptr && P.prefix_ends == nullptr) {  // the first token's window, the last one's reach
        int lo, hi;
        token_keys(P, t.tok0, t.pos0, t.seq_after, first, hi);
        token_keys(P, t.tok0, t.pos0 + t.tokens - 1, t.seq_after, lo, last);
        return;
    }
    first = 0x7fffffff;
    last = -1;
    for (int k = 0; k < t.tokens; ++k) {
        int lo, hi;
        token_keys(P, t.tok0 + k, t.pos0 + k, t.seq_after, lo, hi);
        if (lo <= hi) {
            first = min(first, lo);
            last = max(last, hi);
        }
    }
}
// Half units: 16 keys from a multiple of 16 on, which lie in one page.
__device__ __forceinline__ int tile_halves(int first, int last) { return first <= last ? (last >> 4) - (first >> 4) + 1 : 0; }

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ int wave_prefix(int v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d, 64);
        v += lane >= d ? u : 0;
    }
    return v;
}

// The cut of a batch: chunks of `per` half units, the shortest length with which all tiles together need no more than P.target chunks;
// a live tile has at least one.  halves: [entries] in LDS, -1 for tiles without tokens.
constexpr int kMaxSplitEntries = 512;   // entries of a batch that is split
__device__ __forceinline__ int chunks_of(int halves, int per) { return halves < 0 ? 0 : max(1, fast_div(halves + per - 1, per)); }
__device__ __forceinline__ int chunk_length(const ScoredParams& P, const int* halves, int lane) {
    int total = 0, live = 0, longest = 0;
    for (int e = lane; e < P.entries; e += 64) {
        total += max(halves[e], 0);
        live += halves[e] >= 0 ? 1 : 0;
        longest = max(longest, halves[e]);
    }
    total = __builtin_amdgcn_readfirstlane(wave_sum(total));
    live = __builtin_amdgcn_readfirstlane(wave_sum(live));
    // too short / long enough: sum of ceil(h / per) <= total / per + live
    int low = max(P.min_halves, (total + P.target - 1) / P.target) - 1;
    int high = max(low + 1, (total + P.target - live - 1) / max(P.target - live, 1));
    while (high - low > 1 && P.entries <= 64) {
        const int mid = (low + high) >> 1;
        const int n = wave_sum(lane < P.entries ? chunks_of(halves[lane], mid) : 0);
        if (__builtin_amdgcn_readfirstlane(n) <= P.target) high = mid;
        else low = mid;
    }
    return high;
}
// The tile and chunk of a slot; entry -1: the slot stays empty.
struct ScoredWork {
    int entry, chunk, chunks, first_slot;
};
__device__ __forceinline__ ScoredWork find_work(const ScoredParams& P, const int* halves, int per, int slot, int lane) {
    int before = 0;
    for (int base = 0; base < P.entries; base += 64) {
        const int mine = base + lane < P.entries ? chunks_of(halves[base + lane], per) : 0;
        const int upto = before + wave_prefix(mine, lane);
        const unsigned long long hit = __ballot(slot < upto);
        if (hit != 0ull) {
            const int l = (int)__builtin_ctzll(hit);
            const int n = __builtin_amdgcn_readlane(mine, l), end = __builtin_amdgcn_readlane(upto, l);
            return ScoredWork{base + l, slot - (end - n), n, end - n};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
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

// Joins the chunks of a row: a workgroup of eight waves for each column of each tile that has several; wave w adds up chunks w, w + 8, ...
template <typename TQ, int HD>
__global__ __launch_bounds__(512) void scored_join_kernel(const ScoredParams P, int columns, float value_scale) {
    __shared__ __align__(16) float sums[8][HD];
    const int entry = (int)blockIdx.x, kv_sub = (int)blockIdx.y, col = (int)blockIdx.z;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const ScoredTile t = scored_tile(P, entry);
    const int mine = column_token(col, P);
    if (mine >= t.tokens) return;
    const int tok = t.tok0 + mine;
    if (P.B.valid_token_mask != nullptr && P.B.valid_token_mask[tok] == 0) return;
    const int first = P.table[2 * entry], chunks = P.table[2 * entry + 1];
    if (chunks <= 1) return;
    const int kv_subs = P.L.local_kv_heads * P.q_subgroups;
    const auto record = [&](int c) { return ((size_t)(first + c) * kv_subs + kv_sub) * columns + col; };
    float m = kNegBig;
    for (int c = lane; c < chunks; c += 64) m = fmaxf(m, P.part_ml[2 * record(c)]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    f4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    const int at = (4 * lane) & (HD - 1);
    for (int base = 0; base < chunks; base += 64) {
        const int c = base + lane;
        f2 ml = {kNegBig, 0.f};
        if (c < chunks) ml = *reinterpret_cast<const f2*>(P.part_ml + 2 * record(c));
        const float w = __builtin_amdgcn_exp2f(ml[0] - m);
        l += ml[1] * w;
        // a wave's eight records at most, their loads together
        const int end = min(64, chunks - base);
        f4 part[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (wave + 8 * k < end) part[k] = *reinterpret_cast<const f4*>(P.part_acc + record(base + wave + 8 * k) * HD + at);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (wave + 8 * k < end) acc += part[k] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), wave + 8 * k));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    if (4 * lane < HD) *reinterpret_cast<f4*>(&sums[wave][at]) = acc;
    __syncthreads();
    if (wave != 0) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const f4 s = *reinterpret_cast<const f4*>(&sums[w][at]);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += s[k];
    }
    const int head = (kv_sub / P.q_subgroups) * P.gqa + (kv_sub % P.q_subgroups) * P.q_group + (col - mine * P.q_group);
    finish_row<TQ, HD>(P, tok, head, lane, v, m, l, value_scale);
}

}  // namespace w34
