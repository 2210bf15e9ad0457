// Verification of drafted tokens: acceptance by u * q(x) < p(x), and one token drawn behind the accepted ones,
//
//   x = the lowest index with  sum_{y <= x} w(y) > u * sum_y w(y),   w = max(p - q, 0) behind a refusal, p otherwise,
//
// in 64 bits: a running sum over 10^5 entries in 32 bits is 10^-7 off at each of them, which moves one border in a thousand draws.
//
// One row of p (and of q) a request is all that is read, by as many workgroups as there are tiles of kDraftTile entries; a second launch, a
// wave a request, finds the tile by the tiles' sums and the entry inside it.
// Bound: latency for a few requests, HBM for many.
#include "../../include/warp34_drafts.h"
#include "attn_launch.h"
#include "kv_common.h"

namespace w34 {

constexpr int kDraftThreads = 256, kDraftEntries = 8;      // entries in a row of a thread
constexpr int kDraftTile = kDraftThreads * kDraftEntries;  // of a workgroup
constexpr int kDraftMaxReqs = 1 << 20;

struct DraftRow {
    int lo, n;       // the request's rows
    int accepted;    // drafts
    int refused;     // the token whose refusal ends them, -1: none
};

struct DraftArgs {
    const int32_t *query_start_loc, *tokens;
    const uint8_t* valid_req_mask;
    const float *target, *draft, *accept_u, *sample_u;
    int64_t target_stride, draft_stride;
    int32_t *out_tokens, *counts;
    double2* sums;   // [request][tile] of (p, what a refusal leaves), nullptr: none
    DraftRow* rows;  // [request] beside them
    int total_tokens, vocab, tiles;
};

// What a wave finds out about a request, the same in every lane.
__device__ __forceinline__ DraftRow draft_row(const DraftArgs& a, int req) {
    const int lane = lane_id();
    DraftRow d;
    d.lo = max(0, a.query_start_loc[req]);
    d.n = max(0, min(a.query_start_loc[req + 1], a.total_tokens) - d.lo);
    d.accepted = max(0, d.n - 1);
    d.refused = -1;
    for (int base = 0; base < d.n - 1; base += 64) {
        const int i = base + lane;
        bool ok = true;
        int token = -1;
        if (i < d.n - 1) {
            token = a.tokens[d.lo + i + 1];
            ok = false;
            if (token >= 0 && token < a.vocab) {
                const int64_t row = d.lo + i;
                const double p = a.target[row * a.target_stride + token];
                const double q = a.draft == nullptr ? 1.0 : (double)a.draft[row * a.draft_stride + token];
                ok = (double)a.accept_u[row] * q < p;
            }
        }
        const unsigned long long bad = __ballot(!ok);
        if (bad) {
            const int first = __builtin_ctzll(bad);
            d.accepted = base + first;
            token = __shfl(token, first, 64);
            d.refused = token >= 0 && token < a.vocab ? token : -1;
            break;
        }
    }
    return d;
}

__device__ __forceinline__ double proper(float x) { return x > 0.f && x < INFINITY ? (double)x : 0.0; }

// Weights of a row's entries: p, and what a refusal leaves of it.
struct DraftWeights {
    const float *p, *q;
    int refused, vocab;
};
__device__ __forceinline__ DraftWeights draft_weights(const DraftArgs& a, const DraftRow& d) {
    const int64_t row = d.lo + d.accepted;
    return {a.target + row * a.target_stride, a.draft == nullptr || d.refused < 0 ? nullptr : a.draft + row * a.draft_stride, d.refused, a.vocab};
}
typedef float f4_at4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

// 4 N entries from x0 on.  Behind the vocabulary there is no weight.
template <int N>
struct DraftEntries {
    float p[4 * N], q[4 * N];
    int x0;
    __device__ __forceinline__ void load(const DraftWeights& w, int from) {
        x0 = from;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = x0 + 4 * i;
            f4_at4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
            if (x <= w.vocab - 4) {
                a = *reinterpret_cast<const f4_at4*>(w.p + x);
                if (w.q != nullptr) b = *reinterpret_cast<const f4_at4*>(w.q + x);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (x < w.vocab - k) {
                        a[k] = w.p[x + k];
                        if (w.q != nullptr) b[k] = w.q[x + k];
                    }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) p[4 * i + k] = a[k], q[4 * i + k] = b[k];
        }
    }
    __device__ __forceinline__ double whole(int i) const { return proper(p[i]); }
    __device__ __forceinline__ double rest(const DraftWeights& w, int i) const {
        const double left = w.q != nullptr ? proper(p[i]) - proper(q[i]) : x0 + i == w.refused ? 0.0 : proper(p[i]);
        return left > 0.0 ? left : 0.0;
    }
};

// The value of another lane by CTRL (row_shr n, row_bcast), 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the lanes up to and with this one.
__device__ __forceinline__ double wave_run(double v) {
    v += dpp_f64<0x111, 0xF>(v);
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);  // the last lane of a row to the next row
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sums of a tile's weights by a workgroup.  `waves` is LDS for eight sums.
__device__ __forceinline__ double2 tile_sums(const DraftWeights& w, int tile, double* waves) {
    DraftEntries<kDraftEntries / 4> e;
    e.load(w, tile * kDraftTile + (int)threadIdx.x * kDraftEntries);
    double p = 0.0, rest = 0.0;
#pragma unroll
    for (int i = 0; i < kDraftEntries; ++i) p += e.whole(i), rest += w.refused >= 0 ? e.rest(w, i) : 0.0;
    p = wave_run(p), rest = wave_run(rest);
    __syncthreads();
    if (lane_id() == 63) waves[threadIdx.x >> 6] = p, waves[4 + (threadIdx.x >> 6)] = rest;
    __syncthreads();
    return make_double2(waves[0] + waves[1] + waves[2] + waves[3], waves[4] + waves[5] + waves[6] + waves[7]);
}

__global__ __launch_bounds__(kDraftThreads) void draft_sums_kernel(const DraftArgs a) {
    __shared__ double waves[8];
    const int req = (int)(blockIdx.x / (uint32_t)a.tiles), tile = (int)(blockIdx.x - (uint32_t)req * (uint32_t)a.tiles);
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = draft_row(a, req);
    if (tile == 0 && threadIdx.x == 0) a.rows[req] = d;
    if (d.n == 0) return;
    const double2 s = tile_sums(draft_weights(a, d), tile, waves);
    if (threadIdx.x == 0) a.sums[(int64_t)req * a.tiles + tile] = s;
}

// The token drawn by one wave, the same in every lane.  mine: the sums of the lane's tiles, `each` in a row.
__device__ int draw_token(const DraftWeights& w, double u, double2 mine, int each, int tiles) {
    const int lane = lane_id();
    const double run_p = wave_run(mine.x), run_rest = wave_run(mine.y);
    const double total_p = lane_value(run_p, 63), total_rest = lane_value(run_rest, 63);
    const bool from_rest = w.refused >= 0 && total_rest > 0.0;
    const double total = from_rest ? total_rest : total_p, target = u * total;
    if (!(total > 0.0)) return -1;
    const double have = from_rest ? mine.y : mine.x, run = from_rest ? run_rest : run_p;
    // the lowest lane whose tiles pass the target, or the last one with any weight, which stands in where rounding leaves none
    const unsigned long long weighted = __ballot(have > 0.0), past = __ballot(have > 0.0 && run > target);
    if (weighted == 0) return -1;
    const int owner = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(weighted);
    double before = lane_value(run - have, owner);
    int last = -1;  // the last entry with any weight so far
    constexpr int kStep = 64 * 16;
    for (int64_t x = (int64_t)owner * each * kDraftTile; x < min((int64_t)(owner + 1) * each * kDraftTile, (int64_t)w.vocab); x += 2 * kStep) {
        DraftEntries<4> e[2];
        e[0].load(w, (int)x + lane * 16);
        if (x + kStep < w.vocab) e[1].load(w, (int)x + kStep + lane * 16);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (x + half * kStep >= w.vocab) break;
            double v[16], sum = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = from_rest ? e[half].rest(w, i) : e[half].whole(i), sum += v[i];
            const double upto = wave_run(sum);
            double at = before + (upto - sum);
            int here = -1, some = -1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                at += v[i];
                if (v[i] > 0.0) {
                    some = e[half].x0 + i;
                    if (at > target && here < 0) here = some;
                }
            }
            const unsigned long long hits = __ballot(here >= 0), any = __ballot(some >= 0);
            if (hits) return __builtin_amdgcn_readlane(here, __builtin_ctzll(hits));
            if (any) last = __builtin_amdgcn_readlane(some, 63 - __builtin_clzll(any));
            before += lane_value(upto, 63);
        }
    }
    return last;
}

// By the first wave: the request's tokens.
__device__ __forceinline__ void put_tokens(const DraftArgs& a, int req, const DraftRow& d, int drawn) {
    for (int i = lane_id(); i < d.n; i += 64) a.out_tokens[d.lo + i] = i < d.accepted ? a.tokens[d.lo + i + 1] : i == d.accepted ? drawn : -1;
    if (lane_id() == 0) a.counts[req] = d.n > 0 ? d.accepted + 1 : 0;
}

// Behind the sums: a wave a request.  What it needs of memory it asks for in two steps: the request's row, u and its sums, then the tile.
__global__ __launch_bounds__(64) void draft_draw_kernel(const DraftArgs a) {
    const int req = (int)blockIdx.x;
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = a.rows[req];
    const double u = a.sample_u[req];
    int drawn = -1;
    if (d.n > 0) {
        const int each = (a.tiles + 63) / 64, first = lane_id() * each;
        const double2* stored = a.sums + (int64_t)req * a.tiles;
        double2 mine = make_double2(0.0, 0.0);
        for (int t = first; t < min(first + each, a.tiles); ++t) mine.x += stored[t].x, mine.y += stored[t].y;
        drawn = draw_token(draft_weights(a, d), u, mine, each, a.tiles);
    }
    put_tokens(a, req, d, drawn);
}

// Without a workspace: a workgroup a request, which makes the sums itself.
__global__ __launch_bounds__(kDraftThreads) void draft_alone_kernel(const DraftArgs a) {
    __shared__ double waves[8];
    const int req = (int)blockIdx.x;
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = draft_row(a, req);
    int drawn = -1;
    if (d.n > 0) {
        const DraftWeights w = draft_weights(a, d);
        const int each = (a.tiles + 63) / 64, first = lane_id() * each;
        double2 mine = make_double2(0.0, 0.0);
        for (int t = 0; t < a.tiles; ++t) {
            const double2 s = tile_sums(w, t, waves);
            if (t >= first && t < first + each) mine.x += s.x, mine.y += s.y;
        }
        if (threadIdx.x >= 64) return;
        drawn = draw_token(w, a.sample_u[req], mine, each, a.tiles);
    }
    if (threadIdx.x < 64) put_tokens(a, req, d, drawn);
}

static int draft_tiles(int vocab) { return (int)(((int64_t)vocab + kDraftTile - 1) / kDraftTile); }

}  // namespace w34

using namespace w34;

extern "C" size_t warp34_verify_drafts_scratch_bytes(int num_reqs, int vocab_size) {
    if (num_reqs <= 0 || num_reqs > kDraftMaxReqs || vocab_size <= 0) return 0;
    return (size_t)num_reqs * (sizeof(double2) * (size_t)draft_tiles(vocab_size) + sizeof(DraftRow));
}

extern "C" int warp34_verify_drafts(const warp34_exec* ex, const warp34_draft_batch* batch, const float* target_probs, const float* draft_probs,
                                    const float* accept_uniforms, const float* sample_uniforms, int32_t* out_tokens, int32_t* emitted_counts) {
    if (!ex || !batch || !target_probs || !accept_uniforms || !sample_uniforms || !out_tokens || !emitted_counts || !batch->query_start_loc ||
        !batch->tokens || batch->vocab_size < 1 || batch->target_row_stride < batch->vocab_size ||
        (draft_probs && batch->draft_row_stride < batch->vocab_size) || batch->num_reqs > kDraftMaxReqs)
        return (int)hipErrorInvalidValue;
    if (batch->num_reqs <= 0 || batch->total_tokens <= 0) return 0;
    DraftArgs a{batch->query_start_loc, batch->tokens, batch->valid_req_mask, target_probs, draft_probs, accept_uniforms, sample_uniforms,
                batch->target_row_stride, batch->draft_row_stride, out_tokens, emitted_counts, nullptr, nullptr, batch->total_tokens, batch->vocab_size,
                draft_tiles(batch->vocab_size)};
    const size_t need = warp34_verify_drafts_scratch_bytes(batch->num_reqs, batch->vocab_size);
    if (ex->scratch_ptr && (ex->scratch_ptr & 15u) == 0 && ex->scratch_size >= need && grid_fits((long long)batch->num_reqs * a.tiles, kDraftThreads)) {
        a.sums = (double2*)(uintptr_t)ex->scratch_ptr;
        a.rows = (DraftRow*)(a.sums + (size_t)batch->num_reqs * a.tiles);
        hipLaunchKernelGGL(draft_sums_kernel, dim3((unsigned)((long long)batch->num_reqs * a.tiles)), dim3(kDraftThreads), 0, (hipStream_t)ex->stream, a);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
        hipLaunchKernelGGL(draft_draw_kernel, dim3((unsigned)batch->num_reqs), dim3(64), 0, (hipStream_t)ex->stream, a);
    } else {
        hipLaunchKernelGGL(draft_alone_kernel, dim3((unsigned)batch->num_reqs), dim3(kDraftThreads), 0, (hipStream_t)ex->stream, a);
    }
    return (int)hipGetLastError();
}
