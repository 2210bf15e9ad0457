// Verification of drafted tokens: acceptance by u * q(x) < p(x), and one token drawn behind the accepted ones,
//
//   x = the lowest index with  sum_{y <= x} w(y) > u * sum_y w(y),   w = max(p - q, 0) behind a refusal, p otherwise,
//
// in 64 bits: a running sum over 10^5 entries in 32 bits is 10^-7 off at each of them, which moves one border in a thousand draws.
//
// One row of p (and of q) a request is all that is read, by as many workgroups as there are tiles of kDraftTile entries; a second launch, a
// workgroup a request, finds the tile by the tiles' sums and the entry inside it.
// Bound: latency for a few requests, HBM for many.
#include "../../include/warp34_drafts.h"
#include "attn_launch.h"
#include "kv_common.h"

namespace w34 {

constexpr int kDraftTile = 1024;  // entries of a workgroup of 256 threads, four in a row each
constexpr int kDraftMaxReqs = 1 << 20;

struct DraftArgs {
    const int32_t *query_start_loc, *tokens;
    const uint8_t* valid_req_mask;
    const float *target, *draft, *accept_u, *sample_u;
    int64_t target_stride, draft_stride;
    int32_t *out_tokens, *counts;
    double2* sums;  // [request][tile] of (p, what a refusal leaves), nullptr: none
    int total_tokens, vocab, tiles;
};

struct DraftRow {
    int lo, n;       // the request's rows
    int accepted;    // drafts
    int refused;     // the token whose refusal ends them, -1: none
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

// Weights of an entry: p, and what a refusal leaves of it.
struct DraftWeights {
    const float *p, *q;
    int refused;
    __device__ __forceinline__ double2 at(int x) const {
        const double w = proper(p[x]);
        if (refused < 0) return make_double2(w, 0.0);
        const double rest = q != nullptr ? w - proper(q[x]) : x == refused ? 0.0 : w;
        return make_double2(w, rest > 0.0 ? rest : 0.0);
    }
};
__device__ __forceinline__ DraftWeights draft_weights(const DraftArgs& a, const DraftRow& d) {
    const int64_t row = d.lo + d.accepted;
    return {a.target + row * a.target_stride, a.draft == nullptr ? nullptr : a.draft + row * a.draft_stride, d.refused};
}

__device__ __forceinline__ double shfl_up_f64(double v, int by) { return __shfl_up(v, by, 64); }

// Sum over the threads before this one of a workgroup of 256, and the sum of all.  `waves` is LDS for four sums.
__device__ __forceinline__ double sum_before(double v, double* waves, double& total) {
    const int lane = lane_id(), wave = (int)threadIdx.x >> 6;
    double run = v;
#pragma unroll
    for (int by = 1; by < 64; by *= 2) {
        const double o = shfl_up_f64(run, by);
        if (lane >= by) run += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = run;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    return before + (run - v);
}

// Sums of a tile's weights (both in one reduction's time).
__device__ __forceinline__ double2 tile_sums(const DraftWeights& w, int tile, int vocab, double* waves) {
    double2 s = make_double2(0.0, 0.0);
    const int x0 = tile * kDraftTile + (int)threadIdx.x * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (x0 + k < vocab) {
            const double2 v = w.at(x0 + k);
            s.x += v.x, s.y += v.y;
        }
#pragma unroll
    for (int by = 32; by; by /= 2) {
        s.x += __shfl_xor(s.x, by, 64);
        s.y += __shfl_xor(s.y, by, 64);
    }
    __syncthreads();
    if (lane_id() == 0) waves[threadIdx.x >> 6] = s.x, waves[4 + (threadIdx.x >> 6)] = s.y;
    __syncthreads();
    return make_double2(waves[0] + waves[1] + waves[2] + waves[3], waves[4] + waves[5] + waves[6] + waves[7]);
}

__global__ __launch_bounds__(256) void draft_sums_kernel(const DraftArgs a) {
    __shared__ double waves[8];
    const int req = (int)(blockIdx.x / (uint32_t)a.tiles), tile = (int)(blockIdx.x - (uint32_t)req * (uint32_t)a.tiles);
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = draft_row(a, req);
    if (d.n == 0) return;
    const double2 s = tile_sums(draft_weights(a, d), tile, a.vocab, waves);
    if (threadIdx.x == 0) a.sums[(int64_t)req * a.tiles + tile] = s;
}

// The token drawn, the same in every thread.  Without stored sums they are made again where they are asked for.
__device__ int draw_token(const DraftArgs& a, int req, const DraftRow& d, double* waves, int* found) {
    const DraftWeights w = draft_weights(a, d);
    const double2* stored = a.sums == nullptr ? nullptr : a.sums + (int64_t)req * a.tiles;
    // a thread's tiles stand in a row, so that its sum is one step of the running sum
    const int each = (a.tiles + 255) / 256, first = (int)threadIdx.x * each;
    double2 mine = make_double2(0.0, 0.0);
    if (stored != nullptr) {
        for (int t = first; t < min(first + each, a.tiles); ++t) mine.x += stored[t].x, mine.y += stored[t].y;
    } else {
        for (int t = 0; t < a.tiles; ++t) {
            const double2 s = tile_sums(w, t, a.vocab, waves);
            if (t >= first && t < first + each) mine.x += s.x, mine.y += s.y;
        }
    }
    double total_p, total_rest;
    const double before_p = sum_before(mine.x, waves, total_p), before_rest = sum_before(mine.y, waves, total_rest);
    const bool rest = d.refused >= 0 && total_rest > 0.0;
    const double total = rest ? total_rest : total_p, target = (double)a.sample_u[req] * total;
    if (!(total > 0.0)) return -1;
    const double have = rest ? mine.y : mine.x, before = rest ? before_rest : before_p;
    // found[0]: the lowest thread whose tiles pass the target; [1]: the last one with any weight, which stands in where rounding leaves none
    if (threadIdx.x == 0) found[0] = 256, found[1] = -1;
    __syncthreads();
    if (have > 0.0) {
        if (before + have > target) atomicMin(&found[0], (int)threadIdx.x);
        atomicMax(&found[1], (int)threadIdx.x);
    }
    __syncthreads();
    const int owner = found[0] < 256 ? found[0] : found[1];
    __syncthreads();
    // its tiles one after another
    double* base = waves + 8;
    if ((int)threadIdx.x == owner) *base = before;
    __syncthreads();
    double run = *base;
    int last = -1;  // the last entry with any weight so far
    for (int t = owner * each; t < min(owner * each + each, a.tiles); ++t) {
        const int x0 = t * kDraftTile + (int)threadIdx.x * 4;
        double v[4], sum = 0.0, tile_total;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double2 both = x0 + k < a.vocab ? w.at(x0 + k) : make_double2(0.0, 0.0);
            v[k] = rest ? both.y : both.x;
            sum += v[k];
        }
        double at = run + sum_before(sum, waves, tile_total);
        int here = 1 << 30, weighted = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            at += v[k];
            if (v[k] > 0.0) {
                weighted = x0 + k;
                if (at > target && here == 1 << 30) here = x0 + k;
            }
        }
        if (threadIdx.x == 0) found[0] = 1 << 30, found[1] = last;
        __syncthreads();
        if (here != 1 << 30) atomicMin(&found[0], here);
        if (weighted >= 0) atomicMax(&found[1], weighted);
        __syncthreads();
        const int hit = found[0];
        last = found[1];
        __syncthreads();
        if (hit != 1 << 30) return hit;
        run += tile_total;
    }
    return last;
}

__global__ __launch_bounds__(256) void draft_draw_kernel(const DraftArgs a) {
    __shared__ double waves[9];
    __shared__ int found[2];
    const int req = (int)blockIdx.x;
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = draft_row(a, req);
    int drawn = -1;
    if (d.n > 0) drawn = draw_token(a, req, d, waves, found);
    for (int i = (int)threadIdx.x; i < d.n; i += 256)
        a.out_tokens[d.lo + i] = i < d.accepted ? a.tokens[d.lo + i + 1] : i == d.accepted ? drawn : -1;
    if (threadIdx.x == 0) a.counts[req] = d.n > 0 ? d.accepted + 1 : 0;
}

static int draft_tiles(int vocab) { return (int)(((int64_t)vocab + kDraftTile - 1) / kDraftTile); }

}  // namespace w34

using namespace w34;

extern "C" size_t warp34_verify_drafts_scratch_bytes(int num_reqs, int vocab_size) {
    if (num_reqs <= 0 || num_reqs > kDraftMaxReqs || vocab_size <= 0) return 0;
    return sizeof(double2) * (size_t)num_reqs * (size_t)draft_tiles(vocab_size);
}

extern "C" int warp34_verify_drafts(const warp34_exec* ex, const warp34_draft_batch* batch, const float* target_probs, const float* draft_probs,
                                    const float* accept_uniforms, const float* sample_uniforms, int32_t* out_tokens, int32_t* emitted_counts) {
    if (!ex || !batch || !target_probs || !accept_uniforms || !sample_uniforms || !out_tokens || !emitted_counts || !batch->query_start_loc ||
        !batch->tokens || batch->vocab_size < 1 || batch->target_row_stride < batch->vocab_size ||
        (draft_probs && batch->draft_row_stride < batch->vocab_size) || batch->num_reqs > kDraftMaxReqs)
        return (int)hipErrorInvalidValue;
    if (batch->num_reqs <= 0 || batch->total_tokens <= 0) return 0;
    DraftArgs a{batch->query_start_loc, batch->tokens, batch->valid_req_mask, target_probs, draft_probs, accept_uniforms, sample_uniforms,
                batch->target_row_stride, batch->draft_row_stride, out_tokens, emitted_counts, nullptr, batch->total_tokens, batch->vocab_size,
                draft_tiles(batch->vocab_size)};
    const size_t need = warp34_verify_drafts_scratch_bytes(batch->num_reqs, batch->vocab_size);
    if (ex->scratch_ptr && (ex->scratch_ptr & 15u) == 0 && ex->scratch_size >= need && grid_fits((long long)batch->num_reqs * a.tiles, 256)) {
        a.sums = (double2*)(uintptr_t)ex->scratch_ptr;
        hipLaunchKernelGGL(draft_sums_kernel, dim3((unsigned)((long long)batch->num_reqs * a.tiles)), dim3(256), 0, (hipStream_t)ex->stream, a);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    hipLaunchKernelGGL(draft_draw_kernel, dim3((unsigned)batch->num_reqs), dim3(256), 0, (hipStream_t)ex->stream, a);
    return (int)hipGetLastError();
}
