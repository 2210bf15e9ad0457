// Verification of drafted tokens: acceptance by u * q(x) < p(x), and one token drawn behind the accepted ones,
//
//   x = the lowest index with  sum_{y <= x} w(y) > u * sum_y w(y),   w = max(p - q, 0) behind a refusal, p otherwise,
//
// in 64 bits: a running sum over 10^5 entries in 32 bits is 10^-7 off at each of them, which moves one border in a thousand draws.
//
// One row of p (and of q) a request is all that is read, by as many workgroups as there are tiles of kDraftTile entries; a second launch, a
// workgroup a request, finds the tile by the tiles' sums and the entry inside it.
// Bound: latency for a few requests, HBM for many.  One request of 128 000 entries 7.5 us, two launches (one workgroup a request instead, as without a
// workspace, goes through 63 tiles one after the other, twice); 32 requests of 150 001, 38 MB, 12.6 us: sums 7.7, the rate of a large copy, and draw 3.8.
// Tiles of 2 048 entries: of 4 096, or sums by one wave through LDS, 32 requests took 18 to 29.
#include "../../include/warp34_drafts.h"
#include "attn_launch.h"
#include "kv_common.h"
#include "wave_sums.h"

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

// The entry of tile `owner`, in front of which weigh `before`, at which the running sum passes the target, by a workgroup: the wave whose entries
// pass it, of these the lane, of its entries the one.  Where rounding lets none pass, the last one with any weight stands in (the tile has some).
// The result is that wave's; the others get -1.
__device__ __forceinline__ int draw_entry(DraftWeights w, bool from_rest, double target, int owner, double before, double* waves) {
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (!from_rest) w.q = nullptr, w.refused = -1;
    DraftEntries<kDraftEntries / 4> e;
    e.load(w, owner * kDraftTile + (int)threadIdx.x * kDraftEntries);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kDraftEntries; ++i) sum += e.rest(w, i);
    const double run = wave_run(sum);
    __syncthreads();
    if (lane == 63) waves[wave] = run;
    __syncthreads();
    int mine = -1;
    double at = before;
    for (int k = 0; k < kDraftThreads / 64; ++k) {
        const double have = waves[k];
        if (have > 0.0) mine = k, before = at;
        at += have;
        if (have > 0.0 && at > target) break;
    }
    if (wave != mine) return -1;
    const unsigned long long some = __ballot(sum > 0.0), past = __ballot(sum > 0.0 && before + run > target);
    const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    before += lane_value(run - sum, l);
    const int first = owner * kDraftTile + (wave * 64 + l) * kDraftEntries, x = first + lane;
    double v = 0.0;
    if (lane < kDraftEntries && x < w.vocab) {
        const double p = proper(w.p[x]);
        v = w.q != nullptr ? p - proper(w.q[x]) : x == w.refused ? 0.0 : p;
        v = v > 0.0 ? v : 0.0;
    }
    const double upto = wave_run(v);
    const unsigned long long any = __ballot(v > 0.0), hit = __ballot(v > 0.0 && before + upto > target);
    return first + (hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any));
}

// A request's tokens but for the one drawn, by a workgroup.
__device__ __forceinline__ void put_tokens(const DraftArgs& a, int req, const DraftRow& d, bool drawn) {
    for (int i = (int)threadIdx.x; i < d.n; i += kDraftThreads) {
        if (i != d.accepted) a.out_tokens[d.lo + i] = i < d.accepted ? a.tokens[d.lo + i + 1] : -1;
        else if (!drawn) a.out_tokens[d.lo + i] = -1;
    }
    if (threadIdx.x == 0) a.counts[req] = d.n > 0 ? d.accepted + 1 : 0;
}

// Behind the sums: a workgroup a request.  It asks for the request's row, u and the first sums at once, then for the tile's entries; each wave
// finds the tile for itself.  Four waves and not one: the tile's entries are a quarter of the code, and it is fetched cold.
__global__ __launch_bounds__(kDraftThreads) void draft_draw_kernel(const DraftArgs a) {
    __shared__ double waves[4];
    const int req = (int)blockIdx.x, lane = lane_id();
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const double2* stored = a.sums + (int64_t)req * a.tiles;
    double2 mine[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) mine[k] = stored[min(64 * k + lane, a.tiles - 1)];
    const DraftRow d = a.rows[req];
    const double u = a.sample_u[req];
    const auto tile = [&](int t0) {
        double2 s = t0 == 0 ? mine[0] : mine[1];
        if (t0 >= 128 && t0 + lane < a.tiles) s = stored[t0 + lane];
        return t0 + lane < a.tiles ? s : make_double2(0.0, 0.0);
    };
    int owner = -1;
    if (d.n > 0) {
        const DraftWeights w = draft_weights(a, d);
        double2 all = make_double2(0.0, 0.0);
        for (int t0 = 0; t0 < a.tiles; t0 += 64) {
            const double2 s = tile(t0);
            all.x += s.x, all.y += s.y;
        }
        const double total_p = lane_value(wave_run(all.x), 63), total_rest = lane_value(wave_run(all.y), 63);
        const bool from_rest = w.refused >= 0 && total_rest > 0.0;
        const double target = u * (from_rest ? total_rest : total_p);
        double before = 0.0, base = 0.0;
        for (int t0 = 0; t0 < a.tiles; t0 += 64) {
            const double2 s = tile(t0);
            const double have = from_rest ? s.y : s.x, run = wave_run(have);
            const unsigned long long some = __ballot(have > 0.0), past = __ballot(have > 0.0 && base + run > target);
            if (some) {
                const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
                owner = t0 + l, before = base + lane_value(run - have, l);
            }
            if (past) break;
            base += lane_value(run, 63);
        }
        if (owner >= 0) {
            const int token = draw_entry(w, from_rest, target, owner, before, waves);
            if (token >= 0 && lane == 0) a.out_tokens[d.lo + d.accepted] = token;
        }
    }
    put_tokens(a, req, d, owner >= 0);
}

// Without a workspace: a workgroup a request, which makes the sums itself, once for the total and once to find the tile.
__global__ __launch_bounds__(kDraftThreads) void draft_alone_kernel(const DraftArgs a) {
    __shared__ double waves[8];
    const int req = (int)blockIdx.x;
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const DraftRow d = draft_row(a, req);
    int owner = -1;
    if (d.n > 0) {
        const DraftWeights w = draft_weights(a, d);
        double2 all = make_double2(0.0, 0.0);
        for (int t = 0; t < a.tiles; ++t) {
            const double2 s = tile_sums(w, t, waves);
            all.x += s.x, all.y += s.y;
        }
        const bool from_rest = w.refused >= 0 && all.y > 0.0;
        const double target = (double)a.sample_u[req] * (from_rest ? all.y : all.x);
        double before = 0.0, base = 0.0;
        for (int t = 0; t < a.tiles; ++t) {
            const double2 s = tile_sums(w, t, waves);
            const double have = from_rest ? s.y : s.x;
            if (have > 0.0) owner = t, before = base;
            base += have;
            if (have > 0.0 && base > target) break;
        }
        if (owner >= 0) {
            const int token = draw_entry(w, from_rest, target, owner, before, waves);
            if (token >= 0 && lane_id() == 0) a.out_tokens[d.lo + d.accepted] = token;
        }
    }
    put_tokens(a, req, d, owner >= 0);
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
        hipLaunchKernelGGL(draft_draw_kernel, dim3((unsigned)batch->num_reqs), dim3(kDraftThreads), 0, (hipStream_t)ex->stream, a);
    } else {
        hipLaunchKernelGGL(draft_alone_kernel, dim3((unsigned)batch->num_reqs), dim3(kDraftThreads), 0, (hipStream_t)ex->stream, a);
    }
    return (int)hipGetLastError();
}
