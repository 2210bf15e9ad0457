// What the kernels of linear attention share: their arguments, a request's share of a batch, and the recurrent kernel.
//
//   S = exp(g_t) S + k_t v_t^T        o_t = scale S^T q_t
#pragma once

#include "../../include/warp34_linear.h"
#include "attn_lanes.h"

namespace w34 {

struct LinearArgs {
    const int32_t *query_start_loc, *state_in_slots, *has_initial_state, *state_out_slots, *state_tokens;
    const uint8_t* valid_req_mask;
    const uint16_t *q, *k, *v;
    const float* g;  // nullptr: no decay
    uint16_t* out;   // nullptr: none
    uint64_t state_base, slot_stride;
    int num_reqs, total_tokens, v_heads, v_dim, group;  // group: value heads of a key head
    int q_stride, k_stride, v_stride, out_stride, g_stride;
    float scale;
};

// States: an address that comes out of an integer has to say that it is global memory, or its loads and stores count with those of LDS.
typedef __attribute__((address_space(1))) float linear_float;
typedef __attribute__((address_space(1))) f4 linear_f4;

struct LinearRequest {
    int lo, n;     // its rows
    int kept;      // the state written is the one behind that many of them
    const linear_float* in;  // of the head, nullptr: zeros
    linear_float* out;       // of the head, nullptr: not written
};
__device__ __forceinline__ LinearRequest linear_request(const LinearArgs& a, int req, int head, int state_size) {
    LinearRequest r;
    r.lo = max(0, a.query_start_loc[req]);
    r.n = max(0, min(a.query_start_loc[req + 1], a.total_tokens) - r.lo);
    r.kept = a.state_tokens == nullptr ? r.n : min(max(a.state_tokens[req], 0), r.n);
    const int in = a.state_in_slots == nullptr || (a.has_initial_state != nullptr && a.has_initial_state[req] == 0) ? -1 : a.state_in_slots[req];
    const int out = a.state_out_slots == nullptr ? -1 : a.state_out_slots[req];
    linear_float* base = reinterpret_cast<linear_float*>((uintptr_t)a.state_base);
    const uint64_t stride = a.slot_stride / 4, mine = (uint64_t)head * state_size;
    r.in = in < 0 ? nullptr : base + (uint64_t)in * stride + mine;
    r.out = out < 0 ? nullptr : base + (uint64_t)out * stride + mine;
    return r;
}

// ---- the recurrent kernel --------------------------------------------------------------------------------------------------
// A wave keeps 32 columns of a head's state in registers, lane l columns 4 (l & 7) .. + 3 of rows DK / 8 (l >> 3) .. + DK / 8 - 1, so that a row is
// read in runs of 128 bytes and the state passes once through the chip however many tokens there are.  The waves of a workgroup have the head's
// other columns and the same q and k; nothing is exchanged between them.  All in 32 bits.
// Bound: HBM, the state read once and written once: 64 single tokens of 32 heads of 128 x 128, 270 MB, 53.4 us (5.05 TB/s, the rate of a large copy);
// 16 x 5 tokens 15.8 us, where the tokens' 5 x 64 multiply-adds a lane come to the same; one token 4.2 us, a launch and two round trips.
template <typename T, int DK, int DV>
__global__ __launch_bounds__(2 * DV) void linear_step_kernel(const LinearArgs a) {
    constexpr int R = DK / 8;
    const int req = (int)(blockIdx.x / (uint32_t)a.v_heads), head = (int)(blockIdx.x - (uint32_t)req * (uint32_t)a.v_heads);
    if (a.valid_req_mask != nullptr && a.valid_req_mask[req] == 0) return;
    const int lane = lane_id(), row0 = (lane >> 3) * R, col = ((int)threadIdx.x >> 6) * 32 + (lane & 7) * 4;
    const LinearRequest r = linear_request(a, req, head, DK * DV);
    const int kh = head / a.group, steps = a.out == nullptr ? r.kept : r.n;
    // a token's rows are asked for while the one before it is gone through
    uint4 kx[R / 8], qx[R / 8];
    uint2 vx = {0, 0};
    float gx = 0.f;
    const auto fetch = [&](int t) {
        const int64_t tok = r.lo + t;
#pragma unroll
        for (int i = 0; i < R / 8; ++i) {
            kx[i] = reinterpret_cast<const uint4*>(a.k + tok * a.k_stride + kh * DK + row0)[i];
            qx[i] = reinterpret_cast<const uint4*>(a.q + tok * a.q_stride + kh * DK + row0)[i];
        }
        vx = *reinterpret_cast<const uint2*>(a.v + tok * a.v_stride + head * DV + col);
        if (a.g != nullptr) gx = a.g[tok * a.g_stride + head];
    };
    if (steps > 0) fetch(0);
    f4 s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = f4{0.f, 0.f, 0.f, 0.f};
    if (r.in != nullptr) {
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = *reinterpret_cast<const linear_f4*>(r.in + (row0 + i) * DV + col);
    }
    if (r.kept == 0 && r.out != nullptr) {
#pragma unroll
        for (int i = 0; i < R; ++i) *reinterpret_cast<linear_f4*>(r.out + (row0 + i) * DV + col) = s[i];
    }
    for (int t = 0; t < steps; ++t) {
        const bool keeps = t + 1 == r.kept && r.out != nullptr;
        const int64_t tok = r.lo + t;
        uint32_t kw[R / 2], qw[R / 2];
#pragma unroll
        for (int i = 0; i < R / 8; ++i) {
            kw[4 * i] = kx[i].x, kw[4 * i + 1] = kx[i].y, kw[4 * i + 2] = kx[i].z, kw[4 * i + 3] = kx[i].w;
            qw[4 * i] = qx[i].x, qw[4 * i + 1] = qx[i].y, qw[4 * i + 2] = qx[i].z, qw[4 * i + 3] = qx[i].w;
        }
        const float fade = a.g == nullptr ? 1.f : expf(gx);
        const f4 v = {T::to_f32((uint16_t)vx.x), T::to_f32((uint16_t)(vx.x >> 16)), T::to_f32((uint16_t)vx.y), T::to_f32((uint16_t)(vx.y >> 16))};
        if (t + 1 < steps) fetch(t + 1);
        f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float ki = T::to_f32((uint16_t)(kw[i / 2] >> (i % 2 * 16))), qi = T::to_f32((uint16_t)(qw[i / 2] >> (i % 2 * 16)));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[i][c] = __builtin_fmaf(ki, v[c], fade * s[i][c]);
                o[c] = __builtin_fmaf(qi, s[i][c], o[c]);
            }
            if (keeps) *reinterpret_cast<linear_f4*>(r.out + (row0 + i) * DV + col) = s[i];
        }
        if (a.out == nullptr) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            o[c] += lane_xor<8>(o[c], lane);
            o[c] += lane_xor<16>(o[c], lane);
            o[c] += lane_xor<32>(o[c], lane);
            o[c] *= a.scale;
        }
        if (lane < 8) {
            const uint2 w = {(uint32_t)T::from_f32(o[0]) | (uint32_t)T::from_f32(o[1]) << 16, (uint32_t)T::from_f32(o[2]) | (uint32_t)T::from_f32(o[3]) << 16};
            *reinterpret_cast<uint2*>(a.out + tok * a.out_stride + head * DV + col) = w;
        }
    }
}

}  // namespace w34
