// Running sums over the lanes of a wave in 64 bits, without LDS.
#pragma once

#include <hip/hip_runtime.h>

namespace w34 {

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

}  // namespace w34
