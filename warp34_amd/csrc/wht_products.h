// The 256-point transform of a row as a product of 16 x 16 matrices: with X[r][c] = x[16 r + c] and H[r][c] = (-1)^popcount(r & c), 16 times the
// transformed row is Y = H X H.  Two 16x16x32 MFMAs do it:
//   Z = X H      A = X (lane (n, b) holds X[n][4 b .. 4 b + 3]), B = H; lane (n, b) gets Z[4 b + i][n]
//   Y^T = Z^T H  those registers are the A operand Z^T as they stand; lane (n, b) gets Y[n][4 b + i]
// Operands have two fp16 parts in the halves of the product (22 bits), so the result is as good as the 60 additions a row in 32 bits that
// the MFMAs stand for.
#pragma once

#include "attn_lanes.h"

namespace w34 {

__device__ __forceinline__ h8 two_parts(const float (&x)[4]) {
    u4 r;
    uint32_t hi, lo;
    split_weights(x[0], x[1], hi, lo);
    r[0] = hi, r[2] = lo;
    split_weights(x[2], x[3], hi, lo);
    r[1] = hi, r[3] = lo;
    return __builtin_bit_cast(h8, r);
}
// (-1)^popcount((4 b + i) & n) for i = 0 .. 3 as fp16, twice
__device__ __forceinline__ h8 hadamard_column(int n, int b) {
    const uint32_t of_b = (uint32_t)(b & (n >> 2)), odd = (of_b ^ of_b >> 1) & 1u;
    const uint32_t lo = 0x3C003C00u ^ odd * 0x80008000u ^ ((uint32_t)n & 1u) << 31;  // i = 0, 1
    const uint32_t hi = lo ^ ((uint32_t)n >> 1 & 1u) * 0x80008000u;                  // i = 2, 3
    return __builtin_bit_cast(h8, u4{lo, hi, lo, hi});
}

}  // namespace w34
