// What the attention kernels share beside the definitions of kv_common.h: vector types, divisions without a divide, the 256-point
// transform of a wave, the TQ4 table in LDS, 16-bit operand pairs, and reductions over the rows of an MFMA result.
#pragma once

#include "kv_common.h"

namespace w34 {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

// Bytes of a slab.  An address that comes out of an integer has to say that it is global memory: a flat load is counted with the LDS
// accesses too, and every wait for a look-up would wait for the rows in flight.
typedef __attribute__((address_space(1))) const uint8_t slab_byte;
__device__ __forceinline__ const slab_byte* slab_at(uint64_t address) { return reinterpret_cast<const slab_byte*>((uintptr_t)address); }
template <typename T>
__device__ __forceinline__ T load_as(const slab_byte* p) { return *reinterpret_cast<const __attribute__((address_space(1))) T*>(p); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1.0e30f;  // "minus infinity" that stays finite under subtraction
// The table holds fp16(kLutGain * centroid); the gain is divided out of the query (K side)
// and of the final normalisation (V side).  1.908032 minimises the worst fp16 rounding error
// of the eight centroid magnitudes (9.4e-5 relative instead of 3.7e-4), which is what limits
// the accuracy of the scores.
constexpr float kLutGain = 1.908032f;
constexpr float kLutInvGain = 1.0f / kLutGain;

// a / b for 0 <= a < 2^21 and 0 < b: the float quotient is within one of the exact result,
// one correction step makes it exact.  A runtime integer division costs ~40 dependent
// instructions on this hardware, and the prologue and the per-unit address arithmetic
// divide by block sizes and group sizes that only the descriptors know.
__device__ __forceinline__ int small_div(int a, int b) {  // a < 2^21
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    const int r = a - q * b;
    q += r >= b ? 1 : 0;
    q -= r < 0 ? 1 : 0;
    return q;
}
__device__ __forceinline__ int fast_div(int a, int b) { return a >= (1 << 21) ? a / b : small_div(a, b); }
// for div_block: floor(2^32 / block size)
__host__ inline uint32_t block_magic_for(int block_size) {
    return block_size <= 1 ? 0xFFFFFFFFu : (uint32_t)((1ull << 32) / (uint32_t)block_size);
}

// The 256-point WHT of finished rows and queries: 60 instructions a row (128 with an exchange, two sums and a select per value and lane stage).
// A prefill wave rotates 64 rows: 16 requests of 256 tokens on 512 keys 116.6 / 107.7 us, 2 of 250 on 1 000 46.9 / 45.3.
// One lane stage, H = 1, 2 or 8: lanes with bit H clear take v + v[lane ^ H], the others v[lane ^ H] - v.
// SELECT: the same by both results and a choice, twelve instructions more in all and no sign to keep.  For the two-column-tile form of 8-bit rows: with
// the signs it spills 30 to 50 more scalars, also where nothing is rotated.  us a call, signs / choice: Q8_0 5 requests x 4 tokens on 2 000 keys 17.3 / 16.1, 24 tokens
// on 240 keys 14.3 / 13.0, FP8 16.4 / 15.8, 13.5 / 12.7.  The other forms are as fast with the signs or faster (rotated FP8, 8 x 8 tokens on 240 keys 14.4 / 14.8).
template <int H, bool SELECT = false>
__device__ __forceinline__ void wht_stage(float (&v)[4], int lane) {
    const uint32_t flip = (lane & H) ? 0x80000000u : 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float o = lane_xor<H>(v[k], lane);
        if constexpr (SELECT) v[k] = (lane & H) ? o - v[k] : v[k] + o;
        else v[k] = o + __uint_as_float(__float_as_uint(v[k]) ^ flip);
    }
}
// H = 4: the sum in the groups of four lanes with the bit clear, the difference in the others.  (The compiler does not see that the statement
// reads across lanes: the waits stand in it.)
__device__ __forceinline__ void wht_stage4(float (&v)[4]) {
    float r[4];
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %1, %5, %5 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %2, %6, %6 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %3, %7, %7 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_sub_f32_dpp %0, %4, %4 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_sub_f32_dpp %1, %5, %5 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_sub_f32_dpp %2, %6, %6 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_sub_f32_dpp %3, %7, %7 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "s_nop 1"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]));
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = r[k];
}
// H = 16 or 32, two values at a time: exchanged halves put both sides of a's pairs (and of b's) into the same lane, the sum and the difference
// are the results of both sides, and a second exchange brings them back.
template <int H>
__device__ __forceinline__ void wht_stage_pair(float& a, float& b) {
    const auto swap = [](float x, float y) {
        if constexpr (H == 16) return __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        else return __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    };
    const auto r = swap(a, b);
    const float sum = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const float diff = __uint_as_float(r[0]) - __uint_as_float(r[1]);
    const auto o = swap(sum, diff);
    a = __uint_as_float(o[0]);
    b = __uint_as_float(o[1]);
}

// 256-point WHT over one wave: element e = 4*lane + k, scaled by 1/16.
template <bool SELECT = false>
__device__ __forceinline__ void wht256_wave(float (&v)[4], int lane) {
    {
        const float a0 = v[0] + v[1], a1 = v[0] - v[1], a2 = v[2] + v[3], a3 = v[2] - v[3];
        v[0] = a0 + a2;
        v[1] = a1 + a3;
        v[2] = a0 - a2;
        v[3] = a1 - a3;
    }
    wht_stage<1, SELECT>(v, lane);
    wht_stage<2, SELECT>(v, lane);
    wht_stage4(v);
    wht_stage<8, SELECT>(v, lane);
    wht_stage_pair<16>(v[0], v[1]);
    wht_stage_pair<16>(v[2], v[3]);
    wht_stage_pair<32>(v[0], v[1]);
    wht_stage_pair<32>(v[2], v[3]);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= 0.0625f;
}

// Entry bits of a code: fp16(kLutGain * centroid), by two byte permutes over immediates (no constant-memory load on the critical path; a chain of selects
// is sixty instructions with branches).  Magnitude k is that of centroids 8 + k and 7 - k.
__host__ __device__ constexpr uint32_t centroid_bits_of(int code) { return __builtin_bit_cast(uint16_t, (_Float16)(kLutGain * kCentroids[code])); }
__host__ __device__ constexpr uint32_t magnitude_bytes(int first, int shift) {  // byte `shift / 8` of four magnitudes
    uint32_t r = 0;
    for (int k = 0; k < 4; ++k) r |= (centroid_bits_of(8 + first + k) >> shift & 0xFFu) << (8 * k);
    return r;
}
__device__ __forceinline__ uint32_t centroid_bits(uint32_t code) {
    constexpr uint32_t lo0 = magnitude_bytes(0, 0), lo4 = magnitude_bytes(4, 0), hi0 = magnitude_bytes(0, 8), hi4 = magnitude_bytes(4, 8);
    const bool negative = (code & 8u) == 0u;
    const uint32_t k = (negative ? ~code : code) & 7u;
    return __builtin_amdgcn_perm(lo4, lo0, k | 0x0c0c0c00u) | __builtin_amdgcn_perm(hi4, hi0, k << 8 | 0x0c0c000cu) | (negative ? 0x8000u : 0u);
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    f2 f = {a, b};
    h2 h = __builtin_convertvector(f, h2);
    return __builtin_bit_cast(uint32_t, h);
}
// Two fp16 operands for one fp32 weight pair: hi = fp16(w), lo = fp16(w - hi).  A value scale
// that is folded into the probabilities (w = p * d) reaches every element of a 128-wide scale
// block through ONE number; rounded to fp16 once, its error is the same for the whole block,
// and the inverse rotation gathers such a block-wide error into a single output channel
// (channel c ^ 128 of a channel c with large values).  With the low-order operand the weight
// carries 22 bits and that error disappears; the price is a second MFMA per value tile.
__device__ __forceinline__ void split_h2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const h2 h = __builtin_convertvector(f2{a, b}, h2);
    hi = __builtin_bit_cast(uint32_t, h);
    // lo = fp16(a - hi.x) | fp16(b - hi.y) << 16: one mixed-precision FMA per half (x * 1 - h with
    // h read as fp16), the same value as widening, subtracting (exact) and rounding
    uint32_t l;
    asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(l) : "v"(a), "v"(hi));
    asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(b), "v"(hi));
    lo = l;
}
// An MFMA may read a register two wait states after a vector instruction has written it.  The compiler
// keeps that distance for its own instructions but does not see through an assembly statement, so
// the low-order operands pass through settle() on their way to the MFMAs.
__device__ __forceinline__ void settle(u2v (&a)[8]) {
    asm("s_nop 1" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7]));
}
__device__ __forceinline__ void settle(u4 (&a)[8]) {
    asm("s_nop 1" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7]));
}
// The same for the weights of TQ4 rows, where issue and not registers is short: v_fma_mix_f32 and v_cvt_pk_f16_f32 issue every 4 cycles, v_fma_mixlo_f16 /
// mixhi, which do both, every 8.  (Written as fma, the compiler widens the halves with instructions of their own.)
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_h2(a, b);
    float r0, r1;
    asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(r0) : "v"(a), "v"(hi));
    asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r1) : "v"(b), "v"(hi));
    lo = pack_h2(r0, r1);
}
// a * (fp16 half of w) as one mixed-precision FMA that reads the half in place (v_fma_mix_f32 with
// a zero addend; written as an fma so that the compiler forms it and places the wait states that
// separate it from the instruction that produced a).  A product of -0 comes out as +0.
__device__ __forceinline__ float mul_by_half_lo(float a, uint32_t w) {
    return __builtin_fmaf(a, (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xFFFFu)), 0.0f);
}
__device__ __forceinline__ float mul_by_half_hi(float a, uint32_t w) {
    return __builtin_fmaf(a, (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)), 0.0f);
}
// the larger ones of two pairs of 16-bit numbers
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
// maximum of three finite values in one instruction (fmaxf would first quiet each operand); the
// operands must come from ordinary vector instructions: the compiler places no wait states in
// front of an assembly statement that reads the result of an MFMA
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float half_lo_to_f32(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xFFFFu));
}
__device__ __forceinline__ float half_hi_to_f32(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}
// max / sum over the four 16-lane rows of a wave, result in every lane (pure VALU on gfx950)
__device__ __forceinline__ float max_over_rows(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_rows(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Table lookup: the dequantisation table sits at LDS address 0 (it is the start of the dynamic
// LDS block and the kernel has no static LDS), so the v_perm_b32 result IS the address.
typedef __attribute__((address_space(3))) const uint32_t lds_cu32;
typedef __attribute__((address_space(3))) const h8 lds_ch8;
typedef __attribute__((address_space(1))) const u4 global_cu4;
__device__ __forceinline__ uint32_t lut_read(uint32_t code_word, uint32_t lut_lane, uint32_t sel) {
    const uint32_t addr = __builtin_amdgcn_perm(code_word, lut_lane, sel);
    return *reinterpret_cast<lds_cu32*>((uintptr_t)addr);
}

// The pair table, by 512 threads: entry e = (gain*centroid[e & 15], gain*centroid[e >> 4]) as packed fp16, 64 copies of 4 bytes.
// Thread t writes the 16-byte slots t + 512 i (conflict-free), i.e. entries (t >> 4) + 32 i:
// their low code (t >> 4) & 15 is the thread's own, their high code (t >> 8) + 2 i is the
// same in the whole wave, one of two immediates.
__device__ __forceinline__ void build_pair_table(uint8_t* smem, int tid, int wave) {
    const uint32_t lo = centroid_bits((uint32_t)tid >> 4 & 15u);
    const bool odd = (wave >> 2) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t v = lo | (odd ? centroid_bits_of(2 * i + 1) << 16 : centroid_bits_of(2 * i) << 16);
        *reinterpret_cast<u4*>(smem + (tid + 512 * i) * 16) = u4{v, v, v, v};
    }
}

}  // namespace w34
