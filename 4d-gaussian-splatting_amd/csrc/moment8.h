// Moments of an optimizer in 8 bits (device helpers of adamw.hip).
//
// Blocks of 256 consecutive elements share one exponent byte E, the biased float32 exponent of the block's largest
// magnitude.  A value's code counts the steps of its "key" (float32 bit pattern >> 20: exponent and three mantissa
// bits) above the block's base:
//   second moment: code 1..255 <-> key base + code, base = max(0, 8 (E + 1) - 255)         31.75 powers of two
//   first moment:  sign and code 1..127,            base = max(0, 8 (E + 1) - 127)         15.75 powers of two
// Code 0 is zero.  Because the grid is a cut of the float32 pattern, its points do not move when a block's exponent
// does: a value that is stored, read and stored again stays what it is.  The largest code stands for 2^(E + 1 - 127),
// so a largest value that rounds up has a place: up to E = 253.  With E = 254 that place is infinity's, and a value above
// 1.875 times 2^127 may be read back as such; squares of gradients come there from 10^19 on.
//
// The cut is stochastic (a 16-bit random number is added just below the last kept bit).  With beta2 = 0.999 a step
// moves v by a thousandth of g^2 - v while the grid's points are an eighth to a sixteenth of v apart: a cut to the
// nearest would leave v where it is for good, and on average the cut that is drawn keeps the change.  16 random bits and
// not 8, because that change is about a hundredth of the grid's spacing.  The spread that the draws leave in v is about
// 0.2 v (each step adds 0.09 v * 0.001 |g^2 - v| to the variance, and 1 / (1 - beta2^2) = 500 steps are remembered),
// 0.1 of its root.  v has 3 mantissa bits and 5 of exponent, because its root's range beside eps (2^16 in a block)
// matters more than the third of that spread that a fourth mantissa bit would take away.
// A second moment that is not zero never gets code 0: its root divides.  What a first moment loses below its smallest
// code is 2^-16 of the block's largest.  A block with a value that is not finite gets E = 255 and stands for NaN.
#pragma once
#include "fdgs_common.h"

#define M8_BLOCK 256

// 32 bits from an element's index and a tensor's key of the step.  Three odd multipliers from the fractions of the
// golden ratio and of the roots of 2 and 3, with shifts in between that bring the high bits back down.
// x0: (index + key) * M8_C1 of the element (the next element's is M8_C1 more)
#define M8_C1 0x9E3779B9u
__device__ __forceinline__ uint32_t m8_hash(uint32_t x0) {
    uint32_t x = x0;
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
// the part of the hash that is the same for 2^32 elements
__device__ __forceinline__ uint32_t m8_key(uint32_t key, long long index) {
    return key + (uint32_t)((unsigned long long)index >> 32) * 0x6A09E667u;
}

// The two fields of the hash; 16 times such a field is what is added below the kept bits.
__device__ __forceinline__ uint32_t m8_noise_m(uint32_t h) { return h >> 16; }
__device__ __forceinline__ uint32_t m8_noise_v(uint32_t h) { return h & 0xFFFFu; }

template <bool SIGNED>
__device__ __forceinline__ int m8_base(int e) {
    const int b = 8 * (e + 1) - (SIGNED ? 127 : 255);
    return b > 0 ? b : 0;
}

// The float32 pattern that a code stands for, in a block whose exponent is not 255 (the caller's NaN).
template <bool SIGNED>
__device__ __forceinline__ uint32_t m8_decode(uint32_t code, int base) {
    const uint32_t size = SIGNED ? (code & 127u) : code;
    const uint32_t bits = size ? (size + (uint32_t)base) << 20 : 0u;
    return SIGNED ? bits | ((code & 128u) << 24) : bits;
}

// The code of a magnitude's pattern, without a sign; the caller stores 0 in a block whose exponent is 255.
template <bool SIGNED>
__device__ __forceinline__ uint32_t m8_encode(uint32_t bits, uint32_t noise, int base) {
    // the subtraction saturates: what lies below the base gets code 0
    const uint32_t code = __builtin_elementwise_sub_sat(bits + (noise << 4), (uint32_t)base << 20) >> 20;
    if (SIGNED) return code;
    const uint32_t least = bits < 1u ? bits : 1u;
    return code > least ? code : least;
}
// Bit 7 of each byte: the signs of four values.
__device__ __forceinline__ uint32_t m8_signs(const float* x) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0C0C0703u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07030C0Cu);
    return (lo | hi) & 0x80808080u;
}

typedef unsigned short m8_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t m8_max2(uint32_t v, uint32_t w) {
    const m8_u16x2 a = __builtin_bit_cast(m8_u16x2, v), b = __builtin_bit_cast(m8_u16x2, w);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
}
// Largest of two 16-bit fields over the wave, the exponents of both moments in one reduction: neighbours, quads, rows of
// 16 (a lane reads another of its row without going through LDS), then rows into the rows above; the last lane has it.
__device__ __forceinline__ uint32_t m8_wave_max2(uint32_t v) {
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));    // quad: 1 0 3 2
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));    // quad: 2 3 0 1
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));   // mirrored half rows
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));   // mirrored rows
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, true));   // rows 1 and 3: from 0 and 2
    v = m8_max2(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, true));   // rows 2 and 3: from row 1
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
