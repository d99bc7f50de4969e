// The block-scaled 8-bit KV cache: codes int8 [max_seq, hkv, hd], one exponent byte e for each
// block of `block` consecutive rows and KV head ([ceil(max_seq / block), hkv]); a code stands for
// code * 2^(e - 127), e in 1..254; e = 255 makes the block NaN (it was given a value that is not
// finite).
//
// Why a power of two: an appended row can only raise its block's exponent, and each doubling
// then rounds the block's earlier codes once more, by half a new step at most. A free scale would
// creep upwards a little with every new largest value and round them each time. It also keeps
// every value exact in f16, so that the matrix-core kernels take the codes as they are and the
// scales as exponents.
#pragma once

#include <hip/hip_runtime.h>

#include "eb_common.h"
#include "eb_internal.h"

namespace eb {

constexpr unsigned kNanExponent = 255;

// The exponent byte of a block whose largest magnitude has the f32 bits a (sign cleared): the
// least with |x| <= 127 * 2^(e - 127), 127 * 2^E being 1.984375 * 2^(E + 6).
__device__ __forceinline__ unsigned i8_exponent(unsigned a) {
    if (a >= 0x7F800000u) return kNanExponent;
    const int e = (int)(a >> 23) - 6 + ((a & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
    return (unsigned)(e < 1 ? 1 : e);
}

// x as a code of exponent byte e (0 in a NaN block), in the low 8 bits. Exact scaling, then the
// nearest whole number, ties to even; |x| <= 127 * 2^(e - 127), so it fits.
__device__ __forceinline__ unsigned i8_code(float x, unsigned e) {
    if (e == kNanExponent) return 0u;
    return (unsigned)(int)__builtin_rintf(ldexpf(x, 127 - (int)e)) & 0xFFu;
}

// Byte i of w as a signed number.
__device__ __forceinline__ float i8_f32(unsigned w, int i) {
    return (float)((int)(w << (24 - 8 * i)) >> 24);
}

// Four codes of exponent old_e as codes of exponent e > old_e.
__device__ __forceinline__ unsigned i8_recode(unsigned w, unsigned old_e, unsigned e) {
    unsigned r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= ((unsigned)(int)__builtin_rintf(ldexpf(i8_f32(w, i), (int)old_e - (int)e)) & 0xFFu) << (8 * i);
    return r;
}

// The exponent byte of a block that holds rows of exponent old_e and gets new rows of exponent e.
__device__ __forceinline__ unsigned i8_join(unsigned old_e, unsigned e) {
    return old_e > e ? old_e : e;  // (255 is the largest: NaN stays)
}

// The factor of an exponent byte, as 2^(e - 127 + shift).
__device__ __forceinline__ float i8_scale(unsigned e, int shift) {
    return e == kNanExponent ? __builtin_nanf("") : ldexpf(1.0f, (int)e - 127 + shift);
}

}  // namespace eb
