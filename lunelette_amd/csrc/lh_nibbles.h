// Operands of the 16x16x32 FP16 matrix instructions that the 4-bit operators share:
// nibbles as exact FP16 integers, FP32 values as two FP16 planes.
#pragma once

#include "lh_device.h"
#include "lh_mfma.h"

namespace lh {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The eight codes of a word, minus 8: 0x6400 | c is the half 1024 + c, 0x6400 | 16 c
// is 1024 + 16 c, whose sixteenth less 72 is one fused instruction; all exact.
// low and high: the masks 0x000f000f and 0x00f000f0 in registers, where one
// instruction masks and sets the exponent.
struct NibbleMasks {
    uint32_t low, high;

    __device__ __forceinline__ NibbleMasks() : low(0x000f000fu), high(0x00f000f0u)
    {
        asm("" : "+v"(low), "+v"(high));
    }
};

__device__ __forceinline__ f16x8 codes_minus8(uint32_t w, const NibbleMasks& mask)
{
    const f16x2 low = {(_Float16)1032, (_Float16)1032}, high = {(_Float16)72, (_Float16)72};
    const f16x2 part = {(_Float16)0.0625f, (_Float16)0.0625f};
    const uint32_t x = w >> 8;
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t,
        __builtin_bit_cast(f16x2, (w & mask.low) | 0x64006400u) - low);
    r.y = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (w & mask.high) | 0x64006400u), part, -high));
    r.z = __builtin_bit_cast(uint32_t,
        __builtin_bit_cast(f16x2, (x & mask.low) | 0x64006400u) - low);
    r.w = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (x & mask.high) | 0x64006400u), part, -high));
    return __builtin_bit_cast(f16x8, r);
}

// a and b as two pairs of FP16 planes: hi nearest, lo nearest to the rest. Planes of small
// values are subnormal halves, which the matrix instructions take: they align a sum as if
// such an operand were 2^-14, so 32 products of subnormal and common numbers come out to
// 2^-33 (measured), where the largest of a row's planes stand at 2^14. The rest
// has to be that of the hi which goes into the product: left to itself the compiler
// forms one by a fused multiplication and conversion and the other from the rounded
// product, and the two differ by a whole step at a tie (1 of 2^13 values). The asm
// makes the packed bits one value; v - hi is exact.
__device__ __forceinline__ void planes2(float a, float b, uint32_t& hi, uint32_t& lo)
{
    hi = __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
    asm("" : "+v"(hi));
    float ra, rb;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(rb) : "v"(hi), "v"(b));
    lo = __builtin_bit_cast(uint32_t, (f16x2){(_Float16)ra, (_Float16)rb});
}

__device__ __forceinline__ void planes8(const float* v, f16x8& hi, f16x8& lo)
{
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t a, b;
        planes2(v[2 * i], v[2 * i + 1], a, b);
        h[i] = a;
        l[i] = b;
    }
    hi = __builtin_bit_cast(f16x8, h);
    lo = __builtin_bit_cast(f16x8, l);
}

// Eight values as planes of which the first lies away from 0 by up to a step and the
// second, of the other sign, has the rest: 22 bits where planes8 has 23. Times an
// infinite number the two are Inf and -Inf, so their sum is a NaN whatever the value's
// sign and bits are (planes8 gives an Inf where both have the same sign).
__device__ __forceinline__ void planes8_away(const float* v, f16x8& hi, f16x8& lo)
{
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = v[2 * i], b = v[2 * i + 1];
        // Toward 0, then the next magnitude.
        h[i] = __builtin_bit_cast(uint32_t,
            __builtin_bit_cast(u16x2, __builtin_amdgcn_cvt_pkrtz(a, b)) + (u16x2){1, 1});
        float ra, rb;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h[i]), "v"(a));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=v"(rb) : "v"(h[i]), "v"(b));
        l[i] = __builtin_bit_cast(uint32_t, (f16x2){(_Float16)ra, (_Float16)rb});
    }
    hi = __builtin_bit_cast(f16x8, h);
    lo = __builtin_bit_cast(f16x8, l);
}

}  // namespace lh
