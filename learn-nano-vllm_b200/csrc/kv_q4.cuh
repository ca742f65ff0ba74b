// Records of the 4-bit KV cache, shared by the kernels that write and read them.
//
// One record of 80 bytes stands for the 128 values of one (token, kv head):
//   bytes  0-63  codes, 16 bytes for each of the four groups of 32 head dimensions;
//   bytes 64-79  one 32-bit word per group: scale s (low half) and minimum m (high half)
//                in the model's 16-bit type.
// A value is s * code + m.  A 32-bit word of codes holds eight consecutive dimensions, the
// even ones in its low half and the odd ones in its high half (nibble i of a half is dimension
// 2 i, 2 i + 1): masking a word, shifted by 4 i, with 0x000f000f leaves the codes of two
// neighbouring dimensions in the two halves of a register, where a 16-bit matrix operand
// wants them.  Records of consecutive tokens of one head are contiguous
// ([num_blocks][num_kv_heads][block_size][80]), so that a tile of a head's tokens is one bulk
// copy; the 80-byte stride puts eight records' 16-byte rows into eight different bank groups.
#pragma once

#include <cfloat>

#include "common.cuh"

namespace b200 {
namespace q4 {

constexpr int kD = 128;
constexpr int kGroups = 4;          // groups of 32 dimensions
constexpr int kRecord = 80;         // bytes
constexpr int kParams = 64;         // byte offset of the scales and minima
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100: smaller scales are stored as 0

template <bool BF16>
__device__ __forceinline__ float lo_f(uint32_t w) {
    if constexpr (BF16) return __uint_as_float(w << 16);
    else return __half2float(__ushort_as_half(uint16_t(w)));
}
template <bool BF16>
__device__ __forceinline__ float hi_f(uint32_t w) {
    if constexpr (BF16) return __uint_as_float(w & 0xffff0000u);
    else return __half2float(__ushort_as_half(uint16_t(w >> 16)));
}

// Minimum / maximum of packed pairs; a NaN in either operand gives NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Quantises eight consecutive dimensions per lane (x: four packed pairs); the four lanes of an
// aligned quad hold one group.  Returns the lane's word of codes and the group's parameter word.
//
//   m = min x, s = (max x - m) / 15 rounded to the model's type (0 below 2^-100),
//   code = min(15, rint((x - m) / s)), ties to even; a group whose max - min is not finite
//   gets s = m = NaN and codes 0.
// The codes are those of the correctly rounded quotient (x - m) / s, without a division (after
// Markstein 1990): with y ~ 1/s to 2^-23 and q0 the rounded product (x - m) y, within two units of
// the quotient, the residual (x - m) - q0 s is exact in one fused operation, and q0 + residual * y is
// the quotient to 2^-22 units before its rounding.  No quotient of a 24-bit by an 11-bit number is
// that near the middle between two floats, so the rounding is the quotient's own.  The same
// steps give the span's fifteenth.  (s is 0 or at least 2^-100, so nothing under- or overflows.)
template <bool BF16>
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&x)[4], uint32_t& params) {
    const uint32_t mn = min2_nan<BF16>(min2_nan<BF16>(x[0], x[1]), min2_nan<BF16>(x[2], x[3]));
    const uint32_t mx = max2_nan<BF16>(max2_nan<BF16>(x[0], x[1]), max2_nan<BF16>(x[2], x[3])) ^ 0x80008000u;
    // {min, -max} of the lane, then of the quad: one minimum serves both.
    uint32_t r = min2_nan<BF16>(__byte_perm(mn, mx, 0x5410), __byte_perm(mn, mx, 0x7632));
    r = min2_nan<BF16>(r, __shfl_xor_sync(0xffffffffu, r, 1));
    r = min2_nan<BF16>(r, __shfl_xor_sync(0xffffffffu, r, 2));
    const float lo = lo_f<BF16>(r), span = -hi_f<BF16>(r) - lo;
    const bool finite = span <= FLT_MAX;
    constexpr float kFifteenth = 1.f / 15.f;
    const float f0 = span * kFifteenth;
    uint32_t sbits = to_bits16<BF16>(fmaf(fmaf(-f0, 15.f, span), kFifteenth, f0));
    float s = lo_f<BF16>(sbits), inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    if (s < kMinScale) {
        s = 0.f;
        inv = 0.f;
        sbits = 0;
    }
    params = finite ? (sbits | (r << 16)) : 0x7fff7fffu;  // the all-ones pattern is NaN in both types
    uint32_t even = 0, odd = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const float2 d = fsub2(make_float2(lo_f<BF16>(x[i]), hi_f<BF16>(x[i])), make_float2(lo, lo));
        const float2 q0 = fmul2(d, make_float2(inv, inv));
        const float2 e = ffma2(q0, make_float2(-s, -s), d);
        float2 q = ffma2(e, make_float2(inv, inv), q0);
        if constexpr (!BF16) {  // fp16 scales may be subnormal, off by a third; a bf16 one leaves q below 15.1
            q.x = fminf(q.x, 15.f);
            q.y = fminf(q.y, 15.f);
        }
        // rint by the magic constant 1.5 * 2^23: the code lands in the low mantissa bits.  Shifting
        // moves the constant's own bits (22 and up) past bit 15, which is all that is kept.
        const float2 t = fadd2(q, make_float2(12582912.f, 12582912.f));
        even = even * 16 + __float_as_uint(t.x);
        odd = odd * 16 + __float_as_uint(t.y);
    }
    const uint32_t word = __byte_perm(even, odd, 0x5410);
    return finite ? word : 0u;
}

template <bool BF16>
__device__ __forceinline__ uint32_t fma2_16(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// The eight values s n + m of a word of codes in the model's type (four packed pairs), each rounded once.
// A code in the low mantissa bits of 128 (bf16) or 1024 (fp16) is that number plus n, exactly; taking it
// off again in 16 bits is exact too.  fp16 has room for the next nibble, 16 n, as it stands.  (Gather of four
// sequences of 26k tokens: 109.6 us against 111.9 with the codes taken to fp32.)
template <bool BF16>
__device__ __forceinline__ uint4 dequantise8(uint32_t word, uint32_t params) {
    const uint32_t s = __byte_perm(params, 0, 0x1010), m = __byte_perm(params, 0, 0x3232);
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t n;
        if constexpr (BF16)
            n = fma2_16<BF16>(((word >> (4 * i)) & 0x000f000fu) | 0x43004300u, 0x3f803f80u, 0xc300c300u);
        else if (i & 1)
            n = fma2_16<BF16>(((word >> (4 * i - 4)) & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd400d400u);
        else
            n = fma2_16<BF16>(((word >> (4 * i)) & 0x000f000fu) | 0x64006400u, 0x3c003c00u, 0xe400e400u);
        y[i] = fma2_16<BF16>(n, s, m);
    }
    return make_uint4(y[0], y[1], y[2], y[3]);
}

}  // namespace q4
}  // namespace b200
