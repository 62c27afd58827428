// The 4-bit key/value cache: how its pages lie in memory, and the arithmetic of a group.
//
// A page holds kPage positions of one key/value head of D = 32 NG lanes, as keys or as values, in 40 D bytes.  The lanes lie in
// groups of 32; lane x of a group is d c + m with c in 0..15 and the group's two float16 numbers:
//   lo, hi = least and greatest of the group, each within +-65504 (float16's range: what lies beyond is taken as its end);
//   d = half((hi - lo) (1 / 15)), m = half(lo), c = clamp(rint((x - m) (1 / d)), 0, 15), 1 / 15 and 1 / d rounded to 32 bits, as is each operation; d of 0: c = 0.
// A group that holds a NaN is NaN as a whole (m is).
//
//   key page:    64 rows of D / 2 bytes; then 64 rows of NG pairs (d, m).
//                A row is 32-bit words [4][NG]: word (c, g) holds lanes 32 g + 8 c + i at bits 4 i, i = 0..7.
//   value page:  words [8][8][4][NG]; then 64 rows of NG pairs (d, m).
//                Word (b, r, p, g) holds position 8 b + 2 p in its lower half and 8 b + 2 p + 1 in its upper one, each
//                lanes 32 g + 4 r + i at bits 4 i, i = 0..3.
//
// So that attention_q4.cu reads whole tensor-core operands: in a key row the four lanes of a quad find their words of all groups
// side by side (16 bytes for D = 128), and two codes 16 bits apart are neighbours along the product's inner dimension (lanes of a
// key; positions of a value lane), which one mask and one OR turn into two float16 numbers 1 024 + c.
#pragma once

#include <cuda_fp16.h>

constexpr int kGroup = 32;                 // lanes that share d and m
constexpr float kHalfMax = 65504.0f;

__host__ __device__ __forceinline__ size_t q4_page_bytes(int D) { return (size_t)kPage * D / 8 * 5; }
__host__ __device__ __forceinline__ int q4_scales_at(int D) { return kPage / 2 * D; }    // bytes of a page's codes

// The 32-bit word, and the bit in it, where a key's or a value's code lies.
__device__ __forceinline__ int q4_key_word(int tok, int c, int g, int NG) { return tok * 4 * NG + c * NG + g; }
__device__ __forceinline__ int q4_value_word(int tok, int r, int g, int NG) {
    return (((tok >> 3) * 8 + r) * 4 + ((tok & 7) >> 1)) * NG + g;
}

// Of a group's least and greatest number (both already within float16's range): d and m, and what codes are made with.
struct Q4Scale {
    __half d, m;
    float m32, inv;      // m and 1 / d (0 where d is 0) as 32-bit numbers
};
__device__ __forceinline__ Q4Scale q4_scale(float lo, float hi) {
    Q4Scale s;
    s.d = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    s.m = __float2half_rn(lo);
    const float d = __half2float(s.d);
    s.m32 = __half2float(s.m);
    s.inv = d > 0.0f ? __frcp_rn(d) : 0.0f;
    return s;
}
// (Each operation rounded by itself: a fused one would give other codes next to a border.)
__device__ __forceinline__ uint32_t q4_code(float x, const Q4Scale& s) {
    const float t = rintf(__fmul_rn(__fsub_rn(x, s.m32), s.inv));
    return (uint32_t)fminf(fmaxf(t, 0.0f), 15.0f);      // (a NaN's code is 0)
}
// Four neighbours' codes, the first in the lowest four bits (of 16; the others are not said).  Clamped before it is rounded, which
// gives the same; 1.5 x 2^23 is added, so that the sum's last bits are the rounded number.
__device__ __forceinline__ uint32_t q4_codes(float x0, float x1, float x2, float x3, const Q4Scale& s) {
    auto one = [&](float x) {
        return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(__fsub_rn(x, s.m32), s.inv), 0.0f), 15.0f), 12582912.0f));
    };
    return ((one(x3) * 16 + one(x2)) * 16 + one(x1)) * 16 + one(x0);
}
// x within float16's range; a NaN stays one (fminf and fmaxf would drop it).
__device__ __forceinline__ float q4_in_range(float x) { return fabsf(x) > kHalfMax ? copysignf(kHalfMax, x) : x; }

__device__ __forceinline__ float q4_number(uint32_t code, float2 dm) { return fmaf(dm.x, (float)code, dm.y); }
