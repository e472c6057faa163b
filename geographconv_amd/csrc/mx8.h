// The 8-bit checkpoint format, shared by the kernels that write it and the ones that read it.
// 32 consecutive values of a row share one power-of-two scale 2^s, stored as the byte s + 127; a value is the e4m3 code of x / 2^s (4
// significant bits, round to nearest even).  s is the smallest exponent, -126 at least, with max|x| <= 448 * 2^s (448 = the largest e4m3
// value): no value saturates, so every rounding is off by at most half a step, and the division is exact.  At the largest scale, 2^120, the
// code 256 would stand for 2^128, which is no fp32 number: values from 248 * 2^120 on take the code 240 below it (off by 2^-4 of themselves
// at most, like any other).  A block that holds an infinity or a NaN has the byte 255 and stands for NaN throughout.
#pragma once
#include "common.h"

namespace geogcn {

constexpr int kMxBlock = 32;

__device__ __forceinline__ uint32_t mx8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }      // (as integers NaN > inf > finite)

// scale byte of a block from its largest |x| (bits)
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
    return (uint32_t)(b < 1 ? 1 : b);
}
// 2^-s / 2^s; a NaN block's codes are 0
__device__ __forceinline__ float mx8_inv_scale(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float mx8_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23); }

__device__ __forceinline__ uint32_t mx8_encode4(float x0, float x1, float x2, float x3, float inv, bool finite) {
    // (0 * inf of a NaN block would be NaN: the codes of such a block are written as 0)
    const float top = inv == 0x1p-120f ? 240.f : 448.f;
    const auto code = [&](float x) { return finite ? __builtin_amdgcn_fmed3f(x * inv, -top, top) : 0.f; };
    const float y0 = code(x0), y1 = code(x1), y2 = code(x2), y3 = code(x3);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, w, true);
    return (uint32_t)w;
}
__device__ __forceinline__ float4 mx8_decode4(uint32_t w, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return make_float4(lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale);
}

// ---- bf16 <-> fp32 ------------------------------------------------------------------------------------------------------------------------
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {          // round to nearest even, two at a time
    const mx_f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, mx_bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// four consecutive values x -> their P bf16 terms (P = 3: x = x1 + x2 + x3 exactly, the residuals are exact in fp32; P = 2: to 2^-16 of x; P = 1:
// rounded)
template <int P>
__device__ __forceinline__ void bf16_terms4(const float4& x, uint2 (&t)[P]) {
    t[0] = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    if constexpr (P >= 2) {
        const float r0 = x.x - bf16_lo(t[0].x), r1 = x.y - bf16_hi(t[0].x), r2 = x.z - bf16_lo(t[0].y), r3 = x.w - bf16_hi(t[0].y);
        t[1] = make_uint2(pack_bf16(r0, r1), pack_bf16(r2, r3));
        if constexpr (P == 3) t[2] = make_uint2(pack_bf16(r0 - bf16_lo(t[1].x), r1 - bf16_hi(t[1].x)), pack_bf16(r2 - bf16_lo(t[1].y), r3 - bf16_hi(t[1].y)));
    }
}

// four consecutive values of row r from column c (c % 4 == 0, c < roundup4(F) <= ld) of a matrix of one of the three storage types; columns
// from F on read as zero whatever the pad holds
struct MatIn { int type; const void* p; int64_t ld; const uint8_t* scale; };
template <int TYPE>
__device__ __forceinline__ float4 mat_load4(const MatIn& m, int64_t r, int c) {
    if constexpr (TYPE == GEOGCN_T_F32) {
        return *reinterpret_cast<const float4*>(static_cast<const float*>(m.p) + r * m.ld + c);
    } else if constexpr (TYPE == GEOGCN_T_BF16) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(m.p) + r * m.ld + c);
        return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(m.p) + r * m.ld + c);
        return mx8_decode4(w, mx8_scale(m.scale[r * (m.ld / kMxBlock) + c / kMxBlock]));
    }
}
__device__ __forceinline__ float4 mask4(float4 v, int c, int F) {
    if (c + 3 >= F) {
        if (c >= F) v.x = 0.f;
        if (c + 1 >= F) v.y = 0.f;
        if (c + 2 >= F) v.z = 0.f;
        v.w = 0.f;
    }
    return v;
}

}  // namespace geogcn
