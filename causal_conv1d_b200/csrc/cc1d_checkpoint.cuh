// e4m3 with power-of-two group scales: the arithmetic of include/cc1d_checkpoint.h.
#pragma once

#include "cc1d_common.cuh"

namespace cc1d {

constexpr int kCodeGroup = 32;     // neighbours that share a scale

// Biased exponent of the least power of two s with most / s <= 448 = 1.75 * 2^8; 255 when most is
// infinite or NaN, at least 1 (2^-126, below which 2^-s would leave the normal numbers).
__device__ __forceinline__ uint32_t code_scale(float most) {
    const uint32_t b = __float_as_uint(most), e = b >> 23;
    if (e == 255u) return 255u;
    const int s = (int)e - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(s < 1 ? 1 : s);
}
__device__ __forceinline__ float scale_inverse(uint32_t s) { return __uint_as_float((s < 254u ? 254u - s : 0u) << 23); }
__device__ __forceinline__ float scale_value(uint32_t s) { return __uint_as_float(s == 255u ? 0x7fc00000u : s << 23); }

// A NaN has to come out of the maximum (max itself drops it)
__device__ __forceinline__ float max_abs(float m, float x) { return fabsf(x) <= m ? m : fabsf(x); }

// 4 values already divided by their scale
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// 4 neighbouring values of each of 8 lanes, a group -> this lane's codes, and the group's scale.  The bits of
// a float without their sign are ordered like the values, with infinities above all numbers and NaN above
// those, so the largest magnitude is an integer's (of 16-bit types two at a time).
template <typename T> __device__ __forceinline__ uint32_t codes_of_group(const uint2 &v, uint32_t &s) {
    uint32_t m = __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
    #pragma unroll
    for (int i = 1; i < 8; i <<= 1) m = __vmaxu2(m, __shfl_xor_sync(kFullMask, m, i));
    s = code_scale(unpack_pair<T>(max(m & 0xffffu, m >> 16)).x);
    const float inv = scale_inverse(s);
    const float2 a = unpack_pair<T>(v.x), b = unpack_pair<T>(v.y);
    return to_codes(a.x * inv, a.y * inv, b.x * inv, b.y * inv);
}
template <typename T> __device__ __forceinline__ uint32_t codes_of_group(const uint4 &v, uint32_t &s) {
    uint32_t m = max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
    #pragma unroll
    for (int i = 1; i < 8; i <<= 1) m = max(m, __shfl_xor_sync(kFullMask, m, i));
    s = code_scale(__uint_as_float(m));
    const float inv = scale_inverse(s);
    return to_codes(__uint_as_float(v.x) * inv, __uint_as_float(v.y) * inv, __uint_as_float(v.z) * inv, __uint_as_float(v.w) * inv);
}
// 2 codes (the low 16 bits) times their scale
__device__ __forceinline__ float2 from_codes(uint32_t codes, float scale) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    return make_float2(f.x * scale, f.y * scale);
}
// A rounded-up 65504 stays what fp16 holds (a NaN stays one)
template <typename T> __device__ __forceinline__ float2 fit(float2 v) { return v; }
template <> __device__ __forceinline__ float2 fit<__half>(float2 v) {
    return make_float2(fabsf(v.x) > 65504.f ? copysignf(65504.f, v.x) : v.x, fabsf(v.y) > 65504.f ? copysignf(65504.f, v.y) : v.y);
}
// 4 codes -> 4 packed 16-bit values
template <typename T> __device__ __forceinline__ uint2 expand4(uint32_t codes, float scale) {
    return make_uint2(pack_pair<T>(fit<T>(from_codes(codes, scale))), pack_pair<T>(fit<T>(from_codes(codes >> 16, scale))));
}
template <typename T> __device__ __forceinline__ uint4 expand8(uint2 codes, float scale) {
    const uint2 a = expand4<T>(codes.x, scale), b = expand4<T>(codes.y, scale);
    return make_uint4(a.x, a.y, b.x, b.y);
}

}  // namespace cc1d
