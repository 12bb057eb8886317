// e4m3 with power-of-two group scales: the arithmetic of include/cc1d_checkpoint.h.
#pragma once

#include "cc1d_common.cuh"

namespace cc1d {

constexpr int kCodeGroup = 32;     // neighbours that share a scale

// Biased exponent of the least power of two s with most / s <= 448 = 1.75 * 2^8; 255 when most is
// infinite or NaN, at least 1 (2^-126, below which 2^-s would leave the normal numbers).
__device__ __forceinline__ uint32_t code_scale(float most) {
    const uint32_t b = __float_as_uint(most);       // a mantissa above 1.75's carries into the exponent
    return b >= 0x7f800000u ? 255u : (uint32_t)max((int)((b + 0x1fffffu) >> 23) - 8, 1);
}
__device__ __forceinline__ float scale_inverse(uint32_t s) { return __uint_as_float((uint32_t)max(254 - (int)s, 0) << 23); }
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
// Largest magnitudes.  The bits of a float without their sign are ordered like the values, with infinities above
// all numbers and NaN above those, so they are integers' maxima (of 16-bit types two at a time).
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t most2(const uint4 &v) { return __vmaxu2(most2(v.x, v.y), most2(v.z, v.w)); }
template <typename T> __device__ __forceinline__ float most_of(uint32_t m) { return unpack_pair<T>(max(m & 0xffffu, m >> 16)).x; }

template <typename T> __device__ __forceinline__ uint32_t codes_by(const uint2 &v, float inv) {
    const float2 f = make_float2(inv, inv), a = mul2(unpack_pair<T>(v.x), f), b = mul2(unpack_pair<T>(v.y), f);
    return to_codes(a.x, a.y, b.x, b.y);
}
template <typename T> __device__ __forceinline__ uint32_t codes_by(const uint4 &v, float inv) {
    return to_codes(__uint_as_float(v.x) * inv, __uint_as_float(v.y) * inv, __uint_as_float(v.z) * inv, __uint_as_float(v.w) * inv);
}
// 4 neighbouring values of each of 8 lanes are a group: codes and scales of two groups (two tokens), whose
// maxima go through the shuffles in one register where they are 16-bit
template <typename T> __device__ __forceinline__ void codes_of_groups(const uint2 &u, const uint2 &v, uint32_t (&c)[2], uint32_t (&s)[2]) {
    const uint32_t a = most2(u.x, u.y), b = most2(v.x, v.y);
    uint32_t m = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    #pragma unroll
    for (int i = 1; i < 8; i <<= 1) m = __vmaxu2(m, __shfl_xor_sync(kFullMask, m, i));
    const float2 most = unpack_pair<T>(m);
    s[0] = code_scale(most.x); s[1] = code_scale(most.y);
    c[0] = codes_by<T>(u, scale_inverse(s[0])); c[1] = codes_by<T>(v, scale_inverse(s[1]));
}
template <typename T> __device__ __forceinline__ void codes_of_groups(const uint4 &u, const uint4 &v, uint32_t (&c)[2], uint32_t (&s)[2]) {
    const uint4 w[2] = {u, v};
    #pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t m = max(max(w[k].x & 0x7fffffffu, w[k].y & 0x7fffffffu), max(w[k].z & 0x7fffffffu, w[k].w & 0x7fffffffu));
        #pragma unroll
        for (int i = 1; i < 8; i <<= 1) m = max(m, __shfl_xor_sync(kFullMask, m, i));
        s[k] = code_scale(__uint_as_float(m));
        c[k] = codes_by<T>(w[k], scale_inverse(s[k]));
    }
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
