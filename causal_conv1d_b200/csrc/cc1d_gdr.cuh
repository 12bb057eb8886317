// Shared pieces of the gated delta rule kernels: arguments, gates, sequence lookup.
#pragma once

#include "cc1d_common.cuh"
#include "cc1d_gdr.h"
#include "cc1d_kernels.h"

namespace cc1d {

constexpr int kGdrMaxDim = 128;

// exp(x) to about one unit in the last place: x = n ln 2 + r with ln 2 = 2839 / 4096 + a rest (n times the first
// part is exact), the Taylor series of exp(r) to r^7 / 7! (|r| <= 0.35: what is left out is 5e-9), and 2^n in two
// factors so that it may leave the range.  ex2.approx's 2^-22 shows in the states: the decays of all chunks
// multiply.  Below -176 (and at -inf) the result is 0, a NaN stays one.
__device__ __forceinline__ float gdr_exp(float x) {
    x = x < -176.f ? -176.f : x > 176.f ? 176.f : x;
    const float n = rintf(x * 1.44269504f);
    const float r = fmaf(n, -3.194618494547e-05f, fmaf(n, -2839.f / 4096.f, x));
    float p = 1.f / 5040.f;
    p = fmaf(p, r, 1.f / 720.f);
    p = fmaf(p, r, 1.f / 120.f);
    p = fmaf(p, r, 1.f / 24.f);
    p = fmaf(p, r, 1.f / 6.f);
    p = fmaf(p, r, 0.5f);
    p = fmaf(p, r, 1.f);
    p = fmaf(p, r, 1.f);
    const int i = (int)n, half = i >> 1;
    return p * __uint_as_float((uint32_t)(half + 127) << 23) * __uint_as_float((uint32_t)(i - half + 127) << 23);
}

// A gate as it lies in memory, and its value: a conversion beside the load would wait for it
__device__ __forceinline__ uint32_t load_bits(const void *p, int64_t at, int dtype) {
    return dtype == CC1D_F32 ? __ldg(reinterpret_cast<const uint32_t *>(p) + at) : (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(p) + at);
}
__device__ __forceinline__ float from_bits(uint32_t v, int dtype) {
    return dtype == CC1D_F32 ? __uint_as_float(v) : dtype == CC1D_BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half((unsigned short)v));
}

__device__ __forceinline__ void store_any(void *p, int64_t at, int dtype, float v) {
    if (dtype == CC1D_F32) reinterpret_cast<float *>(p)[at] = v;
    else if (dtype == CC1D_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half *>(p)[at] = __float2half_rn(v);
}

// Tokens [begin, end) of sequence n, and the batch row they lie in.
struct GdrSeq { int64_t row; int32_t begin, end; };

__device__ __forceinline__ GdrSeq gdr_sequence(const cc1d_gdr_params &p, int n) {
    if (p.cu_seqlens == nullptr) return {n, 0, (int32_t)p.seqlen};
    const int32_t last = (int32_t)p.seqlen;
    int32_t a = __ldg(p.cu_seqlens + n), b = __ldg(p.cu_seqlens + n + 1);
    a = min(max(a, 0), last);
    b = min(max(b, a), last);
    return {0, a, b};
}

// State row of sequence n; negative where it has none.
__device__ __forceinline__ int64_t gdr_state_row(const cc1d_gdr_params &p, int64_t n) {
    const int64_t r = p.state_indices != nullptr ? (int64_t)__ldg(p.state_indices + n) : n;
    return r < p.state_rows ? r : -1;
}

__host__ __device__ inline int64_t gdr_sequences(const cc1d_gdr_params &p) { return p.cu_seqlens != nullptr ? p.nseq : p.batch; }

int launch_gdr_update(const cc1d_gdr_params &p, cudaStream_t stream);
size_t gdr_fwd_workspace_bytes(const cc1d_gdr_params &p);
int launch_gdr_fwd(const cc1d_gdr_params &p, cudaStream_t stream);
size_t gdr_bwd_workspace_bytes(const cc1d_gdr_bwd_params &p);
int launch_gdr_bwd(const cc1d_gdr_bwd_params &p, cudaStream_t stream);

}  // namespace cc1d
