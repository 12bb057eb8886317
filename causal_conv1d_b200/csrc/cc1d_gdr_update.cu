// Decode step of the gated delta rule: cc1d_gdr_update (include/cc1d_gdr.h).
#include "cc1d_gdr.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

// One CTA owns 4 * kLanes columns of one state (dim_k x dim_v fp32) and keeps them in registers
// over all tokens: every state element is read once and written once, which is all the traffic
// that matters (64 KB each way per row and head of 128 x 128, q, k, v, out together 1 KB).
//   r = S^T k, y = S^T q (one pass over the old state, one reduction)
//   d = beta (v - a r);  o = scale (a y + (k.q) d);  S <- a S + k d^T
// A warp's load covers 32 / kLanes rows of the slice, 16 bytes per lane; all loads of a thread
// (128 / (4 * 32 / kLanes)) are in flight together.  Bound by HBM: 256 rows x 32 heads, 1.08 GB, 164 us =
// 6.58 TB/s with 64-column slices and 4 CTAs of 128 threads per SM; 128 columns and 2 CTAs 184 us, 32 columns
// 177 us, 256 threads 195-220 us (fewer, longer CTAs leave gaps between load and store).  One row of 32 heads:
// 3.3 us with 32 columns (128 CTAs), 4.1 us with 64.
template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads, kLanes == 16 ? 4 : 6) gdr_update_kernel(const cc1d_gdr_params p, int slices) {
    constexpr int kRows = 32 / kLanes, kIter = kGdrMaxDim / (kWarps * kRows), kCols = 4 * kLanes;
    __shared__ float sk[2][kGdrMaxDim], sq[2][kGdrMaxDim];
    __shared__ float4 red[2][2][kWarps][kLanes];
    pdl_wait();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    uint32_t id = blockIdx.x;
    const int slice = id % slices; id /= slices;
    const int h = id % (uint32_t)p.heads_v;
    const int64_t b = id / (uint32_t)p.heads_v;
    const int dk = (int)p.dim_k, dv = (int)p.dim_v, tokens = (int)p.seqlen;
    const int hk = h / (int)(p.heads_v / p.heads_k);
    const int col = slice * kCols + 4 * (lane % kLanes);
    const bool col_ok = col < dv;
    const int64_t row = gdr_state_row(p, b);
    T *out = reinterpret_cast<T *>(p.out) + b * p.out_batch_stride + h * p.out_h_stride + col;
    if (row < 0) {
        if (warp == 0 && lane < kLanes && col_ok) {
            for (int t = 0; t < tokens; ++t) {
                #pragma unroll
                for (int c = 0; c < 4; ++c) out[t * p.out_l_stride + c] = Elem<T>::from_f(0.f);
            }
        }
        return;
    }
    // A token's inputs do not wait for the state row: they are asked for before it, the next token's while one
    // is computed.
    const T *kp = reinterpret_cast<const T *>(p.k) + b * p.k_batch_stride + hk * p.k_h_stride + tid;
    const T *qp = reinterpret_cast<const T *>(p.q) + b * p.q_batch_stride + hk * p.q_h_stride + tid;
    const T *v = reinterpret_cast<const T *>(p.v) + b * p.v_batch_stride + h * p.v_h_stride + col;
    T k_next = Elem<T>::from_f(0.f), q_next = k_next, v_next[4];
    uint32_t g_next = 0, beta_next = 0;
    #pragma unroll
    for (int c = 0; c < 4; ++c) v_next[c] = k_next;
    auto ask = [&](int t) {
        if (tid < dk) { k_next = kp[t * p.k_l_stride]; q_next = qp[t * p.q_l_stride]; }
        if (col_ok) {
            #pragma unroll
            for (int c = 0; c < 4; ++c) v_next[c] = v[t * p.v_l_stride + c];
        }
        g_next = load_bits(p.g, b * p.g_batch_stride + t * p.g_l_stride + h * p.g_h_stride, p.gtype);
        beta_next = load_bits(p.beta, b * p.beta_batch_stride + t * p.beta_l_stride + h * p.beta_h_stride, p.btype);
    };
    if (tokens > 0) ask(0);
    float *state = p.final_states + row * p.final_states_batch_stride + h * p.final_states_h_stride + col;
    const int row0 = warp * kRows + lane / kLanes;   // rows of this thread: row0 + i * kWarps * kRows
    float4 S[kIter];
    #pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const int r = row0 + i * kWarps * kRows;
        S[i] = col_ok && r < dk ? __ldcs(reinterpret_cast<const float4 *>(state + (int64_t)r * dv)) : make_float4(0, 0, 0, 0);
    }
    for (int t = 0; t < tokens; ++t) {
        const int s = t & 1;
        if (tid < kGdrMaxDim) { sk[s][tid] = Elem<T>::to_f(k_next); sq[s][tid] = Elem<T>::to_f(q_next); }
        const float a = gdr_exp(from_bits(g_next, p.gtype)), beta = from_bits(beta_next, p.btype);
        float vt[4];
        #pragma unroll
        for (int c = 0; c < 4; ++c) vt[c] = Elem<T>::to_f(v_next[c]);
        if (t + 1 < tokens) ask(t + 1);
        __syncthreads();
        float4 r = make_float4(0, 0, 0, 0), y = r;
        #pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float kk = sk[s][row0 + i * kWarps * kRows], qq = sq[s][row0 + i * kWarps * kRows];
            r.x = fmaf(S[i].x, kk, r.x); r.y = fmaf(S[i].y, kk, r.y); r.z = fmaf(S[i].z, kk, r.z); r.w = fmaf(S[i].w, kk, r.w);
            y.x = fmaf(S[i].x, qq, y.x); y.y = fmaf(S[i].y, qq, y.y); y.z = fmaf(S[i].z, qq, y.z); y.w = fmaf(S[i].w, qq, y.w);
        }
        float kq = 0.f;
        #pragma unroll
        for (int i = 0; i < kGdrMaxDim / 32; ++i) kq = fmaf(sk[s][lane + 32 * i], sq[s][lane + 32 * i], kq);
        #pragma unroll
        for (int m = 16; m >= 1; m >>= 1) {
            kq += __shfl_xor_sync(kFullMask, kq, m);
            if (m >= kLanes) {
                r.x += __shfl_xor_sync(kFullMask, r.x, m); r.y += __shfl_xor_sync(kFullMask, r.y, m);
                r.z += __shfl_xor_sync(kFullMask, r.z, m); r.w += __shfl_xor_sync(kFullMask, r.w, m);
                y.x += __shfl_xor_sync(kFullMask, y.x, m); y.y += __shfl_xor_sync(kFullMask, y.y, m);
                y.z += __shfl_xor_sync(kFullMask, y.z, m); y.w += __shfl_xor_sync(kFullMask, y.w, m);
            }
        }
        if (lane < kLanes) { red[s][0][warp][lane] = r; red[s][1][warp][lane] = y; }
        __syncthreads();
        r = y = make_float4(0, 0, 0, 0);
        #pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 u = red[s][0][w][lane % kLanes], z = red[s][1][w][lane % kLanes];
            r.x += u.x; r.y += u.y; r.z += u.z; r.w += u.w;
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        const float4 d = make_float4(beta * (vt[0] - a * r.x), beta * (vt[1] - a * r.y), beta * (vt[2] - a * r.z), beta * (vt[3] - a * r.w));
        if (warp == 0 && lane < kLanes && col_ok) {
            T *o = out + t * p.out_l_stride;
            o[0] = Elem<T>::from_f(p.scale * fmaf(a, y.x, kq * d.x)); o[1] = Elem<T>::from_f(p.scale * fmaf(a, y.y, kq * d.y));
            o[2] = Elem<T>::from_f(p.scale * fmaf(a, y.z, kq * d.z)); o[3] = Elem<T>::from_f(p.scale * fmaf(a, y.w, kq * d.w));
        }
        #pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float kk = sk[s][row0 + i * kWarps * kRows];
            S[i].x = fmaf(a, S[i].x, kk * d.x); S[i].y = fmaf(a, S[i].y, kk * d.y);
            S[i].z = fmaf(a, S[i].z, kk * d.z); S[i].w = fmaf(a, S[i].w, kk * d.w);
        }
    }
    #pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const int r = row0 + i * kWarps * kRows;
        if (col_ok && r < dk) __stcs(reinterpret_cast<float4 *>(state + (int64_t)r * dv), S[i]);
    }
}

}  // namespace

int launch_gdr_update(const cc1d_gdr_params &p, cudaStream_t stream) {
    const int64_t states = p.batch * p.heads_v;
    // 32 columns a CTA while 64 would not give every SM two CTAs
    const int lanes = states * ((p.dim_v + 63) / 64) >= 2 * num_sms() ? 16 : 8;
    const int slices = (int)((p.dim_v + 4 * lanes - 1) / (4 * lanes));
    if (states * slices >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    const dim3 grid((unsigned)(states * slices));
    CC1D_DISPATCH_ITYPE(p.itype, {
        if (lanes == 16) launch_k(gdr_update_kernel<T, 16>, grid, kThreads, 0, stream, p, slices);
        else launch_k(gdr_update_kernel<T, 8>, grid, kThreads, 0, stream, p, slices);
    });
    return check_launch();
}

}  // namespace cc1d
