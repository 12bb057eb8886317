// Tensor-core side of the chunked gated delta rule: tcgen05 wrappers, operand layouts, fp32 values
// as sums of bf16 pieces, and the per-chunk preparation that forward and backward share.
#pragma once

#include "cc1d_gdr.cuh"
#include "cc1d_tma.cuh"

namespace cc1d {

constexpr int kChunk = 64;

// ---- tcgen05 ---------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc512(uint32_t smem_slot) {   // one whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free512(uint32_t tmem) {         // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// all MMAs issued by this thread so far arrive on `bar` when they are done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}

template <int N> __device__ __forceinline__ void tmem_ld(float (&f)[N], uint32_t at);
template <> __device__ __forceinline__ void tmem_ld<16>(float (&f)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
                   "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]) : "r"(at));
}
template <> __device__ __forceinline__ void tmem_ld<32>(float (&f)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
                 "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
                   "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]),
                   "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]),
                   "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31]) : "r"(at));
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "r"(at), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

// Instruction descriptor of kind::f16, bf16 x bf16 -> fp32 (M rows, N columns; MN-major operands
// have their contraction index as the slow one in shared memory).
__device__ __forceinline__ constexpr uint32_t mma_desc(int M, int N, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N / 8) << 17) |
           ((uint32_t)(M / 16) << 24);
}
// Shared-memory operand in the 128-byte swizzle.  K-major (lead unused): rows of 128 bytes, 1024
// bytes from one group of 8 rows to the next.  MN-major: atoms of 64 MN x 8 K elements, 1024 bytes
// from one group of 8 K to the next, `lead` bytes from one 64 of MN to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead = 16) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

// Bounded wait.  When one runs out (never expected) the flag of the translation unit is raised and
// `dead` makes every later wait of the CTA return at once: the CTA then runs to its end on
// incomplete data, releases its tensor memory and returns.
__device__ __forceinline__ void gdr_wait(uint32_t bar, uint32_t parity, volatile int *dead) {
    for (uint32_t i = 0; i < kTmaSpinLimit; ++i) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return;
        if ((i & 255) == 255 && *dead) return;
    }
    *dead = 1;
    g_tma_wait_expired = 1;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
template <int kId, int kThreads> __device__ __forceinline__ void group_sync() {
    asm volatile("bar.sync %0, %1;" :: "n"(kId), "n"(kThreads) : "memory");
}

// ---- fp32 as a sum of bf16 pieces ---------------------------------------------------------------
// x = x1 + x2 + x3 with x1 = bf16(x), x2 = bf16(x - x1), x3 = bf16(x - x1 - x2): 8 + 8 + 8
// significant bits, so three pieces hold an fp32 and two leave 2^-17 of it.  The differences are
// exact.  bf16 inputs are one piece, fp16 inputs two.  A product of two such sums takes the
// pairs of pieces whose orders add up to less than the pieces kept.
__device__ __forceinline__ uint32_t bf16_pair(float2 x) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t *>(&t);
}
// first kPieces pieces of a pair.  An infinite or NaN first piece leaves NaN or infinity in the
// product as the value itself would (later pieces of it are NaN or inf - inf = NaN as well).
template <int kPieces> __device__ __forceinline__ void split_pair(float2 x, uint32_t (&r)[kPieces]) {
    #pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        r[i] = bf16_pair(x);
        if (i + 1 < kPieces) x = add2(x, make_float2(-__uint_as_float(r[i] << 16), -__uint_as_float(r[i] & 0xffff0000u)));
    }
}
// 16 values -> kPieces registers vectors of 8 packed pairs
template <int kPieces> __device__ __forceinline__ void split16(const float (&x)[16], uint32_t (&r)[kPieces][8]) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t p[kPieces];
        split_pair<kPieces>(make_float2(x[2 * i], x[2 * i + 1]), p);
        #pragma unroll
        for (int k = 0; k < kPieces; ++k) r[k][i] = p[k];
    }
}

template <typename T> struct GdrType;
template <> struct GdrType<__nv_bfloat16> { static constexpr int kPieces = 1, kOutPieces = 2; };
template <> struct GdrType<__half> { static constexpr int kPieces = 2, kOutPieces = 2; };
template <> struct GdrType<float> { static constexpr int kPieces = 3, kOutPieces = 3; };

// ---- operand tiles ------------------------------------------------------------------------------
// Token tile of one piece: panels of 64 columns, a panel `rows` x 128 bytes in the 128-byte swizzle.
// Used K-major (contraction over the columns) and MN-major (contraction over the tokens).
__device__ __forceinline__ uint32_t tile_at(int row, int chunk16, uint32_t panel_bytes) {
    return (chunk16 >> 3) * panel_bytes + row * 128 + (((chunk16 & 7) ^ (row & 7)) << 4);
}

// 8 elements of one row -> one 16-byte piece vector each
template <typename T, int kPieces> __device__ __forceinline__ void row_pieces(const T *src, bool ok, uint4 (&out)[kPieces]) {
    if constexpr (sizeof(T) == 2 && kPieces == 1) {
        out[0] = ok ? ld_cached(src) : make_uint4(0, 0, 0, 0);
    } else {
        float f[8];
        if constexpr (sizeof(T) == 2) {
            unpack<T>(ok ? ld_cached(src) : make_uint4(0, 0, 0, 0), f);
        } else {
            unpack<T>(ok ? ld_cached(src) : make_uint4(0, 0, 0, 0), f);
            unpack<T>(ok ? ld_cached(src + 4) : make_uint4(0, 0, 0, 0), f + 4);
        }
        uint32_t r[4][kPieces];
        #pragma unroll
        for (int i = 0; i < 4; ++i) split_pair<kPieces>(make_float2(f[2 * i], f[2 * i + 1]), r[i]);
        #pragma unroll
        for (int k = 0; k < kPieces; ++k) out[k] = make_uint4(r[0][k], r[1][k], r[2][k], r[3][k]);
    }
}

__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Gates of a chunk.  G, the running sum of g, is summed in double and kept as two floats: a
// difference G_i - G_j of near tokens far from the chunk's start keeps its relative accuracy.
struct GdrGates {
    float g_hi[kChunk], g_lo[kChunk], from_start[kChunk], to_end[kChunk], beta[kChunk];
};
__device__ __forceinline__ float gdr_fade(const GdrGates &s, float hi, float lo, int j) {
    return gdr_exp((hi - s.g_hi[j]) + (lo - s.g_lo[j]));
}

// One warp: gates of tokens t0 .. t0 + 63 (those at or after `end` do not exist: g = beta = 0).
__device__ __forceinline__ void load_gates(GdrGates &s, const cc1d_gdr_params &p, const GdrSeq &seq, int h, int t0, int lane) {
    const int64_t ga = seq.row * p.g_batch_stride + h * p.g_h_stride, ba = seq.row * p.beta_batch_stride + h * p.beta_h_stride;
    double v[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = t0 + 2 * lane + i;
        const bool ok = t < seq.end;
        const float g = ok ? load_any(p.g, ga + t * p.g_l_stride, p.gtype) : 0.f;
        v[i] = g < -200.f ? -200.0 : (double)g;
        s.beta[2 * lane + i] = ok ? load_any(p.beta, ba + t * p.beta_l_stride, p.btype) : 0.f;
    }
    v[1] += v[0];
    double sum = v[1];
    #pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(kFullMask, sum, m);
        if (lane >= m) sum += o;
    }
    const double before = sum - v[1], whole = __shfl_sync(kFullMask, sum, 31);
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double G = before + v[i];
        const float hi = (float)G;
        s.g_hi[2 * lane + i] = hi;
        s.g_lo[2 * lane + i] = (float)(G - (double)hi);
        s.from_start[2 * lane + i] = gdr_exp(hi) * (1.f + (float)(G - (double)hi));
        s.to_end[2 * lane + i] = gdr_exp((float)(whole - G));
    }
}

// ---- (I + A)^-1 of a unit lower triangular 64 x 64 matrix ------------------------------------
// Block elimination: four 16 x 16 diagonal blocks column by column, then 16 -> 32 -> 64 with
//   T21 = -T22 (A21 T11).
// a: the strictly lower part (its upper blocks are scratch); t: receives the lower part of the
// inverse, diagonal included.  Rows are kLd floats.  256 threads; ends without a barrier.
constexpr int kLd = kChunk + 4;

template <int kId> __device__ __forceinline__ void invert_unit_lower(float *a, float *t, int tid) {
    if (tid < 64) {
        const int b = (tid >> 4) * 16, c = tid & 15;
        float x[16];
        #pragma unroll
        for (int r = 0; r < 16; ++r) {
            float acc = r == c ? 1.f : 0.f;
            #pragma unroll
            for (int l4 = 0; l4 < r; l4 += 4) {
                const float4 m = *reinterpret_cast<const float4 *>(a + (b + r) * kLd + b + l4);
                acc = fmaf(-m.x, x[l4], acc);
                if (l4 + 1 < r) acc = fmaf(-m.y, x[l4 + 1], acc);
                if (l4 + 2 < r) acc = fmaf(-m.z, x[l4 + 2], acc);
                if (l4 + 3 < r) acc = fmaf(-m.w, x[l4 + 3], acc);
            }
            x[r] = r < c ? 0.f : acc;
            t[(b + r) * kLd + b + c] = x[r];
        }
    }
    group_sync<kId, 256>();
    {   // 16 -> 32, two blocks: 2 outputs per thread
        const int b = (tid >> 7) * 32, r = (tid >> 3) & 15, c = (tid & 7) * 2;
        float2 m = make_float2(0.f, 0.f);
        #pragma unroll
        for (int l = 0; l < 16; ++l) {
            const float x = a[(b + 16 + r) * kLd + b + l];
            const float2 y = *reinterpret_cast<const float2 *>(t + (b + l) * kLd + b + c);
            m.x = fmaf(x, y.x, m.x); m.y = fmaf(x, y.y, m.y);
        }
        *reinterpret_cast<float2 *>(a + (b + r) * kLd + b + 16 + c) = m;   // scratch above the diagonal
        group_sync<kId, 256>();
        float2 n = make_float2(0.f, 0.f);
        #pragma unroll
        for (int l = 0; l < 16; ++l) {
            const float x = t[(b + 16 + r) * kLd + b + 16 + l];
            const float2 y = *reinterpret_cast<const float2 *>(a + (b + l) * kLd + b + 16 + c);
            n.x = fmaf(-x, y.x, n.x); n.y = fmaf(-x, y.y, n.y);
        }
        *reinterpret_cast<float2 *>(t + (b + 16 + r) * kLd + b + c) = n;
        *reinterpret_cast<float2 *>(t + (b + r) * kLd + b + 16 + c) = make_float2(0.f, 0.f);   // zeros above the diagonal
    }
    group_sync<kId, 256>();
    {   // 32 -> 64: 4 outputs per thread
        const int r = tid >> 3, c = (tid & 7) * 4;
        float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll 8
        for (int l = 0; l < 32; ++l) {
            const float x = a[(32 + r) * kLd + l];
            const float4 y = *reinterpret_cast<const float4 *>(t + l * kLd + c);
            m.x = fmaf(x, y.x, m.x); m.y = fmaf(x, y.y, m.y); m.z = fmaf(x, y.z, m.z); m.w = fmaf(x, y.w, m.w);
        }
        *reinterpret_cast<float4 *>(a + r * kLd + 32 + c) = m;
        group_sync<kId, 256>();
        float4 n = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll 8
        for (int l = 0; l < 32; ++l) {
            const float x = t[(32 + r) * kLd + 32 + l];
            const float4 y = *reinterpret_cast<const float4 *>(a + l * kLd + 32 + c);
            n.x = fmaf(-x, y.x, n.x); n.y = fmaf(-x, y.y, n.y); n.z = fmaf(-x, y.z, n.z); n.w = fmaf(-x, y.w, n.w);
        }
        *reinterpret_cast<float4 *>(t + (32 + r) * kLd + c) = n;
        *reinterpret_cast<float4 *>(t + r * kLd + 32 + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

}  // namespace cc1d

namespace cc1d {

// ---- a chunk made ready -------------------------------------------------------------------------
// What the walk over the chunks reads of one chunk:
//   K, Q   token tiles, rows 0-63 k, 64-127 q (kPieces pieces)
//   T      (I + A)^-1, A_ij = beta_i (k_i.k_j) e^{G_i - G_j} for j < i    (3 pieces, row i, column j)
//   P      (q_i.k_j) e^{G_i - G_j} for j <= i                             (kOutPieces pieces)
//   V      as it is, [64][128]
template <typename T> struct GdrStage {
    static constexpr int kPieces = GdrType<T>::kPieces, kOut = GdrType<T>::kOutPieces;
    static constexpr uint32_t kPanel = 128 * 128, kKqPiece = 2 * kPanel;     // panel: 128 rows x 64 columns
    static constexpr uint32_t kKq = 0, kT = kKq + kPieces * kKqPiece, kP = kT + 3 * 8192, kV = kP + kOut * 8192,
                              kGates = kV + kChunk * kGdrMaxDim * sizeof(T), kBytes = kGates + 2048;
};
static_assert(sizeof(GdrGates) <= 2048, "gates of a chunk");
constexpr uint32_t kGdrInverseBytes = 2 * kChunk * kLd * 4;

constexpr uint32_t kColKq = 416;   // tensor-memory columns 416..479: K K^T (lanes 0-63) and Q K^T (lanes 64-127)

// 256 threads (warps 0-7 of the group) fill a stage; bar_kq is theirs.  Ends without a barrier:
// the caller orders its generic-proxy writes before the walk's MMAs.
template <typename T, int kId>
__device__ __forceinline__ void prepare_chunk(unsigned char *stage, float *inv, const cc1d_gdr_params &p, const GdrSeq &seq, int h, int t0,
                                              uint32_t tmem, uint32_t bar_kq, uint32_t kq_parity, volatile int *dead, int tid) {
    using S = GdrStage<T>;
    constexpr int NP = S::kPieces;
    const int warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(stage);
    GdrGates &gates = *reinterpret_cast<GdrGates *>(stage + S::kGates);
    const int hk = h / (int)(p.heads_v / p.heads_k);
    const T *kp = reinterpret_cast<const T *>(p.k) + seq.row * p.k_batch_stride + hk * p.k_h_stride;
    const T *qp = reinterpret_cast<const T *>(p.q) + seq.row * p.q_batch_stride + hk * p.q_h_stride;
    const T *vp = reinterpret_cast<const T *>(p.v) + seq.row * p.v_batch_stride + h * p.v_h_stride;
    if (warp == 0) load_gates(gates, p, seq, h, t0, lane);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = (tid >> 4) + 16 * i, c = tid & 15;
        const int64_t t = t0 + row;
        const bool ok = t < seq.end && c * 8 < p.dim_k;
        uint4 kv[NP], qv[NP];
        row_pieces<T, NP>(kp + t * p.k_l_stride + c * 8, ok, kv);
        row_pieces<T, NP>(qp + t * p.q_l_stride + c * 8, ok, qv);
        const uint32_t at = base + S::kKq + tile_at(row, c, S::kPanel);
        #pragma unroll
        for (int k = 0; k < NP; ++k) { sts128(at + k * S::kKqPiece, kv[k]); sts128(at + k * S::kKqPiece + 64 * 128, qv[k]); }
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = (tid >> 4) + 16 * i, c = tid & 15;
        const int64_t t = t0 + row;
        const bool ok = t < seq.end && c * 8 < p.dim_v;
        const T *src = vp + t * p.v_l_stride + c * 8;
        #pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k)
            sts128(base + S::kV + (row * kGdrMaxDim + c * 8) * sizeof(T) + 16 * k, ok ? ld_cached(src + 4 * k) : make_uint4(0, 0, 0, 0));
    }
    fence_proxy_async_smem();
    group_sync<kId, 256>();
    if (tid == 0) {
        fence_after_sync();
        constexpr uint32_t id = mma_desc(128, 64, false, false);
        const int steps = (int)(p.dim_k + 15) / 16;
        bool add = false;
        #pragma unroll
        for (int a = 0; a < NP; ++a) {
            #pragma unroll
            for (int b = 0; b < NP && a + b < 3; ++b) {
                for (int s = 0; s < steps; ++s) {
                    const uint32_t off = (s >> 2) * S::kPanel + (s & 3) * 32;
                    mma_ss(tmem + kColKq, smem_desc(base + S::kKq + a * S::kKqPiece + off), smem_desc(base + S::kKq + b * S::kKqPiece + off), id, add);
                    add = true;
                }
            }
        }
        mma_commit(bar_kq);
    }
    gdr_wait(bar_kq, kq_parity, dead);
    __syncwarp();
    fence_after_sync();
    {
        const int quad = warp & 3, half = warp >> 2, i = (quad & 1) * 32 + lane;
        const float hi = gates.g_hi[i], lo = gates.g_lo[i], beta = gates.beta[i];
        #pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int j0 = 32 * half + 16 * b;
            float x[16];
            tmem_ld<16>(x, tmem + ((uint32_t)(quad * 32) << 16) + kColKq + j0);
            tmem_wait_ld();
            if (quad < 2) {
                #pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = j0 + j < i ? beta * x[j] * gdr_fade(gates, hi, lo, j0 + j) : 0.f;
                #pragma unroll
                for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4 *>(inv + i * kLd + j0 + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            } else {
                #pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = j0 + j <= i ? x[j] * gdr_fade(gates, hi, lo, j0 + j) : 0.f;
                uint32_t r[S::kOut][8];
                split16<S::kOut>(x, r);
                #pragma unroll
                for (int k = 0; k < S::kOut; ++k) {
                    sts128(base + S::kP + k * 8192 + tile_at(i, j0 / 8, 0), make_uint4(r[k][0], r[k][1], r[k][2], r[k][3]));
                    sts128(base + S::kP + k * 8192 + tile_at(i, j0 / 8 + 1, 0), make_uint4(r[k][4], r[k][5], r[k][6], r[k][7]));
                }
            }
        }
        fence_before_sync();
    }
    group_sync<kId, 256>();
    float *t = inv + kChunk * kLd;
    invert_unit_lower<kId>(inv, t, tid);
    group_sync<kId, 256>();
    {
        const int i = tid >> 2, j0 = (tid & 3) * 16;
        float x[16];
        #pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(t + i * kLd + j0 + j);
            x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
        }
        uint32_t r[3][8];
        split16<3>(x, r);
        #pragma unroll
        for (int k = 0; k < 3; ++k) {
            sts128(base + S::kT + k * 8192 + tile_at(i, j0 / 8, 0), make_uint4(r[k][0], r[k][1], r[k][2], r[k][3]));
            sts128(base + S::kT + k * 8192 + tile_at(i, j0 / 8 + 1, 0), make_uint4(r[k][4], r[k][5], r[k][6], r[k][7]));
        }
    }
    fence_proxy_async_smem();
}

}  // namespace cc1d
