// What the walks over the chunks of the gated delta rule share, made for all chunks at once:
// T = (I + A)^-1, P and the gates of every chunk (cc1d_gdr_mma.cuh says what they are).
#include "cc1d_gdr_mma.cuh"

namespace cc1d {
namespace {

// Gates of two tokens as they lie in memory, converted where they are used.
struct GateRegs { uint32_t g[2], beta[2]; };
struct GateSums { float4 G; float2 beta; };   // (high, low) of G and beta of two tokens
// One warp: gates of tokens t0 .. t0 + 63 (those at or after `end` do not exist: g = beta = 0).
__device__ __forceinline__ void load_gates(GateRegs &r, const cc1d_gdr_params &p, const GdrSeq &seq, int h, int t0, int lane) {
    const int64_t ga = seq.row * p.g_batch_stride + h * p.g_h_stride, ba = seq.row * p.beta_batch_stride + h * p.beta_h_stride;
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t t = t0 + 2 * lane + i;
        r.g[i] = r.beta[i] = 0;            // the bits of 0 in every type
        if (t < seq.end) {
            r.g[i] = load_bits(p.g, ga + t * p.g_l_stride, p.gtype);
            r.beta[i] = load_bits(p.beta, ba + t * p.beta_l_stride, p.btype);
        }
    }
}
// a + b as two floats (Knuth's two-sum: s + e is a + b exactly), low parts added up
__device__ __forceinline__ float2 sum2(float2 a, float2 b) {
    const float s = a.x + b.x, t = s - a.x;
    return make_float2(s, (a.x - (s - t)) + (b.x - t) + (a.y + b.y));
}
__device__ __forceinline__ float2 shfl2(float2 v, int src) { return make_float2(__shfl_sync(kFullMask, v.x, src), __shfl_sync(kFullMask, v.y, src)); }

// One warp: G and beta.  (In double this scan alone took 5000 cycles.)
__device__ __forceinline__ GateSums scan_gates(const GateRegs &r, const cc1d_gdr_params &p, int lane) {
    float2 v[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float g = from_bits(r.g[i], p.gtype);
        v[i] = make_float2(g < -200.f ? -200.f : g, 0.f);
    }
    v[1] = sum2(v[0], v[1]);
    float2 sum = v[1];
    #pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const float2 o = shfl2(sum, lane - m);
        if (lane >= m) sum = sum2(sum, o);
    }
    const float2 o = shfl2(sum, lane - 1), before = lane > 0 ? o : make_float2(0.f, 0.f);
    v[0] = sum2(v[0], before);
    return {make_float4(v[0].x, v[0].y, sum.x, sum.y), make_float2(from_bits(r.beta[0], p.btype), from_bits(r.beta[1], p.btype))};
}
__device__ __forceinline__ void store_gates(GdrGates &s, const GateSums &r, int lane) {
    *reinterpret_cast<float4 *>(&s.g[2 * lane]) = r.G;
    *reinterpret_cast<float2 *>(&s.beta[2 * lane]) = r.beta;
    if (lane == 0) { s.steep = 0; s.bad = kChunk; }
}
// 128 threads, after store_gates: the exponentials
__device__ __forceinline__ void expand_gates(GdrGates &s, int tid) {
    const int t = tid & 63;
    const float2 G = s.g[t];
    if (tid < 64) {
        const float start = gdr_exp(G.x) * (1.f + G.y);
        s.from_start[t] = start;
        s.minus_beta_from_start[t] = -s.beta[t] * start;
        const float2 ref = t < 16 ? make_float2(0.f, 0.f) : s.g[(t & 48) - 1];
        const float span = (ref.x - G.x) + (ref.y - G.y);
        s.row[t] = gdr_exp(-span);
        s.same[t] = gdr_exp(span);
        if (!(fabsf(span) < 60.f)) s.steep = 1;
        if (t < 16) s.column[0][t] = gdr_fade(s.g[15], G);
    } else {
        s.to_end[t] = gdr_fade(s.g[kChunk - 1], G);
        if (t < 32) s.column[1][t] = gdr_fade(s.g[31], G);
        if (t < 48) s.column[2][t] = gdr_fade(s.g[47], G);
    }
}

// ---- (I + A)^-1 of a unit lower triangular 64 x 64 matrix ------------------------------------
// Block elimination: four 16 x 16 diagonal blocks column by column in fp32, then 16 -> 32 -> 64 with
//   T21 = -(T22 A21) T11
// on the TF32 tensor cores, every factor as two TF32 values (11 + 11 bits; three products).  The
// contraction index is taken in the order 0, 2, 4, 6, 1, 3, 5, 7 within a step of 8: a product in
// accumulator layout is then the left factor of the next one as it is.
// In place: a holds the strictly lower part and receives the lower part of the inverse, diagonal
// included, with zeros above it inside the 16 x 16 diagonal blocks; the upper right 32 x 32 block is
// scratch.  Rows are kLd floats.  128 threads; ends with a barrier.
constexpr int kLd = kChunk + 4;

struct Tf32Pair { uint32_t hi, lo; };
// cut, not rounded (a conversion runs at a quarter of the rate of a mask): the low part takes what the
// high one leaves, so 2^-20 of the value is lost at most
__device__ __forceinline__ Tf32Pair tf32_pair(float x) {
    const uint32_t hi = __float_as_uint(x) & 0xffffe000u;
    return {hi, __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u};
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d (16 x 8) += A (16 x 8) B (8 x 8): x = A(g, 2t), A(g+8, 2t), A(g, 2t+1), A(g+8, 2t+1) and y = B(2t, g), B(2t+1, g)
// for g = lane / 4, t = lane % 4
// the three products go to accumulators of their own (d[0] the large one): three short chains instead of a long one
__device__ __forceinline__ void mma_fp32(float (&d)[3][4], const float (&x)[4], const float (&y)[2]) {
    const Tf32Pair a0 = tf32_pair(x[0]), a1 = tf32_pair(x[1]), a2 = tf32_pair(x[2]), a3 = tf32_pair(x[3]), b0 = tf32_pair(y[0]), b1 = tf32_pair(y[1]);
    mma_tf32(d[1], a0.lo, a1.lo, a2.lo, a3.lo, b0.hi, b1.hi);
    mma_tf32(d[2], a0.hi, a1.hi, a2.hi, a3.hi, b0.lo, b1.lo);
    mma_tf32(d[0], a0.hi, a1.hi, a2.hi, a3.hi, b0.hi, b1.hi);
}
__device__ __forceinline__ float total(const float (&d)[3][4], int i) { return d[0][i] + (d[1][i] + d[2][i]); }
__device__ __forceinline__ void left_factor(float (&x)[4], const float *m, int lane) {
    const float2 u = *reinterpret_cast<const float2 *>(m + (lane >> 2) * kLd + 2 * (lane & 3));
    const float2 v = *reinterpret_cast<const float2 *>(m + ((lane >> 2) + 8) * kLd + 2 * (lane & 3));
    x[0] = u.x; x[1] = v.x; x[2] = u.y; x[3] = v.y;
}
__device__ __forceinline__ void right_factor(float (&y)[2], const float *m, int lane) {
    y[0] = m[2 * (lane & 3) * kLd + (lane >> 2)];
    y[1] = m[(2 * (lane & 3) + 1) * kLd + (lane >> 2)];
}
__device__ __forceinline__ void store_product(float *m, const float (&d)[3][4], float sign, int lane) {
    *reinterpret_cast<float2 *>(m + (lane >> 2) * kLd + 2 * (lane & 3)) = make_float2(sign * total(d, 0), sign * total(d, 1));
    *reinterpret_cast<float2 *>(m + ((lane >> 2) + 8) * kLd + 2 * (lane & 3)) = make_float2(sign * total(d, 2), sign * total(d, 3));
}

__device__ __forceinline__ void invert_unit_lower(float *a, int warp, int lane) {
    {
        float *m = a + 16 * warp * (kLd + 1);
        float x[16];
        if (lane < 16) {
            #pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = r == lane ? 1.f : 0.f;
            #pragma unroll
            for (int l = 0; l < 16; l += 4) {
                #pragma unroll
                for (int r = l + 1; r < 16; ++r) {
                    const float4 v = *reinterpret_cast<const float4 *>(m + r * kLd + l);
                    x[r] = fmaf(-v.x, x[l], x[r]);
                    if (r > l + 1) x[r] = fmaf(-v.y, x[l + 1], x[r]);
                    if (r > l + 2) x[r] = fmaf(-v.z, x[l + 2], x[r]);
                    if (r > l + 3) x[r] = fmaf(-v.w, x[l + 3], x[r]);
                }
            }
        }
        __syncwarp();
        if (lane < 16) {
            #pragma unroll
            for (int r = 0; r < 16; ++r) m[r * kLd + lane] = x[r];
        }
    }
    __syncthreads();
    {                        // 16 -> 32: pair warp / 2, columns 8 * (warp % 2) ..
        const int b = 32 * (warp >> 1), n = 8 * (warp & 1);
        float m[2][3][4] = {}, d[3][4] = {};
        #pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x[4], y[2];
            left_factor(x, a + (b + 16) * kLd + b + 16 + 8 * k, lane);
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                right_factor(y, a + (b + 16 + 8 * k) * kLd + b + 8 * c, lane);
                mma_fp32(m[c], x, y);
            }
        }
        #pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float x[4] = {total(m[k], 0), total(m[k], 2), total(m[k], 1), total(m[k], 3)};
            float y[2];
            right_factor(y, a + (b + 8 * k) * kLd + b + n, lane);
            mma_fp32(d, x, y);
        }
        __syncthreads();      // both warps of the pair have read A21
        store_product(a + (b + 16) * kLd + b + n, d, -1.f, lane);
    }
    __syncthreads();
    {                        // 32 -> 64: columns 8 * warp .. of both 16-row halves
        float d[2][3][4] = {};
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            float x[4], y[2];
            right_factor(y, a + (32 + 8 * k) * kLd + 8 * warp, lane);
            #pragma unroll
            for (int row = 0; row < 2; ++row) {
                if (k < 2 || row == 1) {       // T22 is lower triangular
                    left_factor(x, a + (32 + 16 * row) * kLd + 32 + 8 * k, lane);
                    mma_fp32(d[row], x, y);
                }
            }
        }
        #pragma unroll
        for (int row = 0; row < 2; ++row) store_product(a + 16 * row * kLd + 32 + 8 * warp, d[row], 1.f, lane);
        __syncthreads();
        float e[2][3][4] = {};
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= 2 || warp < 2) {          // T11 is lower triangular
                float x[4], y[2];
                right_factor(y, a + 8 * k * kLd + 8 * warp, lane);
                #pragma unroll
                for (int row = 0; row < 2; ++row) {
                    left_factor(x, a + 16 * row * kLd + 32 + 8 * k, lane);
                    mma_fp32(e[row], x, y);
                }
            }
        }
        #pragma unroll
        for (int row = 0; row < 2; ++row) store_product(a + (32 + 16 * row) * kLd + 8 * warp, e[row], -1.f, lane);
    }
    __syncthreads();
}


constexpr int kThreads = 128;

template <typename T, bool kBack> struct Prep {
    using S = GdrStage<T, kBack>;
    // what is computed takes the place of K and Q once their product is there: A and its inverse that of T, P its own;
    // the gates lie beside them till the end
    static constexpr uint32_t kTiles = S::kPieces * S::kKqPiece, kGates = kTiles > S::kImage ? kTiles : S::kImage, kBars = kGates + kGateBytes, kBytes = kBars + 64 + 1024;
    static_assert(kChunk * kLd * 4 <= S::kP - S::kT, "A in the place of T and the image's gates");
};

// One CTA makes one chunk of one value head: K K^T and Q K^T by one MMA with the 128 rows [K; Q], then
// warps 0, 1 the rows of A and warps 2, 3 those of P, the inverse, and the image out by one bulk copy.
// A chain of short dependent steps: what fills the SM is that five CTAs share it (bf16).  8192 chunks of
// 128 x 128 take 142 us: 8,300 warp instructions a chunk at 49 % of the issue slots, the rest barriers, waits for
// results and instruction fetches.  (In the walk itself the same steps took 13,000 cycles a chunk.)
template <typename T, int kSteps, bool kBack>
__global__ void __launch_bounds__(kThreads, 5)
gdr_prep_kernel(const __grid_constant__ cc1d_gdr_params p, unsigned char *images) {
    using S = GdrStage<T, kBack>;
    using L = Prep<T, kBack>;
    constexpr int NP = S::kPieces;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    float *inv = reinterpret_cast<float *>(smem);
    GdrGates &gates = *reinterpret_cast<GdrGates *>(smem + L::kGates);
    const uint32_t base = smem_u32(smem), bar = base + L::kBars;
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::kBars + 8);
    uint32_t *slot_at = reinterpret_cast<uint32_t *>(smem + L::kBars + 12);
    const int tid = threadIdx.x, warp = __shfl_sync(kFullMask, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    const int heads = (int)p.heads_v, h = blockIdx.x % heads;
    const int64_t slot = blockIdx.x / heads;
    int n, c;
    GdrSeq seq;
    if (!gdr_find_chunk(p, slot, n, seq, c)) return;      // the whole CTA
    const int t0 = seq.begin + c * kChunk;

    if (tid == 0) { mbar_init(bar, 1); *dead = 0; fence_mbar_init(); }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 64;" :: "r"(smem_u32(slot_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        GateRegs r;
        load_gates(r, p, seq, h, t0, lane);
        store_gates(gates, scan_gates(r, p, lane), lane);
    }
    const GdrRows<T, kThreads> rows(p, seq, h, p.v, 0, 0);
    rows.load_kq(base, t0, tid);
    copy_async_wait();
    fence_proxy_async_smem();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *slot_at;
    if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t id = mma_desc(128, 64, false, false);
            const uint64_t kq = smem_desc(base);
            bool more = false;
            #pragma unroll
            for (int o = 2; o >= 0; --o) {
                #pragma unroll
                for (int a = 0; a <= o; ++a) {
                    const int b = o - a;
                    if (a >= NP || b >= NP) continue;
                    #pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        const uint32_t off = (s >> 2) * S::kPanel + (s & 3) * 32;
                        mma_ss(tmem, desc_add(kq, a * S::kKqPiece + off), desc_add(kq, b * S::kKqPiece + off), id, again(more));
                    }
                }
            }
            mma_commit(bar);
        }
        __syncwarp();
    }
    expand_gates(gates, tid);
    gdr_wait(bar, 0, dead);
    __syncthreads();                   // the gates are there
    fence_after_sync();
    {
        const int first = (warp & 1) * 32, i = first + lane, block = i >> 4;
        const float2 gi = gates.g[i];
        const float scale = (warp < 2 ? gates.beta[i] : 1.f), row = scale * gates.row[i];
        const bool steep = gates.steep != 0;
        const int last = warp < 2 ? i - 1 : i;
        #pragma unroll 1                                 // (unrolled, the code is fetched slower than it runs: 142 us for 130)
        for (int j0 = 0; j0 < kChunk; j0 += 16) {        // columns j0 .. j0 + 15
            float x[16];
            if (j0 > first + 31) {                       // above the diagonal
                if (warp < 2) continue;
                #pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = 0.f;
            } else {
                tmem_ld<16>(x, tmem + ((uint32_t)(warp * 32) << 16) + j0);
                tmem_wait_ld();
                if (j0 + 16 <= first || !steep) {
                    const float *f = (16 * block > j0 ? gates.column[block - 1] : gates.same) + j0;
                    #pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(f + j);
                        x[j] *= row * v.x; x[j + 1] *= row * v.y; x[j + 2] *= row * v.z; x[j + 3] *= row * v.w;
                    }
                } else {
                    #pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float4 f = *reinterpret_cast<const float4 *>(&gates.g[j0 + j]);
                        x[j] *= scale * gdr_fade(gi, make_float2(f.x, f.y));
                        x[j + 1] *= scale * gdr_fade(gi, make_float2(f.z, f.w));
                    }
                }
                if (j0 + 16 > first) {
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = j0 + j <= last ? x[j] : 0.f;
                }
            }
            if (warp < 2) {
                // an infinite or NaN entry would reach the rows before it through products with zeros: its row is noted
                // (the walk cannot see finite keys whose product overflows), and the walk gives NaN to it and those behind.
                // Where the gates between leave nothing (e^-110 is 0) there is no entry, whatever the product; the last of
                // them is the one that they leave most of.
                if (__builtin_expect(!all_finite(x), 0)) {
                    uint32_t out = 0;
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const bool ok = finite(x[j]);
                        out |= ok ? 0u : 1u << j;
                        x[j] = ok ? x[j] : 0.f;
                    }
                    if (out != 0 && !(gi.x - gates.g[j0 + 31 - __clz(out)].x < -110.f)) atomicMin(&gates.bad, i);
                }
                #pragma unroll
                for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4 *>(inv + i * kLd + j0 + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            } else {
                #pragma unroll
                for (int j = 0; j < 16; j += 8) store_pieces8<S::kOut>(x + j, base + (S::kP - S::kT) + tile_at(i, (j0 + j) / 8, 0));
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 64;" :: "r"(tmem) : "memory");
    invert_unit_lower(inv, warp, lane);
    float x[2][16];
    #pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int i = (tid >> 2) + 32 * half, j0 = (tid & 3) * 16;
        #pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 v = j0 <= i ? *reinterpret_cast<const float4 *>(inv + i * kLd + j0 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[half][j] = v.x; x[half][j + 1] = v.y; x[half][j + 2] = v.z; x[half][j + 3] = v.w;
        }
    }
    __syncthreads();                   // the pieces of T go where the inverse lay
    #pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int i = (tid >> 2) + 32 * half, j0 = (tid & 3) * 16;
        #pragma unroll
        for (int j = 0; j < 16; ++j) if (j0 + j == i) x[half][j] = 0.f;      // T - I
        if (!all_finite(x[half])) {
            atomicMin(&gates.bad, i);
            #pragma unroll
            for (int j = 0; j < 16; ++j) x[half][j] = finite(x[half][j]) ? x[half][j] : 0.f;
        }
        #pragma unroll
        for (int j = 0; j < 16; j += 8) store_pieces8<S::kSolve>(x[half] + j, base + tile_at(i, (j0 + j) / 8, 0));
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (kBack && gates.bad < kChunk) {
        // what goes back through an entry that was left out is not finite either: with this factor dB of the chunk, and with it
        // the gradient of every state before, is NaN (and the state behind, as it is in the forward)
        if (tid < kChunk) gates.to_end[tid] = __uint_as_float(0x7fc00000u);
        fence_proxy_async_smem();
        __syncthreads();
    }
    if (tid == 0) {
        unsigned char *image = images + (slot * heads + h) * (int64_t)S::kImage;
        bulk_store(image, base, S::kSolve * 8192);
        bulk_store(image + S::kSolve * 8192, base + L::kGates, kGateBytes);
        bulk_store(image + (S::kP - S::kT), base + (S::kP - S::kT), S::kOut * 8192);
        bulk_commit();
        bulk_wait_read();
    }
}

// ---- segments ----------------------------------------------------------------------------------------
constexpr int kJoinColumns = 16;

// One CTA carries 16 of the dim_v columns of one sequence and value head from segment to segment, in fp32:
// start of the next = M start + B, or, back, end of the one before = M^T end + back.  Thread: one row of the
// result and half of the sum; the matrix is read in the layout whose rows lie along the threads.
__global__ void __launch_bounds__(256) gdr_join_kernel(const __grid_constant__ cc1d_gdr_params p, const GdrSegments segs, const float *dfinal_states, bool back) {
    __shared__ float4 cur[kGdrMaxDim][kJoinColumns / 4], half_sum[kGdrMaxDim][kJoinColumns / 4];
    pdl_wait();
    const int groups = (int)(p.dim_v + kJoinColumns - 1) / kJoinColumns, heads = (int)p.heads_v, dk = (int)p.dim_k, dv = (int)p.dim_v;
    const bool to_back = back && (blockIdx.x & 1);            // back: both directions, every other CTA
    const unsigned id = back ? blockIdx.x >> 1 : blockIdx.x;
    const int col0 = (int)(id % groups) * kJoinColumns, h = (int)(id / groups) % heads, n = (int)(id / groups) / heads;
    const GdrSeq seq = gdr_sequence(p, n);
    const int chunks = gdr_chunks(seq), count = max(1, (chunks + segs.per - 1) / segs.per);
    if (count == 1) return;
    GdrSegment *at = segs.at + gdr_first_segment(p, seq, n, segs.per) * heads + h;
    const int tid = threadIdx.x, row = tid & 127, half = tid >> 7;
    float *flat = reinterpret_cast<float *>(&cur[row][0]);
    if (half == 0) {
        const float *src = nullptr;
        if (to_back) {
            if (dfinal_states != nullptr) src = dfinal_states + ((int64_t)n * heads + h) * dk * dv;
        } else {
            const int64_t r = gdr_state_row(p, n);
            if (p.initial_states != nullptr && r >= 0 && (p.has_initial_state == nullptr || p.has_initial_state[n] != 0))
                src = p.initial_states + r * p.initial_states_batch_stride + h * p.initial_states_h_stride;
        }
        for (int c = 0; c < kJoinColumns; ++c) flat[c] = src != nullptr && row < dk && col0 + c < dv ? src[(int64_t)row * dv + col0 + c] : 0.f;
        if (!to_back) {
            for (int c = 0; c < kJoinColumns; ++c) at->start[row][col0 + c] = flat[c];
        }
    }
    __syncthreads();
    for (int i = 0; i + 1 < count; ++i) {
        GdrSegment &s = at[(int64_t)(to_back ? count - 1 - i : i) * heads];
        const float(*m)[kGdrMaxDim] = to_back ? s.M : s.Mt;
        float4 sum[kJoinColumns / 4];
        #pragma unroll
        for (int c = 0; c < kJoinColumns / 4; ++c)
            sum[c] = half == 0 ? *reinterpret_cast<const float4 *>(&(to_back ? s.back : s.B)[row][col0 + 4 * c]) : make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll 8
        for (int k = 64 * half; k < 64 * half + 64; ++k) {
            const float f = m[k][row];
            #pragma unroll
            for (int c = 0; c < kJoinColumns / 4; ++c) {
                const float4 v = cur[k][c];
                sum[c].x = fmaf(f, v.x, sum[c].x); sum[c].y = fmaf(f, v.y, sum[c].y); sum[c].z = fmaf(f, v.z, sum[c].z); sum[c].w = fmaf(f, v.w, sum[c].w);
            }
        }
        if (half == 1) {
            #pragma unroll
            for (int c = 0; c < kJoinColumns / 4; ++c) half_sum[row][c] = sum[c];
        }
        __syncthreads();
        if (half == 0) {
            GdrSegment &next = at[(int64_t)(to_back ? count - 2 - i : i + 1) * heads];
            #pragma unroll
            for (int c = 0; c < kJoinColumns / 4; ++c) {
                const float4 v = half_sum[row][c];
                sum[c].x += v.x; sum[c].y += v.y; sum[c].z += v.z; sum[c].w += v.w;
                cur[row][c] = sum[c];
                *reinterpret_cast<float4 *>(&(to_back ? next.end : next.start)[row][col0 + 4 * c]) = sum[c];
            }
        }
        __syncthreads();
    }
}

}  // namespace

// Times in us of a walk's chunk and of a join's step (measured, bf16, 128 x 128), for sequences of the mean length;
// `back`: of the backward's walks as launches of their own.  (In the one launch that they share now a chunk takes 6.3
// to 6.8, so the rule cuts a little less often than it could; and one long sequence among many short ones is not cut.)
// Cut where that is expected to save a quarter: one sequence of 32768 tokens and 4 heads, for example, is one
// wave of 37 segments a head instead of 4 chains of 512 chunks.
int gdr_plan_segments(const cc1d_gdr_params &p, bool back) {
    const int64_t n = gdr_sequences(p), slots = gdr_slots(p);
    if (n == 0 || slots == 0) return 0;
    const int64_t mean = (slots + n - 1) / n, sms = num_sms(), heads = n * p.heads_v;
    if (heads >= sms || mean < 8) return 0;
    const int walks = back ? 2 : 1, sums = back ? 3 : 2;
    const auto waves = [&](int64_t ctas) { return (double)((ctas + sms - 1) / sms); };
    const double chunk = back ? 4.6 : 4.0, sum_chunk = back ? 4.2 : 3.6, step = 3.0, launches = 8.0;
    double best = 0.75 * waves(walks * heads) * (double)mean * chunk;
    int per = 0;
    for (int64_t count = 2; count <= 64 && count * 2 <= mean; ++count) {
        const int64_t m = (mean + count - 1) / count, segments = (mean + m - 1) / m;
        const double t = launches + waves(sums * heads * (segments - 1)) * (double)m * sum_chunk + step * (double)segments + waves(walks * heads * segments) * (double)m * chunk;
        if (t < best) { best = t; per = (int)m; }
    }
    return per;
}

int launch_gdr_join(const cc1d_gdr_params &p, const GdrSegments &segs, const float *dfinal_states, bool back, cudaStream_t stream) {
    const int64_t ctas = gdr_sequences(p) * p.heads_v * ((p.dim_v + kJoinColumns - 1) / kJoinColumns) * (back ? 2 : 1);
    if (ctas >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    launch_k(gdr_join_kernel, dim3((unsigned)ctas), dim3(256), 0, stream, p, segs, dfinal_states, back);
    return check_launch();
}

size_t gdr_image_bytes(const cc1d_gdr_params &p, bool back) {
    size_t one = 0;
    CC1D_DISPATCH_ITYPE(p.itype, { one = back ? GdrStage<T, true>::kImage : GdrStage<T, false>::kImage; });
    return one * (size_t)gdr_slots(p) * (size_t)p.heads_v;
}

int launch_gdr_prep(const cc1d_gdr_params &p, bool back, void *images, cudaStream_t stream) {
    const int64_t ctas = gdr_slots(p) * p.heads_v;
    if (ctas == 0) return CC1D_OK;
    if (ctas >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    CC1D_DISPATCH_ITYPE(p.itype, {
        CC1D_DISPATCH_BOOL(p.dim_k <= 64, kNarrow, {
            CC1D_DISPATCH_BOOL(back, kBack, {
                constexpr int kSteps = kNarrow ? 4 : 8;     // contraction steps of 16 over dim_k
                constexpr uint32_t kBytes = Prep<T, kBack>::kBytes;
                allow_dynamic_smem(reinterpret_cast<const void *>(gdr_prep_kernel<T, kSteps, kBack>), kBytes);
                launch_k(gdr_prep_kernel<T, kSteps, kBack>, dim3((unsigned)ctas), dim3(kThreads), kBytes, stream, p, reinterpret_cast<unsigned char *>(images));
            });
        });
    });
    return check_launch();
}

int gdr_prep_wait_expired() { return read_and_clear_wait_expired(); }

}  // namespace cc1d
