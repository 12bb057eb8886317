// Gradients of the gated delta rule: cc1d_gdr_bwd (include/cc1d_gdr.h).  Three launches:
//   gdr_prep_kernel       T, P and the gates of every chunk (as in the forward)
//   gdr_bwd_walks_kernel  half of the CTAs walk forwards again and leave the state before each chunk and U, half
//                         walk from the last chunk to the first and leave the state's gradient and dB (neither
//                         needs the other: one after the other they took 287 + 312 us where 64 CTAs of each
//                         fit the SMs together)
//   gdr_grads_kernel      all other gradients, every chunk by itself
#include "cc1d_gdr_walk.cuh"

namespace cc1d {
namespace {

// ---- the walk backwards -------------------------------------------------------------------------
// warps 0-15 walk, 16 issues their products, 17 does nothing, 18, 19 load

constexpr uint32_t kColS = 0;      // 3 x 64: pieces of dS^T; later in a chunk
constexpr uint32_t kColDelta = 0;  //   128: E^T Q + F^T K
constexpr uint32_t kColX = 192;    // 64: dS^T K^T, then dU^T (T - I)
constexpr uint32_t kColA = 256;    // 64: dO^T P
constexpr uint32_t kColF = 320;    // 3 x 32: pieces of dU^T, then of F^T = (-beta e^G dB)^T
constexpr uint32_t kColE = 416;    // 3 x 32: pieces of E^T = (scale e^G dO)^T

template <typename T> struct Back {
    using S = GdrStage<T, true>;
    static constexpr int kStages = S::kPieces == 1 ? 2 : 1;
    static constexpr uint32_t kDoPiece = 16384, kDo = S::kPieces * S::kKqPiece, kT = kDo + S::kPieces * kDoPiece, kGates = kT + (S::kGates - S::kT),
                              kP = kT + (S::kP - S::kT), kStage = kT + S::kImage;
    static constexpr uint32_t kBars = kStages * kStage, kBytes = kBars + 128 + sizeof(GdrPart) + 1024;
    static_assert(kBytes <= 232448, "shared memory of a CTA");
};

// One CTA walks one sequence of one value head from its end, with dS^T (dim_v x dim_k) in registers:
//   dU = scale P^T dO + e^{G_C - G} K dS        dB = dU + (T - I)^T dU
//   dS <- e^{G_C} dS + scale (e^G Q)^T dO - (beta e^G K)^T dB
// Same division of work and same precision as the forward walk; P^T dO and Q^T E do not wait for the
// walk and run beside its arithmetic.
// kSum: a segment from zeros, its last gradient only.
template <typename T, int kSteps, bool kSum>
__device__ __forceinline__ void walk_back(const cc1d_gdr_bwd_params &b, const unsigned char *images, GdrRecord *records, const GdrSegments &segs, int64_t block) {
    using L = Back<T>;
    using St = GdrStage<T, true>;
    constexpr int NP = St::kPieces, PO = St::kOut, PT = St::kSolve;
    const cc1d_gdr_params &p = b.fwd;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t bars = smem_u32(smem + L::kBars);
    const uint32_t bar_full = bars, bar_empty = bars + 16, bar_x = bars + 32, bar_u = bars + 40, bar_d = bars + 48, bar_s = bars + 56, bar_e = bars + 64,
                   bar_r = bars + 72, bar_w = bars + 80;
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::kBars + 96);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 100);
    const int tid = threadIdx.x, warp = __shfl_sync(kFullMask, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    const int heads = (int)p.heads_v, h = (int)(block % heads), sequences = (int)gdr_sequences(p);
    GdrPart w;
    if (!gdr_find_part(p, segs, segs.ranked ? gdr_ranked(p, (int)(block / heads), reinterpret_cast<int *>(smem)) : block / heads, w) || (kSum && w.first)) return;
    const GdrSeq seq = w.seq;
    const int n = w.n, chunks = w.chunks, dk = (int)p.dim_k, dv = (int)p.dim_v;
    const int64_t first_slot = w.slot;
    // what the walkers need again at their end (kept in registers over the walk it makes them spill)
    volatile GdrPart *kept = reinterpret_cast<volatile GdrPart *>(smem + L::kBars + 128);
    if (tid == 0) {
        kept->n = w.n; kept->seq.begin = w.seq.begin; kept->seq.end = w.seq.end; kept->segment = w.segment; kept->first = w.first; kept->last = w.last;
        for (int s = 0; s < 2; ++s) { mbar_init(bar_full + 8 * s, kFeeders + 1); mbar_init(bar_empty + 8 * s, kWalkers / 32); }
        mbar_init(bar_x, 1); mbar_init(bar_u, 1); mbar_init(bar_d, 1);
        mbar_init(bar_s, kWalkers / 32); mbar_init(bar_e, kWalkers / 32); mbar_init(bar_r, kWalkers / 32); mbar_init(bar_w, kWalkers / 32);
        *dead = 0;
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc512(smem_u32(slot));
    fence_before_sync();
    __syncthreads();
    fence_after_sync();

    if (warp == kWalkers / 32) {
        for (int i = 0; i < chunks; ++i) {
            const int s = i % L::kStages;
            const uint32_t par = i & 1;
            const uint32_t stage = smem_u32(smem) + s * L::kStage;
            const uint64_t kq = smem_desc(stage), kmn = smem_desc(stage, St::kPanel), dout = smem_desc(stage + L::kDo, 8192);
            constexpr uint32_t id = mma_desc(128, 64, false, false), id_mn = mma_desc(128, 64, false, true), id_mm = mma_desc(128, 64, true, true),
                               idd = mma_desc(128, 128, false, true);
            gdr_wait(bar_full + 8 * s, (i / L::kStages) & 1, dead);
            gdr_wait(bar_s, par, dead);
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = 2; o >= 0; --o) {          // dS^T K^T
                    #pragma unroll
                    for (int x = 0; x <= o; ++x) {
                        const int y = o - x;
                        if (x >= 3 || y >= NP) continue;
                        #pragma unroll
                        for (int k = 0; k < kSteps; ++k)
                            mma_ts(kColX, kColS + 64 * x + 8 * k, desc_add(kq, y * St::kKqPiece + (k >> 2) * St::kPanel + (k & 3) * 32), id, again(more));
                    }
                }
                more = false;
                #pragma unroll
                for (int o = PO - 1; o >= 0; --o) {         // dO^T P, both with the tokens as the slow index
                    #pragma unroll
                    for (int x = 0; x <= o; ++x) {
                        const int y = o - x;
                        if (x >= NP || y >= PO) continue;
                        #pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ss(kColA, desc_add(dout, x * L::kDoPiece + 2048 * k), desc_add(kq, L::kP + y * 8192 + 2048 * k), id_mm, again(more));
                    }
                }
                mma_commit(bar_x);
            }
            __syncwarp();
            gdr_wait(bar_e, par, dead);
            gdr_wait(bar_x, par, dead);                // the columns of dS^T are free for Delta
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = 2; o >= 0; --o) {          // E^T Q
                    #pragma unroll
                    for (int x = 0; x <= o; ++x) {
                        const int y = o - x;
                        if (x >= 3 || y >= NP) continue;
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) mma_ts(kColDelta, kColE + 32 * x + 8 * k, desc_add(kmn, y * St::kKqPiece + 64 * 128 + 2048 * k), idd, again(more));
                    }
                }
            }
            __syncwarp();
            gdr_wait(bar_r, par, dead);
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = PT - 1; o >= 0; --o) {         // dU^T (T - I)
                    #pragma unroll
                    for (int x = 0; x <= o; ++x) {
                        const int y = o - x;
                        if (x >= PT || y >= PT) continue;
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) mma_ts(kColX, kColF + 32 * x + 8 * k, desc_add(kq, L::kT + y * 8192 + 2048 * k), id_mn, again(more));
                    }
                }
                mma_commit(bar_u);
            }
            __syncwarp();
            gdr_wait(bar_w, par, dead);
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                #pragma unroll
                for (int o = 2; o >= 0; --o) {          // + F^T K
                    #pragma unroll
                    for (int x = 0; x <= o; ++x) {
                        const int y = o - x;
                        if (x >= 3 || y >= NP) continue;
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) mma_ts(kColDelta, kColF + 32 * x + 8 * k, desc_add(kmn, y * St::kKqPiece + 2048 * k), idd, true);
                    }
                }
                mma_commit(bar_d);
            }
            __syncwarp();
        }
    } else if (warp > kWalkers / 32 + 1) {
        const int ft = tid - kWalkers - 64;
        const T *dout = reinterpret_cast<const T *>(b.dout) + seq.row * b.dout_batch_stride + h * b.dout_h_stride;
        const GdrRows<T, kFeeders> rows(p, seq, h, dout, 0, b.dout_l_stride);
        const int64_t step = (int64_t)heads * St::kImage;
        const unsigned char *image = images + first_slot * step + h * (int64_t)St::kImage;
        for (int i = 0; i < chunks; ++i) {
            const int s = i % L::kStages, c = chunks - 1 - i;
            const uint32_t stage = smem_u32(smem) + s * L::kStage, full = bar_full + 8 * s;
            gdr_wait(bar_empty + 8 * s, ((i / L::kStages) & 1) ^ 1, dead);
            if (ft == 0) {
                mbar_expect_tx(full, St::kImage);
                bulk_load(stage + L::kT, image + c * step, St::kImage, full);
            }
            rows.load_kq(stage, seq.begin + c * kChunk, ft);
            load_tile<T, NP, kFeeders>(stage + L::kDo, 8192, L::kDoPiece, dout, b.dout_l_stride, seq.begin + c * kChunk, seq.end, dv, ft);
            copy_async_wait();
            fence_proxy_async_smem();
            mbar_arrive(full);
        }
    } else if (warp < kWalkers / 32) {
        const int quad = warp & 3, part = warp >> 2, col = quad * 32 + lane;   // part: a quarter of the dim_k and of the tokens
        const uint32_t mine = (uint32_t)(quad * 32) << 16;
        float S[32];
        {
            const int64_t state_at = ((int64_t)n * heads + h) * dk * dv + (int64_t)(32 * part) * dv + col;
            #pragma unroll
            for (int j = 0; j < 32; ++j)
                S[j] = kSum || 32 * part + j >= dk || col >= dv ? 0.f : !w.last ? w.segment[h].end[32 * part + j][col]
                     : b.dfinal_states != nullptr && n < sequences ? b.dfinal_states[state_at + (int64_t)j * dv] : 0.f;
        }
        auto ready = [&](uint32_t bar) {
            tmem_wait_st();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        GdrRecord *record = records + (first_slot + chunks - 1) * heads + h;
        auto put_state = [&]() {
            if (!kSum) {
                #pragma unroll
                for (int j = 0; j < 32; ++j) record->dS[32 * part + j][col] = S[j];
            }
            #pragma unroll
            for (int i = 0; i < 4; ++i) split8_to_tmem<3>(S + 8 * i, mine + kColS + 16 * part + 4 * i, 64, 128);
            ready(bar_s);
        };
        if (chunks > 0) put_state();
        const int first = 16 * part;               // this thread's tokens of a chunk: first .. first + 15
        for (int i = 0; i < chunks; ++i) {
            const int s = i % L::kStages;
            const uint32_t par = i & 1;
            const unsigned char *stage = smem + s * L::kStage;
            const GdrGates &gates = *reinterpret_cast<const GdrGates *>(stage + L::kGates);
            gdr_wait(bar_full + 8 * s, (i / L::kStages) & 1, dead);
            #pragma unroll
            for (int j = 0; j < 16; j += 8) {      // E
                float x[8];
                #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const unsigned char *at = stage + L::kDo + tile_at(first + j + k, col / 8, 8192) + (col & 7) * 2;
                    x[k] = 0.f;
                    #pragma unroll
                    for (int q = NP - 1; q >= 0; --q) x[k] += Elem<__nv_bfloat16>::to_f(*reinterpret_cast<const __nv_bfloat16 *>(at + q * L::kDoPiece));
                    x[k] *= p.scale * gates.from_start[first + j + k];
                }
                split8_to_tmem<3>(x, mine + kColE + first / 2 + j / 2, 32, 64);
            }
            ready(bar_e);
            gdr_wait(bar_x, par, dead);
            __syncwarp();
            fence_after_sync();
            float R[16];
            #pragma unroll
            for (int j = 0; j < 16; j += 8) {      // dU
                float x[8], y[8];
                tmem_ld<8>(x, mine + kColX + first + j);
                tmem_ld<8>(y, mine + kColA + first + j);
                tmem_wait_ld();
                #pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(gates.to_end + first + j + k);
                    R[j + k] = fmaf(f.x, x[k], p.scale * y[k]); R[j + k + 1] = fmaf(f.y, x[k + 1], p.scale * y[k + 1]);
                    R[j + k + 2] = fmaf(f.z, x[k + 2], p.scale * y[k + 2]); R[j + k + 3] = fmaf(f.w, x[k + 3], p.scale * y[k + 3]);
                }
                split8_to_tmem<PT>(R + j, mine + kColF + first / 2 + j / 2, 32, 64);
            }
            ready(bar_r);
            gdr_wait(bar_u, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int j = 0; j < 16; j += 8) {      // dB and F
                float x[8];
                tmem_ld<8>(x, mine + kColX + first + j);
                tmem_wait_ld();
                #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] += R[j + k];
                    if (!kSum) record->dB[first + j + k][col] = x[k];
                    x[k] *= gates.minus_beta_from_start[first + j + k];
                }
                split8_to_tmem<3>(x, mine + kColF + first / 2 + j / 2, 32, 64);
            }
            ready(bar_w);
            record -= heads;
            const float whole = gates.from_start[kChunk - 1];
            gdr_wait(bar_d, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int j = 0; j < 32; j += 16) {
                float x[16];
                tmem_ld<16>(x, mine + kColDelta + 32 * part + j);
                tmem_wait_ld();
                #pragma unroll
                for (int k = 0; k < 16; ++k) S[j + k] = fmaf(whole, S[j + k], x[k]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + 8 * s);
            fence_before_sync();
            walk_sync<kWalkers>();                 // every thread has read its part of Delta
            fence_after_sync();
            if (i + 1 < chunks) put_state();
        }
        const int head = (int)(block % heads), at = kept->n, all = (int)gdr_sequences(p);
        if (kSum) {
            GdrSegment &to = kept->segment[head];
            #pragma unroll
            for (int j = 0; j < 32; ++j) to.back[32 * part + j][col] = S[j];
        }
        if (!kSum && kept->first && b.dinitial_states != nullptr && at < all) {
            const int64_t state_at = ((int64_t)at * heads + head) * dk * dv + (int64_t)(32 * part) * dv + col;
            const bool from = p.initial_states != nullptr && gdr_state_row(p, at) >= 0 && (p.has_initial_state == nullptr || p.has_initial_state[at] != 0);
            #pragma unroll
            for (int j = 0; j < 32; ++j)
                if (32 * part + j < dk && col < dv) b.dinitial_states[state_at + (int64_t)j * dv] = from ? S[j] : 0.f;
        }
        if (!kSum && p.cu_seqlens != nullptr) {
            const int group = heads / (int)p.heads_k;
            unowned_tokens(p, kept, part, [&](int64_t t) {
                if (col < dv) reinterpret_cast<T *>(b.dv)[(t * heads + head) * dv + col] = Elem<T>::from_f(0.f);
                if (head % group == 0 && col < dk) {
                    reinterpret_cast<T *>(b.dq)[(t * p.heads_k + head / group) * dk + col] = Elem<T>::from_f(0.f);
                    reinterpret_cast<T *>(b.dk)[(t * p.heads_k + head / group) * dk + col] = Elem<T>::from_f(0.f);
                }
                if (col == 0) {
                    store_any(b.dg, t * heads + head, p.gtype, 0.f);
                    store_any(b.dbeta, t * heads + head, p.btype, 0.f);
                }
            });
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_free512();
}

template <typename T, int kSteps>
__global__ void __launch_bounds__(kWalkThreads, 1) gdr_bwd_walks_kernel(const __grid_constant__ cc1d_gdr_bwd_params b, const unsigned char *images, GdrRecord *records, const GdrSegments segs) {
    if (blockIdx.x & 1) walk_forward<T, kSteps, kKeep, true>(b.fwd, images, records, segs, blockIdx.x >> 1, false);
    else walk_back<T, kSteps, false>(b, images, records, segs, blockIdx.x >> 1);
}

// a third of the CTAs each: the gradient's walk from zeros, the state's, M
template <typename T, int kSteps>
__global__ void __launch_bounds__(kWalkThreads, 1) gdr_bwd_summary_kernel(const __grid_constant__ cc1d_gdr_bwd_params b, const unsigned char *images, const GdrSegments segs, unsigned walks) {
    if (blockIdx.x < walks) {
        walk_back<T, kSteps, true>(b, images, nullptr, segs, blockIdx.x);
    } else {
        const unsigned block = blockIdx.x - walks;
        const bool unit = block >= walks;
        walk_forward<T, kSteps, kSummary, true>(b.fwd, images, nullptr, segs, unit ? block - walks : block, unit);
    }
}

// ---- everything else, chunk by chunk --------------------------------------------------------------
constexpr int kGradThreads = 512;

// Tensor memory: lanes 0-63 the rows of q (and dO), lanes 64-127 those of k (and dB).
constexpr uint32_t kColG = 0;      // 128: dO S0^T | dB S0^T, later M_P K | M_A K
constexpr uint32_t kColPa = 128;   // 64: dO U^T | dB U^T
constexpr uint32_t kColQk = 192;   // 64: Q K^T | K K^T
constexpr uint32_t kColU = 256;    // 128: - | U dS^T, later - | M_P^T Q + M_A^T K

template <typename T> struct Grads {
    using S = GdrStage<T, true>;
    static constexpr int NP = S::kPieces;
    // three pieces in every type: the gradient of g, fp32 as a rule, is a difference of larger sums
    static constexpr int NB = 3;
    // dS has a place of its own where that fits (else that of [dO; dB], when their products are done)
    static constexpr bool kOwnDs = NP == 1;
    static constexpr uint32_t kKq = 0, kA = NP * S::kKqPiece, kAPiece = 16384, kB = kA + NB * kAPiece, kBPiece = 192 * 128,
                              kDs = kOwnDs ? kB + NB * kBPiece : kA, kGates = kB + NB * kBPiece + (kOwnDs ? NB * kAPiece : 0),
                              kDots = kGates + kGateBytes, kBars = kDots + 3 * 4 * 128 * 4, kBytes = kBars + 64 + 1024;
    static_assert(kBytes <= 232448, "shared memory of a CTA");
};

// 8 fp32 values -> kPieces vectors of a tile
template <int kPieces> __device__ __forceinline__ void put8(const float (&x)[8], uint32_t at, uint32_t piece_bytes) {
    uint32_t r[4][kPieces];
    #pragma unroll
    for (int i = 0; i < 4; ++i) split_pair<kPieces>(make_float2(x[2 * i], x[2 * i + 1]), r[i]);
    #pragma unroll
    for (int k = 0; k < kPieces; ++k) sts128(at + k * piece_bytes, make_uint4(r[0][k], r[1][k], r[2][k], r[3][k]));
}
__device__ __forceinline__ void get8(float (&x)[8], const float *src) {
    const float4 u = *reinterpret_cast<const float4 *>(src), v = *reinterpret_cast<const float4 *>(src + 4);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}
template <typename T> __device__ __forceinline__ void store8(T *dst, const float *x) {
    *reinterpret_cast<uint4 *>(dst) = pack<T>(x);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(dst + 4) = pack<T>(x + 4);
}
// One CTA: one chunk of one key head, the value heads of its group one after the other (so dq and dk are
// summed in registers in a fixed order).  With the rows [dO; dB] and [Q; K] stacked to 128:
//   [dO; dB] [S0; U]^T -> dO S0^T, dB S0^T, dP = dO U^T, -dA = dB U^T      [Q; K] K^T      U dS^T
//   M_P = scale dP e^{Gi - Gj} (j <= i), M_A = beta dA e^{Gi - Gj} (j < i)
//   dQ = scale e^G dO S0^T + M_P K
//   dK = -beta e^G dB S0^T + e^{G_C - G} U dS^T + M_A K + [M_P; M_A]^T [Q; K]
//   dbeta = dB.V - e^G k.(dB S0^T) + sum_j t_ij,  t = dA (k_i.k_j) e^{Gi - Gj}
//   dG = q.dQ - beta e^G k.(dB S0^T) + beta sum_j t_ij - k.(e^{G_C - G} U dS^T) - k.([M_P; M_A]^T [Q; K])
//        (what q and k see of G they see through their own products, with the sign of their place in e^{Gi - Gj}), and
//        at the chunk's end + sum k.(e^{G_C - G} U dS^T) + e^{G_C} <S0, dS>;
//   dg is its sum from the chunk's end.
// U dS^T has a barrier of its own: dS is split while the first product runs, and the next panel's [dO; dB] and
// S0, or the tile below, are made while it runs itself (training step 2 x 4096 x 32 heads 1355 -> 1311 us).
// Bound by its chain of phases: about 33,000 cycles a head and chunk (one CTA an SM, 215 KB), 12,500 of them
// products; its record, 192 KB a head and chunk written by the walks and read here, is 1.5 TB/s.
// [M_P; M_A] is one tile of shared memory: rows as the contraction's results for the products with K, and
// (read with its rows as the contraction) its own transpose for those with [Q; K].
template <typename T, int kSteps>
__global__ void __launch_bounds__(kGradThreads, 1) gdr_grads_kernel(const __grid_constant__ cc1d_gdr_bwd_params b, const unsigned char *images, const GdrRecord *records) {
    using L = Grads<T>;
    using S = GdrStage<T, true>;
    constexpr int NP = L::NP, NB = L::NB;
    const cc1d_gdr_params &p = b.fwd;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t base = smem_u32(smem), bar = base + L::kBars, bar_state = bar + 8;
    const GdrGates &gates = *reinterpret_cast<const GdrGates *>(smem + L::kGates);
    float(*dots)[4][128] = reinterpret_cast<float(*)[4][128]>(smem + L::kDots);
    // first token whose gradients of q, k, g and beta are NaN, of a head and of the group (a place that no sum takes)
    int *bad = reinterpret_cast<int *>(&dots[2][2][0]);
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::kBars + 16);
    uint32_t *tmem_at = reinterpret_cast<uint32_t *>(smem + L::kBars + 20);
    const int tid = threadIdx.x, warp = __shfl_sync(kFullMask, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    const int heads = (int)p.heads_v, heads_k = (int)p.heads_k, hk = blockIdx.x % heads_k, group = heads / heads_k;
    const int64_t slot = blockIdx.x / heads_k;
    int n, c;
    GdrSeq seq;
    if (!gdr_find_chunk(p, slot, n, seq, c)) return;      // the whole CTA
    const int t0 = seq.begin + c * kChunk, dk = (int)p.dim_k, dv = (int)p.dim_v;
    if (tid == 0) { mbar_init(bar, 1); mbar_init(bar_state, 1); *dead = 0; fence_mbar_init(); }
    if (warp == 0) tmem_alloc512(smem_u32(tmem_at));
    {   // rows 0-63 q, 64-127 k
        const T *kp = reinterpret_cast<const T *>(p.k) + seq.row * p.k_batch_stride + hk * p.k_h_stride;
        const T *qp = reinterpret_cast<const T *>(p.q) + seq.row * p.q_batch_stride + hk * p.q_h_stride;
        load_tile<T, NP, kGradThreads>(base + L::kKq, S::kPanel, S::kKqPiece, qp, p.q_l_stride, t0, seq.end, dk, tid);
        load_tile<T, NP, kGradThreads>(base + L::kKq + 64 * 128, S::kPanel, S::kKqPiece, kp, p.k_l_stride, t0, seq.end, dk, tid);
        copy_async_wait();
    }
    const int quad = warp & 3, part = warp >> 2;           // part: a quarter of the columns
    const bool is_k = quad >= 2;
    const int first = (quad & 1) * 32, i = first + lane;   // this thread's token (as q or as k)
    const uint32_t mine = (uint32_t)(quad * 32) << 16;
    const int panels = dv > 64 ? 2 : 1;
    uint32_t parity = 0, parity_state = 0;
    auto wait_mma = [&]() {
        gdr_wait(bar, parity, dead);
        parity ^= 1;
        __syncwarp();
        fence_after_sync();
    };
    auto wait_state = [&]() {                              // for U dS^T, which has a barrier of its own
        gdr_wait(bar_state, parity_state, dead);
        parity_state ^= 1;
        __syncwarp();
        fence_after_sync();
    };
    auto smem_written = [&]() {
        fence_proxy_async_smem();
        fence_before_sync();
        __syncthreads();
    };
    float total[32];
    #pragma unroll
    for (int j = 0; j < 32; ++j) total[j] = 0.f;

    for (int h = hk * group; h < (hk + 1) * group; ++h) {
        const GdrRecord &record = records[slot * heads + h];
        if (tid < (int)kGateBytes / 16) {
            const uint4 *src = reinterpret_cast<const uint4 *>(images + (slot * heads + h) * (int64_t)S::kImage + S::kGates - S::kT);
            sts128(base + L::kGates + 16 * tid, src[tid]);
        } else if (tid == kGradThreads - 1) {
            const int4 v = *reinterpret_cast<const int4 *>(record.bad);
            bad[0] = min(min(v.x, v.y), min(v.z, v.w));
            bad[1] = h == hk * group ? bad[0] : min(bad[0], bad[1]);
        }
        __syncthreads();
        const T *dout = reinterpret_cast<const T *>(b.dout) + seq.row * b.dout_batch_stride + h * b.dout_h_stride;
        const T *v = reinterpret_cast<const T *>(p.v) + seq.row * p.v_batch_stride + h * p.v_h_stride;
        float state_dot = 0.f, value_dot = 0.f;
        // a panel: 64 of the dim_v; this thread: 8 of them, of token `row` and of the rows `row` and 64 + `row` of the states
        const int row = tid >> 3, c16 = tid & 7;
        const int64_t t = t0 + row;
        uint4 do_raw[sizeof(T) / 2], v_raw[sizeof(T) / 2];
        float d_b[8], u[8], s0[2][8], ds[2][8];
        auto ask = [&](int at) {
            const bool ok = t < seq.end && at < dv;
            load_row<T>(dout + t * b.dout_l_stride + at, ok, do_raw);
            load_row<T>(v + t * p.v_l_stride + at, ok, v_raw);
            get8(d_b, &record.dB[row][at]);
            get8(u, &record.U[row][at]);
            #pragma unroll
            for (int r = 0; r < 2; ++r) get8(s0[r], &record.S0[row + 64 * r][at]);
        };
        auto ask_ds = [&](int at) {
            #pragma unroll
            for (int r = 0; r < 2; ++r) get8(ds[r], &record.dS[row + 64 * r][at]);
        };
        ask(8 * c16);
        ask_ds(8 * c16);
        for (int q = 0; q < panels; ++q) {
            const int at = 64 * q + 8 * c16;
            float x[8], y[8];
            unpack<T>(do_raw[0], x); unpack<T>(v_raw[0], y);
            if constexpr (sizeof(T) == 4) { unpack<T>(do_raw[1], x + 4); unpack<T>(v_raw[1], y + 4); }
            put8<NB>(x, base + L::kA + tile_at(row, c16, 0), L::kAPiece);
            put8<NB>(d_b, base + L::kA + tile_at(64 + row, c16, 0), L::kAPiece);
            #pragma unroll
            for (int j = 0; j < 8; ++j) { value_dot = fmaf(d_b[j], y[j], value_dot); x[j] = gates.beta[row] * d_b[j]; }
            if (t < seq.end && at < dv) store8<T>(reinterpret_cast<T *>(b.dv) + ((seq.row * p.seqlen + t) * heads + h) * dv + at, x);
            #pragma unroll
            for (int r = 0; r < 2; ++r) {
                put8<NB>(s0[r], base + L::kB + tile_at(row + 64 * r, c16, 0), L::kBPiece);
                #pragma unroll
                for (int j = 0; j < 8; ++j) state_dot = fmaf(s0[r][j], ds[r][j], state_dot);
            }
            if (L::kOwnDs && q > 0) wait_state();        // of the last panel's U and dS only now
            put8<NB>(u, base + L::kB + tile_at(128 + row, c16, 0), L::kBPiece);
            smem_written();
            if (warp == 0) {
                if (elect_one()) {
                    fence_after_sync();
                    constexpr uint32_t id = mma_desc(128, 192, false, false), idq = mma_desc(128, 64, false, false);
                    const uint64_t a = smem_desc(base + L::kA), bb = smem_desc(base + L::kB), kq = smem_desc(base + L::kKq);
                    bool more = q > 0;
                    #pragma unroll
                    for (int o = NB - 1; o >= 0; --o) {
                        #pragma unroll
                        for (int m = 0; m <= o; ++m) {
                            #pragma unroll
                            for (int s = 0; s < 4; ++s) mma_ss(kColG, desc_add(a, m * L::kAPiece + 32 * s), desc_add(bb, (o - m) * L::kBPiece + 32 * s), id, again(more));
                        }
                    }
                    if (q == 0 && h == hk * group) {
                        more = false;
                        #pragma unroll
                        for (int o = 2; o >= 0; --o) {
                            #pragma unroll
                            for (int m = 0; m <= o; ++m) {
                                if (m >= NP || o - m >= NP) continue;
                                #pragma unroll
                                for (int s = 0; s < kSteps; ++s) {
                                    const uint32_t off = (s >> 2) * S::kPanel + (s & 3) * 32;
                                    mma_ss(kColQk, desc_add(kq, m * S::kKqPiece + off), desc_add(kq, (o - m) * S::kKqPiece + 64 * 128 + off), idq, again(more));
                                }
                            }
                        }
                    }
                    mma_commit(bar);
                }
                __syncwarp();
            }
            if (q + 1 < panels) ask(at + 64);            // the next panel's loads pass under this one's products
            if constexpr (!L::kOwnDs) wait_mma();
            #pragma unroll
            for (int r = 0; r < 2; ++r) put8<NB>(ds[r], base + L::kDs + tile_at(row + 64 * r, c16, 0), L::kAPiece);
            if (q + 1 < panels) ask_ds(at + 64);
            smem_written();
            if (warp == 0) {
                if (elect_one()) {
                    fence_after_sync();
                    constexpr uint32_t id = mma_desc(128, 128, false, false);
                    // rows 64-191 of [S0; U]: the upper half of the result is U dS^T, the lower one is not used (and the next
                    // panel's S0 may be on its way into its rows)
                    const uint64_t up = smem_desc(base + L::kB + 64 * 128), d = smem_desc(base + L::kDs);
                    bool more = q > 0;
                    #pragma unroll
                    for (int o = NB - 1; o >= 0; --o) {
                        #pragma unroll
                        for (int m = 0; m <= o; ++m) {
                            #pragma unroll
                            for (int s = 0; s < 4; ++s) mma_ss(kColU, desc_add(up, m * L::kBPiece + 32 * s), desc_add(d, (o - m) * L::kAPiece + 32 * s), id, again(more));
                        }
                    }
                    mma_commit(bar_state);
                }
                __syncwarp();
            }
            if constexpr (L::kOwnDs) wait_mma();
            else wait_state();
        }
        if (h + 1 < (hk + 1) * group) {
            // the next head's record into L2, two lines a thread (in registers it would spill)
            const char *next = reinterpret_cast<const char *>(&records[slot * heads + h + 1]);
            for (uint32_t at = tid * 128; at < sizeof(GdrRecord); at += kGradThreads * 128) asm volatile("prefetch.global.L2 [%0];" :: "l"(next + at));
        }
        // row sums whose threads are not those of the rows below
        #pragma unroll
        for (int m = 1; m < 8; m <<= 1) value_dot += __shfl_xor_sync(kFullMask, value_dot, m);
        #pragma unroll
        for (int m = 16; m >= 1; m >>= 1) state_dot += __shfl_xor_sync(kFullMask, state_dot, m);
        if ((lane & 7) == 0) dots[2][1][tid >> 3] = value_dot;
        if (lane == 0) dots[2][0][warp] = state_dot;

        {   // [M_P; M_A], 64 columns
            const int j0 = 16 * part, block = i >> 4;
            const float2 gi = gates.g[i];
            const float factor = is_k ? -gates.beta[i] : p.scale;
            const bool steep = gates.steep != 0;
            float sum = 0.f, x[16];
            #pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = 0.f;
            if (j0 <= first + 31) {
                float y[16];
                tmem_ld<16>(x, mine + kColPa + j0);
                tmem_ld<16>(y, mine + kColQk + j0);
                tmem_wait_ld();
                const float *f = (16 * block > j0 ? gates.column[block - 1] : gates.same) + j0;
                const float row_fade = gates.row[i];
                const int last = is_k ? i - 1 : i;
                #pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float fade = j0 + 16 <= first || !steep ? row_fade * f[j] : gdr_fade(gi, gates.g[j0 + j]);
                    x[j] = j0 + j <= last ? x[j] * fade : 0.f;
                    sum = fmaf(-x[j], y[j], sum);      // of the rows of k: dA (k_i.k_j) e^{Gi - Gj}
                    x[j] *= factor;
                }
            }
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float z[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = x[8 * e + j];
                put8<NB>(z, base + L::kA + tile_at((is_k ? 64 : 0) + i, j0 / 8 + e, 0), L::kAPiece);
            }
            if (is_k) dots[1][part][i] = sum;
        }
        float mineq[32];                                   // this head's dq or dk: token i, dim_k 32 * part ..
        float dot_g = 0.f, dot_u = 0.f;
        const float start = gates.from_start[i], scale_g = is_k ? -gates.beta[i] * start : p.scale * start, scale_u = gates.to_end[i];
        // the row of q or k itself, 8 values at a time
        auto own8 = [&](float (&x)[8], int e) {
            #pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
            #pragma unroll
            for (int k = NP - 1; k >= 0; --k) {
                float y[8];
                unpack<__nv_bfloat16>(*reinterpret_cast<const uint4 *>(smem + L::kKq + k * S::kKqPiece + tile_at((is_k ? 64 : 0) + i, 4 * part + e, S::kPanel)), y);
                #pragma unroll
                for (int j = 0; j < 8; ++j) x[j] += y[j];
            }
        };
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x[8], own[8];
            tmem_ld<8>(x, mine + kColG + 32 * part + 8 * e);
            tmem_wait_ld();
            if (is_k) own8(own, e);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                mineq[8 * e + j] = scale_g * x[j];
                if (is_k) dot_g = fmaf(own[j], x[j], dot_g);
            }
        }
        if constexpr (L::kOwnDs) wait_state();             // (the last panel's; passed under the two blocks above)
        if (is_k) {
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y[8], own[8];
                tmem_ld<8>(y, mine + kColU + 32 * part + 8 * e);
                tmem_wait_ld();
                own8(own, e);
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float z = scale_u * y[j];
                    dot_u = fmaf(own[j], z, dot_u);
                    mineq[8 * e + j] += z;
                }
            }
        }
        smem_written();
        if (warp == 0) {
            if (elect_one()) {
                fence_after_sync();
                constexpr uint32_t id = mma_desc(128, 128, false, true), idt = mma_desc(128, 128, true, true);
                const uint64_t tile = smem_desc(base + L::kA), k_mn = smem_desc(base + L::kKq + 64 * 128, S::kPanel), qk = smem_desc(base + L::kKq, S::kPanel);
                bool more = false;
                #pragma unroll
                for (int o = NB - 1; o >= 0; --o) {
                    #pragma unroll
                    for (int m = 0; m <= o; ++m) {
                        if (o - m >= NP) continue;
                        #pragma unroll
                        for (int s = 0; s < 4; ++s) mma_ss(kColG, desc_add(tile, m * L::kAPiece + 32 * s), desc_add(k_mn, (o - m) * S::kKqPiece + 2048 * s), id, again(more));
                    }
                }
                // the transpose of the tile as lanes 64-127; lanes 0-63 take what lies in K and Q's place, and are not used
                const uint64_t turned = smem_desc(base + L::kKq, L::kA - L::kKq);
                more = false;
                #pragma unroll
                for (int o = NB - 1; o >= 0; --o) {
                    #pragma unroll
                    for (int m = 0; m <= o; ++m) {
                        if (o - m >= NP) continue;
                        #pragma unroll
                        for (int s = 0; s < 8; ++s) mma_ss(kColU, desc_add(turned, m * L::kAPiece + 2048 * s), desc_add(qk, (o - m) * S::kKqPiece + 2048 * s), idt, again(more));
                    }
                }
                mma_commit(bar);
            }
            __syncwarp();
        }
        wait_mma();
        float dot = 0.f;
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x[8], y[8], own[8];
            tmem_ld<8>(x, mine + kColG + 32 * part + 8 * e);
            tmem_ld<8>(y, mine + kColU + 32 * part + 8 * e);
            tmem_wait_ld();
            own8(own, e);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float sum = x[j] + mineq[8 * e + j];
                dot = fmaf(own[j], is_k ? y[j] : sum, dot);
                total[8 * e + j] += is_k ? sum + y[j] : sum;
            }
        }
        fence_before_sync();
        dots[0][part][(is_k ? 64 : 0) + i] = dot;
        if (is_k) { dots[1][part][64 + i] = dot_g; dots[2][part][64 + i] = dot_u; }
        __syncthreads();
        if (warp == 0) {
            // two tokens a lane, from the chunk's end
            float d[2], db[2], u = 0.f, s = lane < kGradThreads / 32 ? dots[2][0][lane] : 0.f;
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = 2 * lane + e;
                float qd = 0.f, kd = 0.f, g2 = 0.f, ts = 0.f, uk = 0.f;
                #pragma unroll
                for (int w = 0; w < 4; ++w) { qd += dots[0][w][k]; kd += dots[0][w][64 + k]; g2 += dots[1][w][64 + k]; ts += dots[1][w][k]; uk += dots[2][w][64 + k]; }
                u += uk;
                const float seen = -gates.from_start[k] * g2;      // -e^G k.(dB S0^T)
                db[e] = dots[2][1][k] + seen + ts;
                d[e] = (qd - kd) - uk + gates.beta[k] * (seen + ts);
            }
            #pragma unroll
            for (int m = 16; m >= 1; m >>= 1) { u += __shfl_xor_sync(kFullMask, u, m); s += __shfl_xor_sync(kFullMask, s, m); }
            float sum = d[0] + d[1];
            #pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const float o = __shfl_down_sync(kFullMask, sum, m);
                if (lane + m < 32) sum += o;
            }
            const float end = u + gates.from_start[kChunk - 1] * s;
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t t = t0 + 2 * lane + e;
                if (t < seq.end) {
                    const int64_t at = (seq.row * p.seqlen + t) * heads + h;
                    const bool lost = 2 * lane + e >= bad[0];
                    store_any(b.dg, at, p.gtype, lost ? __uint_as_float(0x7fc00000u) : (e == 0 ? sum : sum - d[0]) + end);
                    store_any(b.dbeta, at, p.btype, lost ? __uint_as_float(0x7fc00000u) : db[e]);
                }
            }
        }
        __syncthreads();
    }
    {
        const int64_t t = t0 + i;
        if (i >= bad[1]) {
            #pragma unroll
            for (int j = 0; j < 32; ++j) total[j] = __uint_as_float(0x7fc00000u);
        }
        T *dst = reinterpret_cast<T *>(is_k ? b.dk : b.dq) + ((seq.row * p.seqlen + t) * heads_k + hk) * dk + 32 * part;
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            if (t < seq.end && 32 * part + 8 * e < dk) store8<T>(dst + 8 * e, total + 8 * e);
    }
    if (warp == 0) tmem_free512();
}

}  // namespace

static size_t images_bytes(const cc1d_gdr_params &p) { return (gdr_image_bytes(p, true) + 255) / 256 * 256; }

static size_t records_bytes(const cc1d_gdr_params &p) { return (size_t)gdr_slots(p) * (size_t)p.heads_v * sizeof(GdrRecord); }

size_t gdr_bwd_workspace_bytes(const cc1d_gdr_bwd_params &b) {
    const int per = gdr_plan_segments(b.fwd, true);
    return images_bytes(b.fwd) + records_bytes(b.fwd) + (per > 0 ? (size_t)gdr_segment_slots(b.fwd, per) * (size_t)b.fwd.heads_v * sizeof(GdrSegment) : 0);
}

int launch_gdr_bwd(const cc1d_gdr_bwd_params &b, cudaStream_t stream) {
    const cc1d_gdr_params &p = b.fwd;
    unsigned char *images = reinterpret_cast<unsigned char *>(b.workspace);
    GdrRecord *records = reinterpret_cast<GdrRecord *>(images + images_bytes(p));
    GdrSegments segs = {reinterpret_cast<GdrSegment *>(images + images_bytes(p) + records_bytes(p)), gdr_plan_segments(p, true), false};
    const int64_t sequences = gdr_sequences(p), chunks = gdr_slots(p) * p.heads_k;
    const int64_t walks = (segs.per > 0 ? gdr_segment_slots(p, segs.per) : sequences > 0 ? sequences : 1) * p.heads_v;
    if (walks >= (1ll << 29) || chunks >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    segs.ranked = gdr_rank_walks(p, segs.per, 2 * walks);
    int rc = launch_gdr_prep(p, true, images, stream);
    if (rc != CC1D_OK) return rc;
    CC1D_DISPATCH_ITYPE(p.itype, {
        CC1D_DISPATCH_BOOL(p.dim_k <= 64, kNarrow, {
            constexpr int kSteps = kNarrow ? 4 : 8;     // contraction steps of 16 over dim_k
            constexpr uint32_t kBytes = Back<T>::kBytes > Fwd<T, true>::kBytes ? Back<T>::kBytes : Fwd<T, true>::kBytes;
            if (segs.per > 0) {
                allow_dynamic_smem(reinterpret_cast<const void *>(gdr_bwd_summary_kernel<T, kSteps>), kBytes);
                launch_k(gdr_bwd_summary_kernel<T, kSteps>, dim3((unsigned)(3 * walks)), dim3(kWalkThreads), kBytes, stream, b, (const unsigned char *)images, segs, (unsigned)walks);
                rc = launch_gdr_join(p, segs, b.dfinal_states, true, stream);
                if (rc != CC1D_OK) return rc;
            }
            allow_dynamic_smem(reinterpret_cast<const void *>(gdr_bwd_walks_kernel<T, kSteps>), kBytes);
            launch_k(gdr_bwd_walks_kernel<T, kSteps>, dim3((unsigned)(2 * walks)), dim3(kWalkThreads), kBytes, stream, b, (const unsigned char *)images, records, segs);
            allow_dynamic_smem(reinterpret_cast<const void *>(gdr_grads_kernel<T, kSteps>), Grads<T>::kBytes);
            if (chunks > 0)
                launch_k(gdr_grads_kernel<T, kSteps>, dim3((unsigned)chunks), dim3(kGradThreads), Grads<T>::kBytes, stream, b, (const unsigned char *)images, (const GdrRecord *)records);
        });
    });
    return check_launch();
}

int gdr_bwd_wait_expired() { return read_and_clear_wait_expired(); }

}  // namespace cc1d
