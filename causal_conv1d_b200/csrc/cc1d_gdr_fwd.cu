// Gated delta rule over whole sequences: cc1d_gdr_fwd (include/cc1d_gdr.h).
#include "cc1d_gdr_mma.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 512;   // warps 0-7 walk the chunks, warps 8-15 prepare the next one

// Columns of the walk's tensor memory (128 lanes = the dim_v rows of S^T, R^T, U^T, O^T).
constexpr uint32_t kColS = 0;      // 3 x 64: pieces of S^T, two dim_k per column; later in a chunk
constexpr uint32_t kColDelta = 0;  //   128: U''^T K, and
constexpr uint32_t kColU = 128;    //   2 x 32: pieces of U^T (the third, fp32 inputs only, at 480)
constexpr uint32_t kColR = 192;    // 3 x 32: pieces of R^T, then of U''^T
constexpr uint32_t kColX = 288;    // 64: S^T K^T, then U^T, then P U
constexpr uint32_t kColO = 352;    // 64: S^T Q^T
__device__ __forceinline__ uint32_t col_u(int piece) { return piece < 2 ? kColU + 32 * piece : 480; }

template <typename T> struct Fwd {
    using S = GdrStage<T>;
    static constexpr int kStages = S::kPieces == 1 ? 2 : 1;
    static constexpr uint32_t kInv = kStages * S::kBytes, kBars = kInv + kGdrInverseBytes, kBytes = kBars + 128 + 1024;
};

// One CTA walks one sequence of one value head, chunk by chunk, with S^T (dim_v x dim_k) in the
// registers of warps 0-7 (thread: one dim_v, half of the dim_k):
//   X = K S        R = beta (V - e^G X)        U = T R        U'' = e^{G_C - G} U
//   O = scale (e^G Q S + P U)                  S <- e^{G_C} S + K^T U''
// All five products run on tcgen05 with the transposed left factor (S^T, R^T, U^T, U''^T: 128 dim_v
// rows) in tensor memory and the right one (K, Q, T, P) in shared memory, so nothing that the walk
// computes passes through shared memory.  S itself is kept and decayed in fp32 registers; only
// its pieces are rewritten every chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads, 1) gdr_fwd_kernel(const cc1d_gdr_params p) {
    using L = Fwd<T>;
    using St = GdrStage<T>;
    constexpr int NP = St::kPieces, PO = St::kOut;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    float *inv = reinterpret_cast<float *>(smem + L::kInv);
    const uint32_t bars = smem_u32(smem + L::kBars);
    const uint32_t bar_full = bars, bar_empty = bars + 16, bar_kq = bars + 32, bar_x = bars + 40, bar_u = bars + 48, bar_o = bars + 56, bar_d = bars + 64;
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::kBars + 96);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 100);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) { mbar_init(bar_full + 8 * s, 256); mbar_init(bar_empty + 8 * s, 8); }
        mbar_init(bar_kq, 1); mbar_init(bar_x, 1); mbar_init(bar_u, 1); mbar_init(bar_o, 1); mbar_init(bar_d, 1);
        *dead = 0;
        fence_mbar_init();
    }
    pdl_wait();
    if (warp == 0) tmem_alloc512(smem_u32(slot));
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *slot;

    const int heads = (int)p.heads_v, h = blockIdx.x % heads, n = blockIdx.x / heads;
    const int sequences = (int)gdr_sequences(p);
    GdrSeq seq = {0, 0, 0};
    if (n < sequences) seq = gdr_sequence(p, n);
    const int chunks = (seq.end - seq.begin + kChunk - 1) / kChunk;
    const int dk = (int)p.dim_k, dv = (int)p.dim_v;

    if (warp >= 8) {
        for (int c = 0; c < chunks; ++c) {
            const int s = c % L::kStages, round = c / L::kStages;
            gdr_wait(bar_empty + 8 * s, (round & 1) ^ 1, dead);
            prepare_chunk<T, 2>(smem + s * St::kBytes, inv, p, seq, h, seq.begin + c * kChunk, tmem, bar_kq, c & 1, dead, tid - 256);
            mbar_arrive(bar_full + 8 * s);
            group_sync<2, 256>();      // the inverse's scratch is free again
        }
    } else {
        const int quad = warp & 3, half = warp >> 2, col = quad * 32 + lane;
        const uint32_t mine = tmem + ((uint32_t)(quad * 32) << 16);
        const int64_t row = n < sequences ? gdr_state_row(p, n) : -1;
        const int64_t state_at = (int64_t)(64 * half) * dv + col;
        float S[64];
        {
            const bool from = p.initial_states != nullptr && row >= 0 && (p.has_initial_state == nullptr || p.has_initial_state[n] != 0);
            const float *src = p.initial_states + row * p.initial_states_batch_stride + h * p.initial_states_h_stride + state_at;
            #pragma unroll
            for (int j = 0; j < 64; ++j) S[j] = from && 64 * half + j < dk && col < dv ? src[(int64_t)j * dv] : 0.f;
        }
        auto put_state = [&]() {
            #pragma unroll
            for (int b = 0; b < 4; ++b) {
                float x[16];
                uint32_t r[3][8];
                #pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = S[16 * b + j];
                split16<3>(x, r);
                #pragma unroll
                for (int k = 0; k < 3; ++k) tmem_st8(mine + kColS + 64 * k + 32 * half + 8 * b, r[k]);
            }
            tmem_wait_st();
            fence_before_sync();
            group_sync<1, 256>();
        };
        if (chunks > 0) put_state();
        const int steps = (dk + 15) / 16;
        T *out = reinterpret_cast<T *>(p.out) + seq.row * p.out_batch_stride + h * p.out_h_stride + col;
        for (int c = 0; c < chunks; ++c) {
            const int s = c % L::kStages, round = c / L::kStages;
            const uint32_t par = c & 1;
            unsigned char *stage = smem + s * St::kBytes;
            const uint32_t base = smem_u32(stage);
            const GdrGates &gates = *reinterpret_cast<const GdrGates *>(stage + St::kGates);
            const T *V = reinterpret_cast<const T *>(stage + St::kV);
            gdr_wait(bar_full + 8 * s, round & 1, dead);
            if (tid == 0) {
                fence_after_sync();
                constexpr uint32_t id = mma_desc(128, 64, false, false);
                bool add = false;
                #pragma unroll
                for (int a = 0; a < 3; ++a) {
                    #pragma unroll
                    for (int b = 0; b < NP && a + b < 3; ++b) {
                        for (int i = 0; i < steps; ++i) {
                            mma_ts(tmem + kColX, tmem + kColS + 64 * a + 8 * i,
                                   smem_desc(base + St::kKq + b * St::kKqPiece + (i >> 2) * St::kPanel + (i & 3) * 32), id, add);
                            add = true;
                        }
                    }
                }
                mma_commit(bar_x);
                add = false;
                #pragma unroll
                for (int a = 0; a < PO; ++a) {
                    #pragma unroll
                    for (int b = 0; b < NP && a + b < PO; ++b) {
                        for (int i = 0; i < steps; ++i) {
                            mma_ts(tmem + kColO, tmem + kColS + 64 * a + 8 * i,
                                   smem_desc(base + St::kKq + b * St::kKqPiece + 64 * 128 + (i >> 2) * St::kPanel + (i & 3) * 32), id, add);
                            add = true;
                        }
                    }
                }
            }
            __syncwarp();
            gdr_wait(bar_x, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int b = 0; b < 2; ++b) {      // R
                const int t0 = 32 * half + 16 * b;
                float x[16];
                uint32_t r[3][8];
                tmem_ld<16>(x, mine + kColX + t0);
                tmem_wait_ld();
                #pragma unroll
                for (int j = 0; j < 16; ++j)
                    x[j] = gates.beta[t0 + j] * fmaf(-gates.from_start[t0 + j], x[j], Elem<T>::to_f(V[(t0 + j) * kGdrMaxDim + col]));
                split16<3>(x, r);
                #pragma unroll
                for (int k = 0; k < 3; ++k) tmem_st8(mine + kColR + 32 * k + t0 / 2, r[k]);
            }
            tmem_wait_st();
            fence_before_sync();
            group_sync<1, 256>();
            if (tid == 0) {
                fence_after_sync();
                constexpr uint32_t id = mma_desc(128, 64, false, false);
                bool add = false;
                #pragma unroll
                for (int a = 0; a < 3; ++a) {
                    #pragma unroll
                    for (int b = 0; a + b < 3; ++b) {
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_ts(tmem + kColX, tmem + kColR + 32 * a + 8 * i, smem_desc(base + St::kT + b * 8192 + 32 * i), id, add);
                            add = true;
                        }
                    }
                }
                mma_commit(bar_u);
            }
            __syncwarp();
            gdr_wait(bar_u, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int b = 0; b < 2; ++b) {      // U and U''
                const int t0 = 32 * half + 16 * b;
                float x[16];
                uint32_t r[3][8], u[PO][8];
                tmem_ld<16>(x, mine + kColX + t0);
                tmem_wait_ld();
                split16<PO>(x, u);
                #pragma unroll
                for (int k = 0; k < PO; ++k) tmem_st8(mine + col_u(k) + t0 / 2, u[k]);
                #pragma unroll
                for (int j = 0; j < 16; ++j) x[j] *= gates.to_end[t0 + j];
                split16<3>(x, r);
                #pragma unroll
                for (int k = 0; k < 3; ++k) tmem_st8(mine + kColR + 32 * k + t0 / 2, r[k]);
            }
            tmem_wait_st();
            fence_before_sync();
            group_sync<1, 256>();
            if (tid == 0) {
                fence_after_sync();
                constexpr uint32_t id = mma_desc(128, 64, false, false), idd = mma_desc(128, 128, false, true);
                bool add = false;
                #pragma unroll
                for (int a = 0; a < PO; ++a) {
                    #pragma unroll
                    for (int b = 0; a + b < PO; ++b) {
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_ts(tmem + kColX, tmem + col_u(a) + 8 * i, smem_desc(base + St::kP + b * 8192 + 32 * i), id, add);
                            add = true;
                        }
                    }
                }
                mma_commit(bar_o);
                add = false;
                #pragma unroll
                for (int a = 0; a < 3; ++a) {
                    #pragma unroll
                    for (int b = 0; b < NP && a + b < 3; ++b) {
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_ts(tmem + kColDelta, tmem + kColR + 32 * a + 8 * i, smem_desc(base + St::kKq + b * St::kKqPiece + 2048 * i, St::kPanel), idd, add);
                            add = true;
                        }
                    }
                }
                mma_commit(bar_d);
            }
            __syncwarp();
            gdr_wait(bar_o, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int b = 0; b < 2; ++b) {      // out
                const int t0 = 32 * half + 16 * b;
                float x[16], y[16];
                tmem_ld<16>(x, mine + kColO + t0);
                tmem_ld<16>(y, mine + kColX + t0);
                tmem_wait_ld();
                if (col < dv) {
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int64_t t = (int64_t)seq.begin + c * kChunk + t0 + j;
                        if (t < seq.end) out[t * p.out_l_stride] = Elem<T>::from_f(p.scale * fmaf(gates.from_start[t0 + j], x[j], y[j]));
                    }
                }
                __syncwarp();
            }
            gdr_wait(bar_d, par, dead);
            __syncwarp();
            fence_after_sync();
            const float whole = gates.from_start[kChunk - 1];
            #pragma unroll
            for (int b = 0; b < 4; ++b) {
                float x[16];
                tmem_ld<16>(x, mine + kColDelta + 64 * half + 16 * b);
                tmem_wait_ld();
                #pragma unroll
                for (int j = 0; j < 16; ++j) S[16 * b + j] = fmaf(whole, S[16 * b + j], x[j]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + 8 * s);
            fence_before_sync();
            group_sync<1, 256>();              // every thread has read its part of Delta
            fence_after_sync();
            if (c + 1 < chunks) put_state();
        }
        if (p.final_states != nullptr && row >= 0) {
            float *dst = p.final_states + row * p.final_states_batch_stride + h * p.final_states_h_stride + state_at;
            #pragma unroll
            for (int j = 0; j < 64; ++j) if (64 * half + j < dk && col < dv) dst[(int64_t)j * dv] = S[j];
        }
        // tokens that belong to no sequence
        if (p.cu_seqlens != nullptr && n + 1 >= sequences) {
            for (int64_t t = seq.end + half; t < p.seqlen; t += 2)
                if (col < dv) out[t * p.out_l_stride] = Elem<T>::from_f(0.f);
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_free512(tmem);
}

}  // namespace

size_t gdr_fwd_workspace_bytes(const cc1d_gdr_params &p) { (void)p; return 0; }

int launch_gdr_fwd(const cc1d_gdr_params &p, cudaStream_t stream) {
    const int64_t sequences = gdr_sequences(p), ctas = (sequences > 0 ? sequences : 1) * p.heads_v;
    if (ctas >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    CC1D_DISPATCH_ITYPE(p.itype, {
        allow_dynamic_smem(reinterpret_cast<const void *>(gdr_fwd_kernel<T>), Fwd<T>::kBytes);
        launch_k(gdr_fwd_kernel<T>, dim3((unsigned)ctas), dim3(kThreads), Fwd<T>::kBytes, stream, p);
    });
    return check_launch();
}

int gdr_wait_expired() { return read_and_clear_wait_expired(); }

}  // namespace cc1d
