// The forward walk over the chunks of the gated delta rule, for the forward and for the backward.
#pragma once

#include "cc1d_gdr_mma.cuh"

namespace cc1d {
namespace {

constexpr int kWalkers = 512, kWalkThreads = kWalkers + 64 + kFeeders;   // warps 0-15 walk the chunks, 16 issues their products, 17 stores, 18, 19 load

// Columns of the walk's tensor memory (128 lanes = the dim_v rows of S^T, R^T, U^T, O^T).
constexpr uint32_t kFwdColS = 0;      // 2 x 64: pieces of S^T, two dim_k per column (the third: col_s); later in a chunk
constexpr uint32_t kFwdColDelta = 0;  //   128: U''^T K, and
constexpr uint32_t kFwdColU = 128;    // 2 x 32: pieces of U^T (the third, fp32 inputs only, at 480)
constexpr uint32_t kFwdColR = 192;    // 3 x 32: pieces of R^T, then of U''^T
constexpr uint32_t kFwdColX = 288;    // 64: S^T K^T, then R^T (T - I)^T
constexpr uint32_t kFwdColO = 352;    // 64: S^T Q^T
constexpr uint32_t kFwdColY = 416;    // 64: U^T P^T
__device__ __forceinline__ uint32_t col_u(int piece) { return piece < 2 ? kFwdColU + 32 * piece : 480; }
// The third piece of S^T.  U^T P^T of the chunk before may still read U^T when the state is written, so not in U's
// place: in that of R, which is written when S^T K^T is done.  Where S^T Q^T, done later, needs it too (fp32
// inputs) it is in U's place, and the state is written when U^T P^T is done.
template <int kOutPieces> __device__ __forceinline__ constexpr uint32_t col_s(int piece) {
    return piece < 2 ? kFwdColS + 64 * piece : kOutPieces < 3 ? kFwdColR : kFwdColU;
}

// Tokens of a packed row that belong to no sequence, every fourth from `part` on: those before the first sequence, by the
// walk that begins it, and those behind the last one, by the walk that ends it.
template <typename F> __device__ __forceinline__ void unowned_tokens(const cc1d_gdr_params &p, const volatile GdrPart *w, int part, F &&f) {
    if (w->n == 0 && w->first) {
        for (int64_t t = part; t < w->seq.begin; t += 4) f(t);
    }
    if (w->n + 1 >= (int)gdr_sequences(p) && w->last) {
        for (int64_t t = w->seq.end + part; t < p.seqlen; t += 4) f(t);
    }
}

enum GdrMode { kOutput, kKeep, kSummary };
template <typename T, bool kBack> struct Fwd {
    using S = GdrStage<T, kBack>;
    static constexpr int kStages = S::kPieces == 1 ? 2 : 1;
    static constexpr uint32_t kBars = kStages * S::kBytes, kPart = kBars + 128, kBad = kPart + 128, kBytes = kBad + 2 * kGdrMaxDim * 4 + 1024;
    static_assert(sizeof(GdrPart) <= 128, "place between the barriers and the first bad tokens");
};

// One CTA walks one sequence of one value head, chunk by chunk, with S^T (dim_v x dim_k) in the
// registers of warps 0-15 (thread: one dim_v, a quarter of the dim_k):
//   X = K S        R = beta (V - e^G X)        U = R + (T - I) R        U'' = e^{G_C - G} U
//   O = scale (e^G Q S + P U)                  S <- e^{G_C} S + K^T U''
// All five products run on tcgen05 with the transposed left factor (S^T, R^T, U^T, U''^T: 128 dim_v
// rows) in tensor memory and the right one (K, Q, T, P) in shared memory, so nothing that the walk
// computes passes through shared memory.  What bounds it is the chain of a chunk, 7,500 cycles (4.0 us, bf16,
// 128 x 128; 64 chunks of 128 heads and rows 258 us): S^T K^T -> R -> (T - I) R -> U -> K^T U'' -> S, each link a
// product, a wait, and registers split into pieces and put back into tensor memory; 3,200 of them are products
// (33 cycles an instruction of 64 columns, 66 of 128), and the rest fills 47 % of the issue slots.  One sequence
// and head a CTA, so few heads leave SMs idle: cc1d_gdr_prep.cu cuts long sequences into segments then.  S itself is kept and decayed in fp32 registers; only
// its pieces are rewritten every chunk.
// A token whose R or U is infinite or NaN in some column takes part as zero there (as do entries of A and T: GdrGates::bad), for a zero of T or P times NaN
// would reach the tokens before it; `bad` holds the first such token of each column, and from it on the
// outputs of the chunk and the state behind it are NaN in that column.
// kKeep: the backward's walk, which leaves S, U and the first bad token of every chunk in its record instead of an
// output.  The gradients of the tokens before that one do not depend on what stands in its place.
// kSummary: what a segment does to the state: from zeros its last state B, or (unit) without values from the
// identity, dim_k columns instead of dim_v, its M.
template <typename T, int kSteps, GdrMode kMode, bool kBack>
__device__ __forceinline__ void walk_forward(const cc1d_gdr_params &p, const unsigned char *images, GdrRecord *records, const GdrSegments &segs, int64_t block, bool unit) {
    constexpr bool kOut = kMode == kOutput, kFinite = kMode != kSummary;
    using L = Fwd<T, kBack>;
    using St = GdrStage<T, kBack>;
    constexpr int NP = St::kPieces, PO = GdrType<T>::kOutPieces, PT = St::kSolve;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t bars = smem_u32(smem + L::kBars);
    const uint32_t bar_full = bars, bar_empty = bars + 16, bar_x = bars + 56, bar_u = bars + 64, bar_o = bars + 72, bar_d = bars + 80,
                   bar_s = bars + 88, bar_r = bars + 96, bar_w = bars + 104, bar_out = bars + 112;
    volatile int *dead = reinterpret_cast<volatile int *>(smem + L::kBars + 120);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 124);
    const int tid = threadIdx.x, warp = __shfl_sync(kFullMask, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    const int heads = (int)p.heads_v, h = (int)(block % heads), sequences = (int)gdr_sequences(p);
    GdrPart w;
    if (!gdr_find_part(p, segs, segs.ranked ? gdr_ranked(p, (int)(block / heads), reinterpret_cast<int *>(smem)) : block / heads, w)) return;
    // B of a last segment leads nowhere, nor does M of one that is alone (or, forwards, of a last one)
    if (kMode == kSummary && (unit ? (kBack ? w.first && w.last : w.last) : w.last)) return;
    const GdrSeq seq = w.seq;
    const int n = w.n, chunks = w.chunks, dk = (int)p.dim_k, dv = kMode == kSummary && unit ? dk : (int)p.dim_v;
    // what the walkers need again at their end (kept in registers over the walk it makes them spill)
    volatile GdrPart *kept = reinterpret_cast<volatile GdrPart *>(smem + L::kPart);
    if (tid == 0) {
        kept->n = w.n; kept->seq.begin = w.seq.begin; kept->seq.end = w.seq.end; kept->segment = w.segment; kept->first = w.first; kept->last = w.last;
        for (int s = 0; s < 2; ++s) { mbar_init(bar_full + 8 * s, kFeeders + 1); mbar_init(bar_empty + 8 * s, 1); }
        mbar_init(bar_x, 1); mbar_init(bar_u, 1); mbar_init(bar_o, 1); mbar_init(bar_d, 1);
        mbar_init(bar_s, kWalkers / 32); mbar_init(bar_r, kWalkers / 32); mbar_init(bar_w, kWalkers / 32); mbar_init(bar_out, kWalkers / 32);
        *dead = 0;
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc512(smem_u32(slot));
    fence_before_sync();
    __syncthreads();
    fence_after_sync();

    if (warp == kWalkers / 32) {
        // issues the walk's products: a thread that issues is held up while earlier ones still run,
        // which no warp with other work should be
        for (int c = 0; c < chunks; ++c) {
            const int s = c % L::kStages;
            const uint32_t par = c & 1;
            const uint32_t stage = smem_u32(smem) + s * St::kBytes;
            const uint64_t kq = smem_desc(stage + St::kKq), kmn = smem_desc(stage + St::kKq, St::kPanel);
            constexpr uint32_t id = mma_desc(128, 64, false, false), idd = mma_desc(128, 128, false, true);
            gdr_wait(bar_full + 8 * s, (c / L::kStages) & 1, dead);
            gdr_wait(bar_s, par, dead);
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = 2; o >= 0; --o) {
                    #pragma unroll
                    for (int a = 0; a <= o; ++a) {
                        const int b = o - a;
                        if (a >= 3 || b >= NP) continue;
                        #pragma unroll
                        for (int i = 0; i < kSteps; ++i)
                            mma_ts(kFwdColX, col_s<PO>(a) + 8 * i, desc_add(kq, b * St::kKqPiece + (i >> 2) * St::kPanel + (i & 3) * 32), id, again(more));
                    }
                }
                mma_commit(bar_x);
            }
            __syncwarp();
            if (kOut && c > 0) gdr_wait(bar_out, (c - 1) & 1, dead);      // the columns of S^T Q^T have been read
            __syncwarp();
            if (kOut && elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = kOut ? PO - 1 : -1; o >= 0; --o) {
                    #pragma unroll
                    for (int a = 0; a <= o; ++a) {
                        const int b = o - a;
                        if (a >= PO || b >= NP) continue;
                        #pragma unroll
                        for (int i = 0; i < kSteps; ++i)
                            mma_ts(kFwdColO, col_s<PO>(a) + 8 * i, desc_add(kq, b * St::kKqPiece + 64 * 128 + (i >> 2) * St::kPanel + (i & 3) * 32), id, again(more));
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
                for (int o = PT - 1; o >= 0; --o) {
                    #pragma unroll
                    for (int a = 0; a <= o; ++a) {
                        const int b = o - a;
                        if (a >= PT || b >= PT) continue;
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) mma_ts(kFwdColX, kFwdColR + 32 * a + 8 * i, desc_add(kq, St::kT + b * 8192 + 32 * i), id, again(more));
                    }
                }
                mma_commit(bar_u);
            }
            __syncwarp();
            gdr_wait(bar_w, par, dead);
            __syncwarp();
            if (elect_one()) {
                fence_after_sync();
                bool more = false;
                #pragma unroll
                for (int o = 2; o >= 0; --o) {
                    #pragma unroll
                    for (int a = 0; a <= o; ++a) {
                        const int b = o - a;
                        if (a >= 3 || b >= NP) continue;
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) mma_ts(kFwdColDelta, kFwdColR + 32 * a + 8 * i, desc_add(kmn, b * St::kKqPiece + 2048 * i), idd, again(more));
                    }
                }
                mma_commit(bar_d);
                more = false;
                #pragma unroll
                for (int o = kOut ? PO - 1 : -1; o >= 0; --o) {
                    #pragma unroll
                    for (int a = 0; a <= o; ++a) {
                        const int b = o - a;
                        if (a >= PO || b >= PO) continue;
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) mma_ts(kFwdColY, col_u(a) + 8 * i, desc_add(kq, St::kP + b * 8192 + 32 * i), id, again(more));
                    }
                }
                if (kOut) mma_commit(bar_o);        // (an arrival that nothing waits for could come when the CTA is gone)
            }
            __syncwarp();
        }
    } else if (warp == kWalkers / 32 + 1) {
        // stores the output, which the walkers leave in the place of the stage's V, by rows, 16 bytes a
        // lane (64 bulk copies of a row each took 4600 cycles to issue); then the stage is free
        T *out = reinterpret_cast<T *>(p.out) + seq.row * p.out_batch_stride + h * p.out_h_stride;
        constexpr int kVec = 16 / (int)sizeof(T), kLanes = kGdrMaxDim / kVec, kRows = 32 / kLanes;
        const int at = lane % kLanes * kVec;
        for (int c = 0; c < chunks; ++c) {
            const unsigned char *V = smem + (c % L::kStages) * St::kBytes + St::kV;
            gdr_wait(bar_out, c & 1, dead);
            __syncwarp();
            const int rows = min(kChunk, seq.end - seq.begin - c * kChunk);
            if (kOut && at < dv) {
                #pragma unroll 8
                for (int i = lane / kLanes; i < rows; i += kRows) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(V + (i * kGdrMaxDim + at) * sizeof(T));
                    *reinterpret_cast<uint4 *>(out + ((int64_t)seq.begin + c * kChunk + i) * p.out_l_stride + at) = v;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + 8 * (c % L::kStages));
        }
    } else if (warp > kWalkers / 32) {
        GdrRows<T, kFeeders> rows(p, seq, h, p.v, seq.row * p.v_batch_stride + h * p.v_h_stride, p.v_l_stride);
        const int64_t step = (int64_t)heads * St::kImage;
        if (kMode == kSummary && unit) rows.dv = 0;
        feed_walk<T, L::kStages, kBack, kOut>(rows, images + w.slot * step + h * (int64_t)St::kImage, step, smem_u32(smem), seq.begin, chunks,
                                        bar_full, bar_empty, dead, tid - kWalkers - 64);
    } else {
        const int quad = warp & 3, part = warp >> 2, col = quad * 32 + lane;   // part: a quarter of the dim_k and of the tokens
        const uint32_t mine = (uint32_t)(quad * 32) << 16;
        float S[32];
        if (kMode == kSummary) {
            #pragma unroll
            for (int j = 0; j < 32; ++j) S[j] = unit && 32 * part + j == col ? 1.f : 0.f;
        } else if (!(w.first && w.last)) {
            // (a first segment's too: its sequence's last one may already have written the state's row; what is past dim_v the
            // join leaves as it lay in memory, and the gradients sum over all 128 columns)
            #pragma unroll
            for (int j = 0; j < 32; ++j) S[j] = 32 * part + j < dk && col < dv ? w.segment[h].start[32 * part + j][col] : 0.f;
        } else {
            const int64_t row = n < sequences ? gdr_state_row(p, n) : -1, state_at = (int64_t)(32 * part) * dv + col;
            const bool from = p.initial_states != nullptr && row >= 0 && (p.has_initial_state == nullptr || p.has_initial_state[n] != 0);
            const float *src = p.initial_states + row * p.initial_states_batch_stride + h * p.initial_states_h_stride + state_at;
            #pragma unroll
            for (int j = 0; j < 32; ++j) S[j] = from && 32 * part + j < dk && col < dv ? src[(int64_t)j * dv] : 0.f;
        }
        // first token of a chunk whose value is not finite, by column; chunks use the two rows in turn
        int *bad = reinterpret_cast<int *>(smem + L::kBad) + col;
        if (kFinite && part < 2) bad[part * kGdrMaxDim] = kChunk;
        if (kFinite) walk_sync<kWalkers>();
        auto only_finite = [&](float (&x)[16], int first, int par) {
            if (__builtin_expect(!all_finite(x), 0)) {
                uint32_t out = 0;
                #pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const bool ok = finite(x[j]);
                    out |= ok ? 0u : 1u << j;
                    x[j] = ok ? x[j] : 0.f;
                }
                if (out != 0) atomicMin(bad + par * kGdrMaxDim, first + __ffs(out) - 1);
            }
            __syncwarp();
        };
        // this warp's part of an operand is in tensor memory
        auto ready = [&](uint32_t bar) {
            tmem_wait_st();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        GdrRecord *record = kMode == kKeep ? records + w.slot * heads + h : nullptr;
        auto put_state = [&]() {
            if (kMode == kKeep) {
                #pragma unroll
                for (int j = 0; j < 32; ++j) record->S0[32 * part + j][col] = S[j];
            }
            #pragma unroll
            for (int b = 0; b < 4; ++b) split8_to_tmem<3>(S + 8 * b, mine + kFwdColS + 16 * part + 4 * b, 64, col_s<PO>(2) - kFwdColS);
            ready(bar_s);
        };
        if (chunks > 0) put_state();
        for (int c = 0; c < chunks; ++c) {
            const int s = c % L::kStages;
            const uint32_t par = c & 1;
            unsigned char *stage = smem + s * St::kBytes;
            gdr_wait(bar_full + 8 * s, (c / L::kStages) & 1, dead);
            const GdrGates &gates = *reinterpret_cast<const GdrGates *>(stage + St::kGates);
            T *V = reinterpret_cast<T *>(stage + St::kV) + 16 * part * kGdrMaxDim + col;
            const int first = 16 * part;               // this thread's tokens: first .. first + 15
            float R[16];
            #pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 b = *reinterpret_cast<const float4 *>(gates.beta + first + j);
                R[j] = b.x * Elem<T>::to_f(V[j * kGdrMaxDim]); R[j + 1] = b.y * Elem<T>::to_f(V[(j + 1) * kGdrMaxDim]);
                R[j + 2] = b.z * Elem<T>::to_f(V[(j + 2) * kGdrMaxDim]); R[j + 3] = b.w * Elem<T>::to_f(V[(j + 3) * kGdrMaxDim]);
            }
            gdr_wait(bar_x, par, dead);
            __syncwarp();
            fence_after_sync();
            {             // R = beta V - beta e^G X
                float x[16];
                tmem_ld<16>(x, mine + kFwdColX + first);
                tmem_wait_ld();
                #pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(gates.minus_beta_from_start + first + j);
                    const float2 u = fma2(make_float2(f.x, f.y), make_float2(x[j], x[j + 1]), make_float2(R[j], R[j + 1]));
                    const float2 v = fma2(make_float2(f.z, f.w), make_float2(x[j + 2], x[j + 3]), make_float2(R[j + 2], R[j + 3]));
                    R[j] = u.x; R[j + 1] = u.y; R[j + 2] = v.x; R[j + 3] = v.y;
                }
                if (kFinite) only_finite(R, first, par);
                #pragma unroll
                for (int j = 0; j < 16; j += 8) split8_to_tmem<PT>(R + j, mine + kFwdColR + first / 2 + j / 2, 32, 64);
            }
            ready(bar_r);
            gdr_wait(bar_u, par, dead);
            __syncwarp();
            fence_after_sync();
            {             // U and U''
                float x[16];
                tmem_ld<16>(x, mine + kFwdColX + first);
                tmem_wait_ld();
                #pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 v = add2(make_float2(x[j], x[j + 1]), make_float2(R[j], R[j + 1]));
                    x[j] = v.x; x[j + 1] = v.y;
                }
                if (kFinite) only_finite(x, first, par);     // (a finite R may overflow with T)
                if (kMode == kKeep) {
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) record->U[first + j][col] = x[j];
                    record += heads;
                } else if (kOut) {
                    #pragma unroll
                    for (int j = 0; j < 16; j += 8) split8_to_tmem<PO>(x + j, mine + kFwdColU + first / 2 + j / 2, 32, 480 - kFwdColU);
                }
                #pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(gates.to_end + first + j);
                    x[j] *= f.x; x[j + 1] *= f.y; x[j + 2] *= f.z; x[j + 3] *= f.w;
                }
                #pragma unroll
                for (int j = 0; j < 16; j += 8) split8_to_tmem<3>(x + j, mine + kFwdColR + first / 2 + j / 2, 32, 64);
            }
            ready(bar_w);
            const float whole = gates.from_start[kChunk - 1];
            const int bad_row = gates.bad;
            gdr_wait(bar_d, par, dead);
            __syncwarp();
            fence_after_sync();
            #pragma unroll
            for (int b = 0; b < 2; ++b) {
                float x[16];
                tmem_ld<16>(x, mine + kFwdColDelta + 32 * part + 16 * b);
                tmem_wait_ld();
                #pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 v = fma2(splat2(whole), make_float2(S[16 * b + j], S[16 * b + j + 1]), make_float2(x[j], x[j + 1]));
                    S[16 * b + j] = v.x; S[16 * b + j + 1] = v.y;
                }
            }
            if (kFinite && part == 0) bad[(par ^ 1) * kGdrMaxDim] = kChunk;      // (all are done with the chunk before)
            fence_before_sync();
            walk_sync<kWalkers>();                      // every thread has read its part of Delta
            fence_after_sync();
            const int bad_from = kFinite ? min(bad[par * kGdrMaxDim], bad_row) : bad_row;
            if (bad_from < kChunk) {
                #pragma unroll
                for (int j = 0; j < 32; ++j) S[j] = __uint_as_float(0x7fc00000u);
            }
            __syncwarp();
            if (kOut && PO == 3) {
                gdr_wait(bar_o, par, dead);             // U^T has been read (col_s)
                __syncwarp();
                fence_after_sync();
            }
            if (c + 1 < chunks) put_state();
            if (kMode == kKeep && part == 0) {
                const int least = __reduce_min_sync(kFullMask, bad_from);
                if (lane == 0) record[-heads].bad[quad] = least;      // (record: the next chunk's)
            }
            // the output, while the next chunk's first product runs
            if (kOut) {
                gdr_wait(bar_o, par, dead);
                __syncwarp();
                fence_after_sync();
                #pragma unroll
                for (int b = 0; b < 16; b += 8) {
                    float x[8], y[8];
                    tmem_ld<8>(x, mine + kFwdColO + first + b);
                    tmem_ld<8>(y, mine + kFwdColY + first + b);
                    tmem_wait_ld();
                    #pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(gates.from_start + first + b + j);
                        x[j] = fmaf(f.x, x[j], y[j]); x[j + 1] = fmaf(f.y, x[j + 1], y[j + 1]);
                        x[j + 2] = fmaf(f.z, x[j + 2], y[j + 2]); x[j + 3] = fmaf(f.w, x[j + 3], y[j + 3]);
                    }
                    #pragma unroll
                    for (int j = 0; j < 8; ++j)      // where this thread read its v
                        V[(b + j) * kGdrMaxDim] = Elem<T>::from_f(first + b + j < bad_from ? p.scale * x[j] : __uint_as_float(0x7fc00000u));
                }
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_out);
        }
        const int head = (int)(block % heads);
        if (kMode == kSummary) {
            GdrSegment &to = kept->segment[head];
            if (unit) {
                #pragma unroll
                for (int j = 0; j < 32; ++j) to.M[32 * part + j][col] = S[j];
                #pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(&to.Mt[col][32 * part + j]) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
            } else {
                #pragma unroll
                for (int j = 0; j < 32; ++j) to.B[32 * part + j][col] = S[j];
            }
        }
        if (kOut && kept->last) {
            const int at = kept->n, all = (int)gdr_sequences(p);
            const int64_t row = at < all ? gdr_state_row(p, at) : -1;
            if (p.final_states != nullptr && row >= 0) {
                float *dst = p.final_states + row * p.final_states_batch_stride + head * p.final_states_h_stride + (int64_t)(32 * part) * dv + col;
                #pragma unroll
                for (int j = 0; j < 32; ++j) if (32 * part + j < dk && col < dv) dst[(int64_t)j * dv] = S[j];
            }
        }
        if (kOut && p.cu_seqlens != nullptr) {
            T *out = reinterpret_cast<T *>(p.out) + head * p.out_h_stride + col;
            unowned_tokens(p, kept, part, [&](int64_t t) { if (col < dv) out[t * p.out_l_stride] = Elem<T>::from_f(0.f); });
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_free512();
}

}  // namespace
}  // namespace cc1d
