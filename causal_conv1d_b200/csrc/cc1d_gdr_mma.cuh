// Tensor-core side of the chunked gated delta rule: tcgen05 wrappers, operand layouts, fp32 values
// as sums of bf16 pieces, and the per-chunk preparation that forward and backward share.
#pragma once

#include "cc1d_gdr.cuh"
#include "cc1d_tma.cuh"

namespace cc1d {

constexpr int kChunk = 64;

// ---- tcgen05 ---------------------------------------------------------------------------------
// The kernels here take all 512 columns of an SM, so tensor-memory addresses are plain constants:
// column + (lane << 16), from 0.
__device__ __forceinline__ void tmem_alloc512(uint32_t smem_slot) {   // one whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free512() {                      // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(0) : "memory");
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
template <> __device__ __forceinline__ void tmem_ld<8>(float (&f)[8], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]) : "r"(at));
}
template <> __device__ __forceinline__ void tmem_ld<16>(float (&f)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
                   "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]) : "r"(at));
}
__device__ __forceinline__ void tmem_st4(uint32_t at, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
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
__device__ __forceinline__ uint64_t desc_add(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
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

// One lane of a converged warp.  MMAs are issued under this predicate: the compiler then keeps
// their descriptors in uniform registers (under `threadIdx.x == 0` each one is moved there anew,
// which costs more than the MMA).
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

// First product into an accumulator: false, and true from then on.  A sum over pieces starts with the
// smallest products: the tensor core cuts its sums off at 24 bits, and so only the last, large ones
// are cut at the size of the result.
__device__ __forceinline__ bool again(bool &more) {
    const bool was = more;
    more = true;
    return was;
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
template <int kThreads> __device__ __forceinline__ void walk_sync() { asm volatile("bar.sync 1, %0;" :: "n"(kThreads) : "memory"); }

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234e38f; }
__device__ __forceinline__ bool all_finite(const float (&x)[16]) {
    float2 m[2] = {};                          // 0 * x is 0 or NaN
    #pragma unroll
    for (int j = 0; j < 16; j += 4) {
        m[0] = fma2(make_float2(x[j], x[j + 1]), splat2(0.f), m[0]);
        m[1] = fma2(make_float2(x[j + 2], x[j + 3]), splat2(0.f), m[1]);
    }
    return finite((m[0].x + m[0].y) + (m[1].x + m[1].y));
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
        if (i + 1 < kPieces) x = fma2(make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u)), splat2(-1.f), x);
    }
}
// x[0..7] -> columns of tensor memory, two values per column: piece k at `at` + k * step, the third at `at` + third
template <int kPieces> __device__ __forceinline__ void split8_to_tmem(const float *x, uint32_t at, uint32_t step, uint32_t third) {
    uint32_t r[kPieces][4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t p[kPieces];
        split_pair<kPieces>(make_float2(x[2 * i], x[2 * i + 1]), p);
        #pragma unroll
        for (int k = 0; k < kPieces; ++k) r[k][i] = p[k];
    }
    #pragma unroll
    for (int k = 0; k < kPieces; ++k) tmem_st4(at + (k < 2 ? k * step : third), r[k]);
}

// x[0..7] -> shared memory: piece k, 16 bytes, at `at` + k * 8192
template <int kPieces> __device__ __forceinline__ void store_pieces8(const float *x, uint32_t at) {
    uint32_t r[4][kPieces];
    #pragma unroll
    for (int i = 0; i < 4; ++i) split_pair<kPieces>(make_float2(x[2 * i], x[2 * i + 1]), r[i]);
    #pragma unroll
    for (int k = 0; k < kPieces; ++k)
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at + k * 8192), "r"(r[0][k]), "r"(r[1][k]), "r"(r[2][k]), "r"(r[3][k]) : "memory");
}

template <typename T> struct GdrType;
// kPieces: of the inputs; kOutPieces: of the factors of an output of this type; kSolve: of T - I and of what it is
// multiplied with
template <> struct GdrType<__nv_bfloat16> { static constexpr int kPieces = 1, kOutPieces = 2, kSolve = 2; };
template <> struct GdrType<__half> { static constexpr int kPieces = 2, kOutPieces = 2, kSolve = 2; };
template <> struct GdrType<float> { static constexpr int kPieces = 3, kOutPieces = 3, kSolve = 3; };

// ---- operand tiles ------------------------------------------------------------------------------
// Token tile of one piece: panels of 64 columns, a panel `rows` x 128 bytes in the 128-byte swizzle.
// Used K-major (contraction over the columns) and MN-major (contraction over the tokens).
__device__ __forceinline__ uint32_t tile_at(int row, int chunk16, uint32_t panel_bytes) {
    return (chunk16 >> 3) * panel_bytes + row * 128 + (((chunk16 & 7) ^ (row & 7)) << 4);
}

// 8 elements of one row, as they are, and as one 16-byte vector for each piece
template <typename T> __device__ __forceinline__ void load_row(const T *src, bool ok, uint4 (&v)[sizeof(T) / 2]) {
    #pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) v[k] = ok ? ld_cached(src + 4 * k) : make_uint4(0, 0, 0, 0);
}
template <typename T, int kPieces> __device__ __forceinline__ void row_pieces(const uint4 (&v)[sizeof(T) / 2], uint4 (&out)[kPieces]) {
    if constexpr (kPieces == 1) {
        out[0] = v[0];
    } else {
        float f[8];
        unpack<T>(v[0], f);
        if constexpr (sizeof(T) == 4) unpack<T>(v[1], f + 4);
        uint32_t r[4][kPieces];
        #pragma unroll
        for (int i = 0; i < 4; ++i) split_pair<kPieces>(make_float2(f[2 * i], f[2 * i + 1]), r[i]);
        #pragma unroll
        for (int k = 0; k < kPieces; ++k) out[k] = make_uint4(r[0][k], r[1][k], r[2][k], r[3][k]);
    }
}

// bytes (a multiple of 16, both ends 16-byte aligned) from shared to global memory by the copy engine
__device__ __forceinline__ void bulk_store(void *dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" :: "l"(dst), "r"(src), "r"(bytes) : "memory");
}
// the other way; the bytes count on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// 16 bytes from global to shared memory without registers; zeros where !ok
__device__ __forceinline__ void copy16_async(uint32_t at, const void *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(at), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Gates of a chunk.  G, the running sum of g, is kept as two floats: a
// difference G_i - G_j of near tokens far from the chunk's start keeps its relative accuracy.
// e^{G_i - G_j} for i in the 16 tokens of block I is row[i] * column[I][j] for j in an earlier block and
// row[i] * same[j] for j in the same one, all taken from the end of the block before I: row and column
// are below 1, same[j] above.  Where some block decays by more than e^-60, `steep` is set and products
// inside a block take an exponential of their own.
struct GdrGates {
    float2 g[kChunk];                 // high and low part of G
    float from_start[kChunk], to_end[kChunk], beta[kChunk], minus_beta_from_start[kChunk];
    float row[kChunk], same[kChunk], column[3][48];
    int steep;
    int bad;                          // first token whose row of A or T is not finite (64: none); such entries are left out
};
__device__ __forceinline__ float gdr_fade(float2 gi, float2 gj) { return gdr_exp((gi.x - gj.x) + (gi.y - gj.y)); }

}  // namespace cc1d

namespace cc1d {

// ---- a chunk made ready -------------------------------------------------------------------------
// What the walks over the chunks read of one chunk, as it lies in a stage of shared memory:
//   K, Q   token tiles, rows 0-63 k, 64-127 q (kPieces pieces), loaded by the walk itself
//   V      as it is, [64][128]                                                 "
//   T - I  T = (I + A)^-1, A_ij = beta_i (k_i.k_j) e^{G_i - G_j} for j < i   (kSolve pieces, row i, column j)
//   gates
//   P      (q_i.k_j) e^{G_i - G_j} for j <= i    (kOut pieces; kBack: the backward's, where P also leads to fp32
//          gradients, has all three)
// T, P and the gates are one image in the workspace, made by gdr_prep_kernel for all chunks at
// once (inside the walk their chain of short dependent steps, 13,000 cycles a chunk, held it up).
// The product with T is taken as x + (T - I) x, x in fp32: two pieces of both (the forward of 16-bit types) then leave
// 2^-17 of the correction alone, not of x.  The backward has three in every type: the gradients of g, of beta and of
// the state are fp32 (64 x 64 states of order one: 2.6e-6 of the largest off with two pieces, 5e-7 with three; both walks of
// 64 chunks 380 -> 404 us).
template <typename T, bool kBack> struct GdrStage {
    static constexpr int kPieces = GdrType<T>::kPieces, kOut = kBack ? 3 : GdrType<T>::kOutPieces, kSolve = kBack ? 3 : GdrType<T>::kSolve;
    static constexpr uint32_t kPanel = 128 * 128, kKqPiece = 2 * kPanel;     // panel: 128 rows x 64 columns
    static constexpr uint32_t kKq = 0, kV = kPieces * kKqPiece, kT = kV + kChunk * kGdrMaxDim * sizeof(T), kGates = kT + kSolve * 8192,
                              kP = kGates + 4096, kBytes = kP + kOut * 8192, kImage = kBytes - kT;
};
constexpr uint32_t kGateBytes = 2688;            // of the 4096 in an image, which align P (the preparation has them in shared memory besides: another 400 bytes would cost it a CTA an SM)
static_assert(sizeof(GdrGates) <= kGateBytes, "gates of a chunk");

// Chunks of sequence n in the workspace: slots gdr_first_slot(n) .. ; the slots of different sequences
// never meet (a sequence of L tokens takes ceil(L / 64) of the at least floor(L / 64) + 1 there are).
__host__ __device__ inline int64_t gdr_slots(const cc1d_gdr_params &p) {
    return p.cu_seqlens != nullptr ? p.seqlen / kChunk + p.nseq : p.batch * ((p.seqlen + kChunk - 1) / kChunk);
}
__device__ __forceinline__ int64_t gdr_first_slot(const cc1d_gdr_params &p, const GdrSeq &seq, int n) {
    return p.cu_seqlens != nullptr ? (int64_t)(seq.begin / kChunk) + n : n * ((p.seqlen + kChunk - 1) / kChunk);
}

// Sequence and place in it of a slot; false where the slot holds no chunk.
__device__ __forceinline__ bool gdr_find_chunk(const cc1d_gdr_params &p, int64_t slot, int &n, GdrSeq &seq, int &c) {
    n = 0;
    if (p.cu_seqlens == nullptr) {
        n = (int)(slot / ((p.seqlen + kChunk - 1) / kChunk));
    } else {
        if (p.nseq == 0) return false;         // all tokens are behind the last sequence
        int last = (int)p.nseq - 1;            // the last sequence whose first slot is not behind this one
        while (n < last) {
            const int mid = (n + last + 1) / 2;
            if (gdr_first_slot(p, gdr_sequence(p, mid), mid) <= slot) n = mid; else last = mid - 1;
        }
    }
    seq = gdr_sequence(p, n);
    c = (int)(slot - gdr_first_slot(p, seq, n));
    return c >= 0 && c < (seq.end - seq.begin + kChunk - 1) / kChunk;
}

// kN threads: rows t0 .. t0 + 63 of a tensor (those at or after `end` and columns at or after `cols` as
// zeros) into a token tile, one piece `piece_bytes` behind the other.
template <typename T, int NP, int kN>
__device__ __forceinline__ void load_tile(uint32_t dst, uint32_t panel_bytes, uint32_t piece_bytes, const T *src, int64_t step, int t0, int end, int cols, int tid) {
    const int row0 = tid >> 4, c8 = (tid & 15) * 8;
    #pragma unroll 4
    for (int i = 0; i < 1024 / kN; ++i) {
        const int row = row0 + kN / 16 * i;
        const int64_t t = t0 + row;
        const bool ok = t < end && c8 < cols;
        const uint32_t at = dst + tile_at(row, c8 / 8, panel_bytes);
        const T *from = ok ? src + t * step + c8 : src;
        if constexpr (NP == 1) {
            copy16_async(at, from, ok);
        } else {
            uint4 r[sizeof(T) / 2], pieces[NP];
            load_row<T>(from, ok, r);
            row_pieces<T, NP>(r, pieces);
            #pragma unroll
            for (int k = 0; k < NP; ++k) sts128(at + k * piece_bytes, pieces[k]);
        }
    }
}

// kN threads bring rows of q and k (and v) into their tiles: one-piece types by asynchronous
// copies, the others split on the way.  The caller waits for the copies and fences.
template <typename T, int kN> struct GdrRows {
    using S = GdrStage<T, false>;     // K, Q and V lie alike in both
    static constexpr int NP = S::kPieces, kVecs = sizeof(T) / 2;
    const T *kp, *qp, *vp;
    int64_t k_step, q_step, v_step;
    int end, dk, dv;
    // v: 64 x dim_v rows beside k and q (the values, or the output's gradient)
    __device__ __forceinline__ GdrRows(const cc1d_gdr_params &p, const GdrSeq &seq, int h, const void *v, int64_t v_row, int64_t v_step_)
        : k_step(p.k_l_stride), q_step(p.q_l_stride), v_step(v_step_), end(seq.end), dk((int)p.dim_k), dv((int)p.dim_v) {
        const int hk = h / (int)(p.heads_v / p.heads_k);
        kp = reinterpret_cast<const T *>(p.k) + seq.row * p.k_batch_stride + hk * p.k_h_stride;
        qp = reinterpret_cast<const T *>(p.q) + seq.row * p.q_batch_stride + hk * p.q_h_stride;
        vp = reinterpret_cast<const T *>(v) + v_row;
    }
    __device__ __forceinline__ void load_kq(uint32_t stage, int t0, int tid) const {
        load_tile<T, NP, kN>(stage + S::kKq, S::kPanel, S::kKqPiece, kp, k_step, t0, end, dk, tid);
        load_tile<T, NP, kN>(stage + S::kKq + 64 * 128, S::kPanel, S::kKqPiece, qp, q_step, t0, end, dk, tid);
    }
    __device__ __forceinline__ void load_v(uint32_t stage, int t0, int tid) const {
        const int row0 = tid >> 4, c8 = (tid & 15) * 8;
        #pragma unroll 4
        for (int i = 0; i < 1024 / kN; ++i) {
            const int row = row0 + kN / 16 * i;
            const int64_t t = t0 + row;
            const bool ok = t < end && c8 < dv;
            const T *src = ok ? vp + t * v_step + c8 : vp;
            #pragma unroll
            for (int k = 0; k < kVecs; ++k) copy16_async(stage + S::kV + (row * kGdrMaxDim + c8) * sizeof(T) + 16 * k, src + 4 * k, ok);
        }
    }
};

constexpr int kFeeders = 64;
// The last two warps of the forward walk: chunk after chunk into the stages.
// bar_full counts the threads and the one that announces the image.
template <typename T, int kStages, bool kBack, bool kWithP>
__device__ __forceinline__ void feed_walk(const GdrRows<T, kFeeders> &rows, const unsigned char *images, int64_t image_step, uint32_t smem, int begin, int chunks,
                                          uint32_t bar_full, uint32_t bar_empty, volatile int *dead, int tid) {
    using S = GdrStage<T, kBack>;
    constexpr uint32_t kBytes = kWithP ? S::kImage : S::kP - S::kT;      // without an output P is not needed
    for (int c = 0; c < chunks; ++c) {
        const int s = c % kStages;
        const uint32_t stage = smem + s * S::kBytes, full = bar_full + 8 * s;
        gdr_wait(bar_empty + 8 * s, ((c / kStages) & 1) ^ 1, dead);
        if (tid == 0) {
            mbar_expect_tx(full, kBytes);
            bulk_load(stage + S::kT, images + c * image_step, kBytes, full);
        }
        rows.load_kq(stage, begin + c * kChunk, tid);
        rows.load_v(stage, begin + c * kChunk, tid);
        copy_async_wait();
        fence_proxy_async_smem();
        mbar_arrive(full);
    }
}

// What the backward keeps of a chunk and value head, all fp32 and padded to 128 columns: the state before
// it, U, the gradient of the state behind it, and the gradient dB of R.
struct GdrRecord {
    float S0[kGdrMaxDim][kGdrMaxDim], U[kChunk][kGdrMaxDim], dS[kGdrMaxDim][kGdrMaxDim], dB[kChunk][kGdrMaxDim];
    int bad[32];              // first token that is not finite in columns 32 i .. (64: none), i < 4; the rest keeps records 128-byte aligned
};
// ---- long sequences of few heads ------------------------------------------------------------------
// A walk is one chain of chunks; where there are too few of them for the SMs, sequences are cut into segments
// of `per` chunks.  Through a segment the state goes as S -> M S + B: a first launch walks every segment from
// zeros (B) and, with no values, from the identity (M); the gradient of the state goes back as dS -> M^T dS +
// back.  A small kernel then carries the states from segment to segment, and the real walks start from those.
// per == 0: no segments, a walk is a whole sequence.
struct GdrSegment {
    float M[kGdrMaxDim][kGdrMaxDim], Mt[kGdrMaxDim][kGdrMaxDim], B[kGdrMaxDim][kGdrMaxDim], back[kGdrMaxDim][kGdrMaxDim];
    float start[kGdrMaxDim][kGdrMaxDim], end[kGdrMaxDim][kGdrMaxDim];     // the state it starts from; the gradient of the one it ends with
};
struct GdrSegments { GdrSegment *at; int per; bool ranked; };     // ranked: walks take the longest sequence first

// Segments of sequence n take slots gdr_first_segment(n) .., at least one each (as with the chunks' slots).
__host__ __device__ inline int64_t gdr_segment_slots(const cc1d_gdr_params &p, int per) { return gdr_slots(p) / per + gdr_sequences(p); }
__device__ __forceinline__ int64_t gdr_first_segment(const cc1d_gdr_params &p, const GdrSeq &seq, int n, int per) { return gdr_first_slot(p, seq, n) / per + n; }

// What one walk covers
struct GdrPart {
    GdrSeq seq;               // its tokens
    int n, chunks;
    int64_t slot;             // of its first chunk
    GdrSegment *segment;      // [heads_v], or NULL: the whole sequence
    bool first, last;         // of the sequence
};
__device__ __forceinline__ int gdr_chunks(const GdrSeq &seq) { return (seq.end - seq.begin + kChunk - 1) / kChunk; }

// Sequences by falling length (the whole CTA; `scratch`: kGdrRanked + 1 ints of its shared memory, free again on
// return): of walks that do not all fit the SMs at once the long ones should not start last.
constexpr int kGdrRanked = 64;
__device__ __forceinline__ int gdr_ranked(const cc1d_gdr_params &p, int rank, int *scratch) {
    const int n = (int)p.nseq, i = threadIdx.x;
    int mine = 0;
    if (i < n) {
        const GdrSeq seq = gdr_sequence(p, i);
        scratch[i] = mine = seq.end - seq.begin;
    }
    __syncthreads();
    if (i < n) {
        int before = 0;
        for (int j = 0; j < n; ++j) before += scratch[j] > mine || (scratch[j] == mine && j < i);
        if (before == rank) scratch[kGdrRanked] = i;
    }
    __syncthreads();
    const int at = scratch[kGdrRanked];
    __syncthreads();
    return at;
}
inline bool gdr_rank_walks(const cc1d_gdr_params &p, int per, int64_t ctas) {
    return per == 0 && p.cu_seqlens != nullptr && p.nseq > 1 && p.nseq <= kGdrRanked && ctas > num_sms();
}

// False: nothing to walk (the whole CTA leaves)
__device__ __forceinline__ bool gdr_find_part(const cc1d_gdr_params &p, const GdrSegments &segs, int64_t slot, GdrPart &w) {
    const int sequences = (int)gdr_sequences(p);
    w.segment = nullptr;
    w.first = w.last = true;
    if (segs.per == 0) {
        w.n = (int)slot;
        w.seq = {0, 0, 0};
        w.slot = 0;
        if (w.n < sequences) {
            w.seq = gdr_sequence(p, w.n);
            w.slot = gdr_first_slot(p, w.seq, w.n);
        }
        w.chunks = gdr_chunks(w.seq);
        return true;
    }
    int n = 0, last = sequences - 1;            // the last sequence whose first slot is not behind this one
    while (n < last) {
        const int mid = (n + last + 1) / 2;
        if (gdr_first_segment(p, gdr_sequence(p, mid), mid, segs.per) <= slot) n = mid; else last = mid - 1;
    }
    w.n = n;
    w.seq = gdr_sequence(p, n);
    const int chunks = gdr_chunks(w.seq), count = max(1, (chunks + segs.per - 1) / segs.per);
    const int64_t i = slot - gdr_first_segment(p, w.seq, n, segs.per);
    if (i < 0 || i >= count) return false;
    w.slot = gdr_first_slot(p, w.seq, n) + i * segs.per;
    w.segment = segs.at + slot * p.heads_v;
    w.first = i == 0;
    w.last = i + 1 == count;
    const int64_t begin = (int64_t)w.seq.begin + i * segs.per * kChunk;
    w.seq.end = (int32_t)min((int64_t)w.seq.end, begin + (int64_t)segs.per * kChunk);
    w.seq.begin = (int32_t)begin;
    w.chunks = gdr_chunks(w.seq);
    return true;
}

int gdr_plan_segments(const cc1d_gdr_params &p, bool back);          // chunks of a segment, or 0
int launch_gdr_join(const cc1d_gdr_params &p, const GdrSegments &segs, const float *dfinal_states, bool back, cudaStream_t stream);
size_t gdr_image_bytes(const cc1d_gdr_params &p, bool back);          // of all chunks
int launch_gdr_prep(const cc1d_gdr_params &p, bool back, void *images, cudaStream_t stream);

}  // namespace cc1d
