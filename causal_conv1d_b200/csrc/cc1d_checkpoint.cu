// x kept in 8 bits (include/cc1d_checkpoint.h): the calls, and the kernels for what the convolution's own
// kernels do not do on their way.
#include "cc1d_checkpoint.cuh"
#include "cc1d_kernels.h"

namespace cc1d {
namespace {

// x as rows along its contiguous axis: (batch, dim) rows of seqlen, or (batch, seqlen) rows of dim
struct CodeArgs {
    const void *x;
    void *restored;
    uint8_t *codes, *scales;
    int64_t batch_stride, row_stride;
    uint64_t rows;
    uint32_t inner, cols, groups, threads_per_row;   // rows of one batch entry; groups and threads (4 a group) of a row
    uint64_t threads;
    bool vectors, code_vectors;                      // 16-byte access to x, 8-byte access to the codes
};

template <typename T> __device__ __forceinline__ bool place(const CodeArgs &a, uint64_t &row, uint32_t &col, int64_t &at) {
    uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const bool there = i < a.threads;
    if (!there) i = 0;
    uint64_t b;
    uint32_t in_batch;
    if (a.threads < (1ull << 32)) {
        row = (uint32_t)i / a.threads_per_row;
        b = (uint32_t)row / a.inner;
    } else {
        row = i / a.threads_per_row;
        b = row / a.inner;
    }
    in_batch = (uint32_t)(row - b * a.inner);
    col = (uint32_t)(i - row * a.threads_per_row) * 8;
    at = (int64_t)b * a.batch_stride + (int64_t)in_batch * a.row_stride + col;
    return there;
}

// A thread per 8 values, 4 neighbouring lanes per group; bound by the bytes (an element's size + 1).
template <typename T> __global__ void __launch_bounds__(256) checkpoint_kernel(const CodeArgs a) {
    pdl_wait();
    uint64_t row;
    uint32_t col;
    int64_t at;
    const bool there = place<T>(a, row, col, at);
    const T *x = reinterpret_cast<const T *>(a.x) + at;
    float f[8];
    if (there && a.vectors && col + 8 <= a.cols) {
        unpack<T>(ld_stream(x), f);
        if constexpr (sizeof(T) == 4) unpack<T>(ld_stream(x + 4), f + 4);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = there && col + i < a.cols ? Elem<T>::to_f(x[i]) : 0.f;
    }
    float most = 0.f;
    #pragma unroll
    for (int i = 0; i < 8; ++i) most = max_abs(most, f[i]);
    most = max_abs(most, __shfl_xor_sync(kFullMask, most, 1));
    most = max_abs(most, __shfl_xor_sync(kFullMask, most, 2));
    const uint32_t s = code_scale(most);
    const float inv = scale_inverse(s);
    const uint2 codes = make_uint2(to_codes(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), to_codes(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
    if (!there || col >= a.cols) return;
    uint8_t *dst = a.codes + row * a.cols + col;
    if (a.code_vectors && col + 8 <= a.cols) {
        st_stream_raw(dst, codes);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) if (col + i < a.cols) dst[i] = (uint8_t)((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
    }
    if ((threadIdx.x & 3) == 0) a.scales[row * a.groups + col / kCodeGroup] = (uint8_t)s;
}

template <typename T> __global__ void __launch_bounds__(256) restore_kernel(const CodeArgs a) {
    pdl_wait();
    uint64_t row;
    uint32_t col;
    int64_t at;
    if (!place<T>(a, row, col, at) || col >= a.cols) return;
    const uint8_t *src = a.codes + row * a.cols + col;
    uint2 codes = make_uint2(0, 0);
    if (a.code_vectors && col + 8 <= a.cols) {
        ld_stream_raw(codes, src);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) if (col + i < a.cols) (i < 4 ? codes.x : codes.y) |= (uint32_t)src[i] << (8 * (i & 3));
    }
    const float s = scale_value(a.scales[row * a.groups + col / kCodeGroup]);
    float f[8];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = fit<T>(from_codes((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)), s));
        f[2 * i] = v.x; f[2 * i + 1] = v.y;
    }
    T *x = reinterpret_cast<T *>(a.restored) + at;
    if (a.vectors && col + 8 <= a.cols) {
        *reinterpret_cast<uint4 *>(x) = pack<T>(f);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(x + 4) = pack<T>(f + 4);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) if (col + i < a.cols) x[i] = Elem<T>::from_f(f[i]);
    }
}

bool channel_last(int64_t c_stride, int64_t l_stride) { return c_stride == 1 && l_stride > 1; }

int code_args(CodeArgs &a, int itype, int64_t batch, int64_t dim, int64_t seqlen, const void *x, int64_t bs, int64_t cs, int64_t ls, const cc1d_codes *c) {
    if (itype != CC1D_F32 && itype != CC1D_F16 && itype != CC1D_BF16) return CC1D_ERR_DTYPE;
    if (batch < 0 || dim < 0 || seqlen < 0) return CC1D_ERR_SHAPE;
    if (cs != 1 && ls != 1) return CC1D_ERR_STRIDE;
    if (seqlen >= (1ll << 31) - 4096 || dim >= (1ll << 31) - 4096) return CC1D_ERR_TOO_LARGE;
    const bool cl = channel_last(cs, ls);
    if (!cl && ls != 1 && seqlen > 1) return CC1D_ERR_STRIDE;
    a.x = x; a.restored = const_cast<void *>(x);
    a.codes = c->codes; a.scales = c->scales;
    a.inner = (uint32_t)(cl ? seqlen : dim); a.cols = (uint32_t)(cl ? dim : seqlen);
    a.batch_stride = batch > 1 ? bs : 0; a.row_stride = a.inner > 1 ? (cl ? ls : cs) : 0;
    a.rows = (uint64_t)batch * a.inner;
    a.groups = (a.cols + kCodeGroup - 1) / kCodeGroup;
    a.threads_per_row = 4 * a.groups;
    a.threads = a.rows * a.threads_per_row;
    a.vectors = is_aligned16(x) && a.batch_stride % vec_elems(itype) == 0 && a.row_stride % vec_elems(itype) == 0;
    a.code_vectors = a.cols % 8 == 0;
    if (a.threads > 0 && (c->codes == nullptr || c->scales == nullptr || x == nullptr)) return CC1D_ERR_NULL;
    if (!is_aligned16(c->codes) || reinterpret_cast<uintptr_t>(x) % elem_size(itype) != 0) return CC1D_ERR_ALIGN;
    if ((a.threads + 255) / 256 >= (1ull << 31)) return CC1D_ERR_TOO_LARGE;
    return CC1D_OK;
}

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int cc1d_checkpoint_e4m3(const cc1d_fwd_params *p, const cc1d_codes *to, cc1d_stream_t stream) {
    if (p == nullptr || to == nullptr) return CC1D_ERR_NULL;
    CodeArgs a;
    const int rc = code_args(a, p->itype, p->batch, p->dim, p->seqlen, p->x, p->x_batch_stride, p->x_c_stride, p->x_l_stride, to);
    if (rc != CC1D_OK || a.threads == 0) return rc;
    CC1D_DISPATCH_ITYPE(p->itype, {
        launch_k(checkpoint_kernel<T>, dim3((unsigned)((a.threads + 255) / 256)), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), a);
    });
    return check_launch();
}

int cc1d_restore_e4m3(const cc1d_fwd_params *p, void *x, const cc1d_codes *from, cc1d_stream_t stream) {
    if (p == nullptr || from == nullptr) return CC1D_ERR_NULL;
    CodeArgs a;
    const int rc = code_args(a, p->itype, p->batch, p->dim, p->seqlen, x, p->x_batch_stride, p->x_c_stride, p->x_l_stride, from);
    if (rc != CC1D_OK || a.threads == 0) return rc;
    CC1D_DISPATCH_ITYPE(p->itype, {
        launch_k(restore_kernel<T>, dim3((unsigned)((a.threads + 255) / 256)), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), a);
    });
    return check_launch();
}

// In the convolution's own kernel where that can, else behind it; the convolution's checks come first.
int cc1d_fwd_e4m3(const cc1d_fwd_params *p, const cc1d_codes *to, cc1d_stream_t stream) {
    if (p == nullptr || to == nullptr) return CC1D_ERR_NULL;
    if (!is_aligned16(to->codes)) return CC1D_ERR_ALIGN;
    if (p->batch > 0 && p->dim > 0 && p->seqlen > 0 && (to->codes == nullptr || to->scales == nullptr)) return CC1D_ERR_NULL;
    bool kept = false;
    const int rc = cc1d_fwd_keeping(p, to, &kept, stream);
    if (rc != CC1D_OK || kept) return rc;
    return cc1d_checkpoint_e4m3(p, to, stream);
}

// A backward whose x lies dense at `x` (codes themselves where they are read as they are)
static cc1d_bwd_params with_dense_x(const cc1d_bwd_params &p, const void *x) {
    cc1d_bwd_params q = p;
    q.x = x;
    q.x_batch_stride = p.dim * p.seqlen;
    if (channel_last(p.x_c_stride, p.x_l_stride)) { q.x_c_stride = 1; q.x_l_stride = p.dim; }
    else { q.x_c_stride = p.seqlen; q.x_l_stride = 1; }
    return q;
}

static bool reads_codes(const cc1d_bwd_params &p) {
    return channel_last(p.x_c_stride, p.x_l_stride) ? bwd_cl_reads_codes(p) : bwd_reads_codes(p);
}

size_t cc1d_bwd_e4m3_restore_bytes(const cc1d_bwd_params *p) {
    if (p == nullptr || p->batch < 0 || p->dim < 0 || p->seqlen < 0) return 0;
    if (reads_codes(*p)) return 0;
    return (size_t)p->batch * (size_t)p->dim * (size_t)p->seqlen * (size_t)elem_size(p->itype);
}

int cc1d_bwd_e4m3(const cc1d_bwd_params *p, const cc1d_codes *from, void *restored, cc1d_stream_t stream) {
    if (p == nullptr || from == nullptr) return CC1D_ERR_NULL;
    const bool some = p->batch > 0 && p->dim > 0 && p->seqlen > 0;
    if (some && (from->codes == nullptr || from->scales == nullptr)) return CC1D_ERR_NULL;
    if (!is_aligned16(from->codes)) return CC1D_ERR_ALIGN;
    if (reads_codes(*p)) {
        const cc1d_bwd_params q = with_dense_x(*p, from->codes);
        return cc1d_bwd_reading(&q, from, stream);
    }
    if (some && restored == nullptr) return CC1D_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(restored) & 31u) != 0) return CC1D_ERR_ALIGN;
    const cc1d_bwd_params q = with_dense_x(*p, restored);
    const int checked = cc1d_bwd_check(&q);       // before anything is launched
    if (checked != CC1D_OK) return checked;
    if (some && p->phase != 2) {
        cc1d_fwd_params f = {};
        f.itype = p->itype; f.batch = p->batch; f.dim = p->dim; f.seqlen = p->seqlen;
        f.x_batch_stride = q.x_batch_stride; f.x_c_stride = q.x_c_stride; f.x_l_stride = q.x_l_stride;
        const int rc = cc1d_restore_e4m3(&f, restored, from, stream);
        if (rc != CC1D_OK) return rc;
    }
    return cc1d_bwd(&q, stream);
}

}  // extern "C"
