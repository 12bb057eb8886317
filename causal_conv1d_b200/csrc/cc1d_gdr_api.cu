// extern "C" entry points of the gated delta rule (include/cc1d_gdr.h): validation and hand-off.
#include "cc1d.h"
#include "cc1d_gdr.cuh"
#include "cc1d_kernels.h"

namespace cc1d {
namespace {

bool bad_dtype(int d) { return d != CC1D_F32 && d != CC1D_F16 && d != CC1D_BF16; }
bool elem_aligned(const void *p, int dtype) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)elem_size(dtype)) == 0; }

int check_gdr(const cc1d_gdr_params &p) {
    if (bad_dtype(p.itype) || bad_dtype(p.gtype) || bad_dtype(p.btype)) return CC1D_ERR_DTYPE;
    if (p.batch < 0 || p.seqlen < 0 || p.nseq < 0 || p.heads_k < 0 || p.heads_v < 0) return CC1D_ERR_SHAPE;
    if (p.dim_k < 8 || p.dim_k > kGdrMaxDim || p.dim_k % 8 || p.dim_v < 8 || p.dim_v > kGdrMaxDim || p.dim_v % 8) return CC1D_ERR_GDR_DIM;
    if (p.heads_k < 1 || p.heads_v < 1 || p.heads_v % p.heads_k != 0) return CC1D_ERR_GDR_HEADS;
    if (p.seqlen >= (1ll << 31) - 4096 || p.heads_v >= (1 << 20) || p.batch >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    if (p.initial_states != nullptr && (!is_aligned16(p.initial_states) || p.initial_states_batch_stride % 4 || p.initial_states_h_stride % 4)) return CC1D_ERR_ALIGN;
    if (p.final_states != nullptr && (!is_aligned16(p.final_states) || p.final_states_batch_stride % 4 || p.final_states_h_stride % 4)) return CC1D_ERR_ALIGN;
    return CC1D_OK;
}

int check_tensors(const cc1d_gdr_params &p) {
    if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.g == nullptr || p.beta == nullptr || p.out == nullptr) return CC1D_ERR_NULL;
    if (!elem_aligned(p.q, p.itype) || !elem_aligned(p.k, p.itype) || !elem_aligned(p.v, p.itype) || !elem_aligned(p.out, p.itype) ||
        !elem_aligned(p.g, p.gtype) || !elem_aligned(p.beta, p.btype)) return CC1D_ERR_ALIGN;
    return CC1D_OK;
}

// what the chunked kernels' 16-byte loads need
bool rows_aligned(const void *t, int64_t bs, int64_t ls, int64_t hs, int64_t batch, int64_t seqlen, int64_t heads, int dtype) {
    const int v = vec_elems(dtype);
    return is_aligned16(t) && (batch <= 1 || bs % v == 0) && (seqlen <= 1 || ls % v == 0) && (heads <= 1 || hs % v == 0);
}

int check_whole(const cc1d_gdr_params &p) {
    int rc = check_gdr(p);
    if (rc != CC1D_OK) return rc;
    if (p.cu_seqlens != nullptr && p.batch != 1) return CC1D_ERR_SHAPE;
    if (p.cu_seqlens == nullptr && p.nseq != 0) return CC1D_ERR_NULL;
    return CC1D_OK;
}

int check_rows(const cc1d_gdr_params &p) {
    if (!rows_aligned(p.q, p.q_batch_stride, p.q_l_stride, p.q_h_stride, p.batch, p.seqlen, p.heads_k, p.itype) ||
        !rows_aligned(p.k, p.k_batch_stride, p.k_l_stride, p.k_h_stride, p.batch, p.seqlen, p.heads_k, p.itype) ||
        !rows_aligned(p.v, p.v_batch_stride, p.v_l_stride, p.v_h_stride, p.batch, p.seqlen, p.heads_v, p.itype)) return CC1D_ERR_ALIGN;
    return CC1D_OK;
}

}  // namespace

int gdr_prep_wait_expired();   // per translation unit
int gdr_fwd_wait_expired();
int gdr_bwd_wait_expired();
int gdr_wait_expired() {
    const int a = gdr_prep_wait_expired(), b = gdr_fwd_wait_expired(), c = gdr_bwd_wait_expired();
    return a < 0 || b < 0 || c < 0 ? -1 : a | b | c;
}

}  // namespace cc1d

using namespace cc1d;

extern "C" {

int cc1d_gdr_update(const cc1d_gdr_params *p, cc1d_stream_t stream) {
    if (p == nullptr) return CC1D_ERR_NULL;
    cc1d_gdr_params a = *p;
    a.initial_states = nullptr; a.cu_seqlens = nullptr; a.has_initial_state = nullptr;
    int rc = check_gdr(a);
    if (rc != CC1D_OK) return rc;
    if (a.batch == 0 || a.seqlen == 0) return CC1D_OK;
    rc = check_tensors(a);
    if (rc != CC1D_OK) return rc;
    if (a.final_states == nullptr) return CC1D_ERR_NULL;
    return launch_gdr_update(a, reinterpret_cast<cudaStream_t>(stream));
}

size_t cc1d_gdr_fwd_workspace_bytes(const cc1d_gdr_params *p) {
    if (p == nullptr || check_whole(*p) != CC1D_OK) return 0;
    return gdr_fwd_workspace_bytes(*p);
}

int cc1d_gdr_fwd(const cc1d_gdr_params *p, cc1d_stream_t stream) {
    if (p == nullptr) return CC1D_ERR_NULL;
    int rc = check_whole(*p);
    if (rc != CC1D_OK) return rc;
    const int64_t sequences = gdr_sequences(*p);
    if (p->seqlen == 0 || p->batch == 0) {
        // no tokens: nothing but the states of empty sequences, which the kernel copies
        if (sequences == 0 || p->final_states == nullptr) return CC1D_OK;
    } else {
        rc = check_tensors(*p);
        if (rc == CC1D_OK) rc = check_rows(*p);
        if (rc == CC1D_OK && !rows_aligned(p->out, p->out_batch_stride, p->out_l_stride, p->out_h_stride, p->batch, p->seqlen, p->heads_v, p->itype)) rc = CC1D_ERR_ALIGN;
        if (rc != CC1D_OK) return rc;
    }
    const size_t need = gdr_fwd_workspace_bytes(*p);
    if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || !is_aligned16(p->workspace))) return CC1D_ERR_WORKSPACE;
    return launch_gdr_fwd(*p, reinterpret_cast<cudaStream_t>(stream));
}

size_t cc1d_gdr_bwd_workspace_bytes(const cc1d_gdr_bwd_params *p) {
    if (p == nullptr || check_whole(p->fwd) != CC1D_OK) return 0;
    return gdr_bwd_workspace_bytes(*p);
}

int cc1d_gdr_bwd(const cc1d_gdr_bwd_params *p, cc1d_stream_t stream) {
    if (p == nullptr) return CC1D_ERR_NULL;
    const cc1d_gdr_params &f = p->fwd;
    int rc = check_whole(f);
    if (rc != CC1D_OK) return rc;
    if (f.seqlen == 0 || f.batch == 0) {
        if (gdr_sequences(f) == 0 || p->dinitial_states == nullptr) return CC1D_OK;
    } else {
        if (f.q == nullptr || f.k == nullptr || f.v == nullptr || f.g == nullptr || f.beta == nullptr || p->dout == nullptr || p->dq == nullptr ||
            p->dk == nullptr || p->dv == nullptr || p->dg == nullptr || p->dbeta == nullptr) return CC1D_ERR_NULL;
        if (!elem_aligned(f.g, f.gtype) || !elem_aligned(f.beta, f.btype) || !elem_aligned(p->dg, f.gtype) || !elem_aligned(p->dbeta, f.btype)) return CC1D_ERR_ALIGN;
        rc = check_rows(f);
        if (rc != CC1D_OK) return rc;
        if (!rows_aligned(p->dout, p->dout_batch_stride, p->dout_l_stride, p->dout_h_stride, f.batch, f.seqlen, f.heads_v, f.itype) ||
            !is_aligned16(p->dq) || !is_aligned16(p->dk) || !is_aligned16(p->dv)) return CC1D_ERR_ALIGN;
    }
    const size_t need = gdr_bwd_workspace_bytes(*p);
    if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || !is_aligned16(p->workspace))) return CC1D_ERR_WORKSPACE;
    return launch_gdr_bwd(*p, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
