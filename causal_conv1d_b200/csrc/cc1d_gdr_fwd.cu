// Gated delta rule over whole sequences: cc1d_gdr_fwd (include/cc1d_gdr.h).
#include "cc1d_gdr_walk.cuh"

namespace cc1d {
namespace {

template <typename T, int kSteps>
__global__ void __launch_bounds__(kWalkThreads, 1) gdr_fwd_kernel(const __grid_constant__ cc1d_gdr_params p, const unsigned char *images) {
    walk_forward<T, kSteps, false>(p, images, nullptr, blockIdx.x);
}

}  // namespace

size_t gdr_fwd_workspace_bytes(const cc1d_gdr_params &p) { return gdr_image_bytes(p, false); }

int launch_gdr_fwd(const cc1d_gdr_params &p, cudaStream_t stream) {
    const int64_t sequences = gdr_sequences(p), ctas = (sequences > 0 ? sequences : 1) * p.heads_v;
    if (ctas >= (1ll << 31)) return CC1D_ERR_TOO_LARGE;
    const int rc = launch_gdr_prep(p, false, p.workspace, stream);
    if (rc != CC1D_OK) return rc;
    CC1D_DISPATCH_ITYPE(p.itype, {
        CC1D_DISPATCH_BOOL(p.dim_k <= 64, kNarrow, {
            constexpr int kSteps = kNarrow ? 4 : 8;     // contraction steps of 16 over dim_k
            constexpr uint32_t kBytes = Fwd<T, false>::kBytes;
            allow_dynamic_smem(reinterpret_cast<const void *>(gdr_fwd_kernel<T, kSteps>), kBytes);
            launch_k(gdr_fwd_kernel<T, kSteps>, dim3((unsigned)ctas), dim3(kWalkThreads), kBytes, stream, p, reinterpret_cast<const unsigned char *>(p.workspace));
        });
    });
    return check_launch();
}

int gdr_fwd_wait_expired() { return read_and_clear_wait_expired(); }

}  // namespace cc1d
