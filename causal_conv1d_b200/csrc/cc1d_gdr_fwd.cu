// Gated delta rule over whole sequences: cc1d_gdr_fwd (include/cc1d_gdr.h).
#include "cc1d_gdr_walk.cuh"

namespace cc1d {
namespace {

template <typename T, int kSteps>
__global__ void __launch_bounds__(kWalkThreads, 1) gdr_fwd_kernel(const __grid_constant__ cc1d_gdr_params p, const unsigned char *images, const GdrSegments segs) {
    walk_forward<T, kSteps, kOutput, false>(p, images, nullptr, segs, blockIdx.x, false);
}

// half of the CTAs B, half M
template <typename T, int kSteps>
__global__ void __launch_bounds__(kWalkThreads, 1) gdr_fwd_summary_kernel(const __grid_constant__ cc1d_gdr_params p, const unsigned char *images, const GdrSegments segs, unsigned walks) {
    const bool unit = blockIdx.x >= walks;
    walk_forward<T, kSteps, kSummary, false>(p, images, nullptr, segs, unit ? blockIdx.x - walks : blockIdx.x, unit);
}

size_t images_bytes(const cc1d_gdr_params &p) { return (gdr_image_bytes(p, false) + 255) / 256 * 256; }

}  // namespace

size_t gdr_fwd_workspace_bytes(const cc1d_gdr_params &p) {
    const int per = gdr_plan_segments(p, false);
    return images_bytes(p) + (per > 0 ? (size_t)gdr_segment_slots(p, per) * (size_t)p.heads_v * sizeof(GdrSegment) : 0);
}

int launch_gdr_fwd(const cc1d_gdr_params &p, cudaStream_t stream) {
    unsigned char *images = reinterpret_cast<unsigned char *>(p.workspace);
    GdrSegments segs = {reinterpret_cast<GdrSegment *>(images + images_bytes(p)), gdr_plan_segments(p, false), false};
    const int64_t sequences = gdr_sequences(p), walks = (segs.per > 0 ? gdr_segment_slots(p, segs.per) : sequences > 0 ? sequences : 1) * p.heads_v;
    if (walks >= (1ll << 30)) return CC1D_ERR_TOO_LARGE;
    segs.ranked = gdr_rank_walks(p, segs.per, walks);
    int rc = launch_gdr_prep(p, false, images, stream);
    if (rc != CC1D_OK) return rc;
    CC1D_DISPATCH_ITYPE(p.itype, {
        CC1D_DISPATCH_BOOL(p.dim_k <= 64, kNarrow, {
            constexpr int kSteps = kNarrow ? 4 : 8;     // contraction steps of 16 over dim_k
            constexpr uint32_t kBytes = Fwd<T, false>::kBytes;
            if (segs.per > 0) {
                allow_dynamic_smem(reinterpret_cast<const void *>(gdr_fwd_summary_kernel<T, kSteps>), kBytes);
                launch_k(gdr_fwd_summary_kernel<T, kSteps>, dim3((unsigned)(2 * walks)), dim3(kWalkThreads), kBytes, stream, p, (const unsigned char *)images, segs, (unsigned)walks);
                rc = launch_gdr_join(p, segs, nullptr, false, stream);
                if (rc != CC1D_OK) return rc;
            }
            allow_dynamic_smem(reinterpret_cast<const void *>(gdr_fwd_kernel<T, kSteps>), kBytes);
            launch_k(gdr_fwd_kernel<T, kSteps>, dim3((unsigned)walks), dim3(kWalkThreads), kBytes, stream, p, (const unsigned char *)images, segs);
        });
    });
    return check_launch();
}

int gdr_fwd_wait_expired() { return read_and_clear_wait_expired(); }

}  // namespace cc1d
