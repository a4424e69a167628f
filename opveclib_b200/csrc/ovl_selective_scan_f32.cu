// The selective scan's kernels for float32 tensors.
#include "ovl_selective_scan.cuh"

namespace ovl {
int scan_run_f32(const ScanParams& p, const ScanShape& s, bool backward, cudaStream_t stream) {
    return scan_dispatch<float>(p, s, backward, stream);
}
int scan_step_f32(const OvlSelectiveScanStep& a, int lanes, cudaStream_t stream) {
    return scan_step_dispatch<float>(a, lanes, stream);
}
}  // namespace ovl
