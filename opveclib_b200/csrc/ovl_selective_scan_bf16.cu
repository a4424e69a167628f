// The selective scan's kernels for bfloat16 tensors.
#include "ovl_selective_scan.cuh"

namespace ovl {
int scan_run_bf16(const ScanParams& p, const ScanShape& s, bool backward, cudaStream_t stream) {
    return scan_dispatch<__nv_bfloat16>(p, s, backward, stream);
}
int scan_step_bf16(const OvlSelectiveScanStep& a, int lanes, cudaStream_t stream) {
    return scan_step_dispatch<__nv_bfloat16>(a, lanes, stream);
}
}  // namespace ovl
