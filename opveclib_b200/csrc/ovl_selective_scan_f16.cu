// The selective scan's kernels for float16 tensors.
#include "ovl_selective_scan.cuh"

namespace ovl {
int scan_run_f16(const ScanParams& p, const ScanShape& s, bool backward, cudaStream_t stream) {
    return scan_dispatch<__half>(p, s, backward, stream);
}
int scan_step_f16(const OvlSelectiveScanStep& a, int lanes, cudaStream_t stream) {
    return scan_step_dispatch<__half>(a, lanes, stream);
}
}  // namespace ovl
