// The gated recurrence's kernels for fp32 tensors.
#include "gated_scan_kernels.cuh"

namespace yuf {

yuf_status_t gated_scan_f32(const GatedScanArgs& a, bool backward, cudaStream_t st) {
  return run_as<float, 1>(a, backward, st);
}
unsigned int gated_scan_wait_timeouts_f32() { return wait_timeouts(); }

}  // namespace yuf
