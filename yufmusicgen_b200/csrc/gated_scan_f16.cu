// The gated recurrence's kernels for fp16 tensors.
#include "gated_scan_kernels.cuh"

namespace yuf {

yuf_status_t gated_scan_f16(const GatedScanArgs& a, bool backward, cudaStream_t st) {
  return gated_scan_pairs(a) ? run_as<__half, 2>(a, backward, st) : run_as<__half, 1>(a, backward, st);
}
unsigned int gated_scan_wait_timeouts_f16() { return wait_timeouts(); }

}  // namespace yuf
