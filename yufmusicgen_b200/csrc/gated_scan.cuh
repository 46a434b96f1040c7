// Arguments of the gated recurrence's kernels (gated_scan_kernels.cuh) and of dropout
// (dropout.cu), filled by the C ABI (capi.cu), and what their host sides share.
#pragma once
#include "common.cuh"

namespace yuf {

struct GatedScanArgs {
  const void *x, *f, *g, *dy;                        // inputs; g and dy may be NULL
  long long xb, xt, fb, ft, gb, gt, yb, yt;          // batch and token strides of x, f, g, dy (elements)
  const float *lower, *h0;                           // [D], [rows, D]; NULL = zeros
  const int* cu;                                     // [n_seqs + 1] or NULL
  int n_seqs;
  int B, T, D;
  int dtype;
  // forward
  void* y;
  float *h_last, *ckpt;                              // either may be NULL (ckpt is an input of the backward)
  // backward
  const float* dh_last;                              // NULL = zeros
  void *dx, *df, *dg;
  float *dlower, *dh0;
  float* partial;                                    // set from work by the dispatch
  float* work;                                       // gated_scan_workspace_floats
};

// tokens between two saved states
constexpr int GATED_SCAN_BLOCK = 16;
constexpr int GATED_SCAN_WARPS = 16;       // warps per block, at most
constexpr int GATED_SCAN_RANGE_WARPS = 4;  // warps per block of ranges

// How a call shares out its work (gated_scan_kernels.cuh).
struct GatedScanSplit {
  int n_cblk, chunks, runs;  // channel blocks; blocks per column; runs per warp of ranges
};
struct GatedScanPlan {
  GatedScanSplit sp;
  int nw;  // warps per block
  bool ranges;
  long long cols, blocks;
  // floats of the ranges' maps: a row for each warp and one for each block
  long long map_floats(int V) const { return ranges ? cols * sp.chunks * (nw + 1) * 64 * V : 0; }
};
GatedScanPlan gated_scan_plan(int B, int T, int D, int V);
bool gated_scan_pairs(const GatedScanArgs& a);
yuf_status_t gated_scan_dlower(const float* partial, float* dlower, long long rows, int D, cudaStream_t st);
inline bool gated_aligned(const void* q, size_t bytes) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; }
inline int gated_elem_size(int dtype) { return dtype == YUF_DTYPE_F32 ? 4 : 2; }

size_t gated_scan_workspace_floats(int B, int T, int D, int dtype, bool backward);

yuf_status_t gated_scan_forward(const GatedScanArgs& a, cudaStream_t st);
yuf_status_t gated_scan_backward(const GatedScanArgs& a, cudaStream_t st);
yuf_status_t gated_scan_step(const void* x, const void* f, const void* g, long long xs, long long fs,
                             long long gs, const float* lower, float* state, long long ss, void* y, int dtype,
                             int B, int D, cudaStream_t st);

struct DropoutArgs {
  const void *x, *res;        // res may be NULL
  void* out;
  long long xs, rs;           // row strides of x and res (out is contiguous)
  long long rows, cols;
  int x_dtype, out_dtype;     // res has out's type
  uint32_t last_dropped;      // an element is dropped when any && its word <= last_dropped
  bool any;
  float scale;
  uint64_t seed, step;
  const uint64_t* step_ptr;   // device; overrides step when not NULL
};
yuf_status_t dropout_forward(const DropoutArgs& a, cudaStream_t st);

}  // namespace yuf
