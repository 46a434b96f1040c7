// The gated recurrence's host side (which form a call takes, sizes of its workspace)
// and its small kernels: the sum of dlower's shares and the single-token form.  The
// scans themselves are in gated_scan_kernels.cuh.
#include "gated_scan.cuh"

#include "io_types.cuh"

namespace yuf {

constexpr int SMS = 148;
// Which form, by the number of columns (blocks that the whole form has) and T.
// A step of the whole form takes about 3.3 us forward whatever the columns, while
// every SM has at most one block; ranges cost by the element, and 3 us more for their
// second launch.  Measured (bf16, forward / backward, us; whole against ranges):
//   32 columns x 4096 tokens 58 / 91 against 31 / 48;  64 x 4096 58 / 91 : 53 / 80;
//   96 x 4096 60 / 93 : 64 / 108;  128 x 4096 62 / 97 : 93 / 147;
//   40 x 1024 21 / 34 : 19 / 30;  40 x 256 11 / 19 : 13 / 20;  10 x 256 11 / 19 : 11 / 17
// (pairs of channels with a gate, not packed; the other types and packed rows follow the
// same rule without having been measured on both sides).
GatedScanPlan gated_scan_plan(int B, int T, int D, int V) {
  constexpr int L = GATED_SCAN_BLOCK;
  GatedScanPlan p;
  p.sp.n_cblk = (D + 32 * V - 1) / (32 * V);
  p.cols = (long long)B * p.sp.n_cblk;
  p.ranges = (72 - p.cols) * T >= 19000;
  if (p.ranges) {
    // One range for each warp that fits (the slots of 16 warps fill an SM's shared
    // memory); blocks of 4 warps, which leave fewer idle at the end than 8.
    p.nw = GATED_SCAN_RANGE_WARPS;
    const long long runs = (p.cols * T + (long long)L * SMS * 16 - 1) / ((long long)L * SMS * 16);
    p.sp.runs = (int)max(1LL, runs);
    p.sp.chunks = (T + p.nw * L * p.sp.runs - 1) / (p.nw * L * p.sp.runs);
  } else {
    // Up to one block per SM: as many warps as its registers hold.  More blocks: two
    // to an SM, whose phases then overlap (160 columns x 4096: 103 against 113 us).
    const int most = p.cols <= SMS ? GATED_SCAN_WARPS : GATED_SCAN_WARPS / 2;
    p.nw = max(1, min(most, (T + L - 1) / L));
    p.sp.runs = 0;
    p.sp.chunks = 1;
  }
  p.blocks = p.cols * p.sp.chunks;
  return p;
}

// Two channels per lane, 4 bytes of a 16-bit type: even widths and strides, every row
// start aligned to a pair.  fp32 takes one channel, the same 4 bytes.
bool gated_scan_pairs(const GatedScanArgs& a) {
  if (a.dtype == YUF_DTYPE_F32) return false;
  const size_t e = 2 * gated_elem_size(a.dtype);
  const void* t[] = {a.x, a.f, a.g, a.dy, a.y, a.dx, a.df, a.dg};
  const float* s[] = {a.lower, a.h0, a.h_last, a.ckpt, a.dh_last, a.dh0};
  bool ok = a.D % 2 == 0 && ((a.xb | a.xt | a.fb | a.ft | a.gb | a.gt | a.yb | a.yt) & 1) == 0;
  for (const void* q : t) ok = ok && gated_aligned(q, e);
  for (const float* q : s) ok = ok && gated_aligned(q, 8);
  return ok;
}

namespace {

// dlower[c] = sum over rows of partial[rows, D], in 64 bits and a fixed order: 32 warps a block,
// each every 32nd row, as many loads under way as there are rows (592 rows: 3.5 us;
// 5 us with 8 warps)
__global__ void __launch_bounds__(1024)
    gated_scan_dlower_kernel(const float* __restrict__ partial, float* __restrict__ out, long long rows, int D) {
  __shared__ double part[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double sum = 0.;
  if (c < D) {
#pragma unroll 4
    for (long long r = w; r < rows; r += 32) sum += partial[r * D + c];
  }
  part[w][lane] = sum;
  __syncthreads();
  sum = part[lane][w];  // warp w: channel w of the block
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0 && blockIdx.x * 32 + w < D) out[blockIdx.x * 32 + w] = (float)sum;
}

// ---------------------------------------------------------------------------
// One token per row, the state updated in place: 24 bytes of traffic per element at
// most (fp32 with a gate), bound by the launch (replayed as a graph 4.3 us for 256x640
// fp32, whose bytes are worth 0.6, and for one row of 640 alike).
template <typename T, int V>
__global__ void __launch_bounds__(256)
    gated_scan_step_kernel(const T* __restrict__ x, const T* __restrict__ f, const T* __restrict__ g, long long xs,
                           long long fs, long long gs, const float* __restrict__ lower, float* state, long long ss,
                           T* __restrict__ y, long long n, int dv) {
  const long long k = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (k >= n) return;
  const long long b = k / dv;
  const int c = (int)(k % dv) * V;
  const Fv<V> xv = load_raw<T, V>(x + b * xs + c).get();
  const Raw<T, V> fv = load_raw<T, V>(f + b * fs + c);
  Raw<T, V> gv{};
  if (g) gv = load_raw<T, V>(g + b * gs + c);
  Fv<V> lo = splat<V>(0.f), om = splat<V>(1.f), s, m;
  if (lower) {
    lo = load_f32<V>(lower + c);
#pragma unroll
    for (int i = 0; i < V; ++i) om.v[i] = 1.f - lo.v[i];
  }
  float* const sp = state + b * ss + c;
  Fv<V> h = load_f32<V>(sp);
  sigmoid_pair(sigmoid_arg(fv).get(), s, m);
  h = fma(fma(om, s, lo), h, mul(mul(om, m), xv));
  store_f32<V>(sp, h);
  if (g) h = mul(h, sigmoid_of(gv.get()));
  store_raw<T, V>(y + b * (long long)dv * V + c, h);
}

}  // namespace

yuf_status_t gated_scan_dlower(const float* partial, float* dlower, long long rows, int D, cudaStream_t st) {
  gated_scan_dlower_kernel<<<(D + 31) / 32, 1024, 0, st>>>(partial, dlower, rows, D);
  return check_launch("gated_scan_dlower_kernel");
}

yuf_status_t gated_scan_f32(const GatedScanArgs& a, bool backward, cudaStream_t st);
yuf_status_t gated_scan_bf16(const GatedScanArgs& a, bool backward, cudaStream_t st);
yuf_status_t gated_scan_f16(const GatedScanArgs& a, bool backward, cudaStream_t st);
unsigned int gated_scan_wait_timeouts_f32();
unsigned int gated_scan_wait_timeouts_bf16();
unsigned int gated_scan_wait_timeouts_f16();

static yuf_status_t run(const GatedScanArgs& a, bool backward, cudaStream_t st) {
  switch (a.dtype) {
    case YUF_DTYPE_F32: return gated_scan_f32(a, backward, st);
    case YUF_DTYPE_BF16: return gated_scan_bf16(a, backward, st);
    default: return gated_scan_f16(a, backward, st);
  }
}

unsigned int gated_scan_wait_timeouts() {
  const unsigned int a = gated_scan_wait_timeouts_f32(), b = gated_scan_wait_timeouts_bf16(),
                     c = gated_scan_wait_timeouts_f16();
  return a == ~0u || b == ~0u || c == ~0u ? ~0u : a + b + c;
}

// Which form a call takes depends on its tensors' alignment: room for either.
size_t gated_scan_workspace_floats(int B, int T, int D, int dtype, bool backward) {
  long long most = 0;
  for (int V = 1; V <= (dtype == YUF_DTYPE_F32 ? 1 : 2); ++V) {
    const GatedScanPlan p = gated_scan_plan(B, T, D, V);
    most = max(most, p.map_floats(V) + (backward ? (long long)B * p.sp.chunks * D : 0));
  }
  return (size_t)most;
}

yuf_status_t gated_scan_forward(const GatedScanArgs& a, cudaStream_t st) { return run(a, false, st); }
yuf_status_t gated_scan_backward(const GatedScanArgs& a, cudaStream_t st) { return run(a, true, st); }

template <typename T, int V>
static yuf_status_t launch_step(const void* x, const void* f, const void* g, long long xs, long long fs, long long gs,
                                const float* lower, float* state, long long ss, void* y, int B, int D,
                                cudaStream_t st) {
  const long long n = (long long)B * (D / V);
  gated_scan_step_kernel<T, V><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
      static_cast<const T*>(x), static_cast<const T*>(f), static_cast<const T*>(g), xs, fs, gs, lower, state, ss,
      static_cast<T*>(y), n, D / V);
  return check_launch("gated_scan_step_kernel");
}

yuf_status_t gated_scan_step(const void* x, const void* f, const void* g, long long xs, long long fs, long long gs,
                             const float* lower, float* state, long long ss, void* y, int dtype, int B, int D,
                             cudaStream_t st) {
  const size_t e = 2 * gated_elem_size(dtype);
  const bool two = D % 2 == 0 && ((xs | fs | gs | ss) & 1) == 0 && gated_aligned(x, e) && gated_aligned(f, e) &&
                   gated_aligned(g, e) && gated_aligned(y, e) && gated_aligned(lower, 8) && gated_aligned(state, 8);
#define STEP(T, V) launch_step<T, V>(x, f, g, xs, fs, gs, lower, state, ss, y, B, D, st)
  switch (dtype) {
    case YUF_DTYPE_F32: return two ? STEP(float, 2) : STEP(float, 1);
    case YUF_DTYPE_BF16: return two ? STEP(__nv_bfloat16, 2) : STEP(__nv_bfloat16, 1);
    default: return two ? STEP(__half, 2) : STEP(__half, 1);
  }
#undef STEP
}

}  // namespace yuf
