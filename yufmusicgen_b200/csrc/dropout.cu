// Dropout, with an optional residual add, whose mask is never stored:
//   y_i = res_i + (w_i >= floor(p 2^32) ? x_i / (1 - p) : 0)
// w_i = word i % 4 of Philox4x32-10(key = seed, counter = (i / 4, step)), i the
// element's row-major index.  The backward is the same map of dy without the
// residual: it draws the same words again.  One fp32 FMA, rounded once on store;
// a dropped element is a select, so an infinite or NaN x does not get through.
//
// One pass in 16-byte pieces, 8 elements per thread.  The ten rounds for each 4 elements
// (5 wide multiplications per element) cost the same whatever the types: 144 us for
// 131072 x 1024 elements.  10 bytes an element hide them (bf16 onto an fp32 residual:
// 194 us, 6.9 TB/s, bound by HBM); its gradient, 6 bytes an element, takes 145 us
// (5.5 TB/s) and bf16 to bf16, 4 bytes, 144 us (3.7 TB/s): bound by the rounds.
#include "gated_scan.cuh"
#include "io_types.cuh"
#include "philox.cuh"

namespace yuf {

namespace {

template <typename T>
YUF_DEVICE float to_f32(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else return static_cast<float>(x);
}
template <typename T>
YUF_DEVICE T from_f32(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else return T(x);
}

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// G neighbouring elements per thread (a multiple of 4, one counter per 4)
// in one row of x and res.  FLAT: x and res have no gaps, so the whole tensor
// is one row and the index needs no division.  VEC: 16-byte accesses.
template <typename TX, typename TO, bool RES, bool FLAT, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutArgs p, long long n) {
  constexpr int G = VEC ? 8 : 4;
  const long long i0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * G;
  if (i0 >= n) return;
  const TX* const x = static_cast<const TX*>(p.x);
  const TO* const res = static_cast<const TO*>(p.res);
  TO* const out = static_cast<TO*>(p.out);
  const uint64_t step = p.step_ptr ? *p.step_ptr : p.step;
  float xv[G], rv[G];
  const bool whole = VEC && i0 + G <= n;
  if (whole) {
    long long xo = i0, ro = i0;
    if constexpr (!FLAT) {
      const long long r = i0 / p.cols, c = i0 - r * p.cols;
      xo = r * p.xs + c;
      ro = r * p.rs + c;
    }
    const Pack<TX, G> xp = *reinterpret_cast<const Pack<TX, G>*>(x + xo);
#pragma unroll
    for (int k = 0; k < G; ++k) xv[k] = to_f32(xp.v[k]);
    if constexpr (RES) {
      const Pack<TO, G> rp = *reinterpret_cast<const Pack<TO, G>*>(res + ro);
#pragma unroll
      for (int k = 0; k < G; ++k) rv[k] = to_f32(rp.v[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < G; ++k) {
      xv[k] = rv[k] = 0.f;
      const long long i = i0 + k;
      if (i < n) {
        long long xo = i, ro = i;
        if constexpr (!FLAT) {
          const long long r = i / p.cols, c = i - r * p.cols;
          xo = r * p.xs + c;
          ro = r * p.rs + c;
        }
        xv[k] = to_f32(x[xo]);
        if constexpr (RES) rv[k] = to_f32(res[ro]);
      }
    }
  }
  Pack<TO, G> o;
#pragma unroll
  for (int q = 0; q < G / 4; ++q) {
    const uint64_t ctr = (uint64_t)(i0 >> 2) + q;
    const U4 u = philox4x32_10(U4{(uint32_t)ctr, (uint32_t)(ctr >> 32), (uint32_t)step, (uint32_t)(step >> 32)},
                               (uint32_t)p.seed, (uint32_t)(p.seed >> 32));
    const uint32_t word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool keep = !p.any || word[k] > p.last_dropped;
      const float r = RES ? rv[4 * q + k] : 0.f;
      const float v = RES ? fmaf(xv[4 * q + k], p.scale, r) : xv[4 * q + k] * p.scale;
      o.v[4 * q + k] = from_f32<TO>(keep ? v : r);
    }
  }
  if (whole) {
    *reinterpret_cast<Pack<TO, G>*>(out + i0) = o;
  } else {
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (i0 + k < n) out[i0 + k] = o.v[k];
  }
}

template <typename TX, typename TO, bool RES>
yuf_status_t launch(const DropoutArgs& a, cudaStream_t st) {
  const long long n = a.rows * a.cols;
  const bool flat = a.rows == 1 || (a.xs == a.cols && (!RES || a.rs == a.cols));
  const auto at16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  // 16-byte accesses: aligned rows, and no group of 8 across a row's end
  const bool vec = at16(a.x) && at16(a.res) && at16(a.out) &&
                   (flat || (a.cols % 8 == 0 && a.xs * sizeof(TX) % 16 == 0 && (!RES || a.rs * sizeof(TO) % 16 == 0)));
  const long long threads = (n + (vec ? 7 : 3)) / (vec ? 8 : 4);
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) {
    set_error("dropout: tensor too large");
    return YUF_ERR_INVALID_ARGUMENT;
  }
  if (flat && vec) dropout_kernel<TX, TO, RES, true, true><<<(unsigned)blocks, 256, 0, st>>>(a, n);
  else if (flat) dropout_kernel<TX, TO, RES, true, false><<<(unsigned)blocks, 256, 0, st>>>(a, n);
  else if (vec) dropout_kernel<TX, TO, RES, false, true><<<(unsigned)blocks, 256, 0, st>>>(a, n);
  else dropout_kernel<TX, TO, RES, false, false><<<(unsigned)blocks, 256, 0, st>>>(a, n);
  return check_launch("dropout_kernel");
}

template <typename TX, typename TO>
yuf_status_t pick(const DropoutArgs& a, cudaStream_t st) {
  return a.res ? launch<TX, TO, true>(a, st) : launch<TX, TO, false>(a, st);
}

}  // namespace

yuf_status_t dropout_forward(const DropoutArgs& a, cudaStream_t st) {
  // the pairs of types: equal ones, a 16-bit x onto an fp32 residual stream, and
  // the gradient of that (fp32 dy to a 16-bit dx)
  const int x = a.x_dtype, o = a.out_dtype;
  if (x == YUF_DTYPE_F32 && o == YUF_DTYPE_F32) return pick<float, float>(a, st);
  if (x == YUF_DTYPE_BF16 && o == YUF_DTYPE_BF16) return pick<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (x == YUF_DTYPE_F16 && o == YUF_DTYPE_F16) return pick<__half, __half>(a, st);
  if (x == YUF_DTYPE_BF16 && o == YUF_DTYPE_F32) return pick<__nv_bfloat16, float>(a, st);
  if (x == YUF_DTYPE_F16 && o == YUF_DTYPE_F32) return pick<__half, float>(a, st);
  if (x == YUF_DTYPE_F32 && o == YUF_DTYPE_BF16 && !a.res) return launch<float, __nv_bfloat16, false>(a, st);
  if (x == YUF_DTYPE_F32 && o == YUF_DTYPE_F16 && !a.res) return launch<float, __half, false>(a, st);
  set_error("dropout: no kernel for x of type %d and output of type %d%s", x, o, a.res ? " with a residual" : "");
  return YUF_ERR_UNSUPPORTED;
}

}  // namespace yuf
