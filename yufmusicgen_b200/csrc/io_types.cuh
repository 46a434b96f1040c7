// Loads and stores of V neighbouring channels of fp32, bf16 or fp16 tensors as
// fp32 values, and packed arithmetic on them (V = 2 uses the fp32x2 pipe).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace yuf {

template <int V>
struct Fv {
  float v[V];
};

// each operation rounds by itself (no contraction), whatever kernel it stands in
YUF_DEVICE float2 as2(const Fv<2>& a) { return make_float2(a.v[0], a.v[1]); }
YUF_DEVICE Fv<2> of2(float2 a) { return Fv<2>{{a.x, a.y}}; }
YUF_DEVICE Fv<1> mul(Fv<1> a, Fv<1> b) { return Fv<1>{{__fmul_rn(a.v[0], b.v[0])}}; }
YUF_DEVICE Fv<2> mul(Fv<2> a, Fv<2> b) { return of2(fmul2(as2(a), as2(b))); }
YUF_DEVICE Fv<1> fma(Fv<1> a, Fv<1> b, Fv<1> c) { return Fv<1>{{fmaf(a.v[0], b.v[0], c.v[0])}}; }
YUF_DEVICE Fv<2> fma(Fv<2> a, Fv<2> b, Fv<2> c) { return of2(ffma2(as2(a), as2(b), as2(c))); }
YUF_DEVICE Fv<1> add(Fv<1> a, Fv<1> b) { return Fv<1>{{__fadd_rn(a.v[0], b.v[0])}}; }
YUF_DEVICE Fv<2> add(Fv<2> a, Fv<2> b) { return of2(__fadd2_rn(as2(a), as2(b))); }
template <int V>
YUF_DEVICE Fv<V> splat(float x) {
  Fv<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}

// Raw<T, V>: V elements as they lie in memory (4 bytes at most per 16-bit pair).
template <typename T, int V>
struct Raw;
template <>
struct Raw<float, 1> {
  float r;
  YUF_DEVICE Fv<1> get() const { return Fv<1>{{r}}; }
  YUF_DEVICE static Raw put(Fv<1> f) { return Raw{f.v[0]}; }
};
template <>
struct Raw<float, 2> {
  float2 r;
  YUF_DEVICE Fv<2> get() const { return of2(r); }
  YUF_DEVICE static Raw put(Fv<2> f) { return Raw{as2(f)}; }
};
template <>
struct Raw<__nv_bfloat16, 1> {
  unsigned short r;
  YUF_DEVICE Fv<1> get() const { return Fv<1>{{__uint_as_float((unsigned)r << 16)}}; }
  YUF_DEVICE static Raw put(Fv<1> f) { return Raw{__bfloat16_as_ushort(__float2bfloat16_rn(f.v[0]))}; }
};
template <>
struct Raw<__nv_bfloat16, 2> {
  unsigned r;
  YUF_DEVICE Fv<2> get() const { return Fv<2>{{__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u)}}; }
  YUF_DEVICE static Raw put(Fv<2> f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[0], f.v[1]);
    return Raw{*reinterpret_cast<const unsigned*>(&h)};
  }
};
template <>
struct Raw<__half, 1> {
  unsigned short r;
  YUF_DEVICE Fv<1> get() const { return Fv<1>{{__half2float(__ushort_as_half(r))}}; }
  YUF_DEVICE static Raw put(Fv<1> f) { return Raw{__half_as_ushort(__float2half_rn(f.v[0]))}; }
};
template <>
struct Raw<__half, 2> {
  unsigned r;
  YUF_DEVICE Fv<2> get() const { return of2(__half22float2(*reinterpret_cast<const __half2*>(&r))); }
  YUF_DEVICE static Raw put(Fv<2> f) {
    const __half2 h = __floats2half2_rn(f.v[0], f.v[1]);
    return Raw{*reinterpret_cast<const unsigned*>(&h)};
  }
};

// streaming accesses: every element is read or written once
template <typename T, int V>
YUF_DEVICE Raw<T, V> load_raw(const T* p) {
  return Raw<T, V>{__ldcs(reinterpret_cast<const decltype(Raw<T, V>::r)*>(p))};
}
template <typename T, int V>
YUF_DEVICE void store_raw(T* p, Fv<V> f) {
  __stcs(reinterpret_cast<decltype(Raw<T, V>::r)*>(p), Raw<T, V>::put(f).r);
}
template <int V>
YUF_DEVICE Fv<V> load_f32(const float* p) {
  Fv<V> r;
  if constexpr (V == 2)
    r = of2(*reinterpret_cast<const float2*>(p));
  else
    r.v[0] = *p;
  return r;
}
template <int V>
YUF_DEVICE void store_f32(float* p, Fv<V> f) {
  if constexpr (V == 2)
    *reinterpret_cast<float2*>(p) = as2(f);
  else
    *p = f.v[0];
}

// sigmoid(x) and sigmoid(-x) = 1 - sigmoid(x), both to fp32 relative accuracy:
// e = 2^(-x log2 e), s = 1 / (1 + e), 1 - s = e s.  x is kept from below
// SIGMOID_MIN, where e would overflow and e s be inf * 0; NaN goes through.
constexpr float SIGMOID_MIN = -87.f;  // exact in bf16 and fp16
YUF_DEVICE float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
YUF_DEVICE float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int V>
YUF_DEVICE Fv<V> sigmoid_exp(Fv<V> x) {
  Fv<V> z = mul(x, splat<V>(-1.4426950408889634f));
#pragma unroll
  for (int i = 0; i < V; ++i) z.v[i] = exp2_fast(z.v[i]);
  return z;
}
template <int V>
YUF_DEVICE Fv<V> rcp_1p(Fv<V> e) {
  Fv<V> d = add(e, splat<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) d.v[i] = rcp_fast(d.v[i]);
  return d;
}
// of x >= SIGMOID_MIN
template <int V>
YUF_DEVICE void sigmoid_pair(Fv<V> x, Fv<V>& s, Fv<V>& one_minus_s) {
  const Fv<V> e = sigmoid_exp(x);
  s = rcp_1p(e);
  one_minus_s = mul(e, s);
}
template <int V>
YUF_DEVICE Fv<V> sigmoid_of(Fv<V> x) {  // any x
  return rcp_1p(sigmoid_exp(x));
}
// The same reciprocal on the FMA pipe, for kernels whose exponentials and reciprocals
// keep the special function unit busy: 1 / u of a float is near K - bits(u) read as a
// float (the exponent negated, the mantissa on a line; K minimises the largest error
// over [1, 4): 5.05e-2), then Newton's iteration with e = 1 - u r, once to third order
// (r + r (e + e^2): 1.3e-4) and once to second: 1.3 x 2^-24 with roundings.  d = -u =
// -(1 + e^-x), so that e is one FMA; u <= 2^126.
YUF_DEVICE Fv<2> rcp_1p_newton(Fv<2> ex) {
  const Fv<2> one = splat<2>(1.f), d = fma(ex, splat<2>(-1.f), splat<2>(-1.f));
  Fv<2> r;
#pragma unroll
  for (int i = 0; i < 2; ++i) r.v[i] = __uint_as_float(0xFEF311C0u - __float_as_uint(d.v[i]));
  Fv<2> e = fma(d, r, one);
  r = fma(r, fma(e, e, e), r);
  e = fma(d, r, one);
  return fma(r, e, r);
}
// max(x, SIGMOID_MIN) that keeps NaN, on the elements as they lie in memory
template <typename T, int V>
YUF_DEVICE Raw<T, V> sigmoid_arg(Raw<T, V> x) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 1) {
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.r) : "f"(SIGMOID_MIN));
    } else {
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.r.x) : "f"(SIGMOID_MIN));
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.r.y) : "f"(SIGMOID_MIN));
    }
  } else if constexpr (V == 2) {
    if constexpr (std::is_same_v<T, __half>) {
      const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&x.r), __float2half2_rn(SIGMOID_MIN));
      x.r = *reinterpret_cast<const unsigned*>(&m);
    } else {
      const __nv_bfloat162 m =
          __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&x.r), __float2bfloat162_rn(SIGMOID_MIN));
      x.r = *reinterpret_cast<const unsigned*>(&m);
    }
  } else {
    if constexpr (std::is_same_v<T, __half>)
      x.r = __half_as_ushort(__hmax_nan(__ushort_as_half(x.r), __float2half_rn(SIGMOID_MIN)));
    else
      x.r = __bfloat16_as_ushort(__hmax_nan(__ushort_as_bfloat16(x.r), __float2bfloat16_rn(SIGMOID_MIN)));
  }
  return x;
}

}  // namespace yuf
