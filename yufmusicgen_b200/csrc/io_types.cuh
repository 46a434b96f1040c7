// Loads and stores of V neighbouring channels of fp32, bf16 or fp16 tensors as
// fp32 values, and packed arithmetic on them (V = 2 uses the fp32x2 pipe).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace yuf {

template <int V>
struct Fv {
  float v[V];
};

YUF_DEVICE float2 as2(const Fv<2>& a) { return make_float2(a.v[0], a.v[1]); }
YUF_DEVICE Fv<2> of2(float2 a) { return Fv<2>{{a.x, a.y}}; }
YUF_DEVICE Fv<1> mul(Fv<1> a, Fv<1> b) { return Fv<1>{{a.v[0] * b.v[0]}}; }
YUF_DEVICE Fv<2> mul(Fv<2> a, Fv<2> b) { return of2(fmul2(as2(a), as2(b))); }
YUF_DEVICE Fv<1> fma(Fv<1> a, Fv<1> b, Fv<1> c) { return Fv<1>{{fmaf(a.v[0], b.v[0], c.v[0])}}; }
YUF_DEVICE Fv<2> fma(Fv<2> a, Fv<2> b, Fv<2> c) { return of2(ffma2(as2(a), as2(b), as2(c))); }
YUF_DEVICE Fv<1> add(Fv<1> a, Fv<1> b) { return Fv<1>{{a.v[0] + b.v[0]}}; }
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
// e = 2^min(-x log2 e, 126), s = 1 / (1 + e), 1 - s = e s.  The cap keeps e s
// finite for very negative x; NaN goes through.
YUF_DEVICE float sigmoid_exp(float x) {
  float z = x * -1.4426950408889634f, e;
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(126.f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z));
  return e;
}
YUF_DEVICE float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int V>
YUF_DEVICE void sigmoid_pair(Fv<V> x, Fv<V>& s, Fv<V>& one_minus_s) {
  Fv<V> e;
#pragma unroll
  for (int i = 0; i < V; ++i) e.v[i] = sigmoid_exp(x.v[i]);
  const Fv<V> d = add(e, splat<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) s.v[i] = rcp_fast(d.v[i]);
  one_minus_s = mul(e, s);
}
template <int V>
YUF_DEVICE Fv<V> sigmoid_of(Fv<V> x) {
  Fv<V> s, t;
  sigmoid_pair(x, s, t);
  return s;
}

}  // namespace yuf
