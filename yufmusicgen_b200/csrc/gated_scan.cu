// Elementwise gated recurrence over [B, T, D] (per channel), its gradients and
// its single-token form:
//   a_t = lower + (1 - lower) sigmoid(f_t),  i_t = (1 - lower) sigmoid(-f_t) = 1 - a_t
//   h_t = a_t h_{t-1} + i_t x_t,             y_t = h_t sigmoid(g_t)
// All of it in fp32; y and the gradients are rounded once, when they are stored.
//
// The recurrence is affine in h, so a run of tokens is the map h -> A h + H
// (A = product of its a_t, H = its end state from zero) and runs compose:
// (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2).  A warp owns L neighbouring
// tokens of 32 V channels, everything in registers: it loads its tokens once,
// forms its map, the maps of the block's warps meet in shared memory, and each
// warp runs its tokens again from its true start state.  Memory is touched once;
// the second run costs one FMA per element.  A block walks the time axis in
// steps of (warps x L) tokens with the state carried in registers.
//
// Packed sequences (cu_seqlens): at a sequence's first token h_{t-1} is that
// sequence's own start state.  The token's map is then constant, written as
// A = 0 with a flag (CUT): a product with zero would let an infinite or NaN
// state of the sequence before leak into it.
//
// The order of every sum is fixed: results do not depend on timing.
#include "gated_scan.cuh"
#include "io_types.cuh"

namespace yuf {

namespace {

constexpr int NW_MAX = 8;      // warps per block
constexpr float CUT = -1.f;    // A of a run that forgets what came before it (A >= 0 otherwise)

template <int V>
YUF_DEVICE Fv<V> apply(Fv<V> A, Fv<V> H, Fv<V> h) {
  Fv<V> r = fma(A, h, H);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (A.v[i] < 0.f) r.v[i] = H.v[i];
  return r;
}

// Sequence of token t: index of the last boundary <= t, -1 before the first,
// n_seqs at and after the last one.  Any contents of cu give a value in [-1, n_seqs].
YUF_DEVICE int owner_of(const int* cu, int n_seqs, int t, int T) {
  if (t < 0) return -1;
  if (t >= T) return n_seqs;
  int lo = 0, hi = n_seqs + 1;  // boundaries before lo are <= t, from hi on > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}
YUF_DEVICE bool live_owner(int o, int n_seqs) { return o >= 0 && o < n_seqs; }

// ---------------------------------------------------------------------------
// Forward.  blockIdx.x = batch row * channel blocks + channel block.
template <typename T, int V, int L, bool GATE, bool PACKED>
__global__ void __launch_bounds__(32 * NW_MAX, 2)
    gated_scan_forward_kernel(const GatedScanArgs p, int n_cblk) {
  __shared__ float2 maps[2][NW_MAX][32 * V];
  __shared__ int owners[2][PACKED ? NW_MAX * L + 2 : 1];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int b = blockIdx.x / n_cblk, c = (blockIdx.x % n_cblk) * 32 * V + lane * V;
  const bool act = c < p.D;
  const T* const xp = static_cast<const T*>(p.x) + b * p.xb + c;
  const T* const fp = static_cast<const T*>(p.f) + b * p.fb + c;
  const T* const gp = GATE ? static_cast<const T*>(p.g) + b * p.gb + c : nullptr;
  T* const yp = static_cast<T*>(p.y) + (long long)b * p.T * p.D + c;
  const int tile = nw * L;

  Fv<V> lo = splat<V>(0.f), om = splat<V>(1.f), h = splat<V>(0.f);
  if (act && p.lower) {
    lo = load_f32<V>(p.lower + c);
#pragma unroll
    for (int i = 0; i < V; ++i) om.v[i] = 1.f - lo.v[i];
  }
  if (!PACKED && act && p.h0) h = load_f32<V>(p.h0 + (long long)b * p.D + c);
  if constexpr (PACKED) {  // sequences without a token keep their start state
    if (p.h_last && act)
      for (int s = w; s < p.n_seqs; s += nw) {
        const int c0 = __ldg(p.cu + s), c1 = __ldg(p.cu + s + 1);
        if (c0 >= c1 || c0 >= p.T || c1 <= 0)
          store_f32<V>(p.h_last + (long long)s * p.D + c,
                       p.h0 ? load_f32<V>(p.h0 + (long long)s * p.D + c) : splat<V>(0.f));
      }
  }

  int buf = 0;
  for (int base = 0; base < p.T; base += tile, buf ^= 1) {
    const int t0 = base + w * L;
    if constexpr (PACKED) {
      for (int j = threadIdx.x; j < tile + 2; j += blockDim.x)
        owners[buf][j] = owner_of(p.cu, p.n_seqs, base - 1 + j, p.T);
      __syncthreads();
    }
    const int* const own = PACKED ? owners[buf] + w * L + 1 : nullptr;  // own[j]: token t0 + j
    const int n = min(L, p.T - t0);                                     // tokens of this warp (may be <= 0)
    Raw<T, V> x[L], f[L], g[GATE ? L : 1];
    bool ok[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      ok[j] = j < n;
      if constexpr (PACKED) ok[j] = ok[j] && live_owner(own[j], p.n_seqs);
      if (ok[j] && act) {
        x[j] = load_raw<T, V>(xp + (t0 + j) * p.xt);
        f[j] = load_raw<T, V>(fp + (t0 + j) * p.ft);
        if constexpr (GATE) g[j] = load_raw<T, V>(gp + (t0 + j) * p.gt);
      }
    }
    // this warp's map
    Fv<V> a[L], bx[L], A = splat<V>(1.f), H = splat<V>(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      if (ok[j]) {
        Fv<V> s, m;
        sigmoid_pair(f[j].get(), s, m);
        a[j] = fma(om, s, lo);
        bx[j] = mul(mul(om, m), x[j].get());
        bool first = false;
        if constexpr (PACKED) first = own[j] != own[j - 1];
        if (first) {
          if (p.h0 && act) bx[j] = fma(a[j], load_f32<V>(p.h0 + (long long)own[j] * p.D + c), bx[j]);
          A = a[j] = splat<V>(CUT);
          H = bx[j];
        } else {
          H = fma(a[j], H, bx[j]);
          A = mul(A, a[j]);  // CUT times a: its sign stays
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (PACKED && A.v[i] <= 0.f && signbit(A.v[i])) A.v[i] = CUT;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) maps[buf][w][lane * V + i] = make_float2(A.v[i], H.v[i]);
    __syncthreads();
    // start state of this warp, and of the next step
    Fv<V> hw = h;
    for (int k = 0; k < nw; ++k) {
      if (k == w) hw = h;
      Fv<V> Ak, Hk;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 m = maps[buf][k][lane * V + i];
        Ak.v[i] = m.x;
        Hk.v[i] = m.y;
      }
      h = apply(Ak, Hk, h);
    }
    if (!act) continue;
    if (p.ckpt && n > 0)
      store_f32<V>(p.ckpt + ((long long)b * ((p.T + L - 1) / L) + t0 / L) * p.D + c, hw);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      if (ok[j]) {
        hw = PACKED ? apply(a[j], bx[j], hw) : fma(a[j], hw, bx[j]);
        Fv<V> y = hw;
        if constexpr (GATE) y = mul(hw, sigmoid_of(g[j].get()));
        store_raw<T, V>(yp + (long long)(t0 + j) * p.D, y);
        if constexpr (PACKED)
          if (p.h_last && own[j + 1] != own[j]) store_f32<V>(p.h_last + (long long)own[j] * p.D + c, hw);
      } else if (PACKED && j < n) {
        store_raw<T, V>(yp + (long long)(t0 + j) * p.D, splat<V>(0.f));
      }
    }
  }
  if (!PACKED && p.h_last && w == 0 && act) store_f32<V>(p.h_last + (long long)b * p.D + c, h);
}

// ---------------------------------------------------------------------------
// Backward, the time axis from its end: with p_t = dy_t sigmoid(g_t) and G_t the
// gradient that reaches h_t from the tokens after it,
//   dh_t = p_t + G_t,  G_{t-1} = a_t dh_t,  G_T = dL/dh_last
//   dx_t = dh_t i_t,   df_t = dh_t (h_{t-1} - x_t) i_t sigmoid(f_t)
//   dg_t = dy_t h_t sigmoid(g_t) sigmoid(-g_t)
//   dlower = sum dh_t (h_{t-1} - x_t) sigmoid(-f_t),  dL/dh_0 = G_0
// Each warp forms h of its L tokens again from the state the forward saved
// there (one state per L tokens: 1/16 or 1/8 of a tensor's elements in fp32),
// and the maps G -> A G + H of the warps meet as in the forward.
template <typename T, int V, int L, bool GATE, bool PACKED>
__global__ void __launch_bounds__(32 * NW_MAX)
    gated_scan_backward_kernel(const GatedScanArgs p, int n_cblk) {
  __shared__ float2 maps[2][NW_MAX][32 * V];
  __shared__ int owners[2][PACKED ? NW_MAX * L + 2 : 1];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int b = blockIdx.x / n_cblk, c = (blockIdx.x % n_cblk) * 32 * V + lane * V;
  const bool act = c < p.D;
  const T* const xp = static_cast<const T*>(p.x) + b * p.xb + c;
  const T* const fp = static_cast<const T*>(p.f) + b * p.fb + c;
  const T* const gp = GATE ? static_cast<const T*>(p.g) + b * p.gb + c : nullptr;
  const T* const dyp = static_cast<const T*>(p.dy) + b * p.yb + c;
  const long long out0 = (long long)b * p.T * p.D + c;
  T *const dxp = static_cast<T*>(p.dx) + out0, *const dfp = static_cast<T*>(p.df) + out0;
  T* const dgp = GATE ? static_cast<T*>(p.dg) + out0 : nullptr;
  const int tile = nw * L;

  Fv<V> lo = splat<V>(0.f), om = splat<V>(1.f), G = splat<V>(0.f), dlo = splat<V>(0.f);
  if (act && p.lower) {
    lo = load_f32<V>(p.lower + c);
#pragma unroll
    for (int i = 0; i < V; ++i) om.v[i] = 1.f - lo.v[i];
  }
  if (!PACKED && act && p.dh_last) G = load_f32<V>(p.dh_last + (long long)b * p.D + c);
  if constexpr (PACKED) {
    if (p.dh0 && act)
      for (int s = w; s < p.n_seqs; s += nw) {
        const int c0 = __ldg(p.cu + s), c1 = __ldg(p.cu + s + 1);
        if (c0 >= c1 || c0 >= p.T || c1 <= 0)
          store_f32<V>(p.dh0 + (long long)s * p.D + c,
                       p.dh_last ? load_f32<V>(p.dh_last + (long long)s * p.D + c) : splat<V>(0.f));
      }
  }

  int buf = 0;
  for (int base = (p.T - 1) / tile * tile; base >= 0; base -= tile, buf ^= 1) {
    const int t0 = base + w * L;
    if constexpr (PACKED) {
      for (int j = threadIdx.x; j < tile + 2; j += blockDim.x)
        owners[buf][j] = owner_of(p.cu, p.n_seqs, base - 1 + j, p.T);
      __syncthreads();
    }
    const int* const own = PACKED ? owners[buf] + w * L + 1 : nullptr;
    const int n = min(L, p.T - t0);
    Raw<T, V> x[L], f[L], g[GATE ? L : 1], dy[L];
    bool ok[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      ok[j] = j < n;
      if constexpr (PACKED) ok[j] = ok[j] && live_owner(own[j], p.n_seqs);
      if (ok[j] && act) {
        x[j] = load_raw<T, V>(xp + (t0 + j) * p.xt);
        f[j] = load_raw<T, V>(fp + (t0 + j) * p.ft);
        dy[j] = load_raw<T, V>(dyp + (t0 + j) * p.yt);
        if constexpr (GATE) g[j] = load_raw<T, V>(gp + (t0 + j) * p.gt);
      }
    }
    Fv<V> h = splat<V>(0.f);
    if (act && n > 0) h = load_f32<V>(p.ckpt + ((long long)b * ((p.T + L - 1) / L) + t0 / L) * p.D + c);
    // h again, dg, and what the reverse run needs: s = sigmoid(f), m = sigmoid(-f),
    // e = h_{t-1} - x_t, q = p_t
    Fv<V> s[L], m[L], e[L], q[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      if (ok[j]) {
        sigmoid_pair(f[j].get(), s[j], m[j]);
        if constexpr (PACKED)
          if (own[j] != own[j - 1])
            h = p.h0 && act ? load_f32<V>(p.h0 + (long long)own[j] * p.D + c) : splat<V>(0.f);
        const Fv<V> xv = x[j].get();
        e[j] = fma(xv, splat<V>(-1.f), h);
        h = fma(fma(om, s[j], lo), h, mul(mul(om, m[j]), xv));
        q[j] = dy[j].get();
        if constexpr (GATE) {
          Fv<V> sg, mg;
          sigmoid_pair(g[j].get(), sg, mg);
          q[j] = mul(q[j], sg);
          if (act) store_raw<T, V>(dgp + (long long)(t0 + j) * p.D, mul(mul(q[j], h), mg));
        }
      }
    }
    Fv<V> A = splat<V>(1.f), H = splat<V>(0.f);
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      if (ok[j]) {
        const Fv<V> a = fma(om, s[j], lo);
        bool last = false;
        if constexpr (PACKED) last = own[j + 1] != own[j];
        if (last) {
          H = p.dh_last && act ? load_f32<V>(p.dh_last + (long long)own[j] * p.D + c) : splat<V>(0.f);
          A = splat<V>(CUT);
        }
        H = mul(a, add(q[j], H));
        A = mul(A, a);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (PACKED && A.v[i] <= 0.f && signbit(A.v[i])) A.v[i] = CUT;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) maps[buf][w][lane * V + i] = make_float2(A.v[i], H.v[i]);
    __syncthreads();
    Fv<V> Gw = G;
    for (int k = nw - 1; k >= 0; --k) {
      if (k == w) Gw = G;
      Fv<V> Ak, Hk;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 mk = maps[buf][k][lane * V + i];
        Ak.v[i] = mk.x;
        Hk.v[i] = mk.y;
      }
      G = apply(Ak, Hk, G);
    }
    if (!act) continue;
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      if (ok[j]) {
        if constexpr (PACKED)
          if (own[j + 1] != own[j])
            Gw = p.dh_last ? load_f32<V>(p.dh_last + (long long)own[j] * p.D + c) : splat<V>(0.f);
        const Fv<V> dh = add(q[j], Gw), dhm = mul(dh, m[j]), di = mul(dhm, om);
        store_raw<T, V>(dxp + (long long)(t0 + j) * p.D, di);
        store_raw<T, V>(dfp + (long long)(t0 + j) * p.D, mul(mul(di, e[j]), s[j]));
        dlo = fma(dhm, e[j], dlo);
        Gw = mul(fma(om, s[j], lo), dh);
        if constexpr (PACKED)
          if (p.dh0 && own[j] != own[j - 1]) store_f32<V>(p.dh0 + (long long)own[j] * p.D + c, Gw);
      } else if (PACKED && j < n) {
        const long long o = (long long)(t0 + j) * p.D;
        store_raw<T, V>(dxp + o, splat<V>(0.f));
        store_raw<T, V>(dfp + o, splat<V>(0.f));
        if constexpr (GATE) store_raw<T, V>(dgp + o, splat<V>(0.f));
      }
    }
  }
  if (!PACKED && p.dh0 && w == 0 && act) store_f32<V>(p.dh0 + (long long)b * p.D + c, G);
  if (p.partial) {  // the block's share of dlower
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) maps[0][w][lane * V + i].x = dlo.v[i];
    __syncthreads();
    if (w == 0 && act)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float sum = 0.f;
        for (int k = 0; k < nw; ++k) sum += maps[0][k][lane * V + i].x;
        p.partial[(long long)b * p.D + c + i] = sum;
      }
  }
}

// dlower[c] = sum over rows of partial[rows, D], in a fixed order
__global__ void __launch_bounds__(256)
    gated_scan_dlower_kernel(const float* __restrict__ partial, float* __restrict__ out, long long rows, int D) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < D)
    for (long long r = w; r < rows; r += 8) sum += partial[r * D + c];
  part[w][lane] = sum;
  __syncthreads();
  if (w == 0 && c < D) {
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += part[k][lane];
    out[c] = sum;
  }
}

// ---------------------------------------------------------------------------
// One token per row, the state updated in place.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    gated_scan_step_kernel(const T* __restrict__ x, const T* __restrict__ f, const T* __restrict__ g, long long xs,
                           long long fs, long long gs, const float* __restrict__ lower, float* state, long long ss,
                           T* __restrict__ y, long long n, int dv) {
  const long long k = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (k >= n) return;
  const long long b = k / dv;
  const int c = (int)(k % dv) * V;
  const Fv<V> xv = load_raw<T, V>(x + b * xs + c).get(), fv = load_raw<T, V>(f + b * fs + c).get();
  Fv<V> lo = splat<V>(0.f), om = splat<V>(1.f), s, m;
  if (lower) {
    lo = load_f32<V>(lower + c);
#pragma unroll
    for (int i = 0; i < V; ++i) om.v[i] = 1.f - lo.v[i];
  }
  float* const sp = state + b * ss + c;
  Fv<V> h = load_f32<V>(sp);
  sigmoid_pair(fv, s, m);
  h = fma(fma(om, s, lo), h, mul(mul(om, m), xv));
  store_f32<V>(sp, h);
  if (g) h = mul(h, sigmoid_of(load_raw<T, V>(g + b * gs + c).get()));
  store_raw<T, V>(y + b * (long long)dv * V + c, h);
}

bool pair_ok(const void* q, size_t bytes) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; }

int elem_size(int dtype) { return dtype == YUF_DTYPE_F32 ? 4 : 2; }

// two channels per lane: even widths and strides, every row start aligned to a pair
bool pairs(const GatedScanArgs& a) {
  const size_t e = 2 * elem_size(a.dtype);
  const void* t[] = {a.x, a.f, a.g, a.dy, a.y, a.dx, a.df, a.dg};
  const float* s[] = {a.lower, a.h0, a.h_last, a.ckpt, a.dh_last, a.dh0};
  bool ok = a.D % 2 == 0 && ((a.xb | a.xt | a.fb | a.ft | a.gb | a.gt | a.yb | a.yt) & 1) == 0;
  for (const void* q : t) ok = ok && pair_ok(q, e);
  for (const float* q : s) ok = ok && pair_ok(q, 8);
  return ok;
}

struct Plan {
  int n_cblk, nw;
  long long blocks;
};
Plan plan(const GatedScanArgs& a, int V) {
  Plan p;
  const int L = gated_scan_block(a.dtype);
  p.n_cblk = (a.D + 32 * V - 1) / (32 * V);
  p.nw = max(1, min(NW_MAX, (a.T + L - 1) / L));
  p.blocks = (long long)a.B * p.n_cblk;
  return p;
}

template <typename T, int V, int L, bool GATE, bool PACKED>
yuf_status_t launch_forward(const GatedScanArgs& a, cudaStream_t st) {
  const Plan p = plan(a, V);
  gated_scan_forward_kernel<T, V, L, GATE, PACKED><<<(unsigned)p.blocks, 32 * p.nw, 0, st>>>(a, p.n_cblk);
  return check_launch("gated_scan_forward_kernel");
}
template <typename T, int V, int L, bool GATE, bool PACKED>
yuf_status_t launch_backward(const GatedScanArgs& a, cudaStream_t st) {
  const Plan p = plan(a, V);
  gated_scan_backward_kernel<T, V, L, GATE, PACKED><<<(unsigned)p.blocks, 32 * p.nw, 0, st>>>(a, p.n_cblk);
  return check_launch("gated_scan_backward_kernel");
}

template <typename T, int V, int L>
yuf_status_t pick_forward(const GatedScanArgs& a, cudaStream_t st) {
  if (a.g) return a.cu ? launch_forward<T, V, L, true, true>(a, st) : launch_forward<T, V, L, true, false>(a, st);
  return a.cu ? launch_forward<T, V, L, false, true>(a, st) : launch_forward<T, V, L, false, false>(a, st);
}
template <typename T, int V, int L>
yuf_status_t pick_backward(const GatedScanArgs& a, cudaStream_t st) {
  if (a.g) return a.cu ? launch_backward<T, V, L, true, true>(a, st) : launch_backward<T, V, L, true, false>(a, st);
  return a.cu ? launch_backward<T, V, L, false, true>(a, st) : launch_backward<T, V, L, false, false>(a, st);
}

}  // namespace

long long gated_scan_partial_rows(int B, int, int) { return B; }

yuf_status_t gated_scan_forward(const GatedScanArgs& a, cudaStream_t st) {
  const bool two = pairs(a);
  switch (a.dtype) {
    case YUF_DTYPE_F32: return two ? pick_forward<float, 2, 8>(a, st) : pick_forward<float, 1, 8>(a, st);
    case YUF_DTYPE_BF16:
      return two ? pick_forward<__nv_bfloat16, 2, 16>(a, st) : pick_forward<__nv_bfloat16, 1, 16>(a, st);
    default: return two ? pick_forward<__half, 2, 16>(a, st) : pick_forward<__half, 1, 16>(a, st);
  }
}

yuf_status_t gated_scan_backward(const GatedScanArgs& a, cudaStream_t st) {
  const bool two = pairs(a);
  yuf_status_t rc;
  switch (a.dtype) {
    case YUF_DTYPE_F32: rc = two ? pick_backward<float, 2, 8>(a, st) : pick_backward<float, 1, 8>(a, st); break;
    case YUF_DTYPE_BF16:
      rc = two ? pick_backward<__nv_bfloat16, 2, 16>(a, st) : pick_backward<__nv_bfloat16, 1, 16>(a, st);
      break;
    default: rc = two ? pick_backward<__half, 2, 16>(a, st) : pick_backward<__half, 1, 16>(a, st);
  }
  if (rc != YUF_OK || !a.dlower) return rc;
  gated_scan_dlower_kernel<<<(a.D + 31) / 32, 256, 0, st>>>(a.partial, a.dlower,
                                                            gated_scan_partial_rows(a.B, a.T, a.D), a.D);
  return check_launch("gated_scan_dlower_kernel");
}

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
  const size_t e = 2 * elem_size(dtype);
  const bool two = D % 2 == 0 && ((xs | fs | gs | ss) & 1) == 0 && pair_ok(x, e) && pair_ok(f, e) && pair_ok(g, e) &&
                   pair_ok(y, e) && pair_ok(lower, 8) && pair_ok(state, 8);
#define STEP(T, V) launch_step<T, V>(x, f, g, xs, fs, gs, lower, state, ss, y, B, D, st)
  switch (dtype) {
    case YUF_DTYPE_F32: return two ? STEP(float, 2) : STEP(float, 1);
    case YUF_DTYPE_BF16: return two ? STEP(__nv_bfloat16, 2) : STEP(__nv_bfloat16, 1);
    default: return two ? STEP(__half, 2) : STEP(__half, 1);
  }
#undef STEP
}

}  // namespace yuf
