// Kernels of the elementwise gated recurrence over [B, T, D] (per channel) and its
// gradients; each element type's are instantiated in a source file of their own:
//   a_t = lower + (1 - lower) sigmoid(f_t),  i_t = (1 - lower) sigmoid(-f_t) = 1 - a_t
//   h_t = a_t h_{t-1} + i_t x_t,             y_t = h_t sigmoid(g_t)
// All of it in fp32; y and the gradients are rounded once, when they are stored.
//
// The recurrence is affine in h, so a run of tokens is the map h -> A h + H
// (A = product of its a_t, H = its end state from zero) and runs compose:
// (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2).  The backward is the same
// recurrence from the end, in the gradient that reaches h_t.  A warp works on runs
// of L = 16 tokens of 32 V channels, 4 bytes of each row per lane.  Two ways to
// share the time axis:
//
// * whole: a block walks all tokens of its channels, in steps of (warps x L).  Each
//   warp loads its run once, forms its map, the maps meet in shared memory, and the
//   warp runs its tokens again from its true start state (one FMA per element).
//   Memory is touched once, but only B x D / (32 V) blocks can work.
// * ranges, where those blocks would not fill the GPU: every warp owns a contiguous
//   range of the time axis.  One kernel forms the ranges' maps; a second starts each
//   warp from the composition of all maps before it and walks its range, no warp
//   waiting for another.  The inputs that the maps need (x and f; f, g and dy) are
//   read twice, the second time largely from L2.
//
// Packed sequences (cu_seqlens): at a sequence's first token h_{t-1} is that
// sequence's own start state.  The token's map is then constant, written as
// A = 0 with a flag (CUT): a product with zero would let an infinite or NaN
// state of the sequence before leak into it.
//
// The order of every sum is fixed: results do not depend on timing.
#pragma once
#include "gated_scan.cuh"

#include <atomic>
#include <climits>
#include <type_traits>

#include "io_types.cuh"
#include "tma.cuh"

namespace yuf {

namespace {

using Split = GatedScanSplit;
using Plan = GatedScanPlan;

constexpr int L = GATED_SCAN_BLOCK;  // tokens per run; the backward's states are L apart
constexpr int NW_MAX = GATED_SCAN_WARPS;
constexpr int RANGE_WARPS = GATED_SCAN_RANGE_WARPS;
constexpr float CUT = -1.f;          // A of a run that forgets what came before it (A >= 0 otherwise)

__device__ unsigned int g_gated_wait_timeouts;  // of this element type's kernels

// h -> A h + H, or H alone where the run is cut
template <bool PACKED, int V>
YUF_DEVICE Fv<V> apply(Fv<V> A, Fv<V> H, Fv<V> h) {
  Fv<V> r = fma(A, h, H);
  if constexpr (PACKED)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (A.v[i] < 0.f) r.v[i] = H.v[i];
  return r;
}
// (A, H) then (A2, H2), as one map
template <bool PACKED, int V>
YUF_DEVICE void compose(Fv<V>& A, Fv<V>& H, Fv<V> A2, Fv<V> H2) {
  H = apply<PACKED>(A2, H2, H);
  const Fv<V> A1 = A;
  A = mul(A1, A2);
  if constexpr (PACKED)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (A1.v[i] < 0.f || A2.v[i] < 0.f) A.v[i] = CUT;
}

// Maps lie as rows of 32 V float2, a lane's V maps as {A.., H..}.
template <int V>
YUF_DEVICE void put_map(float2* at, Fv<V> A, Fv<V> H) {
  if constexpr (V == 2) *reinterpret_cast<float4*>(at) = make_float4(A.v[0], A.v[1], H.v[0], H.v[1]);
  else *at = make_float2(A.v[0], H.v[0]);
}
template <int V>
YUF_DEVICE void get_map(const float2* at, Fv<V>& A, Fv<V>& H) {
  if constexpr (V == 2) {
    const float4 m = *reinterpret_cast<const float4*>(at);
    A = Fv<2>{{m.x, m.y}};
    H = Fv<2>{{m.z, m.w}};
  } else {
    A.v[0] = at->x;
    H.v[0] = at->y;
  }
}
// Four rows at a time, so that their loads overlap; the identity behind the n-th.
template <int V>
YUF_DEVICE void get_four(const float2* at, int n, Fv<V> (&A)[4], Fv<V> (&H)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    A[u] = splat<V>(1.f);
    H[u] = splat<V>(0.f);
    if (u < n) get_map<V>(at + u * 32 * V, A[u], H[u]);
  }
}
// h through the n maps at `at`
template <bool PACKED, int V>
YUF_DEVICE Fv<V> apply_all(const float2* at, int n, Fv<V> h) {
  for (int k = 0; k < n; k += 4) {
    Fv<V> A[4], H[4];
    get_four<V>(at + k * 32 * V, n - k, A, H);
#pragma unroll
    for (int u = 0; u < 4; ++u) h = apply<PACKED>(A[u], H[u], h);
  }
  return h;
}
template <bool PACKED, int V>
YUF_DEVICE void compose_all(const float2* at, int n, Fv<V>& A, Fv<V>& H) {
  for (int k = 0; k < n; k += 4) {
    Fv<V> A4[4], H4[4];
    get_four<V>(at + k * 32 * V, n - k, A4, H4);
#pragma unroll
    for (int u = 0; u < 4; ++u) compose<PACKED>(A, H, A4[u], H4[u]);
  }
}

// Where a warp stands: order `w` of `nw` among its block's warps and `chunk` of
// `chunks` among its column's blocks, both counted from the end by the backward.
struct Place {
  int lane, w, nw, chunk, chunks;
  long long col;
  unsigned long long limit;  // bound of each wait, ns; cut short once one has expired
};

// A wait that gave up: count it, and do not wait as long again (the results are void,
// yuf_sync_check says so).
YUF_DEVICE void check_wait(Place& q, bool ok) {
  if (__all_sync(0xffffffffu, ok)) return;
  if (q.lane == 0 && q.limit == WAIT_NS) atomicAdd(&g_gated_wait_timeouts, 1u);
  q.limit = 1000;
}

// The end of a kernel in which a wait gave up: its copies get time to land before the
// block's shared memory is given away.
YUF_DEVICE void linger(const Place& q) {
  if (q.limit == WAIT_NS) return;
  const unsigned long long t0 = global_ns();
  while (global_ns() - t0 < 10ull * 1000 * 1000) __nanosleep(1000);
}

// Shared memory of the exchange between a block's warps: two copies of each (a
// step's copy is read while the next step's is written; the one after that comes
// behind a barrier that every reader has passed).
constexpr int join_bytes(int V, int nw) { return 2 * 32 * V * (8 * nw + 4); }
constexpr int maps_bytes(int V, int nw) { return 32 * V * 8 * nw; }  // of ranges: one copy of the maps
constexpr int sums_bytes(int V, int nw) { return 32 * V * 8 * nw; }  // of dlower, a double per lane and channel
template <int V>
struct Joint {
  float2* warp_;
  float* carry_;
  int nw;
  YUF_DEVICE Joint(char* at, int nw) : warp_(reinterpret_cast<float2*>(at)), nw(nw) {
    carry_ = reinterpret_cast<float*>(warp_ + 2 * nw * 32 * V);
  }
  YUF_DEVICE float2* warp(int buf, int k) const { return warp_ + (buf * nw + k) * 32 * V; }
  YUF_DEVICE float* carry(int buf) const { return carry_ + buf * 32 * V; }
};

// Joins the runs of step i.  `h` is the state before the first step; returns the
// state before this warp's run, and leaves the state behind the step in the last
// warp's `h`.  Every warp forms the part before it; the last one hands the state on.
template <bool PACKED, int V>
YUF_DEVICE Fv<V> join(const Joint<V>& m, const Place& q, int i, Fv<V> A, Fv<V> H, Fv<V>& h) {
  const int buf = i & 1, at = q.lane * V;
  put_map<V>(m.warp(buf, q.w) + at, A, H);
  __syncthreads();
  if (i > 0) h = load_f32<V>(m.carry(buf ^ 1) + at);
  const Fv<V> mine = apply_all<PACKED, V>(m.warp(buf, 0) + at, q.w, h);
  if (q.w == q.nw - 1) {
    h = apply<PACKED>(A, H, mine);
    store_f32<V>(m.carry(buf) + at, h);
  }
  return mine;
}

// Maps of all ranges in the workspace: per column and chunk one row for each warp,
// and then one row for each chunk.
template <int V>
struct Ranges {
  float2 *warps, *chunks;  // this column's
  YUF_DEVICE Ranges(float* ws, const Place& q, long long cols) {
    float2* const base = reinterpret_cast<float2*>(ws);
    warps = base + q.col * q.chunks * q.nw * 32 * V;
    chunks = base + (cols * q.chunks * q.nw + q.col * q.chunks) * 32 * V;
  }
};
// End of a maps kernel: this warp's map and, by the last warp, the chunk's.
template <bool PACKED, int V>
YUF_DEVICE void leave_maps(const Joint<V>& m, const Place& q, const Ranges<V>& r, Fv<V> A, Fv<V> H) {
  const int at = q.lane * V;
  put_map<V>(r.warps + (q.chunk * q.nw + q.w) * 32 * V + at, A, H);
  put_map<V>(m.warp(0, q.w) + at, A, H);
  __syncthreads();
  if (q.w == q.nw - 1) {
    Fv<V> Ac = splat<V>(1.f), Hc = splat<V>(0.f);
    compose_all<PACKED, V>(m.warp(0, 0) + at, q.nw, Ac, Hc);
    put_map<V>(r.chunks + q.chunk * 32 * V + at, Ac, Hc);
  }
}
// Start of a ranges kernel: the state before this warp's range.  The chunks before
// this one are shared out among the warps.
template <bool PACKED, int V>
YUF_DEVICE Fv<V> take_maps(const Joint<V>& m, const Place& q, const Ranges<V>& r, Fv<V> h) {
  const int at = q.lane * V, k0 = q.chunk * q.w / q.nw, k1 = q.chunk * (q.w + 1) / q.nw;
  Fv<V> A = splat<V>(1.f), H = splat<V>(0.f);
  compose_all<PACKED, V>(r.chunks + k0 * 32 * V + at, k1 - k0, A, H);
  put_map<V>(m.warp(0, q.w) + at, A, H);
  __syncthreads();
  h = apply_all<PACKED, V>(m.warp(0, 0) + at, q.nw, h);
  return apply_all<PACKED, V>(r.warps + q.chunk * q.nw * 32 * V + at, q.w, h);
}

// What a warp has to know of its L tokens from t0 on: bit j for token t0 + j.
struct Run {
  unsigned inside;  // t0 + j < T
  unsigned live;    // inside, and in a sequence
  unsigned first;   // first / last token of its sequence (packed only: the ends of
  unsigned last;    // the row itself are the caller's)
  int owner;        // lane j + 1: the sequence of token t0 + j, where first or last has bits
  // Known of cu_seqlens: lane i holds boundary base + i (packed only), and from .. to - 1
  // are the tokens of a sequence met lately.
  int base = -1, bound = INT_MAX, from = 0, to = -1;
  YUF_DEVICE bool plain() const { return live == (1u << L) - 1 && !(first | last); }
  YUF_DEVICE int owner_of(int j) const { return __shfl_sync(0xffffffffu, owner, j + 1); }
};

// Boundaries <= t, by the whole warp: each round 32 of them cut the rest to a 32nd.  Any
// contents of cu give a value in [0, n_seqs + 1].
YUF_DEVICE int count_boundaries(const int* cu, int n_seqs, int t, int lane) {
  int lo = 0, hi = n_seqs + 1;  // the answer is in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = min(lo + lane * step, hi);
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && __ldg(cu + min(at, n_seqs)) <= t);
    const int k = __popc(below);
    if (k == 0) return lo;
    hi = min(hi, lo + k * step);
    lo += (k - 1) * step + 1;
  }
  return lo;
}

// Whether lanes' boundaries say all about tokens t0 - 1 .. t0 + L.
YUF_DEVICE bool window_covers(const Run& r, int n_seqs, int t0) {
  const int first = __shfl_sync(0xffffffffu, r.bound, 0), last = __shfl_sync(0xffffffffu, r.bound, 31);
  return r.base >= 0 && (r.base == 0 || first < t0) && (r.base + 32 > n_seqs || last > t0 + L);
}

// Sequence of lane's token t0 - 1 + lane: the last boundary at or before it, -1 before
// the first, n_seqs at and after the last one and behind the row.  With up to 31
// sequences the boundaries are read once.
template <bool REVERSE>
YUF_DEVICE int find_owners(Run& r, const GatedScanArgs& p, int t0, int lane) {
  const int t = t0 - 1 + lane;
  bool covers = window_covers(r, p.n_seqs, t0);
  if (!covers) {
    r.base = 0;
    if (p.n_seqs >= 32) {  // most of the window on the side where the next run lies
      const int before = t0 > 0 ? count_boundaries(p.cu, p.n_seqs, t0 - 1, lane) : 0;
      r.base = max(0, REVERSE ? before - 24 : before - 1);
    }
    r.bound = lane <= p.n_seqs - r.base ? __ldg(p.cu + r.base + lane) : INT_MAX;
    covers = window_covers(r, p.n_seqs, t0);
  }
  int mine;
  if (covers) {
    const int c0 = __popc(__ballot_sync(0xffffffffu, r.bound < t0)),
              c1 = __popc(__ballot_sync(0xffffffffu, r.bound <= t0 + L));
    mine = r.base - 1 + c0;
    for (int k = c0; k < c1; ++k) mine += __shfl_sync(0xffffffffu, r.bound, k) <= t;
  } else {  // empty sequences by the dozen: each lane for itself
    int lo = 0, hi = p.n_seqs + 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu + mid) <= t) lo = mid + 1;
      else hi = mid;
    }
    mine = lo - 1;
    r.base = -1;
  }
  return t < 0 ? -1 : t >= p.T ? p.n_seqs : mine;
}

// REVERSE: the next run lies before this one.  Within a sequence longer than a run this
// takes two comparisons.
template <bool PACKED, bool REVERSE>
YUF_DEVICE void look(Run& r, const GatedScanArgs& p, int t0, int lane) {
  const int n = max(0, min(L, p.T - t0));
  r.inside = r.live = (1u << n) - 1;
  r.first = r.last = 0;
  if constexpr (PACKED) {
    if (n == 0 || (r.from < t0 && t0 + L < r.to && t0 + L < p.T)) return;
    r.owner = find_owners<REVERSE>(r, p, t0, lane);
    const int prev = __shfl_up_sync(0xffffffffu, r.owner, 1), next = __shfl_down_sync(0xffffffffu, r.owner, 1);
    const bool mid = lane >= 1 && lane <= L && r.owner >= 0 && r.owner < p.n_seqs;
    r.live = (__ballot_sync(0xffffffffu, mid) >> 1) & r.inside;
    r.first = (__ballot_sync(0xffffffffu, prev != r.owner) >> 1) & r.live;
    r.last = (__ballot_sync(0xffffffffu, next != r.owner) >> 1) & r.live;
    const int at = __shfl_sync(0xffffffffu, r.owner, REVERSE ? 0 : L + 1) - r.base;
    const bool known = r.base >= 0 && at >= 0 && at < 31 && r.base + at < p.n_seqs;
    const int from = __shfl_sync(0xffffffffu, r.bound, at & 31), to = __shfl_sync(0xffffffffu, r.bound, (at + 1) & 31);
    r.from = known ? from : 0;
    r.to = known ? to : -1;
  }
}

// A sequence without a token keeps what it came with.
template <int V>
YUF_DEVICE void empty_sequences(const GatedScanArgs& p, const float* from, float* to, int c, int at, int stride) {
  for (int s = at; s < p.n_seqs; s += stride) {
    const int c0 = __ldg(p.cu + s), c1 = __ldg(p.cu + s + 1);
    if (c0 >= c1 || c0 >= p.T || c1 <= 0)
      store_f32<V>(to + (long long)s * p.D + c, from ? load_f32<V>(from + (long long)s * p.D + c) : splat<V>(0.f));
  }
}
template <int V>
YUF_DEVICE Fv<V> row_of(const float* rows, int r, int D, int c, bool act) {
  return rows && act ? load_f32<V>(rows + (long long)r * D + c) : splat<V>(0.f);
}

// ---- staging ---------------------------------------------------------------
// TMA, for rows of whole 16-byte pieces: a run is one box of 16 rows x 128 bytes per
// tensor, in slots of shared memory of the warp's own; the next boxes are under way
// while one is worked on, and neither loads nor stores cost address arithmetic
// (a fifth of all instructions otherwise).  Rows and columns past the tensor come as
// zeros and are not stored.  Otherwise: plain loads of the run into registers.
constexpr int SLOT = L * 128;

struct ScanMaps {
  CUtensorMap x, f, g, dy, o1, o2, o3;  // outputs: y, or dx, df, dg
};

YUF_DEVICE void box_load(char* slot, const CUtensorMap* map, uint64_t* bar, int c, int t, int b) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(slot)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c), "r"(t), "r"(b)
      : "memory");
}
YUF_DEVICE void box_store(const CUtensorMap* map, const char* slot, int c, int t, int b) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(slot)), "r"(c), "r"(t), "r"(b)
               : "memory");
}
template <typename T, int V>
YUF_DEVICE Raw<T, V> raw_row(const char* slot, int j, int lane) {
  return reinterpret_cast<const Raw<T, V>*>(slot + j * 128)[lane];
}
// row j of a run, from its slot or from the registers it was loaded to
template <bool TMA, typename T, int V, int N>
YUF_DEVICE Raw<T, V> row_at(const char* slot, const Raw<T, V> (&regs)[N], int j, int lane) {
  if constexpr (TMA) return raw_row<T, V>(slot, j, lane);
  else return regs[j];
}
// GROUP rows from j on.  Passes that also store to the slots read a group of rows before
// they work on it: a load cannot move up across such a store, and token after token
// would wait for its own.
constexpr int GROUP = 8;
template <typename T, int V, int N, typename Get>
YUF_DEVICE void take(Raw<T, V> (&to)[N], const Get& get, int j) {
#pragma unroll
  for (int u = 0; u < N; ++u) to[u] = get(j + u);
}
template <typename T, int V>
YUF_DEVICE void put_row(char* slot, int j, int lane, Fv<V> v) {
  reinterpret_cast<Raw<T, V>*>(slot + j * 128)[lane] = Raw<T, V>::put(v);
}
// a lane's word of row j as fp32, for values kept between two passes
YUF_DEVICE float get_word(const char* slot, int j, int lane) {
  return reinterpret_cast<const float*>(slot + j * 128)[lane];
}
YUF_DEVICE void put_word(char* slot, int j, int lane, float v) { reinterpret_cast<float*>(slot + j * 128)[lane] = v; }

// Plain loads of a warp's tokens: one row each, from `q` on; bit j of `lanes`: this lane has one.
template <typename T, int V>
YUF_DEVICE void load_rows(Raw<T, V> (&x)[L], const T* q, long long stride, unsigned lanes) {
  if (lanes == (1u << L) - 1) {
#pragma unroll
    for (int j = 0; j < L; ++j, q += stride) x[j] = load_raw<T, V>(q);
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j, q += stride) {
      x[j] = Raw<T, V>{};
      if (lanes >> j & 1) x[j] = load_raw<T, V>(q);
    }
  }
}

// The channels of a block, and what every kernel starts from.
template <typename T, int V>
struct Columns {
  int b, c0, c;
  bool act;
  Fv<V> lo, om;  // lower and 1 - lower
  YUF_DEVICE Columns(const GatedScanArgs& p, long long col, int n_cblk, int lane) {
    b = (int)(col / n_cblk);
    c0 = (int)(col % n_cblk) * 32 * V;
    c = c0 + lane * V;
    act = c < p.D;
    lo = splat<V>(0.f);
    om = splat<V>(1.f);
    if (act && p.lower) {
      lo = load_f32<V>(p.lower + c);
#pragma unroll
      for (int i = 0; i < V; ++i) om.v[i] = 1.f - lo.v[i];
    }
  }
};
template <typename T>
YUF_DEVICE const T* row_ptr(const void* t, long long sb, int b, int c) {
  return static_cast<const T*>(t) + b * sb + c;
}

// 1 / (1 + e) of token u.  TURNS: every other pair of channels on the FMA pipe (see
// rcp_1p_newton), which balances the two units in the whole form.
template <bool TURNS, int V>
YUF_DEVICE Fv<V> rcp_turns(Fv<V> e, int u) {
  if constexpr (TURNS && V == 2)
    if (u & 1) return rcp_1p_newton(e);
  return rcp_1p(e);
}
// Rates of a group of tokens, and gates of a group.
template <bool TURNS, typename T, int V, int N>
YUF_DEVICE void group_exps(const Raw<T, V> (&f)[N], Fv<V> (&s)[N], Fv<V> (&ex)[N]) {  // sigmoid(-f) = ex s
#pragma unroll
  for (int u = 0; u < N; ++u) {
    ex[u] = sigmoid_exp(sigmoid_arg(f[u]).get());
    s[u] = rcp_turns<TURNS>(ex[u], u);
  }
}
template <bool TURNS, typename T, int V, int N>
YUF_DEVICE void group_pairs(const Raw<T, V> (&f)[N], Fv<V> (&s)[N], Fv<V> (&m)[N]) {
  group_exps<TURNS>(f, s, m);
#pragma unroll
  for (int u = 0; u < N; ++u) m[u] = mul(m[u], s[u]);
}
template <bool TURNS, typename T, int V, int N>
YUF_DEVICE void group_rates(const Columns<T, V>& k, const Raw<T, V> (&f)[N], Fv<V> (&a)[N], Fv<V> (&in)[N]) {
  group_pairs<TURNS>(f, a, in);
#pragma unroll
  for (int u = 0; u < N; ++u) {
    a[u] = fma(k.om, a[u], k.lo);
    in[u] = mul(k.om, in[u]);
  }
}
template <bool TURNS, typename T, int V, int N>
YUF_DEVICE void group_gates(const Raw<T, V> (&g)[N], Fv<V> (&s)[N]) {
#pragma unroll
  for (int u = 0; u < N; ++u) s[u] = rcp_turns<TURNS>(sigmoid_exp(sigmoid_arg(g[u]).get()), u);
}

// ---------------------------------------------------------------------------
// Forward, whole.  blockIdx.x = batch row * channel blocks + channel block.
// Slots of a warp: two stages of x, f, g; y is put over x.
// Bound by HBM where the columns fill the GPU: 16x8192x1024 bf16 with a gate 181 us,
// 5.9 TB/s of its 1.07 GB.  With few columns by the step: 16 tokens of 16 warps load,
// form their maps, join and run again in 3.3 us, a third of it exponentials and
// reciprocals (two of each per element; 8x2048x640 bf16: 29 us for 84 MB, fp32: 35 us for
// 168 MB).  128 registers hold a and i x of the run between the two passes, which allows
// 16 warps; without slots (plain loads) of pairs not quite, and up to 260 bytes a thread
// are spilled.
constexpr int fwd_slots(bool gate) { return gate ? 6 : 4; }

template <typename T, int V, bool GATE, bool PACKED, bool TMA>
__global__ void __launch_bounds__(32 * NW_MAX, 1)
    gated_scan_forward_kernel(const GatedScanArgs p, const __grid_constant__ ScanMaps tm, int n_cblk) {
  constexpr int NS = GATE ? 3 : 2;
  extern __shared__ __align__(128) char smem[];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const Joint<V> joint(smem + (TMA ? nw * (fwd_slots(GATE) * SLOT + 16) : 0), nw);
  const Columns<T, V> k(p, blockIdx.x, n_cblk, lane);
  Place at{lane, w, nw, 0, 1, blockIdx.x, WAIT_NS};
  const T* const xp = row_ptr<T>(p.x, p.xb, k.b, k.c);
  const T* const fp = row_ptr<T>(p.f, p.fb, k.b, k.c);
  const T* const gp = row_ptr<T>(p.g, p.gb, k.b, k.c);
  T* const yp = static_cast<T*>(p.y) + (long long)k.b * p.T * p.D + k.c;
  const long long n_ck = (p.T + L - 1) / L;
  const int stride = nw * L, steps = (p.T + stride - 1) / stride;
  char* const mine = smem + w * (2 * NS * SLOT);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + nw * fwd_slots(GATE) * SLOT) + 2 * w;  // the stages' loads
  const auto issue = [&](int i) {  // by lane 0
    const int t = i * stride + w * L;
    if (t >= p.T) return;
    char* const s = mine + (i & 1) * NS * SLOT;
    uint64_t* const bar = &full[i & 1];
    mbar_expect_tx(bar, NS * SLOT);
    box_load(s, &tm.x, bar, k.c0, t, k.b);
    box_load(s + SLOT, &tm.f, bar, k.c0, t, k.b);
    if constexpr (GATE) box_load(s + 2 * SLOT, &tm.g, bar, k.c0, t, k.b);
  };
  if constexpr (TMA) {
    if (lane == 0) {
      mbar_init(&full[0], 1);
      mbar_init(&full[1], 1);
      fence_mbar_init();
      fence_proxy_async();
      issue(0);
    }
    __syncwarp();
  }
  Run run{};
  look<PACKED, false>(run, p, w * L, lane);  // while the first loads are under way
  Fv<V> h = splat<V>(0.f);
  if constexpr (PACKED) {
    if (p.h_last && k.act) empty_sequences<V>(p, p.h0, p.h_last, k.c, w, nw);
  } else {
    h = row_of<V>(p.h0, k.b, p.D, k.c, k.act);
  }

  for (int i = 0; i < steps; ++i) {
    const int t0 = i * stride + w * L;
    char* const sx = mine + (i & 1) * NS * SLOT;
    Raw<T, V> xr[TMA ? 1 : L], fr[TMA ? 1 : L], gr[TMA ? 1 : L];
    const auto X = [&](int j) { return row_at<TMA, T, V>(sx, xr, j, lane); };
    const auto F = [&](int j) { return row_at<TMA, T, V>(sx + SLOT, fr, j, lane); };
    const auto Gt = [&](int j) { return row_at<TMA, T, V>(sx + 2 * SLOT, gr, j, lane); };
    const unsigned lanes = k.act ? (1u << max(0, min(L, p.T - t0))) - 1 : 0;
    if constexpr (!TMA) {
      load_rows<T, V>(xr, xp + t0 * p.xt, p.xt, lanes);
      load_rows<T, V>(fr, fp + t0 * p.ft, p.ft, lanes);
      if constexpr (GATE) load_rows<T, V>(gr, gp + t0 * p.gt, p.gt, lanes);
    }
    if (i > 0) look<PACKED, false>(run, p, t0, lane);
    if (TMA && run.inside) check_wait(at, mbar_wait(&full[i & 1], (i >> 1) & 1, at.limit));
    // this warp's map; a dead token is the identity
    Fv<V> a[L], bx[L], A = splat<V>(1.f), H = splat<V>(0.f);
    const auto up = [&](auto fast) {  // fast: every token is live, and none first or last
      constexpr bool F_ = decltype(fast)::value;
#pragma unroll
      for (int j0 = 0; j0 < L; j0 += GROUP) {
        Raw<T, V> xv[GROUP], fv[GROUP];
        Fv<V> ag[GROUP], in[GROUP];
        take(xv, X, j0);
        take(fv, F, j0);
        group_rates<true>(k, fv, ag, in);
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
          const int j = j0 + u;
          a[j] = ag[u];
          bx[j] = mul(in[u], xv[u].get());
          if (!F_ && !(run.live >> j & 1)) {
            a[j] = splat<V>(1.f);
            bx[j] = splat<V>(0.f);
          }
          if (PACKED && !F_ && (run.first >> j & 1)) {
            const Fv<V> h0 = row_of<V>(p.h0, run.owner_of(j), p.D, k.c, k.act);
            if (p.h0) bx[j] = fma(a[j], h0, bx[j]);
            a[j] = splat<V>(CUT);
          }
          compose<PACKED && !F_>(A, H, a[j], bx[j]);
        }
      }
    };
    if (run.plain()) up(std::true_type{});
    else if (run.inside) up(std::false_type{});
    if (TMA && lane == 0) {
      bulk_wait_read<0>();  // y of the step before has left the slots that are loaded now
      issue(i + 1);
    }
    Fv<V> hw = join<PACKED, V>(joint, at, i, A, H, h);
    if (!run.inside) continue;
    if (p.ckpt && k.act) store_f32<V>(p.ckpt + (k.b * n_ck + t0 / L) * p.D + k.c, hw);
    const auto down = [&](auto fast) {
      constexpr bool F_ = decltype(fast)::value;
      T* yq = yp + (long long)t0 * p.D;
#pragma unroll
      for (int j0 = 0; j0 < L; j0 += GROUP) {
        Fv<V> sg[GROUP];
        if constexpr (GATE) {
          Raw<T, V> gv[GROUP];
          take(gv, Gt, j0);
          group_gates<true>(gv, sg);
        }
#pragma unroll
        for (int u = 0; u < GROUP; ++u, yq += p.D) {
          const int j = j0 + u;
          hw = apply<PACKED && !F_>(a[j], bx[j], hw);
          Fv<V> y = hw;
          if constexpr (GATE) y = mul(hw, sg[u]);
          if (!F_ && !(run.live >> j & 1)) y = splat<V>(0.f);
          if constexpr (TMA) put_row<T, V>(sx, j, lane, y);
          else if (F_ ? k.act : lanes >> j & 1) store_raw<T, V>(yq, y);
          if (PACKED && !F_ && (run.last >> j & 1)) {
            const int o = run.owner_of(j);
            if (p.h_last && k.act) store_f32<V>(p.h_last + (long long)o * p.D + k.c, hw);
          }
        }
      }
    };
    if (run.plain()) down(std::true_type{});
    else down(std::false_type{});
    if constexpr (TMA) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        box_store(&tm.o1, sx, k.c0, t0, k.b);
        bulk_commit();
      }
    }
  }
  if (!PACKED && p.h_last && w == nw - 1 && k.act) store_f32<V>(p.h_last + (long long)k.b * p.D + k.c, h);
  if (TMA && lane == 0) bulk_wait_read<0>();
  if constexpr (TMA) linger(at);
}

// ---------------------------------------------------------------------------
// Ranges: block = (column, chunk), each warp `runs` runs of its own.
template <bool REVERSE>
YUF_DEVICE Place range_place(const Split& sp) {
  const int nw = blockDim.x >> 5, w = threadIdx.x >> 5, chunk = blockIdx.x % sp.chunks;
  return Place{(int)threadIdx.x & 31, REVERSE ? nw - 1 - w : w, nw, REVERSE ? sp.chunks - 1 - chunk : chunk, sp.chunks,
               blockIdx.x / sp.chunks, WAIT_NS};
}
// first token of this warp's range
YUF_DEVICE int range_start(const Split& sp) {
  const int nw = blockDim.x >> 5, w = threadIdx.x >> 5, chunk = blockIdx.x % sp.chunks;
  return ((chunk * nw + w) * sp.runs) * L;
}
YUF_DEVICE int range_runs(const Split& sp, int t, int T) { return max(0, min(sp.runs, (T - t + L - 1) / L)); }

// The map of each range, forward: x and f; two stages.  The range is walked from its
// end, H = sum_j (a_{j+1} ... a_last) i_j x_j, so that what the ranges kernel reads
// first was read last here and is still in L2.  (The backward's are the other way
// round by themselves.)  1x16384x1024 bf16: 16 us for 67 MB, started cold; half of it
// is the start of loads and the special function unit (55 % busy).
template <typename T, int V, bool PACKED, bool TMA>
__global__ void __launch_bounds__(32 * RANGE_WARPS, 4)
    gated_scan_forward_maps_kernel(const GatedScanArgs p, const __grid_constant__ ScanMaps tm, const Split sp) {
  extern __shared__ __align__(128) char smem[];
  Place at = range_place<false>(sp);
  const int lane = at.lane, w = threadIdx.x >> 5, nw = at.nw;
  pdl_trigger();
  const Joint<V> joint(smem + (TMA ? nw * (4 * SLOT + 16) : 0), nw);
  const Columns<T, V> k(p, at.col, sp.n_cblk, lane);
  const T* const xp = row_ptr<T>(p.x, p.xb, k.b, k.c);
  const T* const fp = row_ptr<T>(p.f, p.fb, k.b, k.c);
  const int r0 = range_start(sp), n = range_runs(sp, r0, p.T);
  char* const mine = smem + w * (4 * SLOT);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + nw * 4 * SLOT) + 2 * w;
  const auto t_of = [&](int i) { return r0 + (n - 1 - i) * L; };
  const auto issue = [&](int i) {  // by lane 0
    if (i >= n) return;
    char* const s = mine + (i & 1) * 2 * SLOT;
    mbar_expect_tx(&full[i & 1], 2 * SLOT);
    box_load(s, &tm.x, &full[i & 1], k.c0, t_of(i), k.b);
    box_load(s + SLOT, &tm.f, &full[i & 1], k.c0, t_of(i), k.b);
  };
  if constexpr (TMA) {
    if (lane == 0) {
      mbar_init(&full[0], 1);
      mbar_init(&full[1], 1);
      fence_mbar_init();
      fence_proxy_async();
      issue(0);
      issue(1);
    }
    __syncwarp();
  }
  Run run{};
  look<PACKED, true>(run, p, t_of(0), lane);  // while the first loads are under way
  Fv<V> A = splat<V>(1.f), H = splat<V>(0.f);
  bool cut = false;  // before a first token nothing reaches the range's end any more
  int upto = n;  // behind a cut only what is under way is waited for
  for (int i = 0; i < upto; ++i) {
    const int t0 = t_of(i);
    char* const sx = mine + (i & 1) * 2 * SLOT;
    Raw<T, V> xr[TMA ? 1 : L], fr[TMA ? 1 : L];
    const auto X = [&](int j) { return row_at<TMA, T, V>(sx, xr, j, lane); };
    const auto F = [&](int j) { return row_at<TMA, T, V>(sx + SLOT, fr, j, lane); };
    if constexpr (!TMA) {
      const unsigned lanes = k.act ? (1u << max(0, min(L, p.T - t0))) - 1 : 0;
      load_rows<T, V>(xr, xp + t0 * p.xt, p.xt, lanes);
      load_rows<T, V>(fr, fp + t0 * p.ft, p.ft, lanes);
    }
    if (i > 0) look<PACKED, true>(run, p, t0, lane);
    if constexpr (TMA) check_wait(at, mbar_wait(&full[i & 1], (i >> 1) & 1, at.limit));
    const auto pass = [&](auto fast) {
      constexpr bool F_ = decltype(fast)::value;
#pragma unroll
      for (int j0 = L - GROUP; j0 >= 0; j0 -= GROUP) {
        Raw<T, V> xv[GROUP], fv[GROUP];
        Fv<V> a[GROUP], in[GROUP];
        take(xv, X, j0);
        take(fv, F, j0);
        group_rates<false>(k, fv, a, in);
#pragma unroll
        for (int u = GROUP - 1; u >= 0; --u) {
          const int j = j0 + u;
          if (F_ || ((run.live >> j & 1) && !cut)) {
            H = fma(A, mul(in[u], xv[u].get()), H);
            A = mul(A, a[u]);
            if (PACKED && !F_ && (run.first >> j & 1)) {
              const Fv<V> h0 = row_of<V>(p.h0, run.owner_of(j), p.D, k.c, k.act);
              if (p.h0) H = fma(A, h0, H);
              A = splat<V>(CUT);
              cut = true;
            }
          }
        }
      }
    };
    if (!cut) {
      if (run.plain()) pass(std::true_type{});
      else pass(std::false_type{});
    }
    if (PACKED && cut) upto = min(upto, TMA ? i + 2 : i + 1);
    if constexpr (TMA) {
      __syncwarp();
      if (lane == 0 && i + 2 < upto) issue(i + 2);
    }
  }
  leave_maps<PACKED, V>(joint, at, Ranges<V>(p.work, at, (long long)p.B * sp.n_cblk), A, H);
  if constexpr (TMA) linger(at);
}

// Each range from its true start state, in one pass.  Two stages of x, f, g; y is
// stored from registers, so that a stage is loaded again as soon as it is worked off
// (with y staged in a third stage half as many blocks fitted: 62 us for both kernels
// of 1x16384x1024 bf16, 50 without; 41 since).  27 us for 134 MB, started cold.
template <typename T, int V, bool GATE, bool PACKED, bool TMA>
__global__ void __launch_bounds__(32 * RANGE_WARPS, 4)
    gated_scan_forward_ranges_kernel(const GatedScanArgs p, const __grid_constant__ ScanMaps tm, const Split sp) {
  constexpr int NS = GATE ? 3 : 2;
  extern __shared__ __align__(128) char smem[];
  Place at = range_place<false>(sp);
  const int lane = at.lane, w = threadIdx.x >> 5, nw = at.nw;
  const Joint<V> joint(smem + (TMA ? nw * 2 * (NS * SLOT + 8) : 0), nw);
  const Columns<T, V> k(p, at.col, sp.n_cblk, lane);
  const T* const xp = row_ptr<T>(p.x, p.xb, k.b, k.c);
  const T* const fp = row_ptr<T>(p.f, p.fb, k.b, k.c);
  const T* const gp = row_ptr<T>(p.g, p.gb, k.b, k.c);
  T* const yp = static_cast<T*>(p.y) + (long long)k.b * p.T * p.D + k.c;
  const long long n_ck = (p.T + L - 1) / L;
  const int r0 = range_start(sp), n = range_runs(sp, r0, p.T);
  char* const mine = smem + w * (2 * NS * SLOT);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + nw * 2 * NS * SLOT) + 2 * w;
  const auto issue = [&](int i) {  // by lane 0
    if (i >= n) return;
    char* const s = mine + (i & 1) * NS * SLOT;
    uint64_t* const bar = &full[i & 1];
    mbar_expect_tx(bar, NS * SLOT);
    box_load(s, &tm.x, bar, k.c0, r0 + i * L, k.b);
    box_load(s + SLOT, &tm.f, bar, k.c0, r0 + i * L, k.b);
    if constexpr (GATE) box_load(s + 2 * SLOT, &tm.g, bar, k.c0, r0 + i * L, k.b);
  };
  if constexpr (TMA) {
    if (lane == 0) {
      mbar_init(&full[0], 1);
      mbar_init(&full[1], 1);
      fence_mbar_init();
      fence_proxy_async();
      issue(0);
      issue(1);
    }
    __syncwarp();
  }
  Run run{};
  look<PACKED, false>(run, p, r0, lane);  // while the first loads are under way
  Fv<V> h = splat<V>(0.f);
  if constexpr (PACKED) {
    if (p.h_last && k.act) empty_sequences<V>(p, p.h0, p.h_last, k.c, at.chunk * nw + w, sp.chunks * nw);
  } else {
    h = row_of<V>(p.h0, k.b, p.D, k.c, k.act);
  }
  pdl_wait();
  h = take_maps<PACKED, V>(joint, at, Ranges<V>(p.work, at, (long long)p.B * sp.n_cblk), h);

  for (int i = 0; i < n; ++i) {
    const int t0 = r0 + i * L;
    char* const sx = mine + (i & 1) * NS * SLOT;
    Raw<T, V> xr[TMA ? 1 : L], fr[TMA ? 1 : L], gr[TMA ? 1 : L];
    const auto X = [&](int j) { return row_at<TMA, T, V>(sx, xr, j, lane); };
    const auto F = [&](int j) { return row_at<TMA, T, V>(sx + SLOT, fr, j, lane); };
    const auto Gt = [&](int j) { return row_at<TMA, T, V>(sx + 2 * SLOT, gr, j, lane); };
    const unsigned lanes = k.act ? (1u << max(0, min(L, p.T - t0))) - 1 : 0;
    if constexpr (!TMA) {
      load_rows<T, V>(xr, xp + t0 * p.xt, p.xt, lanes);
      load_rows<T, V>(fr, fp + t0 * p.ft, p.ft, lanes);
      if constexpr (GATE) load_rows<T, V>(gr, gp + t0 * p.gt, p.gt, lanes);
    }
    if (i > 0) look<PACKED, false>(run, p, t0, lane);
    if constexpr (TMA) check_wait(at, mbar_wait(&full[i & 1], (i >> 1) & 1, at.limit));
    if (p.ckpt && k.act) store_f32<V>(p.ckpt + (k.b * n_ck + t0 / L) * p.D + k.c, h);
    const auto pass = [&](auto fast) {
      constexpr bool F_ = decltype(fast)::value;
      T* yq = yp + (long long)t0 * p.D;
#pragma unroll
      for (int j0 = 0; j0 < L; j0 += GROUP) {
        Raw<T, V> xv[GROUP], fv[GROUP];
        Fv<V> a[GROUP], in[GROUP], sg[GROUP];
        take(xv, X, j0);
        take(fv, F, j0);
        if constexpr (GATE) {
          Raw<T, V> gv[GROUP];
          take(gv, Gt, j0);
          group_gates<false>(gv, sg);
        }
        group_rates<false>(k, fv, a, in);
#pragma unroll
        for (int u = 0; u < GROUP; ++u, yq += p.D) {
          const int j = j0 + u;
          Fv<V> y = splat<V>(0.f);
          if (F_ || (run.live >> j & 1)) {
            if (PACKED && !F_ && (run.first >> j & 1)) h = row_of<V>(p.h0, run.owner_of(j), p.D, k.c, k.act);
            h = fma(a[u], h, mul(in[u], xv[u].get()));
            y = h;
            if constexpr (GATE) y = mul(h, sg[u]);
          }
          if (F_ ? k.act : lanes >> j & 1) store_raw<T, V>(yq, y);
          if (PACKED && !F_ && (run.last >> j & 1)) {
            const int o = run.owner_of(j);
            if (p.h_last && k.act) store_f32<V>(p.h_last + (long long)o * p.D + k.c, h);
          }
        }
      }
    };
    if (run.plain()) pass(std::true_type{});
    else pass(std::false_type{});
    if constexpr (TMA) {
      __syncwarp();
      if (lane == 0) issue(i + 2);
    }
  }
  // the range that holds the last token
  if (!PACKED && p.h_last && n > 0 && r0 + n * L >= p.T && k.act)
    store_f32<V>(p.h_last + (long long)k.b * p.D + k.c, h);
  if constexpr (TMA) linger(at);
}

// ---------------------------------------------------------------------------
// Backward, the time axis from its end: with p_t = dy_t sigmoid(g_t) and G_t the
// gradient that reaches h_t from the tokens after it,
//   dh_t = p_t + G_t,  G_{t-1} = a_t dh_t,  G_T = dL/dh_last
//   dx_t = dh_t i_t,   df_t = dh_t (h_{t-1} - x_t) i_t sigmoid(f_t)
//   dg_t = dy_t h_t sigmoid(g_t) sigmoid(-g_t)
//   dlower = sum dh_t (h_{t-1} - x_t) sigmoid(-f_t),  dL/dh_0 = G_0
// Each warp forms h of its L tokens again from the state the forward saved there
// (one per L tokens: 1/16 of a tensor's elements).  The same pass stores dg and forms
// the run's map G -> A G + H from its start on, H = sum_j P_j p_j with
// P_j = a_0 ... a_j, A = P_{L-1}.  Then the tokens run from their end.
// Slots: two stages of x and f (e^-f, 4 bytes a channel, is put over both by the first
// pass, dx and df by the second); one of dy, loaded again once h has been formed; one of
// g, which dg is put over, loaded again once dg has left.  e^-f gives both sigmoid(f) and
// sigmoid(-f) their relative accuracy again for one reciprocal, here by the special
// function unit alone (by turns with Newton's iteration 8x2048x640 bf16 took 77.9 us
// forward and backward, now 76.2; the smaller of the two sigmoids kept with a sign 77.7).
// 16x8192x1024 bf16 with a gate: 349 us, 5.4 TB/s of its 1.9 GB; bound by the latency of
// its instructions at 16 warps per SM (h and p of the run fill the registers).  The forms
// without slots keep the raw rows in registers too: of pairs they spill 150 to 350 bytes a
// thread in the whole form, 4 to 130 in ranges; of single channels up to 72.
constexpr int bwd_slots(bool gate) { return gate ? 6 : 5; }

// The block's share of dlower, the sum over its warps, to row `row` of `partial`.
// dlower sums over all tokens and rows: in fp32 within a run only, its 16 terms; runs,
// warps and blocks are added in 64 bits, where rounding does not grow with their number.
template <int V>
YUF_DEVICE void write_partial(const double* sums, const GatedScanArgs& p, const Place& q, long long row, int c,
                              bool act) {
  __syncthreads();
  if (q.w == 0 && act) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      double sum = 0.;
      for (int k = 0; k < q.nw; ++k) sum += sums[(k * V + i) * 32 + q.lane];
      p.partial[row * p.D + c + i] = (float)sum;
    }
  }
}

template <typename T, int V, bool GATE, bool PACKED, bool TMA, bool RANGES>
__global__ void __launch_bounds__(32 * NW_MAX, 1)
    gated_scan_backward_kernel(const GatedScanArgs p, const __grid_constant__ ScanMaps tm, const Split sp) {
  // Ranges store from registers, so that a slot is loaded again as soon as it is worked
  // off; the whole form puts the gradients over the inputs and has the join to wait behind.
  constexpr bool OUT_SLOT = TMA && !RANGES;
  extern __shared__ __align__(128) char smem[];
  Place at = range_place<true>(sp);
  const int lane = at.lane, w = threadIdx.x >> 5, nw = at.nw;
  constexpr int PER_WARP = TMA ? bwd_slots(GATE) * SLOT + 32 : 0;
  const Joint<V> joint(smem + nw * PER_WARP, nw);
  // The warps' sums of dlower: of packed rows, whose kernels have no register left, in
  // shared memory of their own (forward and backward of packed 8192x4096 bf16: 298 us
  // against 314), otherwise in registers until the end (1x16384x1024: 105 against 111).
  double* const sums = reinterpret_cast<double*>(
      smem + nw * PER_WARP + (!PACKED ? 0 : RANGES ? maps_bytes(V, nw) : join_bytes(V, nw)));
  double* const my_sum = sums + w * V * 32 + lane;
  double dlo[V] = {};
  if (PACKED && p.partial)
#pragma unroll
    for (int u = 0; u < V; ++u) my_sum[u * 32] = 0.;
  const Columns<T, V> k(p, at.col, sp.n_cblk, lane);
  const T* const xp = row_ptr<T>(p.x, p.xb, k.b, k.c);
  const T* const fp = row_ptr<T>(p.f, p.fb, k.b, k.c);
  const T* const gp = row_ptr<T>(p.g, p.gb, k.b, k.c);
  const T* const dyp = row_ptr<T>(p.dy, p.yb, k.b, k.c);
  const long long out0 = (long long)k.b * p.T * p.D + k.c, n_ck = (p.T + L - 1) / L;
  // runs of this warp, from the end; in the whole form the first may lie past T
  const int stride = nw * L, r0 = range_start(sp);
  const int steps = RANGES ? range_runs(sp, r0, p.T) : (p.T + stride - 1) / stride;
  const auto t_of = [&](int i) { return RANGES ? r0 + (steps - 1 - i) * L : (steps - 1 - i) * stride + w * L; };
  const auto has = [&](int i) { return i < steps && t_of(i) < p.T; };
  char* const mine = smem + w * (bwd_slots(GATE) * SLOT);
  char *const sdy = mine + 4 * SLOT, *const sg = mine + 5 * SLOT;
  // loads of x and f (two stages), dy, g
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + nw * bwd_slots(GATE) * SLOT) + 4 * w;
  // by lane 0
  const auto issue_xf = [&](int i) {
    if (!has(i)) return;
    char* const s = mine + (i & 1) * 2 * SLOT;
    mbar_expect_tx(&full[i & 1], 2 * SLOT);
    box_load(s, &tm.x, &full[i & 1], k.c0, t_of(i), k.b);
    box_load(s + SLOT, &tm.f, &full[i & 1], k.c0, t_of(i), k.b);
  };
  const auto issue_one = [&](int i, char* slot, const CUtensorMap* map, uint64_t* bar) {
    if (!has(i)) return;
    mbar_expect_tx(bar, SLOT);
    box_load(slot, map, bar, k.c0, t_of(i), k.b);
  };
  if constexpr (TMA) {
    if (lane == 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) mbar_init(&full[u], 1);
      fence_mbar_init();
      fence_proxy_async();
      issue_xf(0);
      if constexpr (RANGES) issue_xf(1);
      issue_one(0, sdy, &tm.dy, &full[2]);
      if constexpr (GATE) issue_one(0, sg, &tm.g, &full[3]);
    }
    __syncwarp();
  }
  Run run{};
  look<PACKED, true>(run, p, t_of(0), lane);  // while the first loads are under way
  Fv<V> G = splat<V>(0.f);
  if constexpr (PACKED) {
    if (p.dh0 && k.act) empty_sequences<V>(p, p.dh_last, p.dh0, k.c, at.chunk * nw + w, sp.chunks * nw);
  } else {
    G = row_of<V>(p.dh_last, k.b, p.D, k.c, k.act);
  }
  if constexpr (RANGES) {
    pdl_wait();
    G = take_maps<PACKED, V>(joint, at, Ranges<V>(p.work, at, (long long)p.B * sp.n_cblk), G);
  }

  int seen = 0;  // steps with tokens
  for (int i = 0; i < steps; ++i) {
    const int t0 = t_of(i);
    char* const sx = mine + (i & 1) * 2 * SLOT;
    char* const sf = sx + SLOT;
    Raw<T, V> xr[TMA ? 1 : L], fr[TMA ? 1 : L], gr[TMA ? 1 : L], dr[TMA ? 1 : L];
    const auto X = [&](int j) { return row_at<TMA, T, V>(sx, xr, j, lane); };
    const auto F = [&](int j) { return row_at<TMA, T, V>(sf, fr, j, lane); };
    const auto Gt = [&](int j) { return row_at<TMA, T, V>(sg, gr, j, lane); };
    const auto Dy = [&](int j) { return row_at<TMA, T, V>(sdy, dr, j, lane); };
    const unsigned lanes = k.act ? (1u << max(0, min(L, p.T - t0))) - 1 : 0;
    Fv<V> h = splat<V>(0.f);
    if (lanes & 1) h = load_f32<V>(p.ckpt + (k.b * n_ck + t0 / L) * p.D + k.c);
    if constexpr (OUT_SLOT) {
      if (lane == 0) {
        bulk_wait_read<0>();  // dx and df of the step before have left the slots that are loaded now
        issue_xf(i + 1);
        if (!has(i)) {  // nothing to work on in this step: the single slots are free
          issue_one(i + 1, sdy, &tm.dy, &full[2]);
          if constexpr (GATE) issue_one(i + 1, sg, &tm.g, &full[3]);
        }
      }
    }
    if constexpr (!TMA) {
      load_rows<T, V>(xr, xp + t0 * p.xt, p.xt, lanes);
      load_rows<T, V>(fr, fp + t0 * p.ft, p.ft, lanes);
      load_rows<T, V>(dr, dyp + t0 * p.yt, p.yt, lanes);
      if constexpr (GATE) load_rows<T, V>(gr, gp + t0 * p.gt, p.gt, lanes);
    }
    if (i > 0) look<PACKED, true>(run, p, t0, lane);
    const bool plain = run.plain();
    if (TMA && run.inside) {
      const int miss = i - seen;  // 0, or 1 where the first step had no tokens
      bool ok = mbar_wait(&full[i & 1], ((i >> 1) - ((miss && !(i & 1)) ? 1 : 0)) & 1, at.limit);
      ok = mbar_wait(&full[2], seen & 1, at.limit) && ok;
      if constexpr (GATE) ok = mbar_wait(&full[3], seen & 1, at.limit) && ok;
      check_wait(at, ok);
      ++seen;
    }
    const long long row0 = out0 + (long long)t0 * p.D;
    // e = h_{t-1} - x_t, q = p_t
    Fv<V> e[L], q[L], A = splat<V>(1.f), H = splat<V>(0.f);
    bool cut = false;  // a last token was passed: what lies behind it does not reach the run's start
    const auto up = [&](auto fast) {  // fast: every token is live, and none first or last
      constexpr bool F_ = decltype(fast)::value;
      T* dgq = GATE ? static_cast<T*>(p.dg) + row0 : nullptr;
      const auto token = [&](int j, Fv<V> xv, Fv<V> s, Fv<V> ex, Fv<V> dyv, Fv<V> sgm, Fv<V> mgm, T* dg_at) {
        const Fv<V> a = fma(k.om, s, k.lo);
        if constexpr (TMA) {
          put_word(sx, j, lane, ex.v[0]);
          if constexpr (V == 2) put_word(sf, j, lane, ex.v[V - 1]);
        }
        if (!F_ && !(run.live >> j & 1)) {
          e[j] = q[j] = splat<V>(0.f);
          if constexpr (GATE && OUT_SLOT) put_row<T, V>(sg, j, lane, e[j]);
          else if (GATE && (lanes >> j & 1)) store_raw<T, V>(dg_at, e[j]);
          return;
        }
        if (PACKED && !F_ && (run.first >> j & 1)) h = row_of<V>(p.h0, run.owner_of(j), p.D, k.c, k.act);
        e[j] = fma(xv, splat<V>(-1.f), h);
        h = fma(a, h, mul(mul(k.om, mul(ex, s)), xv));
        q[j] = dyv;
        if constexpr (GATE) {
          q[j] = mul(q[j], sgm);
          const Fv<V> dg = mul(mul(q[j], h), mgm);
          if constexpr (OUT_SLOT) put_row<T, V>(sg, j, lane, dg);
          else if (k.act) store_raw<T, V>(dg_at, dg);
        }
        if (!RANGES && !(PACKED && !F_ && cut)) {
          A = mul(A, a);
          H = fma(A, q[j], H);
          if (PACKED && !F_ && (run.last >> j & 1)) {
            const Fv<V> end = row_of<V>(p.dh_last, run.owner_of(j), p.D, k.c, k.act);
            if (p.dh_last) H = fma(A, end, H);
            A = splat<V>(CUT);
            cut = true;
          }
        }
      };
      if constexpr (F_ || (PACKED && (TMA || V == 1))) {
        constexpr int N = 4;  // as many as the registers hold beside e and q (spills of 44 bytes at most)
#pragma unroll
        for (int j0 = 0; j0 < L; j0 += N) {
          Raw<T, V> xv[N], fv[N], dv[N];
          Fv<V> s[N], ex[N], sgm[N], mgm[N];
          take(xv, X, j0);
          take(fv, F, j0);
          take(dv, Dy, j0);
          if constexpr (GATE) {
            Raw<T, V> gv[N];
            take(gv, Gt, j0);
            group_pairs<!RANGES>(gv, sgm, mgm);
          }
          group_exps<!RANGES>(fv, s, ex);
#pragma unroll
          for (int u = 0; u < N; ++u, dgq += p.D)
            token(j0 + u, xv[u].get(), s[u], ex[u], dv[u].get(), sgm[u], mgm[u], dgq);
        }
      } else {  // a row's end; pairs without slots, whose raw rows leave no registers for a group
#pragma unroll
        for (int j = 0; j < L; ++j, dgq += p.D) {
          e[j] = q[j] = splat<V>(0.f);
          if (run.live >> j & 1) {
            Fv<V> sgm, mgm;
            const Fv<V> ex = sigmoid_exp(sigmoid_arg(F(j)).get()), s = rcp_1p(ex);
            if constexpr (GATE) sigmoid_pair(sigmoid_arg(Gt(j)).get(), sgm, mgm);
            token(j, X(j).get(), s, ex, Dy(j).get(), sgm, mgm, dgq);
          } else if (GATE && (lanes >> j & 1)) {
            store_raw<T, V>(dgq, splat<V>(0.f));
          }
        }
      }
    };
    if (plain) up(std::true_type{});
    else if (run.inside) up(std::false_type{});  // a step without tokens leaves its slots alone
    if (TMA && run.inside) {
      if constexpr (GATE && OUT_SLOT) fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if constexpr (GATE && OUT_SLOT) {
          box_store(&tm.o3, sg, k.c0, t0, k.b);
          bulk_commit();
        }
        issue_one(i + 1, sdy, &tm.dy, &full[2]);
        if constexpr (GATE && !OUT_SLOT) issue_one(i + 1, sg, &tm.g, &full[3]);
      }
    }
    Fv<V> Gw = G;
    if constexpr (!RANGES) Gw = join<PACKED, V>(joint, at, i, A, H, G);
    if (!run.inside) continue;
    if (GATE && OUT_SLOT && lane == 0) {
      bulk_wait_read<0>();
      issue_one(i + 1, sg, &tm.g, &full[3]);
    }
    Fv<V> dl = splat<V>(0.f);  // this run's share of dlower
    const auto down = [&](auto fast) {
      constexpr bool F_ = decltype(fast)::value;
      T* dxq = static_cast<T*>(p.dx) + row0 + (long long)(L - 1) * p.D;
      T* dfq = static_cast<T*>(p.df) + row0 + (long long)(L - 1) * p.D;
#pragma unroll
      for (int j0 = L - GROUP; j0 >= 0; j0 -= GROUP) {
        [[maybe_unused]] Fv<V> sv[GROUP], mv[GROUP];
        if constexpr (TMA) {
#pragma unroll
          for (int u = 0; u < GROUP; ++u) {
            mv[u].v[0] = get_word(sx, j0 + u, lane);
            if constexpr (V == 2) mv[u].v[V - 1] = get_word(sf, j0 + u, lane);
            sv[u] = rcp_1p(mv[u]);
            mv[u] = mul(mv[u], sv[u]);
          }
        }
#pragma unroll
        for (int u = GROUP - 1; u >= 0; --u, dxq -= p.D, dfq -= p.D) {
          const int j = j0 + u;
          Fv<V> dx = splat<V>(0.f), df = dx;
          if (F_ || (run.live >> j & 1)) {
            if (PACKED && !F_ && (run.last >> j & 1)) Gw = row_of<V>(p.dh_last, run.owner_of(j), p.D, k.c, k.act);
            Fv<V> s, m;
            if constexpr (TMA) {
              s = sv[u];
              m = mv[u];
            } else {
              sigmoid_pair(sigmoid_arg(fr[j]).get(), s, m);
            }
            const Fv<V> dh = add(q[j], Gw), dhm = mul(dh, m);
            dx = mul(dhm, k.om);
            df = mul(mul(dx, e[j]), s);
            dl = fma(dhm, e[j], dl);
            Gw = mul(fma(k.om, s, k.lo), dh);
            if (PACKED && !F_ && (run.first >> j & 1)) {
              const int o = run.owner_of(j);
              if (p.dh0 && k.act) store_f32<V>(p.dh0 + (long long)o * p.D + k.c, Gw);
            }
          }
          if constexpr (OUT_SLOT) {
            put_row<T, V>(sx, j, lane, dx);
            put_row<T, V>(sf, j, lane, df);
          } else if (F_ ? k.act : lanes >> j & 1) {
            store_raw<T, V>(dxq, dx);
            store_raw<T, V>(dfq, df);
          }
        }
      }
    };
    if (plain) down(std::true_type{});
    else down(std::false_type{});
    if constexpr (PACKED) {
      if (p.partial)
#pragma unroll
        for (int u = 0; u < V; ++u) my_sum[u * 32] += dl.v[u];
    } else {
#pragma unroll
      for (int u = 0; u < V; ++u) dlo[u] += dl.v[u];
    }
    if constexpr (RANGES) G = Gw;
    if constexpr (OUT_SLOT) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        box_store(&tm.o1, sx, k.c0, t0, k.b);
        box_store(&tm.o2, sf, k.c0, t0, k.b);
        bulk_commit();
      }
    } else if constexpr (TMA) {
      fence_proxy_async();  // e^-f was put over the slots
      __syncwarp();
      if (lane == 0) issue_xf(i + 2);
    }
  }
  // G_0: of the whole form in its last warp, of ranges where token 0 is
  if (!PACKED && p.dh0 && k.act && (RANGES ? r0 == 0 : w == 0)) store_f32<V>(p.dh0 + (long long)k.b * p.D + k.c, G);
  if (!PACKED && p.partial) {
    __syncthreads();  // the maps in this place have been read
#pragma unroll
    for (int u = 0; u < V; ++u) my_sum[u * 32] = dlo[u];
  }
  if (p.partial) write_partial<V>(sums, p, at, (long long)k.b * sp.chunks + blockIdx.x % sp.chunks, k.c, k.act);
  if (OUT_SLOT && lane == 0) bulk_wait_read<0>();
  if constexpr (TMA) linger(at);
}

// The map of each range, backward: f, dy and g; two stages.  h is not needed.
// 1x16384x1024 bf16: 24 us for 101 MB, started cold.
template <typename T, int V, bool GATE, bool PACKED, bool TMA>
__global__ void __launch_bounds__(32 * RANGE_WARPS, 4)
    gated_scan_backward_maps_kernel(const GatedScanArgs p, const __grid_constant__ ScanMaps tm, const Split sp) {
  constexpr int NS = GATE ? 3 : 2;
  extern __shared__ __align__(128) char smem[];
  Place at = range_place<true>(sp);
  const int lane = at.lane, w = threadIdx.x >> 5, nw = at.nw;
  pdl_trigger();
  const Joint<V> joint(smem + (TMA ? nw * 2 * (NS * SLOT + 8) : 0), nw);
  const Columns<T, V> k(p, at.col, sp.n_cblk, lane);
  const T* const fp = row_ptr<T>(p.f, p.fb, k.b, k.c);
  const T* const gp = row_ptr<T>(p.g, p.gb, k.b, k.c);
  const T* const dyp = row_ptr<T>(p.dy, p.yb, k.b, k.c);
  const int r0 = range_start(sp), n = range_runs(sp, r0, p.T);
  char* const mine = smem + w * (2 * NS * SLOT);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + nw * 2 * NS * SLOT) + 2 * w;
  const auto issue = [&](int i) {  // by lane 0
    if (i >= n) return;
    char* const s = mine + (i & 1) * NS * SLOT;
    mbar_expect_tx(&full[i & 1], NS * SLOT);
    box_load(s, &tm.f, &full[i & 1], k.c0, r0 + i * L, k.b);
    box_load(s + SLOT, &tm.dy, &full[i & 1], k.c0, r0 + i * L, k.b);
    if constexpr (GATE) box_load(s + 2 * SLOT, &tm.g, &full[i & 1], k.c0, r0 + i * L, k.b);
  };
  if constexpr (TMA) {
    if (lane == 0) {
      mbar_init(&full[0], 1);
      mbar_init(&full[1], 1);
      fence_mbar_init();
      fence_proxy_async();
      issue(0);
      issue(1);
    }
    __syncwarp();
  }
  Run run{};
  look<PACKED, false>(run, p, r0, lane);  // while the first loads are under way
  Fv<V> A = splat<V>(1.f), H = splat<V>(0.f);
  bool cut = false;  // behind a last token nothing reaches the range's start any more
  int upto = n;  // behind a cut only what is under way is waited for
  for (int i = 0; i < upto; ++i) {
    const int t0 = r0 + i * L;
    char* const sf = mine + (i & 1) * NS * SLOT;
    Raw<T, V> fr[TMA ? 1 : L], dr[TMA ? 1 : L], gr[TMA ? 1 : L];
    const auto F = [&](int j) { return row_at<TMA, T, V>(sf, fr, j, lane); };
    const auto Dy = [&](int j) { return row_at<TMA, T, V>(sf + SLOT, dr, j, lane); };
    const auto Gt = [&](int j) { return row_at<TMA, T, V>(sf + 2 * SLOT, gr, j, lane); };
    if constexpr (!TMA) {
      const unsigned lanes = k.act ? (1u << max(0, min(L, p.T - t0))) - 1 : 0;
      load_rows<T, V>(fr, fp + t0 * p.ft, p.ft, lanes);
      load_rows<T, V>(dr, dyp + t0 * p.yt, p.yt, lanes);
      if constexpr (GATE) load_rows<T, V>(gr, gp + t0 * p.gt, p.gt, lanes);
    }
    if (i > 0) look<PACKED, false>(run, p, t0, lane);
    if constexpr (TMA) check_wait(at, mbar_wait(&full[i & 1], (i >> 1) & 1, at.limit));
    const auto pass = [&](auto fast) {
      constexpr bool F_ = decltype(fast)::value;
#pragma unroll
      for (int j0 = 0; j0 < L; j0 += GROUP) {
        Raw<T, V> fv[GROUP], dv[GROUP];
        Fv<V> a[GROUP], in[GROUP], sg[GROUP];
        take(fv, F, j0);
        take(dv, Dy, j0);
        if constexpr (GATE) {
          Raw<T, V> gv[GROUP];
          take(gv, Gt, j0);
          group_gates<false>(gv, sg);
        }
        group_rates<false>(k, fv, a, in);
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
          const int j = j0 + u;
          if (F_ || ((run.live >> j & 1) && !cut)) {
            A = mul(A, a[u]);
            H = fma(A, GATE ? mul(dv[u].get(), sg[u]) : dv[u].get(), H);
            if (PACKED && !F_ && (run.last >> j & 1)) {
              const Fv<V> end = row_of<V>(p.dh_last, run.owner_of(j), p.D, k.c, k.act);
              if (p.dh_last) H = fma(A, end, H);
              A = splat<V>(CUT);
              cut = true;
            }
          }
        }
      }
    };
    if (!cut) {
      if (run.plain()) pass(std::true_type{});
      else pass(std::false_type{});
    }
    if (PACKED && cut) upto = min(upto, TMA ? i + 2 : i + 1);
    if constexpr (TMA) {
      __syncwarp();
      if (lane == 0 && i + 2 < upto) issue(i + 2);
    }
  }
  leave_maps<PACKED, V>(joint, at, Ranges<V>(p.work, at, (long long)p.B * sp.n_cblk), A, H);
  if constexpr (TMA) linger(at);
}

// ---- host -------------------------------------------------------------------

constexpr int SMEM_MAX = 227 * 1024;
static_assert(NW_MAX * (bwd_slots(true) * SLOT + 32) + join_bytes(2, NW_MAX) + sums_bytes(2, NW_MAX) <= SMEM_MAX,
              "shared memory of a block");

// A kernel's dynamic shared memory, allowed once per device.
bool allow_smem(const void* kernel, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

// `after`: the kernel waits for the one before it by itself (programmatic dependent launch)
template <auto KERNEL, typename Third>
yuf_status_t launch(const char* what, const GatedScanArgs& a, const ScanMaps& m, const Third& third, const Plan& p,
                    int smem, bool after, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(reinterpret_cast<const void*>(KERNEL), done)) {
    set_error("gated scan: cannot set the shared memory of %s", what);
    return YUF_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.blocks);
  cfg.blockDim = dim3(32 * p.nw);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 1 : 0;
  cudaLaunchKernelEx(&cfg, KERNEL, a, m, third);
  return check_launch(what);
}

// [B, T, D] with element strides st (tokens) and sb (rows) as boxes of 16 tokens x 128 bytes
bool scan_map(CUtensorMap* m, int dtype, const void* base, const GatedScanArgs& a, long long sb, long long st) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const int e = gated_elem_size(dtype);
  if (a.B == 1) sb = st;
  const cuuint64_t dim[3] = {(cuuint64_t)a.D, (cuuint64_t)a.T, (cuuint64_t)a.B};
  const cuuint64_t stride[2] = {(cuuint64_t)(st * e), (cuuint64_t)(sb * e)};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / e), (cuuint32_t)L, 1}, one[3] = {1, 1, 1};
  const CUtensorMapDataType t = dtype == YUF_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == YUF_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(m, t, 3, const_cast<void*>(base), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Maps of a call's tensors; false where TMA cannot take them: rows that are not
// whole 16-byte pieces, tokens or rows that share memory (stride 0), or whatever
// else the driver refuses.
bool scan_maps(ScanMaps& m, const GatedScanArgs& a, bool backward) {
  const long long piece = 16 / gated_elem_size(a.dtype), td = (long long)a.T * a.D;
  struct Item {
    CUtensorMap* map;
    const void* base;
    long long sb, st;
  };
  const Item items[] = {{&m.x, a.x, a.xb, a.xt},  {&m.f, a.f, a.fb, a.ft}, {&m.g, a.g, a.gb, a.gt},
                        {&m.dy, a.dy, a.yb, a.yt}, {&m.o1, backward ? a.dx : a.y, td, a.D},
                        {&m.o2, a.df, td, a.D},    {&m.o3, a.dg, td, a.D}};
  if (a.T == 0 || a.D % piece != 0) return false;
  for (const Item& t : items)
    if (t.base && (!gated_aligned(t.base, 16) || t.st == 0 || t.st % piece != 0 ||
                   (a.B > 1 && (t.sb == 0 || t.sb % piece != 0))))
      return false;
  for (const Item& t : items)
    if (t.base && !scan_map(t.map, a.dtype, t.base, a, t.sb, t.st)) return false;
  return true;
}

template <typename T, int V, bool GATE, bool PACKED, bool TMA>
yuf_status_t forward_with(const GatedScanArgs& a, const ScanMaps& m, cudaStream_t st) {
  const Plan p = gated_scan_plan(a.B, a.T, a.D, V);
  const int j = p.ranges ? maps_bytes(V, p.nw) : join_bytes(V, p.nw);
  if (!p.ranges)
    return launch<gated_scan_forward_kernel<T, V, GATE, PACKED, TMA>>(
        "gated_scan_forward_kernel", a, m, p.sp.n_cblk, p, (TMA ? p.nw * (fwd_slots(GATE) * SLOT + 16) : 0) + j, false,
        st);
  const yuf_status_t rc = launch<gated_scan_forward_maps_kernel<T, V, PACKED, TMA>>(
      "gated_scan_forward_maps_kernel", a, m, p.sp, p, (TMA ? p.nw * (4 * SLOT + 16) : 0) + j, false, st);
  if (rc != YUF_OK) return rc;
  return launch<gated_scan_forward_ranges_kernel<T, V, GATE, PACKED, TMA>>(
      "gated_scan_forward_ranges_kernel", a, m, p.sp, p,
      (TMA ? p.nw * 2 * ((GATE ? 3 : 2) * SLOT + 8) : 0) + j, true, st);
}
template <typename T, int V, bool GATE, bool PACKED, bool TMA>
yuf_status_t backward_with(const GatedScanArgs& a, const ScanMaps& m, cudaStream_t st) {
  const Plan p = gated_scan_plan(a.B, a.T, a.D, V);
  const int j = p.ranges ? maps_bytes(V, p.nw) : join_bytes(V, p.nw);
  const int s = (TMA ? p.nw * (bwd_slots(GATE) * SLOT + 32) : 0) + j + (PACKED ? sums_bytes(V, p.nw) : 0);
  GatedScanArgs b = a;
  const long long shares = (long long)a.B * p.sp.chunks;  // of dlower
  if (a.dlower) b.partial = shares == 1 ? a.dlower : a.work + p.map_floats(V);
  yuf_status_t rc;
  if (!p.ranges) {
    rc = launch<gated_scan_backward_kernel<T, V, GATE, PACKED, TMA, false>>("gated_scan_backward_kernel", b, m, p.sp, p,
                                                                            s, false, st);
  } else {
    rc = launch<gated_scan_backward_maps_kernel<T, V, GATE, PACKED, TMA>>(
        "gated_scan_backward_maps_kernel", b, m, p.sp, p, (TMA ? p.nw * 2 * ((GATE ? 3 : 2) * SLOT + 8) : 0) + j, false,
        st);
    if (rc == YUF_OK)
      rc = launch<gated_scan_backward_kernel<T, V, GATE, PACKED, TMA, true>>("gated_scan_backward_kernel (ranges)", b, m,
                                                                             p.sp, p, s, true, st);
  }
  if (rc != YUF_OK || !a.dlower || shares == 1) return rc;
  return gated_scan_dlower(b.partial, a.dlower, shares, a.D, st);
}

template <typename T, int V, bool GATE, bool PACKED>
yuf_status_t run_with(const GatedScanArgs& a, bool backward, cudaStream_t st) {
  ScanMaps m{};
  if constexpr (sizeof(T) * V == 4)
    if (scan_maps(m, a, backward))
      return backward ? backward_with<T, V, GATE, PACKED, true>(a, m, st)
                      : forward_with<T, V, GATE, PACKED, true>(a, m, st);
  return backward ? backward_with<T, V, GATE, PACKED, false>(a, m, st)
                  : forward_with<T, V, GATE, PACKED, false>(a, m, st);
}
template <typename T, int V>
yuf_status_t run_as(const GatedScanArgs& a, bool backward, cudaStream_t st) {
  if (a.g) return a.cu ? run_with<T, V, true, true>(a, backward, st) : run_with<T, V, true, false>(a, backward, st);
  return a.cu ? run_with<T, V, false, true>(a, backward, st) : run_with<T, V, false, false>(a, backward, st);
}
unsigned int wait_timeouts() {
  unsigned int n = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&n, g_gated_wait_timeouts, sizeof(n)) != cudaSuccess ||
      cudaMemcpyToSymbol(g_gated_wait_timeouts, &zero, sizeof(zero)) != cudaSuccess) {
    cudaGetLastError();
    return ~0u;
  }
  return n;
}

}  // namespace

}  // namespace yuf
