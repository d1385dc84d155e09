// Log probabilities of a row of scores: of given labels, with the entropy and the best
// alternatives, and the scores' gradient.
//
// For row x of m scores and z_j = scale * x_j (a squared distance takes a negative scale):
//   M = max z,  S = sum exp(z_j - M),  T = sum exp(z_j - M) (z_j - M),  L = log S
//   log p_j = z_j - M - L        entropy H = L - T / S
//   dz_j = g_l ([j = l] - p_j) - g_H p_j (log p_j + H),  dx_j = scale * dz_j
// z_j - M is formed as (y_j - max y) |scale| with y = sign(scale) x, which loses nothing
// to a common offset of the scores.  T and H are sums of terms of one sign.
//
// Masked scores (z = -inf) have probability 0 and add nothing.  A row with no score left
// has log probabilities of -inf, entropy 0 and a zero gradient; a row that holds a NaN or
// z = +inf has NaN in all of them.  Alternatives go by y, equal ones by the lower index;
// NaN counts as the largest value.
#include "common.cuh"
#include "engine.h"
#include "rows.cuh"

#include <algorithm>

namespace euc {

// y's order as an unsigned integer; -0 and 0 are equal, NaN is above +inf
__device__ __forceinline__ uint32_t order_of(float y) {
  if (y != y) return 0xffffffffu;
  const uint32_t b = __float_as_uint(y + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double y) {
  if (y != y) return ~0ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(y + 0.0));
  return b >> 63 ? ~b : b | (1ull << 63);
}

// Exponents are held in units of log 2 for fp32 (t = d log2 e, one ex2 a score; ex2.approx
// is off by at most 2^-22 of the result and flushes results below 2^-126), in natural units
// for fp64.  `per_nat` converts mag into a factor of such a unit, `unit` a unit back.
template <typename A> struct Expo;
template <> struct Expo<float> {
  static constexpr float per_nat = 1.4426950408889634f, unit = 0.6931471805599453f;
  static constexpr float floor = -200.f;  // ex2 of it is 0
  static __device__ __forceinline__ float exp(float t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
  }
};
template <> struct Expo<double> {
  static constexpr double per_nat = 1.0, unit = 1.0;
  static constexpr double floor = -1000.0;
  static __device__ __forceinline__ double exp(double t) { return ::exp(t); }
};
__device__ __forceinline__ float log_acc(float d) { return logf(d); }
__device__ __forceinline__ double log_acc(double d) { return log(d); }

template <typename A> __device__ __forceinline__ A neg_inf() { return -static_cast<A>(INFINITY); }

// the larger; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) { return fmax_nan(a, b); }
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : (b > a || b != b ? b : a); }
__device__ __forceinline__ double max_nan(double a, double b, double c) { return max_nan(max_nan(a, b), c); }

template <typename A> __device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ double warp_max_nan(double v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}

// The warp's values in descending order over the lanes (bitonic exchanges).
template <typename A> __device__ __forceinline__ A warp_sort_desc(A v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const A o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool up = ((lane & k) == 0) == ((lane & j) == 0);  // this lane keeps the larger
      v = up ? (o > v ? o : v) : (o < v ? o : v);
    }
  return v;
}

template <typename T> struct ScoreArgs {
  const T* x;
  int64_t ld;
  const void* labels;
  int labels_i64;
  int64_t n;
  int m;
  Acc<T> sign, mag;
  int top;
  Acc<T>* log_probs;
  Acc<T>* entropy;
  Acc<T>* stats;
  Acc<T>* top_log_probs;
  int64_t* top_labels;
};

template <typename T> __device__ __forceinline__ int64_t label_of(const void* labels, int i64, int64_t i) {
  return i64 ? static_cast<const long long*>(labels)[i] : static_cast<const int*>(labels)[i];
}

// the row's outputs from its M (as max y), S and T
template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs<T>& a, int64_t i, Acc<T> hi, Acc<T> S, Acc<T> Tm) {
  using A = Acc<T>;
  const bool empty = hi == neg_inf<A>();
  const A L = empty ? neg_inf<A>() : log_acc(S);
  const A H = empty ? A(0) : L - Tm / S;
  if (a.entropy) a.entropy[i] = H;
  if (a.stats) {
    a.stats[3 * i] = hi;
    a.stats[3 * i + 1] = L;
    a.stats[3 * i + 2] = H;
  }
  if (a.log_probs) {
    const int64_t l = label_of<T>(a.labels, a.labels_i64, i);
    A lp = A(0);
    if (l >= 0 && l < a.m) lp = empty ? neg_inf<A>() : (a.sign * to_acc(a.x[i * a.ld + l]) - hi) * a.mag - L;
    a.log_probs[i] = lp;
  }
}

template <typename A> struct Best {
  decltype(order_of(A())) o;
  int j;
};
template <typename A> __device__ __forceinline__ bool before(const Best<A>& p, const Best<A>& q) {
  return p.o > q.o || (p.o == q.o && p.j < q.j);
}

// ------------------------------------------------------------------ a row as vectors
// Vector v of a row is the 16 bytes at its v-th 16-byte boundary, counted from the one at or
// before the row's start (`off` elements before it).  Elements outside the row read as -inf
// in y, which adds nothing to any sum; nothing outside the row is read.
template <typename T> struct RowVecs {
  static constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const T* x;
  int m, off;
  __device__ __forceinline__ RowVecs(const T* x_, int m_) : x(x_), m(m_) {
    off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  }
  __device__ __forceinline__ int64_t count() const { return (static_cast<int64_t>(m) + off + VE - 1) / VE; }
  __device__ __forceinline__ int64_t first(int64_t v) const { return v * VE - off; }
  // the 16 bytes; `negate` flips the signs (y = -x)
  __device__ __forceinline__ void load(int64_t v, bool negate, Acc<T>* y) const {
    const int64_t j = first(v);
    Vec<T, VE> w;
    if (j >= 0 && j + VE <= m) {
      w.raw = load_keep(reinterpret_cast<const uint4*>(x + j));
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = to_acc(w.e[e]);
      if (negate) {
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = -y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        y[e] = neg_inf<Acc<T>>();
        if (j + e >= 0 && j + e < m) y[e] = negate ? -to_acc(x[j + e]) : to_acc(x[j + e]);
      }
    }
  }
};

template <typename A, int N> __device__ __forceinline__ A max_of(const A* y) {
  A r = y[0];
#pragma unroll
  for (int e = 1; e + 1 < N; e += 2) r = max_nan(r, y[e], y[e + 1]);
  if (N % 2 == 0) r = max_nan(r, y[N - 1]);
  return r;
}

// S += exp(t), T += exp(t) t over N scores, t = (y - shift) c; two interleaved partial sums
template <typename A> struct Sums {
  A s[2], t[2];
  __device__ __forceinline__ Sums() : s{A(0), A(0)}, t{A(0), A(0)} {}
  template <int N> __device__ __forceinline__ void add(const A* y, A shift, A c) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      A u = (y[e] - shift) * c;
      u = u > Expo<A>::floor ? u : Expo<A>::floor;
      const A x = Expo<A>::exp(u);
      s[e & 1] += x;
      t[e & 1] += x * u;
    }
  }
  // the same sums about a larger shift: every t falls by `drop` (<= 0)
  __device__ __forceinline__ void move(A drop) {
    const A f = Expo<A>::exp(drop > Expo<A>::floor ? drop : Expo<A>::floor);
    const A d = drop > Expo<A>::floor ? drop : A(0);  // f is 0 below
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      t[q] = f * (t[q] + s[q] * d);
      s[q] *= f;
    }
  }
};
template <> struct Sums<float> {
  uint64_t s, t;
  __device__ __forceinline__ Sums() : s(0), t(0) {}
  template <int N> __device__ __forceinline__ void add(const float* y, float shift, float c) {
    const uint64_t sh = f2_pack(shift, shift), cc = f2_pack(c, c);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float u0, u1;
      f2_unpack(f2_mul(f2_sub(f2_pack(y[e], y[e + 1]), sh), cc), u0, u1);
      u0 = fmaxf(u0, Expo<float>::floor);
      u1 = fmaxf(u1, Expo<float>::floor);
      const uint64_t x = f2_pack(Expo<float>::exp(u0), Expo<float>::exp(u1));
      s = f2_add(s, x);
      t = f2_fma(x, f2_pack(u0, u1), t);
    }
  }
  __device__ __forceinline__ void move(float drop) {
    const float f = Expo<float>::exp(fmaxf(drop, Expo<float>::floor));
    const float d = drop > Expo<float>::floor ? drop : 0.f;
    const uint64_t ff = f2_pack(f, f), dd = f2_pack(d, d);
    t = f2_mul(ff, f2_fma(s, dd, t));
    s = f2_mul(s, ff);
  }
};
__device__ __forceinline__ void both(const Sums<float>& p, float& s, float& t) {
  float a, b;
  f2_unpack(p.s, a, b);
  s = a + b;
  f2_unpack(p.t, a, b);
  t = a + b;
}
__device__ __forceinline__ void both(const Sums<double>& p, double& s, double& t) {
  s = p.s[0] + p.s[1];
  t = p.t[0] + p.t[1];
}

// ------------------------------------------------------------------ the alternatives
// The `top` best of a row without sorting it: any number t that at least `top` scores reach
// bounds the last of them from below, and few scores reach a good one.  t comes from the
// lanes' maxima, which the softmax needs anyhow; the scores that reach it go to a list in
// shared memory (in any order), and a candidate's place is the number of candidates before
// it.  More candidates than the list holds (many equal scores), or a NaN, take the plain way:
// the best one behind the last one, `top` times.
template <typename A> struct Cand {
  A y;
  int j;
};
template <typename A> __device__ __forceinline__ bool ahead(const Cand<A>& p, const Cand<A>& q) {
  return p.y > q.y || (p.y == q.y && p.j < q.j);
}

template <typename T>
__device__ __forceinline__ void write_top(const ScoreArgs<T>& a, int64_t i, int place, Acc<T> y, int j, Acc<T> hi,
                                          Acc<T> L) {
  a.top_labels[i * a.top + place] = j;
  a.top_log_probs[i * a.top + place] = hi == neg_inf<Acc<T>>() ? hi : (y - hi) * a.mag - L;
}

// ------------------------------------------------------------------ one warp per row
// Rows of up to 32 EPL scores: the row stays in registers, so its scores are read once and
// its maximum is known before the first exponential.
constexpr int kWarpCands = 128;

template <typename T, int EPL>
__global__ void __launch_bounds__(128) scores_warp_kernel(ScoreArgs<T> a) {
  using A = Acc<T>;
  constexpr int VE = RowVecs<T>::VE, NV = EPL / VE;
  __shared__ Cand<A> cands[4][kWarpCands];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool negate = a.sign < A(0);
  const A c = a.mag * Expo<A>::per_nat;
  Cand<A>* list = cands[warp];
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + warp; i < a.n; i += static_cast<int64_t>(gridDim.x) * 4) {
    const RowVecs<T> row(a.x + i * a.ld, a.m);
    A y[EPL];
#pragma unroll
    for (int v = 0; v < NV; ++v) row.load(v * 32 + lane, negate, y + v * VE);
    const A mine = max_of<A, EPL>(y);
    const A hi = warp_max_nan(mine);
    Sums<A> sums;
    sums.template add<EPL>(y, hi == neg_inf<A>() ? A(0) : hi, c);
    A S, Tm;
    both(sums, S, Tm);
    S = warp_sum(S);
    Tm = warp_sum(Tm) * Expo<A>::unit;
    const bool odd = hi != hi || hi == -neg_inf<A>();
    if (odd) S = Tm = static_cast<A>(NAN);
    if (lane == 0) write_row(a, i, hi, S, Tm);
    if (a.top == 0) continue;
    const A L = hi == neg_inf<A>() ? hi : log_acc(S);
    bool slow = hi != hi;
    int count = 0;
    if (!slow) {
      const A t = __shfl_sync(0xffffffffu, warp_sort_desc(mine, lane), a.top - 1);
      const bool none = t == neg_inf<A>();  // fewer than `top` lanes hold a score
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        const bool in = none ? y[q] > t : y[q] >= t;
        const unsigned b = __ballot_sync(0xffffffffu, in);
        if (b == 0u) continue;
        const int at = count + __popc(b & ((1u << lane) - 1u));
        if (in && at < kWarpCands) {
          list[at].y = y[q];
          list[at].j = static_cast<int>(row.first((q / VE) * 32 + lane)) + q % VE;
        }
        count += __popc(b);
      }
      if (none) {  // masked scores by index: the first 2 top hold enough of them
        for (int j0 = 0; j0 < min(a.m, 2 * a.top); j0 += 32) {
          const int j = j0 + lane;
          const bool in = j < min(a.m, 2 * a.top) && a.sign * to_acc(row.x[j]) == neg_inf<A>();
          const unsigned b = __ballot_sync(0xffffffffu, in);
          const int at = count + __popc(b & ((1u << lane) - 1u));
          if (in && at < kWarpCands) {
            list[at].y = neg_inf<A>();
            list[at].j = j;
          }
          count += __popc(b);
        }
      }
      slow = count > kWarpCands;
    }
    __syncwarp();
    if (!slow) {
      for (int q = lane; q < count; q += 32) {
        const Cand<A> me = list[q];
        int place = 0;
        for (int r = 0; r < count; ++r) place += ahead(list[r], me) ? 1 : 0;
        if (place < a.top) write_top(a, i, place, me.y, me.j, hi, L);
      }
    } else {
      Best<A> last{};
      for (int k = 0; k < a.top; ++k) {
        Best<A> best;
        best.o = 0;
        best.j = 0x7fffffff;
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
          const int64_t j = row.first((q / VE) * 32 + lane) + q % VE;
          if (j < 0 || j >= a.m) continue;
          Best<A> o;
          o.o = order_of(y[q]);
          o.j = static_cast<int>(j);
          if ((k == 0 || before(last, o)) && before(o, best)) best = o;
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
          Best<A> o;
          o.o = __shfl_xor_sync(0xffffffffu, best.o, s);
          o.j = __shfl_xor_sync(0xffffffffu, best.j, s);
          if (before(o, best)) best = o;
        }
        last = best;
        if (lane == 0) write_top(a, i, k, a.sign * to_acc(row.x[best.j]), best.j, hi, L);
      }
    }
    __syncwarp();
  }
}

// v to the same shared variable of the cluster's first block
template <typename V> __device__ __forceinline__ void store_cluster(const V* at, const V& v) {
  static_assert(sizeof(V) % 4 == 0, "whole words");
  const uint32_t to = cluster_addr(at, 0);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (uint32_t q = 0; q < sizeof(V) / 4; ++q)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4 * q), "r"(w[q]) : "memory");
}

// ------------------------------------------------------------------ blocks per row
// Longer rows are streamed once by a cluster of 1 to 8 blocks (several where the rows are
// too few to fill the SMs), each with a slice of the row's vectors.  A thread keeps its own
// maximum and sums about it, moved when the maximum grows (rarely, after the first
// vectors), and, for the alternatives, the maximum of each of its kGroups groups of
// vectors: after the sweep only the groups that reach the bound are read again (from L2).
// The blocks' results are joined in the first block's shared memory, in rank order.
constexpr int kGroups = 32;       // groups of vectors per thread
constexpr int kBlockVecs = 4;     // vectors in flight per thread
constexpr int kBlockCands = 512;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;

template <typename A> struct Part {  // one block's share of a row
  A hi, S, T;
  int count;  // alternatives listed
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT) scores_block_kernel(ScoreArgs<T> a, int cluster, int per_group) {
  using A = Acc<T>;
  constexpr int VE = RowVecs<T>::VE, U = kBlockVecs, W = NT / 32;
  extern __shared__ __align__(16) unsigned char dyn[];
  A* group_max = reinterpret_cast<A*>(dyn);  // [kGroups][NT], with alternatives only
  __shared__ Cand<A> cands[kBlockCands];
  __shared__ Cand<A> lists[kMaxCluster][kMaxTop];
  __shared__ Part<A> parts[kMaxCluster];
  __shared__ A red[3][W];
  __shared__ int count_sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = blockIdx.x / cluster;
  const int rank = static_cast<int>(blockIdx.x - i * cluster);
  const bool negate = a.sign < A(0);
  const A c = a.mag * Expo<A>::per_nat;
  const RowVecs<T> row(a.x + i * a.ld, a.m);
  const int64_t all = row.count(), per = (all + cluster - 1) / cluster;
  const int64_t v0 = min(all, rank * per), v1 = min(all, v0 + per);
  const int steps = static_cast<int>((v1 - v0 + U * NT - 1) / (U * NT));
  if (threadIdx.x == 0) count_sh = 0;
  if (cluster > 1) cluster_arrive();  // waited for before the first store to another block

  A mine = neg_inf<A>(), gm = neg_inf<A>();
  Sums<A> sums;
  int g = 0, in_group = 0;
  for (int s = 0; s < steps; ++s) {
    A y[U * VE];
    const int64_t v = v0 + static_cast<int64_t>(s) * (U * NT) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v + u * NT < v1) {
        row.load(v + u * NT, negate, y + u * VE);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) y[u * VE + e] = neg_inf<A>();
      }
    }
    const A most = max_of<A, U * VE>(y);
    gm = max_nan(gm, most);
    if (!(most <= mine)) {  // larger, or a NaN
      if (mine > neg_inf<A>()) sums.move((mine - most) * c);
      mine = max_nan(mine, most);
    }
    sums.template add<U * VE>(y, mine == neg_inf<A>() ? A(0) : mine, c);
    if (++in_group == per_group) {
      if (a.top) group_max[g * NT + threadIdx.x] = gm;
      ++g;
      in_group = 0;
      gm = neg_inf<A>();
    }
  }
  if (in_group && a.top) group_max[g * NT + threadIdx.x] = gm;

  // the block's maximum and sums, and the alternatives' bound
  const A wmax = warp_max_nan(mine);
  const int want = static_cast<int>(min(static_cast<int64_t>(a.top), (v1 - v0) * VE));
  A some = neg_inf<A>(), each = neg_inf<A>();
  if (a.top && want > 0) {
    // `want` scores reach the warp's want-th largest lane maximum; ceil(want / W) in every
    // warp reach the smallest of the warps' ceil(want / W)-th largest
    const A sorted = warp_sort_desc(mine, lane);
    some = __shfl_sync(0xffffffffu, sorted, want - 1);
    each = __shfl_sync(0xffffffffu, sorted, (want + W - 1) / W - 1);
  }
  if (lane == 0) {
    red[0][warp] = wmax;
    red[1][warp] = some;
    red[2][warp] = each;
  }
  __syncthreads();
  A hi = red[0][0], bound = red[1][0], least = red[2][0];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    hi = max_nan(hi, red[0][w]);
    bound = red[1][w] > bound ? red[1][w] : bound;
    least = red[2][w] < least ? red[2][w] : least;
  }
  bound = least > bound ? least : bound;
  __syncthreads();
  if (mine > neg_inf<A>()) sums.move((mine - hi) * c);
  A S, Tm;
  both(sums, S, Tm);
  S = warp_sum(S);
  Tm = warp_sum(Tm);
  if (lane == 0) {
    red[0][warp] = S;
    red[1][warp] = Tm;
  }
  __syncthreads();
  S = Tm = A(0);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    S += red[0][w];
    Tm += red[1][w];
  }

  // this block's best `want` scores, in order, in list[rank]
  Cand<A>* list = lists[rank];
  const bool has_nan = hi != hi;
  if (a.top && want > 0) {
    const bool none = bound == neg_inf<A>();
    bool slow = has_nan;
    if (!slow) {
      for (int q = 0; q * per_group < steps; ++q) {
        const A top_of = group_max[q * NT + threadIdx.x];
        if (none ? !(top_of > bound) : !(top_of >= bound)) continue;
        for (int s = q * per_group; s < min(steps, (q + 1) * per_group); ++s)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int64_t v = v0 + static_cast<int64_t>(s) * (U * NT) + u * NT + threadIdx.x;
            if (v >= v1) continue;
            A y[VE];
            row.load(v, negate, y);
#pragma unroll
            for (int e = 0; e < VE; ++e)
              if (none ? y[e] > bound : y[e] >= bound) {
                const int at = atomicAdd(&count_sh, 1);
                if (at < kBlockCands) {
                  cands[at].y = y[e];
                  cands[at].j = static_cast<int>(row.first(v)) + e;
                }
              }
          }
      }
      if (none) {  // masked scores by index, from the slice's first 2 want
        const int64_t j = max(static_cast<int64_t>(0), row.first(v0)) + threadIdx.x;
        if (threadIdx.x < 2 * want && j < a.m && j < row.first(v1) && a.sign * to_acc(row.x[j]) == neg_inf<A>()) {
          const int at = atomicAdd(&count_sh, 1);
          if (at < kBlockCands) {
            cands[at].y = neg_inf<A>();
            cands[at].j = static_cast<int>(j);
          }
        }
      }
      __syncthreads();
      slow = count_sh > kBlockCands;
    }
    if (!slow) {
      const int count = count_sh;
      for (int q = threadIdx.x; q < count; q += NT) {
        const Cand<A> me = cands[q];
        int place = 0;
        for (int r = 0; r < count; ++r) place += ahead(cands[r], me) ? 1 : 0;
        if (place < want) list[place] = me;
      }
      if (threadIdx.x == 0) parts[rank].count = min(count, want);
    } else {
      Best<A>* redb = reinterpret_cast<Best<A>*>(cands);
      Best<A> last{};
      int k = 0;
      for (; k < want; ++k) {
        Best<A> best;
        best.o = 0;
        best.j = 0x7fffffff;
        for (int64_t v = v0 + threadIdx.x; v < v1; v += NT) {
          A y[VE];
          row.load(v, negate, y);
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int64_t j = row.first(v) + e;
            if (j < 0 || j >= a.m) continue;
            Best<A> o;
            o.o = order_of(y[e]);
            o.j = static_cast<int>(j);
            if ((k == 0 || before(last, o)) && before(o, best)) best = o;
          }
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
          Best<A> o;
          o.o = __shfl_xor_sync(0xffffffffu, best.o, s);
          o.j = __shfl_xor_sync(0xffffffffu, best.j, s);
          if (before(o, best)) best = o;
        }
        __syncthreads();
        if (lane == 0) redb[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (before(redb[w], best)) best = redb[w];
        if (best.j == 0x7fffffff) break;  // the slice is shorter than `want`
        last = best;
        if (threadIdx.x == 0) {
          list[k].y = a.sign * to_acc(row.x[best.j]);
          list[k].j = best.j;
        }
      }
      if (threadIdx.x == 0) parts[rank].count = k;
    }
  } else if (threadIdx.x == 0) {
    parts[rank].count = 0;
  }
  if (threadIdx.x == 0) {
    parts[rank].hi = hi;
    parts[rank].S = S;
    parts[rank].T = Tm;
  }
  __syncthreads();
  if (cluster > 1) {
    cluster_wait();
    if (rank > 0) {
      if (threadIdx.x == 0) store_cluster(&parts[rank], parts[rank]);
      for (int q = threadIdx.x; q < parts[rank].count; q += NT) store_cluster(&list[q], list[q]);
    }
    __syncthreads();
    cluster_sync();
    if (rank > 0) return;
  }

  // the row's results, by the first block
  bool any_nan = false;
  hi = neg_inf<A>();
  for (int r = 0; r < cluster; ++r) {
    any_nan |= parts[r].hi != parts[r].hi;
    hi = max_nan(hi, parts[r].hi);
  }
  S = Tm = A(0);
  for (int r = 0; r < cluster; ++r) {
    if (!(parts[r].hi > neg_inf<A>())) continue;
    const A drop = (parts[r].hi - hi) * c;
    const bool far = !(drop > Expo<A>::floor);
    const A f = far ? A(0) : Expo<A>::exp(drop);
    S += f * parts[r].S;
    Tm += f * (parts[r].T + parts[r].S * (far ? A(0) : drop));
  }
  Tm *= Expo<A>::unit;
  if (any_nan || hi == -neg_inf<A>()) S = Tm = static_cast<A>(NAN);
  if (threadIdx.x == 0) write_row(a, i, hi, S, Tm);
  if (!a.top) return;
  const A L = hi == neg_inf<A>() ? hi : log_acc(S);
  for (int q = threadIdx.x; q < cluster * a.top; q += NT) {
    const int r = q / a.top, k = q - r * a.top;
    if (k >= parts[r].count) continue;
    const Cand<A> me = lists[r][k];
    int place = k;  // the lists are in order: only the others' candidates are counted
    for (int o = 0; o < cluster; ++o) {
      if (o == r) continue;
      for (int z = 0; z < parts[o].count; ++z) {
        const Cand<A> he = lists[o][z];
        bool first;
        if (any_nan) {
          Best<A> p, w;
          p.o = order_of(he.y);
          p.j = he.j;
          w.o = order_of(me.y);
          w.j = me.j;
          first = before(p, w);
        } else {
          first = ahead(he, me);
        }
        place += first ? 1 : 0;
      }
    }
    if (place < a.top) write_top(a, i, place, me.y, me.j, hi, L);
  }
}

template <typename T> struct ScoreGradArgs {
  const T* x;
  int64_t ld;
  const void* labels;
  int labels_i64;
  int64_t n;
  int m;
  Acc<T> sign, mag;
  const Acc<T>* stats;
  const Acc<T>* g_log_probs;
  const Acc<T>* g_entropy;
  T* grad;
};

// The gradient reads and writes every score once: bound by HBM.  With t = log p in the
// exponent's unit, dx = p (A + B t) with A = -scale (g_l + g_H H), B = -scale g_H, and
// scale g_l more at the label: per score a subtraction, two fused multiply-adds, one
// exponential and a product.  One warp per (row, kGradVecs 16-byte vectors a lane) of the
// output, whose alignment decides where the vectors begin; scores whose row starts elsewhere
// in its 16 bytes are read element by element.
constexpr int kGradVecs = 4;

template <typename T> __global__ void __launch_bounds__(256) scores_grad_kernel(ScoreGradArgs<T> a, int64_t chunks) {
  using A = Acc<T>;
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t i = unit / chunks;
  if (i >= a.n) return;
  const int64_t chunk = unit - i * chunks;
  T* out = a.grad + i * a.m;
  const T* x = a.x + i * a.ld;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
  const bool same = (reinterpret_cast<uintptr_t>(x) & 15u) == (reinterpret_cast<uintptr_t>(out) & 15u);
  const int64_t j0 = chunk * (32 * kGradVecs * VE) + lane * VE - off;
  Vec<T, VE> v[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int64_t j = j0 + u * 32 * VE;
    if (same && j >= 0 && j + VE <= a.m) {
      v[u].raw = load_once(reinterpret_cast<const uint4*>(x + j));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (j + e >= 0 && j + e < a.m) v[u].e[e] = x[j + e];
    }
  }
  const A hi = a.stats[3 * i], L = a.stats[3 * i + 1], H = a.stats[3 * i + 2];
  const int64_t l = a.labels ? label_of<T>(a.labels, a.labels_i64, i) : -1;
  const A gl = l >= 0 && l < a.m && a.g_log_probs ? a.g_log_probs[i] : A(0);
  const A gh = a.g_entropy ? a.g_entropy[i] : A(0);
  const A scale = a.sign * a.mag, c = a.mag * Expo<A>::per_nat, L2 = L * Expo<A>::per_nat;
  const bool empty = hi == neg_inf<A>();
  const A ca = -scale * (gl + gh * H), cb = -scale * gh * Expo<A>::unit;
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int64_t j = j0 + u * 32 * VE;
    if (j >= a.m || j + VE <= 0) continue;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      A t = (a.sign * to_acc(v[u].e[e]) - hi) * c - L2;
      t = t > Expo<A>::floor ? t : Expo<A>::floor;
      A dx = Expo<A>::exp(t) * (ca + cb * t);
      if (j + e == l) dx += scale * gl;
      v[u].e[e] = from_acc<T>(empty ? A(0) : dx);
    }
    if (j >= 0 && j + VE <= a.m) {
      store_once(reinterpret_cast<uint4*>(out + j), v[u].raw);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (j + e >= 0 && j + e < a.m) out[j + e] = v[u].e[e];
    }
  }
}

// ------------------------------------------------------------------ launches
template <typename T, int EPL> static cudaError_t scores_warp(const ScoreArgs<T>& a, cudaStream_t st) {
  const int64_t blocks = std::min<int64_t>((a.n + 3) / 4, static_cast<int64_t>(num_sms()) * 64);
  scores_warp_kernel<T, EPL><<<static_cast<unsigned>(blocks), 128, 0, st>>>(a);
  return cudaGetLastError();
}

// Blocks per row: as many as it takes to give every SM two blocks, while each keeps 16 KiB
// of the row (below that the join costs more than the sweep).
template <typename T> static int scores_cluster(const ScoreArgs<T>& a) {
  int c = 1;
  while (c < kMaxCluster && a.n * c * 2 <= 2 * num_sms() &&
         static_cast<int64_t>(a.m) * static_cast<int64_t>(sizeof(T)) >= 2 * c * 16384)
    c *= 2;
  return c;
}

template <typename T, int NT> static cudaError_t scores_block(const ScoreArgs<T>& a, cudaStream_t st) {
  const int cluster = scores_cluster(a);
  constexpr int VE = RowVecs<T>::VE;
  const int64_t vecs = (static_cast<int64_t>(a.m) + 2 * VE - 2) / VE;  // at any alignment
  const int64_t steps = ((vecs + cluster - 1) / cluster + kBlockVecs * NT - 1) / (kBlockVecs * NT);
  const int per_group = static_cast<int>(std::max<int64_t>(1, (steps + kGroups - 1) / kGroups));
  const size_t groups = static_cast<size_t>((steps + per_group - 1) / per_group);
  const size_t smem = a.top ? groups * NT * sizeof(Acc<T>) : 0;
  cudaError_t e = cudaFuncSetAttribute(scores_block_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(kGroups * NT * sizeof(Acc<T>)));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.n * cluster));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, scores_block_kernel<T, NT>, a, cluster, per_group);
}

template <typename T> static cudaError_t scores_t(const ScoreJob& j, cudaStream_t st) {
  ScoreArgs<T> a{};
  a.x = static_cast<const T*>(j.x);
  a.ld = j.ld;
  a.labels = j.labels;
  a.labels_i64 = j.labels_i64;
  a.n = j.n;
  a.m = static_cast<int>(j.m);
  a.sign = j.scale < 0 ? -1 : 1;
  a.mag = static_cast<Acc<T>>(j.scale < 0 ? -j.scale : j.scale);
  a.top = j.top;
  a.log_probs = static_cast<Acc<T>*>(j.log_probs);
  a.entropy = static_cast<Acc<T>*>(j.entropy);
  a.stats = static_cast<Acc<T>*>(j.stats);
  a.top_log_probs = static_cast<Acc<T>*>(j.top_log_probs);
  a.top_labels = j.top_labels;
  // a row in one warp's registers where it fits at any alignment of its rows
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ld * sizeof(T))) & 15u) == 0;
  const int64_t span = a.m + (aligned ? 0 : RowVecs<T>::VE - 1);
  if (span <= 32 * 8) return scores_warp<T, 8>(a, st);
  if (span <= 32 * 16) return scores_warp<T, 16>(a, st);
  if (span <= 32 * 32) return scores_warp<T, 32>(a, st);
  if constexpr (sizeof(T) < 8)
    if (span <= 32 * 64) return scores_warp<T, 64>(a, st);
  if (span <= 16384) return scores_block<T, 128>(a, st);
  return scores_block<T, 256>(a, st);
}

template <typename T> static cudaError_t scores_grad_t(const ScoreGradJob& j, cudaStream_t st) {
  ScoreGradArgs<T> a{};
  a.x = static_cast<const T*>(j.x);
  a.ld = j.ld;
  a.labels = j.labels;
  a.labels_i64 = j.labels_i64;
  a.n = j.n;
  a.m = static_cast<int>(j.m);
  a.sign = j.scale < 0 ? -1 : 1;
  a.mag = static_cast<Acc<T>>(j.scale < 0 ? -j.scale : j.scale);
  a.stats = static_cast<const Acc<T>*>(j.stats);
  a.g_log_probs = static_cast<const Acc<T>*>(j.g_log_probs);
  a.g_entropy = static_cast<const Acc<T>*>(j.g_entropy);
  a.grad = static_cast<T*>(j.grad);
  // chunks of a row at any alignment of the output's rows
  constexpr int64_t per = 32 * kGradVecs * (16 / sizeof(T));
  const int64_t chunks = (a.m + 16 / static_cast<int64_t>(sizeof(T)) - 1 + per - 1) / per;
  scores_grad_kernel<T><<<static_cast<unsigned>((a.n * chunks + 7) / 8), 256, 0, st>>>(a, chunks);
  return cudaGetLastError();
}

cudaError_t launch_label_log_probs(RowType t, const ScoreJob& j, cudaStream_t st) {
  switch (t) {
    case ROW_F32: return scores_t<float>(j, st);
    case ROW_F64: return scores_t<double>(j, st);
    case ROW_F16: return scores_t<__half>(j, st);
    default: return scores_t<__nv_bfloat16>(j, st);
  }
}

cudaError_t launch_label_log_probs_grad(RowType t, const ScoreGradJob& j, cudaStream_t st) {
  switch (t) {
    case ROW_F32: return scores_grad_t<float>(j, st);
    case ROW_F64: return scores_grad_t<double>(j, st);
    case ROW_F16: return scores_grad_t<__half>(j, st);
    default: return scores_grad_t<__nv_bfloat16>(j, st);
  }
}

}  // namespace euc
