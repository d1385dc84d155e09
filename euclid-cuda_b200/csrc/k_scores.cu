// Log probabilities of a row of scores: of given labels, with the entropy and the best
// alternatives, and the scores' gradient.
//
// For row x of m scores and z_j = scale * x_j (a squared distance takes a negative scale):
//   M = max z,  S = sum exp(z_j - M),  T = sum exp(z_j - M) (z_j - M),  L = log S
//   log p_j = z_j - M - L        entropy H = L - T / S
//   dz_j = g_l ([j = l] - p_j) - g_H p_j (log p_j + H),  dx_j = scale * dz_j
// z_j - M is formed as (y_j - max y) |scale| with y = sign(scale) x, which loses nothing
// to a common offset of the scores.  Where the difference is beyond the type, p_j is 0: the
// smallest |scale| that is taken makes it so.  T and H are sums of terms of one sign.
//
// Masked scores (z = -inf) have probability 0 and add nothing.  A row with no score left
// has log probabilities of -inf, entropy 0 and a zero gradient; a row that holds a NaN or
// z = +inf has NaN in all of them.  Alternatives go by y, equal ones by the lower index;
// NaN counts as the largest value.
//
// The scores are read once, so HBM is the bound: 131072 x 1024 fp32 without alternatives take
// 85 us (6.3 TB/s), 4096 x 131072 bf16 179 (6.0).  The alternatives cost instructions, some
// hundreds a row whatever its length: with the 8 best the first takes 132 us (840 instructions a
// row and warp, the issue slots 76 % busy, HBM 50 %), with the 20 best the second 205.  One row
// of 131072 is bound by latency: 4.9 us, 10.5 with 20 alternatives.
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

__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0xffffffffu ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ double value_of(unsigned long long o) {
  return o == ~0ull ? static_cast<double>(NAN)
                    : __longlong_as_double(static_cast<long long>(o >> 63 ? o & ~(1ull << 63) : ~o));
}

// A score and its column, ordered as the alternatives are: y first, equal ones by the lower
// column.  fp32: one 64-bit number.
template <typename A> struct Key;
template <> struct Key<float> {
  unsigned long long k;
  __device__ __forceinline__ static Key of(float y, int j) {
    Key r;
    r.k = (static_cast<unsigned long long>(order_of(y)) << 32) | (0xffffffffu - static_cast<uint32_t>(j));
    return r;
  }
  __device__ __forceinline__ static Key none() {
    Key r;
    r.k = 0;
    return r;
  }
  __device__ __forceinline__ uint32_t order() const { return static_cast<uint32_t>(k >> 32); }
  __device__ __forceinline__ float y() const { return value_of(order()); }
  __device__ __forceinline__ int j() const { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
  __device__ __forceinline__ bool ahead(const Key& o) const { return k > o.k; }
  __device__ __forceinline__ Key other(int s) const {
    Key r;
    r.k = __shfl_xor_sync(0xffffffffu, k, s);
    return r;
  }
};
template <> struct Key<double> {
  unsigned long long o;
  long long col;
  __device__ __forceinline__ static Key of(double y, int j) {
    Key r;
    r.o = order_of(y);
    r.col = j;
    return r;
  }
  __device__ __forceinline__ static Key none() {
    Key r;
    r.o = 0;
    r.col = 0x7fffffff;
    return r;
  }
  __device__ __forceinline__ unsigned long long order() const { return o; }
  __device__ __forceinline__ double y() const { return value_of(o); }
  __device__ __forceinline__ int j() const { return static_cast<int>(col); }
  __device__ __forceinline__ bool ahead(const Key& q) const { return o > q.o || (o == q.o && col < q.col); }
  __device__ __forceinline__ Key other(int s) const {
    Key r;
    r.o = __shfl_xor_sync(0xffffffffu, o, s);
    r.col = __shfl_xor_sync(0xffffffffu, col, s);
    return r;
  }
};

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

template <typename A> __device__ __forceinline__ A lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ double lowest<double>() { return -1.7976931348623157e308; }

// the larger; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) { return fmax_nan(a, b); }
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : (b > a || b != b ? b : a); }
__device__ __forceinline__ double max_nan(double a, double b, double c) { return max_nan(max_nan(a, b), c); }

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

// the largest over the TEAM lanes of this lane's team
template <int TEAM, typename A> __device__ __forceinline__ A team_max_nan(A v) {
  if constexpr (TEAM == 32) {
    return warp_max_nan(v);
  } else {
#pragma unroll
    for (int s = TEAM / 2; s > 0; s >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, s));
    return v;
  }
}
template <int TEAM, typename A> __device__ __forceinline__ A team_sum(A v) {
#pragma unroll
  for (int s = TEAM / 2; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
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

// (y - hi) mag - L of a row.  Above 1, hi may be so large that the difference is beyond the type
// and its product with mag is not: half the difference is taken twice as often then, which
// rounds as the whole one does.
template <typename A> struct LogProb {
  A part, hi, mag, L;
  __device__ __forceinline__ LogProb(A hi_, A mag_, A L_)
      : part(hi_ > A(1) ? A(0.5) : A(1)), hi(hi_ * part), mag(hi_ > A(1) ? mag_ * A(2) : mag_), L(L_) {}
  __device__ __forceinline__ A operator()(A y) const { return fma(y, part, -hi) * mag - L; }
};

// the row's outputs from its M (as max y), S, T, L = log S (-inf for an empty row), and the
// score at its label (`in`: the label is one of the columns)
template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs<T>& a, int64_t i, Acc<T> hi, Acc<T> S, Acc<T> Tm, Acc<T> L,
                                          bool in, Acc<T> at_label) {
  using A = Acc<T>;
  const bool empty = hi == neg_inf<A>();
  const A H = empty ? A(0) : L - Tm / S;
  if (a.entropy) a.entropy[i] = H;
  if (a.stats) {
    a.stats[3 * i] = hi;
    a.stats[3 * i + 1] = L;
    a.stats[3 * i + 2] = H;
  }
  if (a.log_probs) a.log_probs[i] = !in ? A(0) : empty ? neg_inf<A>() : LogProb<A>(hi, a.mag, L)(at_label);
}

// ------------------------------------------------------------------ a row as vectors
// the elements of 16 bytes
template <typename T> __device__ __forceinline__ void unpack(const uint4& w, Acc<T>* y) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      y[2 * q] = __uint_as_float(r[q] << 16);
      y[2 * q + 1] = __uint_as_float(r[q] & 0xffff0000u);
    }
  } else if constexpr (std::is_same<T, __half>::value) {
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[q]));
      y[2 * q] = f.x;
      y[2 * q + 1] = f.y;
    }
  } else {
    Vec<T, 16 / static_cast<int>(sizeof(T))> v;
    v.raw = w;
#pragma unroll
    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) y[e] = v.e[e];
  }
}

// Vector v of a row is the 16 bytes at its v-th 16-byte boundary, counted from the one at or
// before the row's start (`off` elements before it): [0, all) of them, of which [lo, hi) lie
// in the row whole.  The others are read element by element; nothing outside the row is read.
// y = -x where the scale is negative: the sign bits are flipped in the 16 bytes.
template <typename T> struct RowVecs {
  static constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const T* x;
  const uint4* base;
  int m, off, all, lo, hi;
  uint32_t flip_even, flip_odd;  // of the words 0, 2 and 1, 3
  __device__ __forceinline__ RowVecs(const T* x_, int m_, bool negate) : x(x_), m(m_) {
    off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    base = reinterpret_cast<const uint4*>(x - off);
    all = (m + off + VE - 1) / VE;
    lo = off > 0 ? 1 : 0;
    hi = (m + off) / VE;
    const uint32_t odd = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
    flip_odd = negate ? odd : 0u;
    flip_even = sizeof(T) == 8 ? 0u : flip_odd;
  }
  __device__ __forceinline__ uint4 read(int v) const { return load_keep(base + v); }
  // 16 bytes of masked scores
  __device__ __forceinline__ uint4 masked() const {
    Vec<T, VE> v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v.e[e] = from_acc<T>(flip_odd ? -neg_inf<Acc<T>>() : neg_inf<Acc<T>>());
    return v.raw;
  }
  __device__ __forceinline__ void values(uint4 w, Acc<T>* y) const {
    w.x ^= flip_even;
    w.y ^= flip_odd;
    w.z ^= flip_even;
    w.w ^= flip_odd;
    unpack<T>(w, y);
  }
  __device__ __forceinline__ Acc<T> at(int j) const { return flip_odd ? -to_acc(x[j]) : to_acc(x[j]); }
  // any vector of [0, all); elements outside the row are -inf
  __device__ __forceinline__ void load(int v, Acc<T>* y) const {
    if (v >= lo && v < hi) {
      values(read(v), y);
      return;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int j = v * VE - off + e;
      y[e] = j >= 0 && j < m ? at(j) : neg_inf<Acc<T>>();
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
// The `top` best of a row without sorting it: any number that at least `top` scores reach
// bounds the last of them from below, and few scores reach a good one.  The bound comes from
// maxima that the softmax needs anyhow: the row is cut into lists of maxima (over the lanes),
// and with q = ceil(top / lists) the smallest of the lists' q-th largest is reached by q of
// every list.  The scores that reach it go to a candidate list in shared memory (in any
// order), and a candidate's place is the number of candidates before it.  Where they are more
// than the list holds (sorted rows, or a finite mask, which a list with nothing else makes the
// bound), a better bound is looked for: a block takes the last place among those it holds, a
// team halves the range of values.  Scores that are equal beyond the list's size bound
// themselves: those above them are listed, and the places left go to the first of the equal
// ones.  A row with a NaN has its first ones first, and then the best one behind the last one, a
// pass over the row each.
// (50 scores side by side, all others masked by -1e4, the 20 best: 4096 x 131072 bf16 0.23 ms,
// 131072 x 1024 fp32 0.47; by a pass over the row for each 41.7 and 5.5.)

// The q-th largest over the team's lanes of each list, the smallest over the lists: q - 1
// rounds strike each list's largest (and its equals, which only lowers the bound).  No NaN.
// A row that is masked but for fewer scores gives the lowest finite number.
template <int TEAM, int LISTS, typename A> __device__ __forceinline__ A team_bound(A* lists, int q) {
  A t[LISTS];
#pragma unroll
  for (int l = 0; l < LISTS; ++l) t[l] = team_max_nan<TEAM>(lists[l]);
  for (int k = 1; k < q; ++k) {
#pragma unroll
    for (int l = 0; l < LISTS; ++l) lists[l] = lists[l] == t[l] ? neg_inf<A>() : lists[l];
#pragma unroll
    for (int l = 0; l < LISTS; ++l) t[l] = team_max_nan<TEAM>(lists[l]);
  }
#pragma unroll
  for (int l = 1; l < LISTS; ++l) t[0] = t[l] < t[0] ? t[l] : t[0];
  return t[0] > lowest<A>() ? t[0] : lowest<A>();
}

template <typename T>
__device__ __forceinline__ void write_top(const ScoreArgs<T>& a, int64_t i, int place, const Key<Acc<T>>& k, Acc<T> hi,
                                          Acc<T> L) {
  a.top_labels[i * a.top + place] = k.j();
  a.top_log_probs[i * a.top + place] = hi == neg_inf<Acc<T>>() ? hi : LogProb<Acc<T>>(hi, a.mag, L)(k.y());
}

// how many of list[0, count) are ahead of `me`
template <typename A> __device__ __forceinline__ int place_of(const Key<A>* list, int count, const Key<A>& me) {
  int place = 0;
#pragma unroll 4
  for (int r = 0; r < count; ++r) place += list[r].ahead(me) ? 1 : 0;
  return place;
}

// ------------------------------------------------------------------ a team of lanes per row
// Rows of up to TEAM EPL scores, a team of 8, 16 or 32 lanes each: the row stays in registers, so
// its scores are read once and its maximum is known before the first exponential; a warp
// reads its next rows while it works on these, into shared memory, which leaves the registers
// to more warps (131072 x 1024 fp32 with the 8 best: 156 us with the next row in registers
// and five blocks an SM, 131 with seven).  FLAT: every row is whole 16-byte vectors;
// other rows are read element by element, neighbouring lanes neighbouring elements.
template <int TEAM> constexpr int kTeamCands = TEAM == 8 ? 64 : TEAM == 16 ? 96 : 128;

__device__ __forceinline__ void copy_async_16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T, int TEAM, int EPL, bool FLAT>
__global__ void __launch_bounds__(128, EPL * sizeof(Acc<T>) > 128 ? (sizeof(T) == 8 ? 2 : 5) : (FLAT ? 7 : 5))
    scores_team_kernel(ScoreArgs<T> a) {
  using A = Acc<T>;
  constexpr int VE = FLAT ? RowVecs<T>::VE : 1, NV = EPL / VE, RPW = 32 / TEAM, CAP = kTeamCands<TEAM>;
  // FLAT: where a lane's vectors of the next row land; each lane reads its own alone
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Key<A> cands[4][CAP * RPW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tl = lane % TEAM, team = lane / TEAM;
  const unsigned team_lanes = (TEAM == 32 ? 0xffffffffu : (1u << (TEAM & 31)) - 1u) << (team * TEAM);
  const unsigned before_me = team_lanes & ((1u << lane) - 1u);
  const bool negate = a.sign < A(0);
  const A c = a.mag * Expo<A>::per_nat;
  Key<A>* list = cands[warp] + team * CAP;
  uint4* slot = reinterpret_cast<uint4*>(dyn) + (warp * NV) * 32 + lane;  // (v-th vector: slot[v * 32])
  const int64_t step = static_cast<int64_t>(gridDim.x) * (4 * RPW);
  int64_t first = (static_cast<int64_t>(blockIdx.x) * 4 + warp) * RPW;
  if (first >= a.n) return;
  T next[FLAT ? 1 : EPL];
  int64_t next_label = -1;
  // elements behind the row's end hold z = -inf from the start, and no load changes them
  const RowVecs<T> any(a.x, a.m, negate);
  if constexpr (FLAT) {
#pragma unroll
    for (int v = 0; v < NV; ++v) slot[v * 32] = any.masked();
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) next[v] = from_acc<T>(negate ? -neg_inf<A>() : neg_inf<A>());
  }
  auto fetch = [&](int64_t row) {
    row = min(row, a.n - 1);
    const T* x = a.x + row * a.ld;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if ((v * TEAM + tl) * VE < a.m) {
        if constexpr (FLAT) copy_async_16(slot + v * 32, reinterpret_cast<const uint4*>(x) + v * TEAM + tl);
        else next[v] = load_keep(x + v * TEAM + tl);
      }
    if (a.log_probs) next_label = label_of<T>(a.labels, a.labels_i64, row);
  };
  fetch(first + team);
  for (; first < a.n; first += step) {
    const bool live = first + team < a.n, more = first + step < a.n;
    const int64_t i = live ? first + team : a.n - 1;
    const RowVecs<T> row(a.x + i * a.ld, a.m, negate);
    A y[EPL];
    if constexpr (FLAT) {
      copy_async_wait();
#pragma unroll
      for (int v = 0; v < NV; ++v) row.values(slot[v * 32], y + v * VE);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) y[v] = negate ? -to_acc(next[v]) : to_acc(next[v]);
    }
    const bool labelled = next_label >= 0 && next_label < a.m;
    const A at_label = labelled ? row.at(static_cast<int>(next_label)) : A(0);  // ready by the time it is needed
    // the next row is on its way while this one is worked on; with alternatives, a row in
    // shared memory stays until its candidates are read from there
    const bool early = !FLAT || a.top == 0;
    if (early && more) fetch(first + step + team);
    A lists[4];
#pragma unroll
    for (int l = 0; l < 4; ++l) lists[l] = max_of<A, EPL / 4>(y + l * (EPL / 4));
    const A hi = team_max_nan<TEAM>(max_nan(max_nan(lists[0], lists[1]), lists[2], lists[3]));
    Sums<A> sums;
    sums.template add<EPL>(y, hi == neg_inf<A>() ? A(0) : hi, c);
    A S, Tm;
    both(sums, S, Tm);
    S = team_sum<TEAM>(S);
    Tm = team_sum<TEAM>(Tm) * Expo<A>::unit;
    if (hi != hi || hi == -neg_inf<A>()) S = Tm = static_cast<A>(NAN);
    const A L = hi == neg_inf<A>() ? hi : log_acc(S);
    if (tl == 0 && live) write_row(a, i, hi, S, Tm, L, labelled, at_label);
    if (a.top == 0) continue;
    const bool slow = hi != hi;
    int count = 0;
    // fewer lists give a better bound, more of them fewer rounds
    A t;
    if (a.top <= 4) {
      lists[0] = max_nan(max_nan(lists[0], lists[1]), lists[2], lists[3]);
      t = team_bound<TEAM, 1>(lists, a.top);
    } else if (a.top <= 16) {
      lists[0] = max_nan(lists[0], lists[1]);
      lists[1] = max_nan(lists[2], lists[3]);
      t = team_bound<TEAM, 2>(lists, (a.top + 1) / 2);
    } else {
      t = team_bound<TEAM, 4>(lists, (a.top + 3) / 4);
    }
#pragma unroll
    for (int w = 0; w < EPL; w += 32) {
      uint32_t part[4] = {0u, 0u, 0u, 0u};  // (four chains of dependent instructions instead of one)
#pragma unroll
      for (int q = 0; q < (EPL < 32 ? EPL : 32); ++q) part[q % 4] |= y[w + q] >= t ? 1u << q : 0u;
      uint32_t in = (part[0] | part[1]) | (part[2] | part[3]);
      while (true) {
        const unsigned b = __ballot_sync(0xffffffffu, in != 0u);
        if (b == 0u) break;
        if (in != 0u) {
          const int at = count + __popc(b & before_me), q = w + __ffs(in) - 1;
          const int j = ((q / VE) * TEAM + tl) * VE + q % VE;
          if (at < CAP) {
            A z;
            if constexpr (FLAT) {
              z = to_acc(reinterpret_cast<const T*>(slot + (q / VE) * 32)[q % VE]);
              if (negate) z = -z;
            } else {
              z = row.at(j);
            }
            list[at] = Key<A>::of(z, j);
          }
          in &= in - 1u;
        }
        count += __popc(b & team_lanes);
      }
    }
    const bool over = !slow && count > CAP;
    const bool odd = __any_sync(0xffffffffu, over || slow || count < a.top);
    A tie = neg_inf<A>();  // the places that the listed scores leave go to the first that equal it
    if (odd && __any_sync(0xffffffffu, over)) {
      // More than the list holds: a value that at least `top` scores reach and the list holds is
      // looked for, halfway between one that more reach and one that fewer than `top` do.  Before
      // that the smallest of the lanes' maxima, which is a finite mask, and the next number
      // behind it.  Where no value lies between the two, the scores above the lower one are listed.
      // (The scores are read again, which leaves the usual way its registers.)
      const int vecs = (a.m + TEAM * VE - 1) / (TEAM * VE);  // of a lane
      auto read = [&](int v, A* z) {
        if constexpr (FLAT) row.values(slot[v * 32], z);
        else z[0] = v * TEAM + tl < a.m ? row.at(v * TEAM + tl) : neg_inf<A>();
      };
      A least = neg_inf<A>();
      for (int v = 0; v < vecs; ++v) {
        A z[VE];
        read(v, z);
        const A most = max_of<A, VE>(z);
        least = most > least ? most : least;
      }
#pragma unroll
      for (int s = TEAM / 2; s > 0; s >>= 1) {
        const A o = __shfl_xor_sync(0xffffffffu, least, s);
        least = o < least ? o : least;
      }
      bool open = over;
      auto low = order_of(t), high = order_of(hi) + 1, mid = least > t ? order_of(least) : low + 1;
      for (int turn = 0; __any_sync(0xffffffffu, open); ++turn) {
        const A bound = value_of(mid);
        int reach = 0;
#pragma unroll 4
        for (int v = 0; v < vecs; ++v) {
          A z[VE];
          read(v, z);
#pragma unroll
          for (int e = 0; e < VE; ++e) reach += z[e] >= bound ? 1 : 0;
        }
        reach = team_sum<TEAM>(reach);
        if (open) {
          if (reach > CAP) {
            low = mid;
          } else if (reach < a.top) {
            high = mid;
          } else {
            t = bound;
            open = false;
          }
          if (open && high - low == 1) {
            tie = value_of(low);
            t = value_of(high);
            open = false;
          }
          mid = turn == 0 ? low + 1 : low + (high - low) / 2;
        }
      }
      __syncwarp();  // the list's first entries are in, before they are written again
      if (over) count = 0;
      for (int v = 0; v < vecs; ++v) {
        A z[VE];
        read(v, z);
        uint32_t in = 0u;
#pragma unroll
        for (int e = 0; e < VE; ++e) in |= over && z[e] >= t ? 1u << e : 0u;
        if (!__any_sync(0xffffffffu, in != 0u)) continue;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const bool here = in >> e & 1u;
          const unsigned b = __ballot_sync(0xffffffffu, here);
          const int at = count + __popc(b & before_me);
          if (here && at < CAP) list[at] = Key<A>::of(z[e], (v * TEAM + tl) * VE + e);
          count = min(count + __popc(b & team_lanes), CAP);
        }
      }
    }
    if (!early && more) fetch(first + step + team);
    if (odd) {
      // the first that equal `tie`: masked ones where t is the lowest number; of a row with a NaN
      // the first NaN
      __syncwarp();  // the list's first entries are in, before some are written again
      if (slow) count = 0;
      bool fill = count < a.top;
      for (int j0 = 0; __any_sync(0xffffffffu, fill); j0 += TEAM) {
        const int j = j0 + tl;
        const A z = fill && j < a.m ? row.at(j) : A(0);
        const bool here = fill && j < a.m && (slow ? z != z : z == tie);
        const unsigned b = __ballot_sync(0xffffffffu, here);
        const int at = count + __popc(b & before_me);
        if (here && at < a.top) list[at] = Key<A>::of(z, j);
        if (fill) count = min(count + __popc(b & team_lanes), a.top);
        fill = fill && count < a.top && j0 + TEAM < a.m;
      }
      // and then, of such a row, the best one behind the last one
      while (__any_sync(0xffffffffu, slow && count < a.top)) {
        __syncwarp();
        const Key<A> last = list[max(count - 1, 0)];
        Key<A> best = Key<A>::none();
        for (int j = tl; j < a.m; j += TEAM) {
          const Key<A> o = Key<A>::of(row.at(j), j);
          if (last.ahead(o) && o.ahead(best)) best = o;
        }
#pragma unroll
        for (int s = TEAM / 2; s > 0; s >>= 1) {
          const Key<A> o = best.other(s);
          if (o.ahead(best)) best = o;
        }
        if (slow && count < a.top) {
          if (tl == 0) list[count] = best;
          ++count;
        }
      }
    }
    __syncwarp();
    if (live) {
      for (int q = tl; q < count; q += TEAM) {
        const Key<A> me = list[q];
        const int place = place_of(list, count, me);
        if (place < a.top) write_top(a, i, place, me, hi, L);
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
// The blocks' results are joined in the first block's shared memory, in rank order.  Vectors
// are read a step ahead (4096 x 131072 bf16: 196 us without, 184 with).
constexpr int kGroups = 32;       // groups of vectors per thread
constexpr int kBlockVecs = 4;     // vectors in flight per thread
constexpr int kBlockCands = 512;
constexpr int kBlockHits = 256;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;

template <typename A> struct Part {  // one block's share of a row
  A hi, S, T;
  int count;  // alternatives listed
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT, sizeof(T) <= 4 ? 1024 / NT : 1)
    scores_block_kernel(ScoreArgs<T> a, int log_cluster, int per_group) {
  using A = Acc<T>;
  constexpr int VE = RowVecs<T>::VE, U = kBlockVecs, W = NT / 32, LISTS = W == 1 ? U : 1;
  extern __shared__ __align__(16) unsigned char dyn[];
  A* group_max = reinterpret_cast<A*>(dyn);  // [kGroups][NT], with alternatives only
  __shared__ Key<A> cands[kBlockCands];
  __shared__ uint32_t hits[kBlockHits];  // (group of vectors, thread) with a score that reaches the bound
  __shared__ Key<A> lists[kMaxCluster][kMaxTop];
  __shared__ Part<A> parts[kMaxCluster];
  __shared__ A red[2][W];
  __shared__ int count_sh, hits_sh, equals[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cluster = 1 << log_cluster;
  const int64_t i = blockIdx.x >> log_cluster;
  const int rank = static_cast<int>(blockIdx.x) & (cluster - 1);
  const A c = a.mag * Expo<A>::per_nat;
  const RowVecs<T> row(a.x + i * a.ld, a.m, a.sign < A(0));
  const int per = (row.all + cluster - 1) >> log_cluster;
  const int v0 = min(row.all, rank * per), v1 = min(row.all, v0 + per);
  const int j0 = max(0, v0 * VE - row.off), j1 = max(j0, min(a.m, v1 * VE - row.off));  // the slice's scores
  const int i0 = max(v0, row.lo), i1 = max(i0, min(v1, row.hi));                        // its whole vectors
  const int steps = (i1 - i0 + U * NT - 1) / (U * NT);
  // the first and the last vector where they are not whole: the first and the last thread
  int edge = -1;
  if (threadIdx.x == 0 && row.lo > 0 && v0 == 0) edge = 0;
  if (threadIdx.x == NT - 1 && row.hi < row.all && v1 == row.all && v0 < v1 && !(row.lo > 0 && row.all == 1))
    edge = row.all - 1;
  if (threadIdx.x == 0) count_sh = hits_sh = 0;
  __syncwarp();
  if (cluster > 1) cluster_arrive();  // waited for before the first store to another block

  // the label's score, read ahead of its use
  bool labelled = false;
  A at_label = A(0);
  if (rank == 0 && threadIdx.x == 0 && a.log_probs) {
    const int64_t l = label_of<T>(a.labels, a.labels_i64, i);
    labelled = l >= 0 && l < a.m;
    if (labelled) at_label = row.at(static_cast<int>(l));
  }

  A mine = neg_inf<A>(), gm = neg_inf<A>(), edge_max = neg_inf<A>();
  A slot_max[LISTS];  // of one warp's lists: a maximum per vector in flight
#pragma unroll
  for (int l = 0; l < LISTS; ++l) slot_max[l] = neg_inf<A>();
  Sums<A> sums;
  auto take = [&](A most) {  // a new maximum of the thread: larger, or a NaN
    if (!(most <= mine)) {
      if (mine > neg_inf<A>()) sums.move((mine - most) * c);
      mine = max_nan(mine, most);
    }
  };
  if (edge >= 0) {
    A y[VE];
    row.load(edge, y);
    edge_max = max_of<A, VE>(y);
    take(edge_max);
    sums.template add<VE>(y, mine == neg_inf<A>() ? A(0) : mine, c);
  }
  int g = 0, in_group = 0;
  // vectors behind the slice hold z = -inf; a step's vectors are read while the one before it
  // is worked on
  const uint4 fill = row.masked();
  const uint4* from = row.base + i0 + threadIdx.x;
  uint4 next[U];
  auto fetch = [&](int s) {
    if ((s + 1) * (U * NT) <= i1 - i0) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = load_keep(from + s * (U * NT) + u * NT);
    } else {
      const int left = i1 - i0 - s * (U * NT) - static_cast<int>(threadIdx.x);
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = u * NT < left ? load_keep(from + s * (U * NT) + u * NT) : fill;
    }
  };
  if (steps > 0) fetch(0);
  for (int s = 0; s < steps; ++s) {
    A y[U * VE];
#pragma unroll
    for (int u = 0; u < U; ++u) row.values(next[u], y + u * VE);
    if (s + 1 < steps) fetch(s + 1);
    A most;
    if constexpr (LISTS > 1) {
      A m4[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        m4[u] = max_of<A, VE>(y + u * VE);
        slot_max[u] = max_nan(slot_max[u], m4[u]);
      }
      most = max_of<A, U>(m4);
    } else {
      most = max_of<A, U * VE>(y);
    }
    gm = max_nan(gm, most);
    take(most);
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
  const int want = min(a.top, j1 - j0);
  A bound = lowest<A>();
  if (want > 0) {
    constexpr int ALL = W * LISTS;
    if constexpr (LISTS == 1) slot_max[0] = mine;
    else slot_max[0] = max_nan(slot_max[0], edge_max);
    bound = team_bound<32, LISTS>(slot_max, (want + ALL - 1) / ALL);
    // 32 scores reach the smallest of the lanes' maxima: a finite mask, where all lists' largest
    // are equal
    const A least = -warp_max_nan(-mine);
    bound = least > bound ? least : bound;
  }
  if (lane == 0) {
    red[0][warp] = wmax;
    red[1][warp] = bound;
  }
  __syncthreads();
  A hi = red[0][0];
  bound = red[1][0];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    hi = max_nan(hi, red[0][w]);
    bound = red[1][w] < bound ? red[1][w] : bound;
  }
  if (want == 1 && hi > bound) bound = hi;
  __syncthreads();
  if (mine > neg_inf<A>()) sums.move((mine - hi) * c);
  A S, Tm;
  both(sums, S, Tm);
  S = team_sum<32>(S);
  Tm = team_sum<32>(Tm);
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

  // this block's best `want` scores, in order, in lists[rank]
  Key<A>* list = lists[rank];
  if (want > 0) {
    const bool slow = hi != hi;
    A tie = neg_inf<A>();  // the places that the listed scores leave go to the first that equal it
    bool above = false;    // whether the bound is the next number above `tie`
    int found = want;
    // Two turns that do not list all leave out at least 256 - kMaxTop of the slice's scores: the
    // limit is never reached, unless the scores change while they are read.
    for (int turns = (j1 - j0) / 64 + 8; !slow && turns > 0; --turns) {
      auto add = [&](A y, int j) {
        const int at = atomicAdd(&count_sh, 1);
        if (at < kBlockCands) cands[at] = Key<A>::of(y, j);
      };
      if (mine >= bound)
        for (int q = 0; q * per_group < steps; ++q)
          if (group_max[q * NT + threadIdx.x] >= bound) {
            const int at = atomicAdd(&hits_sh, 1);
            if (at < kBlockHits) hits[at] = static_cast<uint32_t>(q) * NT + threadIdx.x;
          }
      if (edge >= 0 && edge_max >= bound)
        for (int e = 0; e < VE; ++e) {
          const int j = edge * VE - row.off + e;
          if (j >= 0 && j < a.m && row.at(j) >= bound) add(row.at(j), j);
        }
      __syncthreads();
      // the groups' vectors over all threads, R reads in flight each, until the list is full
      constexpr int R = VE == 8 ? 2 : 4;
      const int per_hit = per_group * U, all = min(hits_sh, kBlockHits) * per_hit;
      for (int z0 = threadIdx.x; z0 < all; z0 += R * NT) {
        if (*static_cast<volatile int*>(&count_sh) > kBlockCands) break;
        uint4 w[R];
        int v[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
          v[q] = i1;
          const int z = z0 + q * NT;
          if (z < all) {
            const uint32_t hit = hits[z / per_hit];
            const int in_hit = z % per_hit, s = static_cast<int>(hit / NT) * per_group + in_hit / U;
            v[q] = i0 + s * (U * NT) + in_hit % U * NT + static_cast<int>(hit % NT);
          }
          w[q] = v[q] < i1 ? row.read(v[q]) : fill;
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
          A y[VE];
          row.values(w[q], y);
          if (max_of<A, VE>(y) < bound) continue;
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (y[e] >= bound) add(y[e], v[q] * VE - row.off + e);
        }
      }
      __syncthreads();
      const int count = min(count_sh, kBlockCands);
      const bool whole = count_sh <= kBlockCands && hits_sh <= kBlockHits;
      // too many for the list: only those above the bound, since more may equal it than the list
      // holds; if those are too many as well, the last place among those listed bounds the row's
      // better
      const bool rank = whole || above;
      if (rank)
        for (int q = threadIdx.x; q < count; q += NT) {
          const Key<A> me = cands[q];
          const int place = place_of(cands, count, me);
          if (place < want) list[place] = me;
        }
      if (whole) {
        found = count;
        break;
      }
      __syncthreads();
      const A better = rank ? list[want - 1].y() : bound;
      above = !(better > bound);
      if (above) tie = bound;
      bound = above ? value_of(order_of(bound) + 1) : better;
      __syncthreads();
      if (threadIdx.x == 0) count_sh = hits_sh = 0;
      __syncthreads();
    }
    // the first that equal `tie` (masked ones where the bound is the lowest number), a vector a
    // thread and turn; of a slice with a NaN the first NaN
    if (slow) found = 0;
    for (int v = v0; found < want && v < v1; v += NT) {
      uint32_t here = 0u;
      if (v + static_cast<int>(threadIdx.x) < v1) {
        A y[VE];
        row.load(v + static_cast<int>(threadIdx.x), y);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int j = (v + static_cast<int>(threadIdx.x)) * VE - row.off + e;
          here |= (slow ? y[e] != y[e] : y[e] == tie) && j >= j0 && j < j1 ? 1u << e : 0u;
        }
      }
      int before = __popc(here);
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, before, s);
        if (lane >= s) before += o;
      }
      __syncthreads();  // (the last turn's counts are read)
      if (lane == 31) equals[warp] = before;
      before -= __popc(here);
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < warp) before += equals[w];
        all += equals[w];
      }
      for (int place = found + before; here != 0u && place < want; ++place) {
        list[place] = Key<A>::of(slow ? hi : tie, (v + static_cast<int>(threadIdx.x)) * VE - row.off + __ffs(here) - 1);
        here &= here - 1u;
      }
      found += all;
    }
    // and then, of such a slice, the best one behind the last one
    for (; slow && found < want; ++found) {
      __syncthreads();
      const Key<A> last = list[max(found - 1, 0)];
      Key<A> best = Key<A>::none();
      for (int v = v0 + static_cast<int>(threadIdx.x); v < v1; v += NT) {
        A y[VE];
        row.load(v, y);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int j = v * VE - row.off + e;
          const Key<A> o = Key<A>::of(y[e], j);
          if (j >= j0 && j < j1 && last.ahead(o) && o.ahead(best)) best = o;
        }
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) {
        const Key<A> o = best.other(s);
        if (o.ahead(best)) best = o;
      }
      if (lane == 0) cands[warp] = best;
      __syncthreads();
      if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < W; ++w)
          if (cands[w].ahead(best)) best = cands[w];
        list[found] = best;
      }
    }
  }
  if (cluster > 1) {
    if (threadIdx.x == 0) {
      parts[rank].hi = hi;
      parts[rank].S = S;
      parts[rank].T = Tm;
      parts[rank].count = want;
    }
    __syncthreads();
    cluster_wait();
    if (rank > 0) {
      if (threadIdx.x == 0) store_cluster(&parts[rank], parts[rank]);
      for (int q = threadIdx.x; q < want; q += NT) store_cluster(&list[q], list[q]);
    }
    __syncthreads();
    cluster_sync();
    if (rank > 0) return;
    // the row's results, by the first block
    hi = neg_inf<A>();
    for (int r = 0; r < cluster; ++r) hi = max_nan(hi, parts[r].hi);
    S = Tm = A(0);
    for (int r = 0; r < cluster; ++r) {
      if (!(parts[r].hi > neg_inf<A>())) continue;
      const A drop = (parts[r].hi - hi) * c;
      const bool far = !(drop > Expo<A>::floor);
      const A f = far ? A(0) : Expo<A>::exp(drop);
      S += f * parts[r].S;
      Tm += f * (parts[r].T + parts[r].S * (far ? A(0) : drop));
    }
  } else {
    __syncthreads();
  }
  Tm *= Expo<A>::unit;
  if (hi != hi || hi == -neg_inf<A>()) S = Tm = static_cast<A>(NAN);
  const A L = hi == neg_inf<A>() ? hi : log_acc(S);
  if (threadIdx.x == 0) write_row(a, i, hi, S, Tm, L, labelled, at_label);
  if (cluster == 1) {
    if (static_cast<int>(threadIdx.x) < a.top) write_top(a, i, static_cast<int>(threadIdx.x), list[threadIdx.x], hi, L);
    return;
  }
  for (int q = threadIdx.x; q < cluster * kMaxTop; q += NT) {
    const int r = q / kMaxTop, k = q % kMaxTop;
    if (k >= parts[r].count) continue;
    const Key<A> me = lists[r][k];
    int place = k;  // the lists are in order: only the others' candidates are counted
    for (int o = 0; o < cluster; ++o)
      if (o != r) place += place_of(lists[o], parts[o].count, me);
    if (place < a.top) write_top(a, i, place, me, hi, L);
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

// The gradient reads and writes every score once: bound by HBM (131072 x 1024 fp32 166 us, 6.5
// TB/s; 4096 x 131072 bf16 358, 6.0).  With t = log p in the
// exponent's unit, dx = p (A + B t) with A = -scale (g_l + g_H H), B = -scale g_H, and
// scale g_l more at the label: per score a subtraction, two fused multiply-adds, one
// exponential and a product, fp32 in pairs.  One warp per (row, kGradVecs 16-byte vectors a
// lane) of the output, whose alignment decides where the vectors begin; scores whose row
// starts elsewhere in its 16 bytes are put together from two aligned reads.
constexpr int kGradVecs = 4;

template <typename A> struct GradRow {
  A h, c, nL, ca, cb;  // t = (x - h) c + nL, h and c with the scale's sign
};

// y <- p (A + B t)
template <int N> __device__ __forceinline__ void grad_values(float* y, const GradRow<float>& r) {
  const uint64_t h = f2_pack(r.h, r.h), c = f2_pack(r.c, r.c), nl = f2_pack(r.nL, r.nL), ca = f2_pack(r.ca, r.ca),
                 cb = f2_pack(r.cb, r.cb);
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    float t0, t1;
    f2_unpack(f2_fma(f2_sub(f2_pack(y[e], y[e + 1]), h), c, nl), t0, t1);
    t0 = fmaxf(t0, Expo<float>::floor);
    t1 = fmaxf(t1, Expo<float>::floor);
    const uint64_t p = f2_pack(Expo<float>::exp(t0), Expo<float>::exp(t1));
    f2_unpack(f2_mul(p, f2_fma(cb, f2_pack(t0, t1), ca)), y[e], y[e + 1]);
  }
}
template <int N> __device__ __forceinline__ void grad_values(double* y, const GradRow<double>& r) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    double t = (y[e] - r.h) * r.c + r.nL;
    t = t > Expo<double>::floor ? t : Expo<double>::floor;
    y[e] = Expo<double>::exp(t) * (r.ca + r.cb * t);
  }
}

template <typename T> __device__ __forceinline__ uint4 pack(const Acc<T>* y) {
  Vec<T, 16 / static_cast<int>(sizeof(T))> v;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&v.raw);
#pragma unroll
    for (int q = 0; q < 4; ++q) p[q] = __floats2bfloat162_rn(y[2 * q], y[2 * q + 1]);
  } else if constexpr (std::is_same<T, __half>::value) {
    __half2* p = reinterpret_cast<__half2*>(&v.raw);
#pragma unroll
    for (int q = 0; q < 4; ++q) p[q] = __floats2half2_rn(y[2 * q], y[2 * q + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) v.e[e] = y[e];
  }
  return v.raw;
}

template <typename T> __global__ void __launch_bounds__(256) scores_grad_kernel(ScoreGradArgs<T> a, int chunks) {
  using A = Acc<T>;
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t i = unit / chunks;
  if (i >= a.n) return;
  const int chunk = static_cast<int>(unit - i * chunks);
  T* out = a.grad + i * a.m;
  const T* x = a.x + i * a.ld;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int j0 = (chunk * (32 * kGradVecs) + lane) * VE - off;
  const bool whole = j0 >= 0 && j0 + (kGradVecs - 1) * 32 * VE + VE <= a.m;
  uint4 w[kGradVecs];
  if (whole && same) {
    const uint4* from = reinterpret_cast<const uint4*>(x + j0);
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) w[u] = load_once(from + u * 32);
  } else {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) {
      const int j = j0 + u * 32 * VE;
      if (j >= 0 && j + VE <= a.m) {
        w[u] = load_any_16(x + j, a.x, a.x + (a.n - 1) * a.ld + a.m);
      } else {
        Vec<T, VE> v;
        v.raw = raw_zero<uint4>();
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (j + e >= 0 && j + e < a.m) v.e[e] = x[j + e];
        w[u] = v.raw;
      }
    }
  }
  const A hi = a.stats[3 * i], L = a.stats[3 * i + 1], H = a.stats[3 * i + 2];
  const int64_t label = a.labels ? label_of<T>(a.labels, a.labels_i64, i) : -1;
  const bool has = label >= 0 && label < a.m && a.g_log_probs;
  const A gl = has ? a.g_log_probs[i] : A(0);
  const A gh = a.g_entropy ? a.g_entropy[i] : A(0);
  const A scale = a.sign * a.mag;
  GradRow<A> r;  // of an empty row (hi = -inf) every t is the floor, and p 0
  r.h = a.sign * hi;
  r.c = a.sign * (a.mag * Expo<A>::per_nat);
  r.nL = -L * Expo<A>::per_nat;
  r.ca = -scale * (gl + gh * H);
  r.cb = -scale * gh * Expo<A>::unit;
  const int hit = has && hi != neg_inf<A>() ? static_cast<int>(label) - j0 : -1;
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    A y[VE];
    unpack<T>(w[u], y);
    grad_values<VE>(y, r);
    if (static_cast<unsigned>(hit - u * 32 * VE) < static_cast<unsigned>(VE)) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e == hit - u * 32 * VE) y[e] += scale * gl;
    }
    const int j = j0 + u * 32 * VE;
    if (whole || (j >= 0 && j + VE <= a.m)) {
      store_once(reinterpret_cast<uint4*>(out + j), pack<T>(y));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (j + e >= 0 && j + e < a.m) out[j + e] = from_acc<T>(y[e]);
    }
  }
}

// ------------------------------------------------------------------ launches
// whether every row is whole 16-byte vectors
template <typename T> static bool rows_are_vectors(const ScoreArgs<T>& a) {
  return a.m % RowVecs<T>::VE == 0 &&
         ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ld * sizeof(T))) & 15u) == 0;
}

template <typename T, int TEAM, int EPL> static cudaError_t scores_team(const ScoreArgs<T>& a, cudaStream_t st) {
  const unsigned blocks =
      static_cast<unsigned>(std::min<int64_t>((a.n * TEAM + 127) / 128, static_cast<int64_t>(num_sms()) * 28));
  constexpr size_t rows = 128 * EPL * sizeof(T);  // a row per team
  if (rows_are_vectors(a)) {
    if (rows > 32 * 1024 - 1) {  // near 48 KiB with the candidates
      const cudaError_t e = cudaFuncSetAttribute(scores_team_kernel<T, TEAM, EPL, true>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(rows));
      if (e != cudaSuccess) return e;
    }
    scores_team_kernel<T, TEAM, EPL, true><<<blocks, 128, rows, st>>>(a);
  } else if constexpr (EPL <= 32) {
    scores_team_kernel<T, TEAM, EPL, false><<<blocks, 128, 0, st>>>(a);
  } else {
    return cudaErrorInvalidValue;
  }
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
  if (smem > 32 * 1024) {  // beyond 48 KiB with the static arrays
    const cudaError_t e = cudaFuncSetAttribute(scores_block_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(kGroups * NT * sizeof(Acc<T>)));
    if (e != cudaSuccess) return e;
  }
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
  int log_cluster = 0;
  while ((1 << log_cluster) < cluster) ++log_cluster;
  return cudaLaunchKernelEx(&cfg, scores_block_kernel<T, NT>, a, log_cluster, per_group);
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
  // a row in one team's registers where it fits; 8 lanes bound few alternatives well
  if (a.top <= 8 && a.m <= 64) return scores_team<T, 8, 8>(a, st);
  if (a.top <= 8 && a.m <= 256) return scores_team<T, 8, 32>(a, st);
  if (a.top <= 16 && a.m <= 512 && a.m > 256) return scores_team<T, 16, 32>(a, st);
  if (a.m <= 256) return scores_team<T, 32, 8>(a, st);
  if (a.m <= 512) return scores_team<T, 32, 16>(a, st);
  if (a.m <= 1024) return scores_team<T, 32, 32>(a, st);
  if constexpr (sizeof(T) < 8)
    if (a.m <= 2048 && a.n >= num_sms() * 4 && rows_are_vectors(a)) return scores_team<T, 32, 64>(a, st);
  // Small blocks for short rows of which there are enough: what a block does once a row costs
  // every one of its warps (65536 x 3000 bf16 top 8: 227 us with 32 threads, 253 with 64, 343
  // with 128), long rows need their vectors in flight (16384 x 8192 fp32 top 8: 137, 110 and 133;
  // 4096 x 131072 bf16 top 20: 204 with 128 and 215 with 256).
  const int64_t bytes = static_cast<int64_t>(a.m) * static_cast<int64_t>(sizeof(T));
  if (bytes <= 8192 && a.n >= num_sms() * 8) return scores_block<T, 32>(a, st);
  if (bytes <= 32768 && a.n >= num_sms() * 8) return scores_block<T, 64>(a, st);
  if (a.n >= num_sms() * 4) return scores_block<T, 128>(a, st);
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
  constexpr int64_t VE = 16 / sizeof(T);
  const bool aligned = (reinterpret_cast<uintptr_t>(a.grad) & 15u) == 0 && a.m % VE == 0;
  const int chunks = static_cast<int>((a.m + (aligned ? 0 : VE - 1) + per - 1) / per);
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
