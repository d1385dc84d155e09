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

__device__ __forceinline__ float exp_acc(float d) { return __expf(d); }
__device__ __forceinline__ double exp_acc(double d) { return exp(d); }
__device__ __forceinline__ float log_acc(float d) { return logf(d); }
__device__ __forceinline__ double log_acc(double d) { return log(d); }

template <typename A> __device__ __forceinline__ A neg_inf() { return -static_cast<A>(INFINITY); }

// exp(d) d, 0 where exp(d) is 0
template <typename A> __device__ __forceinline__ A weighted(A e, A d) { return e > A(0) ? e * d : A(0); }

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

// ------------------------------------------------------------------ one block per row
template <typename T> __global__ void __launch_bounds__(256) scores_block_kernel(ScoreArgs<T> a) {
  using A = Acc<T>;
  __shared__ A red[8];
  __shared__ Best<A> redb[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const T* x = a.x + i * a.ld;
    A hi = neg_inf<A>();
    bool nan = false;
    for (int j = threadIdx.x; j < a.m; j += 256) {
      const A y = a.sign * to_acc(x[j]);
      nan |= y != y;
      hi = y > hi ? y : hi;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      const A o = __shfl_xor_sync(0xffffffffu, hi, s);
      hi = o > hi ? o : hi;
    }
    if (lane == 0) red[warp] = hi;
    nan = __syncthreads_or(nan);
#pragma unroll
    for (int w = 0; w < 8; ++w) hi = red[w] > hi ? red[w] : hi;
    __syncthreads();
    const A shift = hi == neg_inf<A>() ? A(0) : hi;
    A S = A(0), Tm = A(0);
    for (int j = threadIdx.x; j < a.m; j += 256) {
      const A d = (a.sign * to_acc(x[j]) - shift) * a.mag;
      const A e = exp_acc(d);
      S += e;
      Tm += weighted(e, d);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, s);
      Tm += __shfl_xor_sync(0xffffffffu, Tm, s);
    }
    if (lane == 0) red[warp] = S;
    __syncthreads();
    S = A(0);
#pragma unroll
    for (int w = 0; w < 8; ++w) S += red[w];
    __syncthreads();
    if (lane == 0) red[warp] = Tm;
    __syncthreads();
    Tm = A(0);
#pragma unroll
    for (int w = 0; w < 8; ++w) Tm += red[w];
    if (nan) hi = S = Tm = static_cast<A>(NAN);
    if (threadIdx.x == 0) write_row(a, i, hi, S, Tm);
    const A L = hi == neg_inf<A>() ? neg_inf<A>() : log_acc(S);
    // the alternatives one by one: the best of those behind the last one
    Best<A> last;
    for (int t = 0; t < a.top; ++t) {
      Best<A> best;
      best.o = 0;
      best.j = 0x7fffffff;
      for (int j = threadIdx.x; j < a.m; j += 256) {
        Best<A> c;
        c.o = order_of(a.sign * to_acc(x[j]));
        c.j = j;
        if ((t == 0 || before(last, c)) && before(c, best)) best = c;
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
      for (int w = 0; w < 8; ++w)
        if (before(redb[w], best)) best = redb[w];
      last = best;
      if (threadIdx.x == 0) {
        const A y = a.sign * to_acc(x[best.j]);
        a.top_labels[i * a.top + t] = best.j;
        a.top_log_probs[i * a.top + t] = hi == neg_inf<A>() ? hi : (y - hi) * a.mag - L;
      }
    }
    __syncthreads();
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

template <typename T> __global__ void __launch_bounds__(256) scores_grad_kernel(ScoreGradArgs<T> a) {
  using A = Acc<T>;
  for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const A hi = a.stats[3 * i], L = a.stats[3 * i + 1], H = a.stats[3 * i + 2];
    const bool empty = hi == neg_inf<A>();
    const int64_t l = a.labels ? label_of<T>(a.labels, a.labels_i64, i) : -1;
    const A gl = l >= 0 && l < a.m && a.g_log_probs ? a.g_log_probs[i] : A(0);
    const A gh = a.g_entropy ? a.g_entropy[i] : A(0);
    const A scale = a.sign * a.mag;
    const T* x = a.x + i * a.ld;
    for (int j = threadIdx.x; j < a.m; j += 256) {
      const A lp = (a.sign * to_acc(x[j]) - hi) * a.mag - L;
      const A p = exp_acc(lp);
      A dz = p == A(0) ? A(0) : -p * (gl + gh * (lp + H));
      if (j == l) dz += gl;
      a.grad[i * a.m + j] = from_acc<T>(empty ? A(0) : scale * dz);
    }
  }
}

// ------------------------------------------------------------------ launches
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
  const unsigned g = static_cast<unsigned>(std::min<int64_t>(j.n, 1 << 30));
  scores_block_kernel<T><<<g, 256, 0, st>>>(a);
  return cudaGetLastError();
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
  const unsigned g = static_cast<unsigned>(std::min<int64_t>(j.n, 1 << 30));
  scores_grad_kernel<T><<<g, 256, 0, st>>>(a);
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
