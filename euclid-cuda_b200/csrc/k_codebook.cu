// Codebook lookup with scaling, and its gradient by sorted labels.
//
//   out[i] = s * C[l_i]                (a zero row where l_i lies outside [0, k))
//   dC[c]  = s * sum of G[i] over the rows with l_i = c   (zero where there is none)
//
// The lookup reads each row of C that the labels name and writes n rows: bound by HBM, or
// by L2 where the table fits there.  One thread per 16-byte vector of an output row.
//
// The gradient is the center update's sum without the mean, in 32 bits (64 for fp64) and
// in a fixed order: over the rows sorted by label (k_groups.cu), cut into chunks of equal
// length so that a frequent label costs no more than rare ones.  One thread per (chunk,
// vector of the row) adds the chunk's rows in order; a label that lies inside the chunk is
// rounded and written at once, one that crosses a chunk's border leaves its sum in the
// workspace (slot 0 of the chunk if it began before the chunk, else slot 1), and a second
// kernel adds those in chunk order and clears the rows of labels without rows.
#include "engine.h"
#include "rows.cuh"

#include <algorithm>

namespace euc {

template <typename T, int N, typename TL>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ C, int64_t k, const TL* __restrict__ labels,
                                                     int64_t n, int64_t nv, Acc<T> scale, T* __restrict__ out) {
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  const Raw* Cr = reinterpret_cast<const Raw*>(C);
  Raw* Or = reinterpret_cast<Raw*>(out);
  RowWalk w(static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, static_cast<int64_t>(gridDim.x) * blockDim.x,
            nv);
  while (w.row < n) {
    // four vectors in flight: their labels, then the table's vectors, before any is stored
    int64_t at[4], src[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = -1;
      src[u] = -1;
      if (w.row < n) {
        at[u] = w.row * nv + w.v;
        const int64_t c = static_cast<int64_t>(labels[w.row]);
        if (c >= 0 && c < k) src[u] = c * nv + w.v;
        w.next();
      }
    }
    V v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u].raw = src[u] >= 0 ? load_keep(Cr + src[u]) : raw_zero<Raw>();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (at[u] < 0) continue;
      if (src[u] >= 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[u].e[e] = from_acc<T>(scale * to_acc(v[u].e[e]));
      }
      store_once(Or + at[u], v[u].raw);
    }
  }
}

// ------------------------------------------------------------------ gradient
struct GradArgs {
  const int32_t* offsets;
  const int32_t* order;
  const int32_t* labels;  // of the sorted rows
  int64_t n, k, nv;
  int seg;
  int64_t chunks;
};

template <typename T, int N>
__global__ void __launch_bounds__(256) grad_chunks_kernel(const T* __restrict__ G, GradArgs a, Acc<T> scale,
                                                          T* __restrict__ out, Acc<T>* __restrict__ part) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  const Raw* Gr = reinterpret_cast<const Raw*>(G);
  const int64_t total = min(a.n, static_cast<int64_t>(a.offsets[a.k]));
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t chunk = t / a.nv, v = t - chunk * a.nv;
  const int64_t p0 = chunk * a.seg;
  if (p0 >= total) return;
  const int64_t p1 = min(total, p0 + a.seg);
  A acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = A(0);
  int64_t c = a.labels[p0];
  auto flush = [&]() {
    if (c >= 0 && c < a.k) {
      const int64_t lo = a.offsets[c], hi = a.offsets[c + 1];
      if (lo >= p0 && hi <= p1) {
        V o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(scale * acc[e]);
        store_once(reinterpret_cast<Raw*>(out) + c * a.nv + v, o.raw);
      } else {
        A* to = part + ((2 * chunk + (lo < p0 ? 0 : 1)) * a.nv + v) * N;
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = acc[e];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
  };
  constexpr int RB = 8;  // rows in flight
  for (int64_t pb = p0; pb < p1; pb += RB) {
    V g[RB];
    int32_t lab[RB];
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const int64_t q = pb + u;
      const int64_t row = q < p1 ? a.order[q] : -1;
      lab[u] = q < p1 ? a.labels[q] : -1;
      g[u].raw = row >= 0 && row < a.n ? load_once(Gr + row * a.nv + v) : raw_zero<Raw>();
    }
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      if (pb + u >= p1) break;
      if (lab[u] != c) {
        flush();
        c = lab[u];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += to_acc(g[u].e[e]);
    }
  }
  flush();
}

template <typename T, int N>
__global__ void __launch_bounds__(256) grad_join_kernel(GradArgs a, Acc<T> scale, const Acc<T>* __restrict__ part,
                                                        T* __restrict__ out) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  RowWalk w(static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, static_cast<int64_t>(gridDim.x) * blockDim.x,
            a.nv);
  for (; w.row < a.k; w.next()) {
    const int64_t lo = max(0, a.offsets[w.row]), hi = min(a.n, static_cast<int64_t>(a.offsets[w.row + 1]));
    Raw* to = reinterpret_cast<Raw*>(out) + w.row * a.nv + w.v;
    if (hi <= lo) {
      store_once(to, raw_zero<Raw>());
      continue;
    }
    const int64_t c0 = lo / a.seg, c1 = (hi - 1) / a.seg;
    if (c0 == c1) continue;  // written by its chunk
    A acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
    for (int64_t c = c0; c <= c1; ++c) {
      const A* from = part + ((2 * c + (lo < c * a.seg ? 0 : 1)) * a.nv + w.v) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += from[e];
    }
    V o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(scale * acc[e]);
    store_once(to, o.raw);
  }
}

// ------------------------------------------------------------------ launches
static unsigned grid_for(int64_t items, int waves) {
  const int64_t most = static_cast<int64_t>(num_sms()) * waves;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, most)));
}

// Rows per chunk.
static int grad_seg(int64_t n) {
  int seg = 16;
  while (seg < 256 && n / seg > 8192) seg *= 2;
  return seg;
}

size_t codebook_grad_ws_bytes(RowType t, int64_t n, int64_t dim) {
  if (n <= 0) return 0;
  const int64_t chunks = (n + grad_seg(n) - 1) / grad_seg(n);
  return static_cast<size_t>(2 * chunks) * dim * (t == ROW_F64 ? 8 : 4);
}

template <typename T, int N, typename TL>
static cudaError_t lookup_go(const T* C, int64_t k, const TL* labels, int64_t n, int64_t dim, double scale, T* out,
                             cudaStream_t st) {
  const int64_t nv = dim / N;
  lookup_kernel<T, N, TL><<<grid_for((n * nv + 3) / 4, 64), 256, 0, st>>>(C, k, labels, n, nv,
                                                                        static_cast<Acc<T>>(scale), out);
  return cudaGetLastError();
}

template <typename T, int N>
static cudaError_t lookup_n(const T* C, int64_t k, const void* labels, bool i64, int64_t n, int64_t dim, double scale,
                            T* out, cudaStream_t st) {
  return i64 ? lookup_go<T, N>(C, k, static_cast<const long long*>(labels), n, dim, scale, out, st)
             : lookup_go<T, N>(C, k, static_cast<const int*>(labels), n, dim, scale, out, st);
}

template <typename T, int N>
static cudaError_t grad_n(const T* G, GradArgs a, int64_t dim, double scale, T* out, void* ws, cudaStream_t st) {
  a.nv = dim / N;
  Acc<T>* part = static_cast<Acc<T>*>(ws);
  const Acc<T> s = static_cast<Acc<T>>(scale);
  if (a.n > 0) {
    const int64_t threads = a.chunks * a.nv;
    grad_chunks_kernel<T, N><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, st>>>(G, a, s, out, part);
  }
  grad_join_kernel<T, N><<<grid_for(a.k * a.nv, 64), 256, 0, st>>>(a, s, part, out);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t lookup_t(const void* C, int64_t k, const void* labels, bool i64, int64_t n, int64_t dim,
                            double scale, void* out, cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(out));
  EUC_ROW_VEC(T, b, lookup_n, static_cast<const T*>(C), k, labels, i64, n, dim, scale, static_cast<T*>(out), st);
}

template <typename T>
static cudaError_t grad_t(const void* G, const GradArgs& a, int64_t dim, double scale, void* out, void* ws,
                          cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(G) | reinterpret_cast<uintptr_t>(out));
  EUC_ROW_VEC(T, b, grad_n, static_cast<const T*>(G), a, dim, scale, static_cast<T*>(out), ws, st);
}

cudaError_t launch_codebook_lookup(RowType t, const void* C, int64_t k, const void* labels, bool labels_i64, int64_t n,
                                   int64_t dim, double scale, void* out, cudaStream_t st) {
  switch (t) {
    case ROW_F32: return lookup_t<float>(C, k, labels, labels_i64, n, dim, scale, out, st);
    case ROW_F64: return lookup_t<double>(C, k, labels, labels_i64, n, dim, scale, out, st);
    case ROW_F16: return lookup_t<__half>(C, k, labels, labels_i64, n, dim, scale, out, st);
    default: return lookup_t<__nv_bfloat16>(C, k, labels, labels_i64, n, dim, scale, out, st);
  }
}

cudaError_t launch_codebook_grad(RowType t, const void* G, const int32_t* offsets, const int32_t* order,
                                 const int32_t* sorted, int64_t n, int64_t k, int64_t dim, double scale, void* out,
                                 void* ws, cudaStream_t st) {
  GradArgs a{};
  a.offsets = offsets;
  a.order = order;
  a.labels = sorted;
  a.n = n;
  a.k = k;
  a.seg = grad_seg(n);
  a.chunks = (n + a.seg - 1) / a.seg;
  switch (t) {
    case ROW_F32: return grad_t<float>(G, a, dim, scale, out, ws, st);
    case ROW_F64: return grad_t<double>(G, a, dim, scale, out, ws, st);
    case ROW_F16: return grad_t<__half>(G, a, dim, scale, out, ws, st);
    default: return grad_t<__nv_bfloat16>(G, a, dim, scale, out, ws, st);
  }
}

}  // namespace euc
