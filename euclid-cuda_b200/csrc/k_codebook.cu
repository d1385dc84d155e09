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
// kernel adds those in a fixed order.  The rows of labels without rows are cleared beside the
// sums.  Bound by HBM where rows are many (1048576 of 128 fp32 to 1024: 100 us, 5.4 TB/s;
// 65536 of 1024 bf16 to 131072, the frequent ones' rows in 60 chunks: 91, 4.4), and by the
// latency of the join where they are few.
#include "engine.h"
#include "rows.cuh"

#include <algorithm>

namespace euc {

// R U vectors a lane in flight: their rows' labels, then the table's vectors, before any is
// stored
template <typename T, int N, typename TL, int R, int U, bool WIDE>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ C, int64_t k, const TL* __restrict__ labels,
                                                     int64_t n, int64_t nv, int64_t chunks, Acc<T> scale,
                                                     T* __restrict__ out) {
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  const Raw* Cr = reinterpret_cast<const Raw*>(C);
  Raw* Or = reinterpret_cast<Raw*>(out);
  V x[R][U];
  auto scaled = [&](V v) {
#pragma unroll
    for (int e = 0; e < N; ++e) v.e[e] = from_acc<T>(scale * to_acc(v.e[e]));
    return v.raw;
  };
  if constexpr (WIDE) {
    const WideRows<R, U> w(chunks);
    int64_t c[R];
#pragma unroll
    for (int r = 0; r < R; ++r) c[r] = w.row + r < n ? static_cast<int64_t>(__ldg(labels + w.row + r)) : -1;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[r][u].raw = raw_zero<Raw>();
        if (c[r] >= 0 && c[r] < k && w.v + 32 * u < nv) x[r][u].raw = load_keep(Cr + c[r] * nv + w.v + 32 * u);
      }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (w.row + r < n && w.v + 32 * u < nv)
          store_once(Or + (w.row + r) * nv + w.v + 32 * u, c[r] >= 0 && c[r] < k ? scaled(x[r][u]) : raw_zero<Raw>());
  } else {
    const NarrowRows<U> w(nv);
    int64_t row[U], c[U];
    uint32_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w.at(u, row[u], v[u]);
      c[u] = row[u] < n ? static_cast<int64_t>(__ldg(labels + row[u])) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[0][u].raw = raw_zero<Raw>();
      if (c[u] >= 0 && c[u] < k) x[0][u].raw = load_keep(Cr + c[u] * nv + v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] < n) store_once(Or + row[u] * nv + v[u], c[u] >= 0 && c[u] < k ? scaled(x[0][u]) : raw_zero<Raw>());
  }
}

// Rows that are not whole 16-byte words, 16 bytes at a time all the same: a vector holds the
// elements between two 16-byte boundaries of the output, and the table's row is read at the
// same elements, wherever those lie.  (35703 rows of 991 fp16: 77 us element by element.)
template <typename T, typename TL>
__global__ void __launch_bounds__(256) lookup_any_kernel(const T* __restrict__ C, int64_t k,
                                                         const TL* __restrict__ labels, int64_t n, int dim,
                                                         int64_t nv, Acc<T> scale, T* __restrict__ out) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));
  using V = Vec<T, N>;
  const NarrowRows<2> w(nv);
  int64_t row[2], c[2];
  int at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t v;
    w.at(u, row[u], v);
    c[u] = row[u] < n ? static_cast<int64_t>(__ldg(labels + row[u])) : -1;
    at[u] = static_cast<int>(v) * N -
            static_cast<int>((reinterpret_cast<uintptr_t>(out + row[u] * dim) & 15u) / sizeof(T));
    if (row[u] >= n) at[u] = dim;
  }
  V x[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    x[u].raw = raw_zero<uint4>();
    if (at[u] >= dim || c[u] < 0 || c[u] >= k) continue;
    const T* from = C + c[u] * dim + at[u];
    if (at[u] >= 0 && at[u] + N <= dim) {
      x[u].raw = load_any_16(from, C, C + k * dim);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (at[u] + e >= 0 && at[u] + e < dim) x[u].e[e] = from[e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[u].e[e] = from_acc<T>(scale * to_acc(x[u].e[e]));
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (at[u] >= dim) continue;
    T* to = out + row[u] * dim + at[u];
    if (at[u] >= 0 && at[u] + N <= dim) {
      store_once(reinterpret_cast<uint4*>(to), x[u].raw);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (at[u] + e >= 0 && at[u] + e < dim) to[e] = x[u].e[e];
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

// zero rows for the labels without rows: a warp takes 32 labels (whose emptiness is one
// ballot) times a chunk of at most kClearVecs vectors
constexpr int kClearVecs = 128;

template <typename Raw>
__device__ __forceinline__ void clear_rows(const GradArgs& a, int64_t block, int64_t blocks, Raw* out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunks = (a.nv + kClearVecs - 1) / kClearVecs, units = (a.k + 31) / 32 * chunks;
  for (int64_t unit = block * 8 + warp; unit < units; unit += blocks * 8) {
    const int64_t c0 = unit / chunks * 32, v0 = unit % chunks * kClearVecs;
    const int64_t c = c0 + lane;
    const bool empty = c < a.k && a.offsets[c + 1] <= a.offsets[c];
    unsigned todo = __ballot_sync(0xffffffffu, empty);
    if (a.nv < 32) {  // short rows: neighbouring lanes over the vectors of all 32 labels
      const uint32_t nv = static_cast<uint32_t>(a.nv);
      for (uint32_t f = lane; f < 32 * nv && todo; f += 32)
        if (todo >> (f / nv) & 1u) store_once(out + c0 * a.nv + f, raw_zero<Raw>());
      continue;
    }
    while (todo) {
      Raw* row = out + (c0 + __ffs(todo) - 1) * a.nv;
#pragma unroll
      for (int u = 0; u < kClearVecs / 32; ++u)
        if (v0 + u * 32 + lane < a.nv) store_once(row + v0 + u * 32 + lane, raw_zero<Raw>());
      todo &= todo - 1;
    }
  }
}

// Blocks that clear and blocks that sum take turns, so that one's writes and the other's
// reads overlap.
struct Role {
  int64_t block;  // among the blocks of its kind
  bool clears;
  __device__ __forceinline__ Role(int64_t chunk_blocks) : block(blockIdx.x) {
    const int64_t clear_blocks = gridDim.x - chunk_blocks, both = 2 * min(chunk_blocks, clear_blocks);
    clears = chunk_blocks < clear_blocks;
    if (block < both) {
      clears = block & 1;
      block >>= 1;
    } else {
      block -= both / 2;
    }
  }
};

template <typename T, int N>
__global__ void __launch_bounds__(256, N * sizeof(T) == 16 && sizeof(T) == 2 ? 3 : 4)
    grad_chunks_kernel(const T* __restrict__ G, GradArgs a, int64_t chunk_blocks, Acc<T> scale, T* __restrict__ out,
                       Acc<T>* __restrict__ part) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  const Raw* Gr = reinterpret_cast<const Raw*>(G);
  Raw* Or = reinterpret_cast<Raw*>(out);
  let_next_start();
  const Role role(chunk_blocks);
  if (role.clears) {
    clear_rows<Raw>(a, role.block, gridDim.x - chunk_blocks, Or);
    return;
  }
  const int64_t total = min(a.n, static_cast<int64_t>(a.offsets[a.k]));
  const int64_t t = role.block * blockDim.x + threadIdx.x;
  const int64_t chunk = t < 0x80000000ll ? static_cast<uint32_t>(t) / static_cast<uint32_t>(a.nv) : t / a.nv;
  const int64_t v = t - chunk * a.nv;
  const int64_t p0 = chunk * a.seg;
  if (p0 >= total) return;
  const int64_t p1 = min(total, p0 + a.seg);
  A acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = A(0);
  int c = a.labels[p0];
  // only the chunk's first label can have begun before it, only its last can go on behind it
  bool from_left = p0 > 0 && a.labels[p0 - 1] == c;
  const int behind = p1 < total ? a.labels[p1] : -1;
  auto flush = [&]() {
    if (c >= 0 && c < a.k) {
      if (!from_left && c != behind) {
        V o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(scale * acc[e]);
        store_once(Or + c * a.nv + v, o.raw);
      } else {
        A* to = part + ((2 * chunk + (from_left ? 0 : 1)) * a.nv + v) * N;
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = acc[e];
      }
    }
    from_left = false;
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
      const int64_t row = q < p1 ? __ldg(a.order + q) : -1;
      lab[u] = q < p1 ? __ldg(a.labels + q) : -1;
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

// The same for 16-bit rows of odd length (a.nv of them): a thread adds the 16 bytes of the row
// from element 8 v on, shifted out of the two aligned words that hold them, and leaves its
// sums by elements, as the kernel above does with N = 1 (33588 rows of 999 bf16 to 30 and 1000
// labels: 75 and 96 us element by element, 46 and 66 so; rows that 4 bytes divide are no
// faster so).
template <typename T>
__global__ void __launch_bounds__(256, 3)
    grad_chunks_any_kernel(const T* __restrict__ G, GradArgs a, int vecs, int64_t chunk_blocks, Acc<T> scale,
                           T* __restrict__ out, Acc<T>* __restrict__ part) {
  using A = Acc<T>;
  constexpr int N = 8;
  let_next_start();
  const Role role(chunk_blocks);
  if (role.clears) {
    clear_rows(a, role.block, gridDim.x - chunk_blocks, reinterpret_cast<unsigned short*>(out));
    return;
  }
  const int64_t total = min(a.n, static_cast<int64_t>(a.offsets[a.k]));
  const int64_t t = role.block * blockDim.x + threadIdx.x;
  const int64_t chunk = t < 0x80000000ll ? static_cast<uint32_t>(t) / static_cast<uint32_t>(vecs) : t / vecs;
  const int64_t p0 = chunk * a.seg;
  if (p0 >= total) return;
  const int64_t p1 = min(total, p0 + a.seg);
  const int64_t at = (t - chunk * vecs) * N;
  const int count = static_cast<int>(min(static_cast<int64_t>(N), a.nv - at));  // elements of the row
  const void *begin = G, *end = G + a.n * a.nv;
  A acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = A(0);
  int c = a.labels[p0];
  bool from_left = p0 > 0 && a.labels[p0 - 1] == c;
  const int behind = p1 < total ? a.labels[p1] : -1;
  auto flush = [&]() {
    if (c >= 0 && c < a.k) {
      const bool whole = !from_left && c != behind;
      T* o = out + c * a.nv + at;
      A* to = part + (2 * chunk + (from_left ? 0 : 1)) * a.nv + at;
      if (whole && count == N) {  // four 4-byte words, or three between two elements
        Vec<T, N> x;
#pragma unroll
        for (int e = 0; e < N; ++e) x.e[e] = from_acc<T>(scale * acc[e]);
        const bool even = (reinterpret_cast<uintptr_t>(o) & 2u) == 0;
        if (!even) {
          o[0] = x.e[0];
          o[N - 1] = x.e[N - 1];
          x.raw = shift_16(x.raw, x.raw, 2u);
        }
        uint32_t* words = reinterpret_cast<uint32_t*>(o + (even ? 0 : 1));
        store_once(words, x.raw.x);
        store_once(words + 1, x.raw.y);
        store_once(words + 2, x.raw.z);
        if (even) store_once(words + 3, x.raw.w);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (e < count) {
            if (whole) o[e] = from_acc<T>(scale * acc[e]);
            else to[e] = acc[e];
          }
      }
    }
    from_left = false;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
  };
  constexpr int RB = 4;  // rows in flight
  for (int64_t pb = p0; pb < p1; pb += RB) {
    Words16 g[RB];
    int32_t lab[RB];
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const int64_t q = pb + u;
      const int64_t row = q < p1 ? __ldg(a.order + q) : -1;
      lab[u] = q < p1 ? __ldg(a.labels + q) : -1;
      g[u].clear();
      if (row >= 0 && row < a.n) g[u].load(G + row * a.nv + at, 0, count, begin, end);
    }
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      if (pb + u >= p1) break;
      if (lab[u] != c) {
        flush();
        c = lab[u];
      }
      Vec<T, N> x;
      x.raw = g[u].get();
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += to_acc(x.e[e]);
    }
  }
  flush();
}

// A label that crosses chunks' borders is joined at the first border inside it: by the
// lanes of (border, vector) if it has fewer than kLongChunks chunks more, else by the block
// that belongs to the first multiple of kLongChunks among its chunks, whose lanes take
// neighbouring vectors, its other threads every so-manyth chunk, and whose sums are added in
// a fixed order.
constexpr int kLongChunks = 64;
constexpr int kJoinThreads = 512;
constexpr int kJoinCandidates = 4;  // multiples of kLongChunks that a block looks at

// sum over chunks [c, c1], every `step`-th, of the label that starts at position lo
template <typename A, int N>
__device__ __forceinline__ void add_parts(const A* part, int64_t c, int64_t c1, int64_t step, int64_t lo, int seg,
                                          int64_t nv, int64_t v, A* acc) {
  constexpr int P = N * sizeof(A) >= 32 ? 4 : 8;  // in flight
  for (; c <= c1; c += P * step) {
    A from[P][N];
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int64_t q = c + u * step;
      const A* at = part + ((2 * q + (lo < q * seg ? 0 : 1)) * nv + v) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) from[u][e] = q <= c1 ? __ldcg(at + e) : A(0);
    }
#pragma unroll
    for (int u = 0; u < P; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += from[u][e];
  }
}

template <typename T, int N>
__device__ __forceinline__ void join_long(const GradArgs& a, int64_t block, Acc<T> scale,
                                          const Acc<T>* __restrict__ part, T* __restrict__ out) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  __shared__ A sums[kJoinThreads][N];
  __shared__ int owner[kJoinCandidates];  // the candidate's label, or -1
  // lanes over vectors: the power of two that holds the row, at most a warp
  int width = 32;
  while (width > 1 && width / 2 >= a.nv) width /= 2;
  const int64_t tiles = (a.nv + width - 1) / width;
  const int64_t first = block / tiles * kJoinCandidates;
  const int64_t total = min(a.n, static_cast<int64_t>(a.offsets[a.k]));
  if (threadIdx.x < kJoinCandidates) {
    const int64_t at = (first + threadIdx.x) * kLongChunks * a.seg;
    int label = -1;
    if (at < total) {
      const int64_t c = a.labels[at];
      if (c >= 0 && c < a.k) {
        const int64_t lo = max(0, a.offsets[c]), hi = min(a.n, static_cast<int64_t>(a.offsets[c + 1]));
        // (the chunk's first row has the label, so the multiple before it is the only other candidate)
        if (hi > lo && (hi - 1) / a.seg - lo / a.seg >= kLongChunks && at - static_cast<int64_t>(kLongChunks) * a.seg < lo)
          label = static_cast<int>(c);
      }
    }
    owner[threadIdx.x] = label;
  }
  __syncthreads();
  const int groups = kJoinThreads / width, group = static_cast<int>(threadIdx.x) / width,
            lane = static_cast<int>(threadIdx.x) % width;
  const int64_t v = block % tiles * width + lane;
  for (int q = 0; q < kJoinCandidates; ++q) {
    const int64_t c = owner[q];
    if (c < 0) continue;
    const int64_t lo = max(0, a.offsets[c]), hi = min(a.n, static_cast<int64_t>(a.offsets[c + 1]));
    const int64_t c0 = lo / a.seg, c1 = (hi - 1) / a.seg;
    A acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
    if (v < a.nv) add_parts<A, N>(part, c0 + group, c1, groups, lo, a.seg, a.nv, v, acc);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) sums[threadIdx.x][e] = acc[e];
    for (int half = groups / 2; half > 0; half /= 2) {
      __syncthreads();
      if (group < half)
#pragma unroll
        for (int e = 0; e < N; ++e) sums[threadIdx.x][e] += sums[threadIdx.x + half * width][e];
    }
    if (group == 0 && v < a.nv) {
      V o;
#pragma unroll
      for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(scale * sums[threadIdx.x][e]);
      store_once(reinterpret_cast<typename V::Raw*>(out) + c * a.nv + v, o.raw);
    }
  }
}

template <typename T, int N, int SUB>
__global__ void __launch_bounds__(kJoinThreads) grad_join_kernel(GradArgs a, int64_t long_blocks, Acc<T> scale,
                                                        const Acc<T>* __restrict__ part, T* __restrict__ out) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  wait_for_previous();
  if (static_cast<int64_t>(blockIdx.x) < long_blocks) {  // the longest work starts first
    join_long<T, N>(a, blockIdx.x, scale, part, out);
    return;
  }
  // SUB 4: a warp takes 32 neighbouring vectors at one border, eight at a time, its four lanes
  // of a vector every fourth chunk; SUB 1 (rows of fewer vectors): a thread per vector and border
  constexpr int VW = 32 / SUB;
  const int lane = threadIdx.x & 31, sub = SUB == 1 ? 0 : lane / VW;
  const int64_t t = static_cast<int64_t>(blockIdx.x - long_blocks) * blockDim.x + threadIdx.x;
  const int64_t unit = SUB == 1 ? t : t >> 5, tiles = SUB == 1 ? a.nv : (a.nv + 31) / 32;
  const int64_t border =
      1 + (unit < 0x80000000ll ? static_cast<uint32_t>(unit) / static_cast<uint32_t>(tiles) : unit / tiles);
  const int64_t tile = unit - (border - 1) * tiles, at = border * a.seg;
  if (at >= min(a.n, static_cast<int64_t>(a.offsets[a.k]))) return;
  const int64_t c = a.labels[at];
  if (c < 0 || c >= a.k || a.labels[at - 1] != c) return;
  const int64_t lo = max(0, a.offsets[c]), hi = min(a.n, static_cast<int64_t>(a.offsets[c + 1]));
  const int64_t c0 = lo / a.seg, c1 = (hi - 1) / a.seg;
  if (c0 != border - 1 || c1 - c0 >= kLongChunks) return;  // an earlier border's, or a block's
  // (a warp of SUB 4 is at one border: all of its lanes are here)
  for (int q = 0; q < SUB; ++q) {
    const int64_t v = SUB == 1 ? tile : tile * 32 + q * VW + lane % VW;
    A acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
    if (v < a.nv) add_parts<A, N>(part, c0 + sub, c1, SUB, lo, a.seg, a.nv, v, acc);
    if constexpr (SUB > 1) {
#pragma unroll
      for (int s = VW; s < 32; s <<= 1)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], s);
    }
    if (sub != 0 || v >= a.nv) continue;
    V o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(scale * acc[e]);
    store_once(reinterpret_cast<Raw*>(out) + c * a.nv + v, o.raw);
  }
}

// ------------------------------------------------------------------ launches
// Rows per chunk: as many as leave 16 warps per SM, since every chunk may cost two partial
// sums and their join.  `row_bytes` / 16 stands for the row's vectors at any alignment.
static int grad_seg(int64_t n, int64_t row_bytes) {
  const int64_t nv = std::max<int64_t>(1, row_bytes / 16);
  int seg = 16;
  while (seg < 256 && n / (2 * seg) * nv >= static_cast<int64_t>(num_sms()) * 512) seg *= 2;
  return seg;
}

size_t codebook_grad_ws_bytes(RowType t, int64_t n, int64_t dim) {
  if (n <= 0) return 0;
  const int64_t seg = grad_seg(n, dim * (t == ROW_F64 ? 8 : t == ROW_F32 ? 4 : 2));
  const int64_t chunks = (n + seg - 1) / seg;
  return static_cast<size_t>(2 * chunks) * dim * (t == ROW_F64 ? 8 : 4);
}

template <typename T, int N, typename TL>
static cudaError_t lookup_go(const T* C, int64_t k, const TL* labels, int64_t n, int64_t dim, double scale, T* out,
                             cudaStream_t st) {
  const int64_t nv = dim / N;
  const Acc<T> s = static_cast<Acc<T>>(scale);
  auto wide = [&](auto kernel, int R, int U) {
    kernel<<<static_cast<unsigned>(wide_blocks(n, nv, R, U)), 256, 0, st>>>(C, k, labels, n, nv,
                                                                          (nv + 32 * U - 1) / (32 * U), s, out);
    return cudaGetLastError();
  };
  if (nv < 32) {
    lookup_kernel<T, N, TL, 1, 4, false>
        <<<static_cast<unsigned>(narrow_blocks(n, nv, 4)), 256, 0, st>>>(C, k, labels, n, nv, 1, s, out);
    return cudaGetLastError();
  }
  // few rows are spread over more warps: latency counts there, not what a warp has in flight
  if (n * nv <= static_cast<int64_t>(num_sms()) * 2048) return wide(lookup_kernel<T, N, TL, 1, 1, true>, 1, 1);
  if (nv <= 32) return wide(lookup_kernel<T, N, TL, 4, 1, true>, 4, 1);
  if (nv <= 64) return wide(lookup_kernel<T, N, TL, 2, 2, true>, 2, 2);
  // (57934 rows of 554 fp32, 8 bytes at a time: 44 us with two vectors a lane)
  if (N * sizeof(T) < 16) return wide(lookup_kernel<T, N, TL, 1, 4, true>, 1, 4);
  return wide(lookup_kernel<T, N, TL, 1, 2, true>, 1, 2);
}

template <typename T, int N>
static cudaError_t lookup_n(const T* C, int64_t k, const void* labels, bool i64, int64_t n, int64_t dim, double scale,
                            T* out, cudaStream_t st) {
  return i64 ? lookup_go<T, N>(C, k, static_cast<const long long*>(labels), n, dim, scale, out, st)
             : lookup_go<T, N>(C, k, static_cast<const int*>(labels), n, dim, scale, out, st);
}

// `vecs`: vectors of a row of odd length that is read 16 bytes at a time (N = 1), else 0
template <typename T, int N>
static cudaError_t grad_n(const T* G, GradArgs a, int64_t dim, int64_t vecs, double scale, T* out, void* ws,
                          cudaStream_t st) {
  a.nv = dim / N;
  Acc<T>* part = static_cast<Acc<T>*>(ws);
  const Acc<T> s = static_cast<Acc<T>>(scale);
  const int64_t sums = (a.chunks * (vecs ? vecs : a.nv) + 255) / 256;
  const int64_t clears = std::min<int64_t>(
      ((a.k + 31) / 32 * ((a.nv + kClearVecs - 1) / kClearVecs) + 7) / 8, static_cast<int64_t>(num_sms()) * 16);
  const unsigned blocks = static_cast<unsigned>(sums + clears);
  bool any = false;
  if constexpr (N == 1 && sizeof(T) == 2) {
    any = vecs > 0;
    if (any)
      grad_chunks_any_kernel<T><<<blocks, 256, 0, st>>>(G, a, static_cast<int>(vecs), sums, s, out, part);
  }
  if (!any) grad_chunks_kernel<T, N><<<blocks, 256, 0, st>>>(G, a, sums, s, out, part);
  if (a.chunks > 1) {
    int width = 32;
    while (width > 1 && width / 2 >= a.nv) width /= 2;
    const int64_t longs =
        a.chunks > kLongChunks
            ? (a.chunks + kLongChunks * kJoinCandidates - 1) / (kLongChunks * kJoinCandidates) * ((a.nv + width - 1) / width)
            : 0;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // four lanes a vector where the row has eight vectors to fill the warp's others
    const bool four = a.nv >= 8;
    const int64_t threads = (a.chunks - 1) * (four ? (a.nv + 31) / 32 * 32 : a.nv);
    const unsigned g = static_cast<unsigned>(longs + (threads + kJoinThreads - 1) / kJoinThreads);
    return four ? launch_after(true, grad_join_kernel<T, N, 4>, g, kJoinThreads, 0, st, a, longs, s, part, out)
                : launch_after(true, grad_join_kernel<T, N, 1>, g, kJoinThreads, 0, st, a, longs, s, part, out);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t lookup_t(const void* C, int64_t k, const void* labels, bool i64, int64_t n, int64_t dim,
                            double scale, void* out, cudaStream_t st) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));
  const T* c = static_cast<const T*>(C);
  T* o = static_cast<T*>(out);
  const int64_t row_bytes = dim * static_cast<int64_t>(sizeof(T));
  const int b = row_vec_bytes(row_bytes, reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(out));
  // (short rows are mostly ends: 1000000 rows of 2 fp32 take 7.4 us by 8 bytes and 13.4 so)
  if (b >= 8 || row_bytes < 128) {
    EUC_ROW_VEC(T, b, lookup_n, c, k, labels, i64, n, dim, scale, o, st);
  }
  const int64_t nv = (dim + 2 * N - 2) / N;  // vectors that cover a row at any alignment
  const unsigned g = static_cast<unsigned>(narrow_blocks(n, nv, 2));
  const Acc<T> s = static_cast<Acc<T>>(scale);
  if (i64)
    lookup_any_kernel<T, long long><<<g, 256, 0, st>>>(c, k, static_cast<const long long*>(labels), n,
                                                      static_cast<int>(dim), nv, s, o);
  else
    lookup_any_kernel<T, int><<<g, 256, 0, st>>>(c, k, static_cast<const int*>(labels), n, static_cast<int>(dim), nv, s,
                                                o);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t grad_t(const void* G, const GradArgs& a, int64_t dim, double scale, void* out, void* ws,
                          cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(G) | reinterpret_cast<uintptr_t>(out));
  // (with fewer threads, latency counts: 30011 rows of 77 to 4099 labels 13.7 us by elements and
  // 19 so, 94720 to 11840 35 and 31; a million rows of 5: 26 and 29)
  if (b == 2 && dim >= 32 && a.chunks * ((dim + 7) / 8) >= static_cast<int64_t>(num_sms()) * 320)
    return grad_n<T, 1>(static_cast<const T*>(G), a, dim, (dim + 7) / 8, scale, static_cast<T*>(out), ws, st);
  EUC_ROW_VEC(T, b, grad_n, static_cast<const T*>(G), a, dim, 0, scale, static_cast<T*>(out), ws, st);
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
  a.seg = grad_seg(n, dim * (t == ROW_F64 ? 8 : t == ROW_F32 ? 4 : 2));
  a.chunks = (n + a.seg - 1) / a.seg;
  switch (t) {
    case ROW_F32: return grad_t<float>(G, a, dim, scale, out, ws, st);
    case ROW_F64: return grad_t<double>(G, a, dim, scale, out, ws, st);
    case ROW_F16: return grad_t<__half>(G, a, dim, scale, out, ws, st);
    default: return grad_t<__nv_bfloat16>(G, a, dim, scale, out, ws, st);
  }
}

}  // namespace euc
