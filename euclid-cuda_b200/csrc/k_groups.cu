// Rows sorted by label and back, with weights applied, and their gradients.
//
// n rows have p labels each; slot s = i * p + j is label j of row i.  The slots whose label
// lies in [0, k) are sorted by label, slots of one label in slot order (a stable sort, so
// that every result is the same on every run):
//   order[r] = slot at sorted position r, position[s] = r (its inverse),
//   offsets[c] = first position of label c, offsets[k] = number of slots kept.
// Rows there and back, and the gradients:
//   Y[position[i, j]] = X[i]              out[i] = sum_j w[i, j] Z[position[i, j]]
//   dZ[position[i, j]] = w[i, j] dOut[i]  dw[i, j] = <dOut[i], Z[position[i, j]]>
// and dX[i] = sum_j dY[position[i, j]], the second with weights of one.
//
// The sort is a counting sort in passes of up to kMaxBins bins (one pass for k < kMaxBins,
// else 2 or 3 by digits, least significant first): per tile of slots a histogram, a scan
// of each bin over the tiles, and a scatter that ranks a slot among its tile's equal keys
// by __match_any_sync within 32 slots, in slot order.  It moves 4 to 8 bytes a slot where
// the rows move kilobytes; the row kernels are bound by HBM, and read and write every row
// once: a row's copies are written from registers after one read, and its weighted sum is
// formed from p reads and written once.
#include "engine.h"
#include "rows.cuh"

#include <algorithm>

namespace euc {

// ------------------------------------------------------------------ the sort
constexpr int kMaxBins = 4097;   // k + 1 bins (the last for labels outside [0, k)) in one pass
constexpr int kSortWarps = 8;
constexpr int kSortItems = 16;   // slots per thread
constexpr int kTile = kSortWarps * 32 * kSortItems;

struct SortPass {
  int64_t n;
  uint32_t k;       // keys lie in [0, k]; k marks a dropped slot
  int shift;
  uint32_t mask;
  int bins;
  int tiles;
  uint32_t* T;      // [bins][tiles] counts, then exclusive prefixes over the tiles
  uint32_t* total;  // [bins]
};

template <typename TL> __device__ __forceinline__ uint32_t key_of(TL label, uint32_t k) {
  return label >= 0 && label < static_cast<TL>(k) ? static_cast<uint32_t>(label) : k;
}
// the keys of a later pass
template <> __device__ __forceinline__ uint32_t key_of<uint32_t>(uint32_t key, uint32_t) { return key; }

template <typename TL>
__global__ void __launch_bounds__(kSortWarps * 32) sort_hist_kernel(const TL* __restrict__ in, SortPass a) {
  extern __shared__ uint32_t cnt[];
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) cnt[c] = 0u;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t s = base + u * (kSortWarps * 32) + threadIdx.x;
    if (s < a.n) atomicAdd(&cnt[(key_of(in[s], a.k) >> a.shift) & a.mask], 1u);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) a.T[static_cast<int64_t>(c) * a.tiles + blockIdx.x] = cnt[c];
}

// one warp per bin: T[bin][.] becomes its exclusive prefix over the tiles
__global__ void __launch_bounds__(256) sort_tiles_kernel(SortPass a) {
  const int bin = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (bin >= a.bins) return;
  uint32_t* row = a.T + static_cast<int64_t>(bin) * a.tiles;
  uint32_t run = 0u;
  for (int b0 = 0; b0 < a.tiles; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t v = b < a.tiles ? row[b] : 0u;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (b < a.tiles) row[b] = run + x - v;
    run += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) a.total[bin] = run;
}

// exclusive scan of v[0, m) in shared memory by the whole block (m of any size)
__device__ __forceinline__ void block_scan(uint32_t* v, int m, uint32_t* warp_sums) {
  const int nt = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = nt >> 5;
  const int per = (m + nt - 1) / nt;
  const int lo = min(m, static_cast<int>(threadIdx.x) * per), hi = min(m, lo + per);
  uint32_t sum = 0u;
  for (int c = lo; c < hi; ++c) sum += v[c];
  uint32_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0u;
  for (int w = 0; w < nw; ++w) before += w < warp ? warp_sums[w] : 0u;
  uint32_t run = before + x - sum;
  for (int c = lo; c < hi; ++c) {
    const uint32_t t = v[c];
    v[c] = run;
    run += t;
  }
  __syncthreads();
}

struct SortOut {
  uint32_t* keys;      // a pass that is not the last: keys and slots in the pass's order
  uint32_t* slots;
  int32_t* order;      // the last pass
  int32_t* position;
  int32_t* labels;
  int32_t* offsets;    // the last pass of a one-pass sort, else null
};

template <typename TL, bool FIRST, bool LAST>
__global__ void __launch_bounds__(kSortWarps * 32) sort_scatter_kernel(const TL* __restrict__ in,
                                                                      const uint32_t* __restrict__ in_slots,
                                                                      SortPass a, SortOut o) {
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t warp_sums[kSortWarps];
  uint32_t* start = sm;                                             // [bins] first position of the tile's bin
  unsigned short* cnt = reinterpret_cast<unsigned short*>(sm + a.bins);  // [warps][bins]
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) start[c] = a.total[c];
  for (int c = threadIdx.x; c < a.bins * kSortWarps; c += blockDim.x) cnt[c] = 0;
  __syncthreads();
  block_scan(start, a.bins, warp_sums);
  if (LAST && o.offsets && blockIdx.x == 0)
    for (int c = threadIdx.x; c < a.bins; c += blockDim.x) o.offsets[c] = static_cast<int32_t>(start[c]);

  // a warp's slots are contiguous, 32 at a time in slot order
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned short* mine = cnt + warp * a.bins;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile + warp * (32 * kSortItems);
  uint32_t key[kSortItems];
  unsigned short rank[kSortItems];
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t s = base + u * 32 + lane;
    key[u] = s < a.n ? key_of(in[s], a.k) : 0xffffffffu;
  }
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const bool in_range = base + u * 32 + lane < a.n;
    const uint32_t d = in_range ? (key[u] >> a.shift) & a.mask : 0xffffffffu;
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    const int before = __popc(peers & ((1u << lane) - 1u));
    if (in_range) rank[u] = static_cast<unsigned short>(mine[d] + before);
    __syncwarp();
    if (in_range && before == 0) mine[d] = static_cast<unsigned short>(mine[d] + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) {  // counts -> prefixes over the warps
    start[c] += a.T[static_cast<int64_t>(c) * a.tiles + blockIdx.x];
    unsigned short run = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const unsigned short t = cnt[w * a.bins + c];
      cnt[w * a.bins + c] = run;
      run = static_cast<unsigned short>(run + t);
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t s = base + u * 32 + lane;
    if (s >= a.n) continue;
    const uint32_t d = (key[u] >> a.shift) & a.mask;
    const uint32_t pos = start[d] + mine[d] + rank[u];
    const uint32_t slot = FIRST ? static_cast<uint32_t>(s) : in_slots[s];
    if (LAST) {
      const bool kept = key[u] < a.k;
      o.order[pos] = kept ? static_cast<int32_t>(slot) : -1;
      o.labels[pos] = kept ? static_cast<int32_t>(key[u]) : -1;
      o.position[slot] = kept ? static_cast<int32_t>(pos) : -1;
    } else {
      o.keys[pos] = key[u];
      o.slots[pos] = slot;
    }
  }
}

// offsets of a sort of several passes: first position whose key is not below c
__global__ void sort_offsets_kernel(const int32_t* __restrict__ labels, int64_t n, int64_t k,
                                    int32_t* __restrict__ offsets) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c > k) return;
  int64_t lo = 0, hi = n;  // dropped slots (-1, at the end) count as k
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    const int64_t v = labels[mid] < 0 ? k : labels[mid];
    if (v < c) lo = mid + 1; else hi = mid;
  }
  offsets[c] = static_cast<int32_t>(lo);
}

static inline size_t al(size_t b) { return (b + 255) & ~size_t(255); }

struct SortPlan {
  int passes, bits, bins, tiles;
};

static SortPlan sort_plan(int64_t n, int64_t k) {
  SortPlan p{};
  p.tiles = static_cast<int>((n + kTile - 1) / kTile);
  if (k + 1 <= kMaxBins) {
    p.passes = 1;
    p.bins = static_cast<int>(k + 1);
    return p;
  }
  int bits = 1;
  while ((1ll << bits) <= k) ++bits;  // keys 0 .. k
  p.passes = (bits + 11) / 12;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.bins = 1 << p.bits;
  return p;
}

size_t group_ws_bytes(int64_t n, int64_t k) {
  if (n <= 0) return 0;
  const SortPlan p = sort_plan(n, k);
  size_t b = al(static_cast<size_t>(p.bins) * p.tiles * 4) + al(static_cast<size_t>(p.bins) * 4);
  if (p.passes > 1) b += 2 * al(static_cast<size_t>(n) * 4);
  if (p.passes > 2) b += 2 * al(static_cast<size_t>(n) * 4);
  return b;
}

template <typename TL, bool FIRST, bool LAST>
static cudaError_t sort_pass(const TL* in, const uint32_t* in_slots, const SortPass& a, const SortOut& o,
                             cudaStream_t st) {
  const size_t hist_sm = static_cast<size_t>(a.bins) * 4;
  const size_t sm = static_cast<size_t>(a.bins) * (4 + 2 * kSortWarps);
  cudaError_t e = cudaSuccess;
  if (sm > 48 * 1024)
    e = cudaFuncSetAttribute(sort_scatter_kernel<TL, FIRST, LAST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sm));
  if (e != cudaSuccess) return e;
  sort_hist_kernel<TL><<<a.tiles, kSortWarps * 32, hist_sm, st>>>(in, a);
  sort_tiles_kernel<<<(a.bins + 7) / 8, 256, 0, st>>>(a);
  sort_scatter_kernel<TL, FIRST, LAST><<<a.tiles, kSortWarps * 32, sm, st>>>(in, in_slots, a, o);
  return cudaGetLastError();
}

template <typename TL>
static cudaError_t group_t(const TL* labels, int64_t n, int64_t k, int32_t* offsets, int32_t* order, int32_t* position,
                           int32_t* sorted, uint8_t* ws, cudaStream_t st) {
  const SortPlan p = sort_plan(n, k);
  SortPass a{};
  a.n = n;
  a.k = static_cast<uint32_t>(k);
  a.bins = p.bins;
  a.tiles = p.tiles;
  a.T = reinterpret_cast<uint32_t*>(ws);
  ws += al(static_cast<size_t>(p.bins) * p.tiles * 4);
  a.total = reinterpret_cast<uint32_t*>(ws);
  ws += al(static_cast<size_t>(p.bins) * 4);
  SortOut o{};
  o.order = order;
  o.position = position;
  o.labels = sorted;
  if (p.passes == 1) {
    a.mask = 0xffffffffu;
    o.offsets = offsets;
    return sort_pass<TL, true, true>(labels, nullptr, a, o, st);
  }
  uint32_t* buf[4];
  for (int i = 0; i < 2 * std::min(p.passes - 1, 2); ++i) {
    buf[i] = reinterpret_cast<uint32_t*>(ws);
    ws += al(static_cast<size_t>(n) * 4);
  }
  a.mask = static_cast<uint32_t>(p.bins - 1);
  o.keys = buf[0];
  o.slots = buf[1];
  cudaError_t e = sort_pass<TL, true, false>(labels, nullptr, a, o, st);
  const uint32_t *keys = buf[0], *slots = buf[1];
  if (e == cudaSuccess && p.passes == 3) {
    a.shift = p.bits;
    o.keys = buf[2];
    o.slots = buf[3];
    e = sort_pass<uint32_t, false, false>(keys, slots, a, o, st);
    keys = buf[2];
    slots = buf[3];
  }
  if (e != cudaSuccess) return e;
  a.shift = p.bits * (p.passes - 1);
  e = sort_pass<uint32_t, false, true>(keys, slots, a, o, st);
  if (e != cudaSuccess) return e;
  sort_offsets_kernel<<<static_cast<unsigned>((k + 1 + 255) / 256), 256, 0, st>>>(sorted, n, k, offsets);
  return cudaGetLastError();
}

cudaError_t launch_group_rows(const void* labels, bool labels_i64, int64_t n, int64_t k, int32_t* offsets,
                              int32_t* order, int32_t* position, int32_t* sorted, void* ws, cudaStream_t st) {
  if (n == 0) return cudaMemsetAsync(offsets, 0, static_cast<size_t>(k + 1) * 4, st);
  uint8_t* w = static_cast<uint8_t*>(ws);
  if (labels_i64) return group_t(static_cast<const long long*>(labels), n, k, offsets, order, position, sorted, w, st);
  return group_t(static_cast<const int*>(labels), n, k, offsets, order, position, sorted, w, st);
}

// ------------------------------------------------------------------ rows there
// One thread per vector of a row: the vector is read once and stored at each of the row's
// kept positions.  Rows [n, n + n p) of the walk are the output's own rows, of which those
// behind the last kept slot are set to zero.
template <typename R>
__global__ void __launch_bounds__(256) rows_to_groups_kernel(const R* __restrict__ X,
                                                             const int32_t* __restrict__ position,
                                                             const int32_t* __restrict__ kept, int64_t n, int p,
                                                             int64_t nv, R* __restrict__ Y) {
  const int64_t slots = n * p;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  RowWalk w(first, step, nv);
  for (; w.row < n; w.next()) {
    const R v = load_once(X + w.row * nv + w.v);
    const int32_t* pos = position + w.row * p;
    for (int j = 0; j < p; ++j) {
      const int64_t r = pos[j];
      if (r >= 0 && r < slots) store_once(Y + r * nv + w.v, v);
    }
  }
  const int64_t filled = max(0, *kept);
  if (filled >= slots) return;
  RowWalk z(first, step, nv);
  for (; z.row + filled < slots; z.next()) store_once(Y + (z.row + filled) * nv + z.v, raw_zero<R>());
}

// ------------------------------------------------------------------ rows back
// One thread per vector of an output row, the p vectors it sums in order of j; slots that
// were dropped (position -1) add nothing.
template <typename T, int N, bool WEIGHTED>
__global__ void __launch_bounds__(256) rows_from_groups_kernel(const T* __restrict__ Z,
                                                               const int32_t* __restrict__ position,
                                                               const Acc<T>* __restrict__ weights, int64_t n, int p,
                                                               int64_t nv, T* __restrict__ out) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  const int64_t slots = n * p;
  const typename V::Raw* Zr = reinterpret_cast<const typename V::Raw*>(Z);
  RowWalk w(static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, static_cast<int64_t>(gridDim.x) * blockDim.x,
            nv);
  for (; w.row < n; w.next()) {
    A acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = A(0);
    const int32_t* pos = position + w.row * p;
    for (int j0 = 0; j0 < p; j0 += 4) {
      V z[4];
      A wt[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t r = j0 + u < p ? pos[j0 + u] : -1;
        const bool ok = r >= 0 && r < slots;
        z[u].raw = ok ? load_once(Zr + r * nv + w.v) : raw_zero<typename V::Raw>();
        wt[u] = ok ? (WEIGHTED ? weights[w.row * p + j0 + u] : A(1)) : A(0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += wt[u] * to_acc(z[u].e[e]);
    }
    V o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(acc[e]);
    store_once(reinterpret_cast<typename V::Raw*>(out) + w.row * nv + w.v, o.raw);
  }
}

// ------------------------------------------------------------------ the way back's gradient
// A team of 32 TEAM_WARPS threads per row: dOut[i] stays in L1 while the row's picks are
// walked; each thread keeps the partial products of up to 4 picks, summed over the team in
// a fixed order.
template <typename T, int N, int TEAM_WARPS>
__global__ void __launch_bounds__(256) rows_from_groups_grad_kernel(
    const T* __restrict__ G, const T* __restrict__ Z, const int32_t* __restrict__ position,
    const Acc<T>* __restrict__ weights, const int32_t* __restrict__ kept, int64_t n, int p, int64_t nv,
    T* __restrict__ gZ, Acc<T>* __restrict__ gW) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  constexpr int TEAMS = 8 / TEAM_WARPS;
  __shared__ A part[8][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = warp / TEAM_WARPS, in_team = threadIdx.x - team * TEAM_WARPS * 32;
  const int64_t slots = n * p;
  const Raw* Gr = reinterpret_cast<const Raw*>(G);
  const Raw* Zr = reinterpret_cast<const Raw*>(Z);
  Raw* gZr = reinterpret_cast<Raw*>(gZ);
  // every team of a block takes the same number of turns, for the block barriers below
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * TEAMS; i0 < n; i0 += static_cast<int64_t>(gridDim.x) * TEAMS) {
    const int64_t i = i0 + team;
    for (int j0 = 0; j0 < p; j0 += 4) {
      A dot[4] = {A(0), A(0), A(0), A(0)};
      if (i < n) {
        int64_t r[4];
        A wt[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          r[u] = j0 + u < p ? position[i * p + j0 + u] : -1;
          if (r[u] >= slots) r[u] = -1;
          wt[u] = r[u] >= 0 ? (weights ? weights[i * p + j0 + u] : A(1)) : A(0);
        }
        for (int64_t v = in_team; v < nv; v += TEAM_WARPS * 32) {
          V g, z[4];
          g.raw = load_keep(Gr + i * nv + v);
          if (gW) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              z[u].raw = r[u] >= 0 ? load_once(Zr + r[u] * nv + v) : raw_zero<Raw>();
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (r[u] >= 0) {
#pragma unroll
                for (int e = 0; e < N; ++e) dot[u] += to_acc(g.e[e]) * to_acc(z[u].e[e]);
              }
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (r[u] >= 0) {
              V o;
#pragma unroll
              for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(wt[u] * to_acc(g.e[e]));
              store_once(gZr + r[u] * nv + v, o.raw);
            }
        }
      }
      if (gW) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int s = 16; s > 0; s >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], s);
        if (TEAM_WARPS == 1) {
          if (lane == 0 && i < n)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (j0 + u < p) gW[i * p + j0 + u] = dot[u];
        } else {
          if (lane == 0)
#pragma unroll
            for (int u = 0; u < 4; ++u) part[warp][u] = dot[u];
          __syncthreads();
          if (in_team < 4 && i < n && j0 + in_team < p) {
            A s = A(0);
#pragma unroll
            for (int q = 0; q < TEAM_WARPS; ++q) s += part[team * TEAM_WARPS + q][in_team];
            gW[i * p + j0 + in_team] = s;
          }
          __syncthreads();
        }
      }
    }
  }
  const int64_t filled = max(0, *kept);
  if (filled >= slots) return;
  RowWalk z(static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, static_cast<int64_t>(gridDim.x) * blockDim.x,
            nv);
  for (; z.row + filled < slots; z.next()) store_once(gZr + (z.row + filled) * nv + z.v, raw_zero<Raw>());
}

// ------------------------------------------------------------------ launches
static unsigned grid_for(int64_t items, int per_block, int waves) {
  const int64_t most = static_cast<int64_t>(num_sms()) * waves;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((items + per_block - 1) / per_block, most)));
}

template <typename R>
static cudaError_t to_groups_t(const void* X, const int32_t* position, const int32_t* kept, int64_t n, int p,
                               int64_t row_bytes, void* Y, cudaStream_t st) {
  const int64_t nv = row_bytes / static_cast<int64_t>(sizeof(R));
  rows_to_groups_kernel<R><<<grid_for(n * nv, 256, 64), 256, 0, st>>>(static_cast<const R*>(X), position, kept, n, p,
                                                                      nv, static_cast<R*>(Y));
  return cudaGetLastError();
}

cudaError_t launch_rows_to_groups(int esize, const void* X, const int32_t* position, const int32_t* kept, int64_t n,
                                  int p, int64_t dim, void* Y, cudaStream_t st) {
  const int64_t rb = dim * esize;
  switch (row_vec_bytes(rb, reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(Y))) {
    case 16: return to_groups_t<uint4>(X, position, kept, n, p, rb, Y, st);
    case 8: return to_groups_t<uint2>(X, position, kept, n, p, rb, Y, st);
    case 4: return to_groups_t<uint32_t>(X, position, kept, n, p, rb, Y, st);
    default: return to_groups_t<unsigned short>(X, position, kept, n, p, rb, Y, st);
  }
}

template <typename T, int N>
static cudaError_t from_groups_n(const T* Z, const int32_t* position, const void* weights, int64_t n, int p,
                                 int64_t dim, T* out, cudaStream_t st) {
  const int64_t nv = dim / N;
  const unsigned g = grid_for(n * nv, 256, 64);
  const Acc<T>* w = static_cast<const Acc<T>*>(weights);
  if (w)
    rows_from_groups_kernel<T, N, true><<<g, 256, 0, st>>>(Z, position, w, n, p, nv, out);
  else
    rows_from_groups_kernel<T, N, false><<<g, 256, 0, st>>>(Z, position, w, n, p, nv, out);
  return cudaGetLastError();
}

template <typename T, int N>
static cudaError_t from_groups_grad_n(const T* G, const T* Z, const int32_t* position, const void* weights,
                                      const int32_t* kept, int64_t n, int p, int64_t dim, T* gZ, void* gW,
                                      cudaStream_t st) {
  const int64_t nv = dim / N;
  const Acc<T>* w = static_cast<const Acc<T>*>(weights);
  Acc<T>* gw = static_cast<Acc<T>*>(gW);
  if (nv <= 64)
    rows_from_groups_grad_kernel<T, N, 1>
        <<<grid_for(n, 8, 64), 256, 0, st>>>(G, Z, position, w, kept, n, p, nv, gZ, gw);
  else
    rows_from_groups_grad_kernel<T, N, 8>
        <<<grid_for(n, 1, 64), 256, 0, st>>>(G, Z, position, w, kept, n, p, nv, gZ, gw);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t from_groups_t(const void* Z, const int32_t* position, const void* weights, int64_t n, int p,
                                 int64_t dim, void* out, cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(Z) | reinterpret_cast<uintptr_t>(out));
  EUC_ROW_VEC(T, b, from_groups_n, static_cast<const T*>(Z), position, weights, n, p, dim, static_cast<T*>(out), st);
}

template <typename T>
static cudaError_t from_groups_grad_t(const void* G, const void* Z, const int32_t* position, const void* weights,
                                      const int32_t* kept, int64_t n, int p, int64_t dim, void* gZ, void* gW,
                                      cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(Z) | reinterpret_cast<uintptr_t>(G) |
                                  reinterpret_cast<uintptr_t>(gZ));
  EUC_ROW_VEC(T, b, from_groups_grad_n, static_cast<const T*>(G), static_cast<const T*>(Z), position, weights, kept, n,
              p, dim, static_cast<T*>(gZ), gW, st);
}

cudaError_t launch_rows_from_groups(RowType t, const void* Z, const int32_t* position, const void* weights, int64_t n,
                                    int p, int64_t dim, void* out, cudaStream_t st) {
  switch (t) {
    case ROW_F32: return from_groups_t<float>(Z, position, weights, n, p, dim, out, st);
    case ROW_F64: return from_groups_t<double>(Z, position, weights, n, p, dim, out, st);
    case ROW_F16: return from_groups_t<__half>(Z, position, weights, n, p, dim, out, st);
    default: return from_groups_t<__nv_bfloat16>(Z, position, weights, n, p, dim, out, st);
  }
}

cudaError_t launch_rows_from_groups_grad(RowType t, const void* G, const void* Z, const int32_t* position,
                                         const void* weights, const int32_t* kept, int64_t n, int p, int64_t dim,
                                         void* gZ, void* gW, cudaStream_t st) {
  switch (t) {
    case ROW_F32: return from_groups_grad_t<float>(G, Z, position, weights, kept, n, p, dim, gZ, gW, st);
    case ROW_F64: return from_groups_grad_t<double>(G, Z, position, weights, kept, n, p, dim, gZ, gW, st);
    case ROW_F16: return from_groups_grad_t<__half>(G, Z, position, weights, kept, n, p, dim, gZ, gW, st);
    default: return from_groups_grad_t<__nv_bfloat16>(G, Z, position, weights, kept, n, p, dim, gZ, gW, st);
  }
}

}  // namespace euc
