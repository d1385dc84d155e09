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
// The sort is a counting sort in passes of up to kMaxBins bins (one pass where shared memory
// holds k + 1 bins, else 2 or 3 by digits, least significant first); a slot is ranked among
// its warp's equal keys by ballots, 32 slots at a time in slot order, with 16-bit
// counters per warp and bin.  Up to kBlockSlots slots one block runs all passes, 64 slots in
// 2.8 us.  More take three kernels a pass (histograms of tiles, scan of each bin over the
// tiles, scatter through shared memory so that a bin's run is stored together): 131072 slots
// of 128 labels in 6.3 us (one cluster of 8 blocks took 54: eight SMs scatter no faster),
// 8192 of 256 in 6.8 (one block: 23).  One pass reads a slot's label twice and writes its three
// results, 20 to 28 bytes a slot, each further pass about as many again; the rows move kilobytes.
//
// The row kernels are bound by HBM, and read and write every row once: a row's copies are
// written from registers after one read, its weighted sum is formed from p reads (16384 rows
// of 2048 bf16, 8 picks: there 100 us at 6.0 TB/s, back 102 at 5.9, the way back's gradient
// 201 at 5.7).  Rows that are not whole 16-byte words go by the widest part that divides them
// (5003 rows of 1001 fp32, 3 picks, by 4 bytes: 15, 18 and 32 us, 4.3 to 5.2 TB/s).
#include "engine.h"
#include "rows.cuh"

#include <algorithm>

namespace euc {

// ------------------------------------------------------------------ the sort
// k + 1 bins (the last for labels outside [0, k)) that one pass may have: of a block, and of
// three kernels, what shared memory holds per warp and bin; of more than kManySlots slots,
// what their histograms cost (262144 of 2900 labels: 22 us in one pass, 27 in two; 1048576 of
// 4000: 94 in one, 50 in two).  Below kManySlots the limit weighs the device against the host's
// four launches more: 5000 to 60000 slots of 2100, 3100 and 4600 labels take 16 to 20, 18 to 25
// and 21 to 31 us in one pass and 17 to 19 in two as part of a captured graph, but 24 to 26, 24
// to 31 and 27 to 35 in one and 33 in two as calls of their own.
constexpr int kBlockBins = 2049;
constexpr int kMaxBins = 4609;
constexpr int kManyBins = 1537;
constexpr int64_t kManySlots = 1 << 18;
constexpr int kPassBits = 11;  // digits of a sort of several passes, at most

struct SortOut {
  uint32_t* keys;  // a pass that is not the last: keys and slots in the pass's order
  uint32_t* slots;
  int32_t* order;  // the last pass
  int32_t* position;
  int32_t* labels;
  int32_t* offsets;  // a sort of one pass, else null
};

template <typename TL> __device__ __forceinline__ uint32_t key_of(TL label, uint32_t k) {
  return label >= 0 && label < static_cast<TL>(k) ? static_cast<uint32_t>(label) : k;
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
  uint32_t run = x - sum;
  for (int w = 0; w < nw; ++w) run += w < warp ? warp_sums[w] : 0u;
  for (int c = lo; c < hi; ++c) {
    const uint32_t t = v[c];
    v[c] = run;
    run += t;
  }
  __syncthreads();
}

// rank[u] <- slots of the warp before (u, lane) with its digit; counts <- slots per digit.
// The lanes with a lane's digit come from a ballot per bit: match_any, whose lanes take turns,
// costs more from a few labels up (1048576 slots of 4, 64 and 1024: 12.6, 18.4 and 26.7 us with
// it, 13.9, 15.9 and 24.5 so).
template <int ITEMS>
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[ITEMS], unsigned short (&rank)[ITEMS],
                                           unsigned short* counts, int lane, int bits) {
  unsigned peers[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) peers[u] = __ballot_sync(0xffffffffu, digit[u] != 0xffffffffu);
  for (int b = 0; b < bits; ++b)
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const bool one = digit[u] >> b & 1u;
      const unsigned ones = __ballot_sync(0xffffffffu, one);
      peers[u] &= one ? ones : ~ones;
    }
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const bool in = digit[u] != 0xffffffffu;
    const int before = __popc(peers[u] & ((1u << lane) - 1u));
    unsigned short base = 0;
    if (in) base = counts[digit[u]];
    __syncwarp();
    if (in && before == 0) counts[digit[u]] = static_cast<unsigned short>(base + __popc(peers[u]));
    rank[u] = static_cast<unsigned short>(base + before);
    __syncwarp();
  }
}

// bits of the digits below `bins`
__device__ __forceinline__ int digit_bits(int bins) { return 32 - __clz(bins - 1); }

// ---- all passes in one block
struct BlockSort {
  int n;
  uint32_t k;
  int passes, bits, bins;
  uint32_t *keys[2], *slots[2];  // between passes
};

constexpr int64_t kBlockSlots = 1024;

template <typename TL>
__global__ void __launch_bounds__(1024) sort_block_kernel(const TL* __restrict__ in, BlockSort a, SortOut o) {
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t warp_sums[32];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* start = sm;  // [bins] first position of the digit
  unsigned short* cnt = reinterpret_cast<unsigned short*>(sm + a.bins);  // [warps][bins]
  unsigned short* mine = cnt + warp * a.bins;
  const int s = static_cast<int>(threadIdx.x);
  for (int pass = 0; pass < a.passes; ++pass) {
    const bool last = pass == a.passes - 1;
    const int shift = pass * a.bits;
    const uint32_t mask = a.passes == 1 ? 0xffffffffu : (1u << a.bits) - 1u;
    const uint32_t* from_keys = a.keys[(pass + 1) & 1];
    const uint32_t* from_slots = a.slots[(pass + 1) & 1];
    const uint32_t key = s >= a.n ? 0u : pass == 0 ? key_of(in[s], a.k) : __ldcg(from_keys + s);
    const uint32_t digit[1] = {s >= a.n ? 0xffffffffu : (key >> shift) & mask};
    unsigned short rank[1];
    for (int c = threadIdx.x; c < a.bins * warps; c += blockDim.x) cnt[c] = 0;
    __syncthreads();
    warp_ranks<1>(digit, rank, mine, lane, digit_bits(a.bins));
    __syncthreads();
    for (int c = threadIdx.x; c < a.bins; c += blockDim.x) {  // counts -> prefixes over the warps
      uint32_t run = 0;
      for (int w = 0; w < warps; ++w) {
        const unsigned short t = cnt[w * a.bins + c];
        cnt[w * a.bins + c] = static_cast<unsigned short>(run);
        run += t;
      }
      start[c] = run;
    }
    __syncthreads();
    block_scan(start, a.bins, warp_sums);
    if (last && o.offsets)
      for (int c = threadIdx.x; c < a.bins; c += blockDim.x) o.offsets[c] = static_cast<int32_t>(start[c]);
    if (s < a.n) {
      const uint32_t pos = start[digit[0]] + mine[digit[0]] + rank[0];
      const uint32_t slot = pass == 0 ? static_cast<uint32_t>(s) : __ldcg(from_slots + s);
      if (last) {
        const bool kept = key < a.k;
        o.order[pos] = kept ? static_cast<int32_t>(slot) : -1;
        o.labels[pos] = kept ? static_cast<int32_t>(key) : -1;
        o.position[slot] = kept ? static_cast<int32_t>(pos) : -1;
      } else {
        a.keys[pass & 1][pos] = key;
        a.slots[pass & 1][pos] = slot;
      }
    }
    __syncthreads();  // the next pass reads what this one wrote
  }
}

// ---- three kernels a pass
// A tile is WARPS x 32 x ITEMS slots (at most 4096: 16 bits index one of them), sorted by a
// block of WARPS warps.
struct SortPass {
  int64_t n;
  uint32_t k;  // keys lie in [0, k]; k marks a dropped slot
  int shift;
  uint32_t mask;
  int bins;
  int tiles;        // rounded up to whole 16 bytes of T
  uint32_t* T;      // [bins][tiles] counts, then exclusive prefixes over the tiles
  uint32_t* total;  // [bins]
};

template <typename TL, bool FIRST> __device__ __forceinline__ uint32_t load_key(const TL* in, int64_t s, uint32_t k) {
  if constexpr (FIRST) return key_of(in[s], k);
  else return static_cast<uint32_t>(__ldcg(in + s));
}

template <typename TL, bool FIRST, int WARPS, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32) sort_hist_kernel(const TL* __restrict__ in, SortPass a) {
  extern __shared__ uint32_t cnt[];
  let_next_start();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) cnt[c] = 0u;
  if (!FIRST) wait_for_previous();
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (WARPS * 32 * ITEMS) + threadIdx.x;
  uint32_t key[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t s = base + u * (WARPS * 32);
    key[u] = s < a.n ? load_key<TL, FIRST>(in, s, a.k) : 0u;
  }
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (base + u * (WARPS * 32) < a.n) atomicAdd(&cnt[(key[u] >> a.shift) & a.mask], 1u);
  __syncthreads();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) {
    uint32_t* row = a.T + static_cast<int64_t>(c) * a.tiles;
    row[blockIdx.x] = cnt[c];
    if (blockIdx.x == gridDim.x - 1)  // the padding
      for (int t = gridDim.x; t < a.tiles; ++t) row[t] = 0u;
  }
}

// one warp per bin: T[bin][.] becomes its exclusive prefix over the tiles, 512 tiles at a time
__global__ void __launch_bounds__(256) sort_tiles_kernel(SortPass a) {
  const int bin = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  let_next_start();
  wait_for_previous();
  if (bin >= a.bins) return;
  uint4* row = reinterpret_cast<uint4*>(a.T + static_cast<int64_t>(bin) * a.tiles);
  const int quads = a.tiles / 4;
  uint32_t run = 0u;
  for (int b0 = 0; b0 < quads; b0 += 128) {
    uint4 v[4];
    uint32_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int b = b0 + u * 32 + lane;
      v[u] = b < quads ? __ldcg(row + b) : make_uint4(0u, 0u, 0u, 0u);
      x[u] = v[u].x + v[u].y + v[u].z + v[u].w;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x[u], o);
        if (lane >= o) x[u] += y;
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int b = b0 + u * 32 + lane;
      uint4 w;
      w.x = run + x[u] - (v[u].x + v[u].y + v[u].z + v[u].w);
      w.y = w.x + v[u].x;
      w.z = w.y + v[u].y;
      w.w = w.z + v[u].z;
      if (b < quads) row[b] = w;
      run += __shfl_sync(0xffffffffu, x[u], 31);
    }
  }
  if (lane == 0) a.total[bin] = run;
}

template <typename TL, bool FIRST, bool LAST, int WARPS, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32) sort_scatter_kernel(const TL* __restrict__ in,
                                                                      const uint32_t* __restrict__ in_slots,
                                                                      SortPass a, SortOut o) {
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t warp_sums[WARPS];
  uint32_t* start = sm;                  // [bins] global position of the tile's first slot of the bin,
  uint32_t* local = sm + a.bins;         // [bins] less its position in the tile
  uint32_t* stage = sm + 2 * a.bins;     // [tile] digit and slot, in the tile's order
  unsigned short* cnt = reinterpret_cast<unsigned short*>(stage + (WARPS * 32 * ITEMS));  // [warps][bins]
  let_next_start();
  for (int c = threadIdx.x; c < a.bins * (WARPS / 2); c += blockDim.x) reinterpret_cast<uint32_t*>(cnt)[c] = 0u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned short* mine = cnt + warp * a.bins;
  const int64_t tile = static_cast<int64_t>(blockIdx.x) * (WARPS * 32 * ITEMS);
  const int first = warp * (32 * ITEMS) + lane;
  // the ranks within the tile need the labels alone (of a first pass: what came before the
  // sort), so they are formed while the histograms are still being summed
  if (!FIRST) wait_for_previous();
  uint32_t digit[ITEMS];
  unsigned short rank[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t s = tile + first + u * 32;
    digit[u] = s < a.n ? (load_key<TL, FIRST>(in, s, a.k) >> a.shift) & a.mask : 0xffffffffu;
  }
  __syncthreads();
  warp_ranks<ITEMS>(digit, rank, mine, lane, digit_bits(a.bins));
  __syncthreads();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) {  // counts -> prefixes over the warps
    uint32_t run = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const unsigned short t = cnt[w * a.bins + c];
      cnt[w * a.bins + c] = static_cast<unsigned short>(run);
      run += t;
    }
    local[c] = run;
  }
  __syncthreads();
  block_scan(local, a.bins, warp_sums);
  if (FIRST) wait_for_previous();
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x) start[c] = __ldcg(a.total + c);
  __syncthreads();
  block_scan(start, a.bins, warp_sums);
  if (LAST && o.offsets && blockIdx.x == 0)
    for (int c = threadIdx.x; c < a.bins; c += blockDim.x) o.offsets[c] = static_cast<int32_t>(start[c]);
  for (int c = threadIdx.x; c < a.bins; c += blockDim.x)  // (every thread its own bins, as above)
    start[c] += __ldcg(a.T + static_cast<int64_t>(c) * a.tiles + blockIdx.x) - local[c];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (digit[u] != 0xffffffffu) {
      const uint32_t l = local[digit[u]] + mine[digit[u]] + rank[u];
      stage[l] = (digit[u] << 16) | static_cast<uint32_t>(first + u * 32);
      // of a sort of one pass the digit is the key, and neighbouring lanes have neighbouring slots
      if (FIRST && LAST)
        o.position[tile + first + u * 32] = digit[u] < a.k ? static_cast<int32_t>(start[digit[u]] + l) : -1;
    }
  __syncthreads();
  const int here = static_cast<int>(min(static_cast<int64_t>((WARPS * 32 * ITEMS)), a.n - tile));
  for (int l = threadIdx.x; l < here; l += blockDim.x) {
    const uint32_t w = stage[l], d = w >> 16;
    const int64_t s = tile + (w & 0xffffu);
    const uint32_t pos = start[d] + l;
    const uint32_t key = FIRST && LAST ? d : load_key<TL, FIRST>(in, s, a.k);
    const uint32_t slot = FIRST ? static_cast<uint32_t>(s) : __ldcg(in_slots + s);
    if (LAST) {
      const bool kept = key < a.k;
      o.order[pos] = kept ? static_cast<int32_t>(slot) : -1;
      o.labels[pos] = kept ? static_cast<int32_t>(key) : -1;
      if (!FIRST) o.position[slot] = kept ? static_cast<int32_t>(pos) : -1;
    } else {
      o.keys[pos] = key;
      o.slots[pos] = slot;
    }
  }
}

// offsets of a sort of several passes: first position whose key is not below c, between two
// of kSamples evenly spaced positions, whose keys the block holds
constexpr int kSamples = 256;

__global__ void sort_offsets_kernel(const int32_t* __restrict__ labels, int64_t n, int k,
                                    int32_t* __restrict__ offsets) {
  __shared__ int32_t sample[kSamples];
  wait_for_previous();
  auto key = [&](int64_t at) {  // dropped slots (-1, at the end) count as k
    const int32_t l = __ldcg(labels + at);
    return l < 0 ? k : l;
  };
  const int64_t step = (n + kSamples - 1) / kSamples;
  for (int i = threadIdx.x; i < kSamples; i += blockDim.x) sample[i] = i * step < n ? key(i * step) : k;
  __syncthreads();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c > k) return;
  int below = 0;  // samples below c
  for (int half = kSamples / 2; half > 0; half /= 2)
    if (sample[below + half - 1] < c) below += half;
  below += sample[below] < c;
  int64_t lo = below > 0 ? (below - 1) * step + 1 : 0, hi = min(n, below * step);
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (key(mid) < c) lo = mid + 1; else hi = mid;
  }
  offsets[c] = static_cast<int32_t>(lo);
}

static inline size_t al(size_t b) { return (b + 255) & ~size_t(255); }

struct SortPlan {
  int passes, bits, bins, tiles;
  int warps, items;  // of a tile
  bool block;
};

// Tiles: small ones fill the SMs, and are cheap to begin while the bins are few; large ones
// leave fewer histograms to add up (131072 slots of 128 labels: 6.3, 7.5 and 9.5 us with
// 8 x 4, 16 x 4 and 16 x 8; 65536 of 1024: 13.3, 14.1, 19.2; 1048576 of 1024: 36, 32, 24.5).
// Where only 16 x 4 are at most one per SM, their kernels overlap (200000 of 128: 9.5, 7.5, 9.5).
constexpr int64_t kSmsOfB200 = 148;

static void set_tiles(SortPlan& p, int64_t n) {
  const bool many = n > (1 << 19), one_each = n > kSmsOfB200 * 1024 && n <= kSmsOfB200 * 2048;
  p.warps = !many && !one_each && p.bins <= 1025 ? 8 : 16;
  p.items = many ? 8 : 4;
  const int tile = p.warps * 32 * p.items;
  p.tiles = static_cast<int>(((n + tile - 1) / tile + 3) / 4 * 4);
}

static SortPlan sort_plan(int64_t n, int64_t k) {
  SortPlan p{};
  p.block = n <= kBlockSlots;
  if (k + 1 <= (p.block ? kBlockBins : n <= kManySlots ? kMaxBins : kManyBins)) {
    p.passes = 1;
    p.bins = static_cast<int>(k + 1);
    set_tiles(p, n);
    return p;
  }
  int bits = 1;
  while ((1ll << bits) <= k) ++bits;  // keys 0 .. k
  p.passes = (bits + kPassBits - 1) / kPassBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.bins = 1 << p.bits;
  set_tiles(p, n);
  return p;
}

size_t group_ws_bytes(int64_t n, int64_t k) {
  if (n <= 0) return 0;
  const SortPlan p = sort_plan(n, k);
  size_t b = 0;
  if (!p.block) b += al(static_cast<size_t>(p.bins) * p.tiles * 4) + al(static_cast<size_t>(p.bins) * 4);
  if (p.passes > 1) b += 2 * al(static_cast<size_t>(n) * 4);
  if (p.passes > 2) b += 2 * al(static_cast<size_t>(n) * 4);
  return b;
}

// dynamic shared memory beyond the 48 KiB that a launch may ask for unannounced, of which the
// kernels' static arrays take a little; always the most that the kernel takes, so that calls
// of different sizes from several threads do not lower one another's limit
static cudaError_t more_smem(const void* kernel, size_t bytes, int most) {
  if (bytes <= 47 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

template <typename TL>
static cudaError_t sort_block(const TL* in, const BlockSort& a, const SortOut& o, cudaStream_t st) {
  const int nt = (a.n + 31) / 32 * 32;
  const size_t smem = static_cast<size_t>(a.bins) * (4 + 2 * (nt / 32));
  constexpr int kMost = std::max(kBlockBins, 1 << kPassBits) * (4 + 2 * static_cast<int>(kBlockSlots / 32));
  const cudaError_t e = more_smem(reinterpret_cast<const void*>(sort_block_kernel<TL>), smem, kMost);
  if (e != cudaSuccess) return e;
  sort_block_kernel<TL><<<1, nt, smem, st>>>(in, a, o);
  return cudaGetLastError();
}

template <typename TL, bool FIRST, bool LAST, int WARPS, int ITEMS>
static cudaError_t sort_pass_t(const TL* in, const uint32_t* in_slots, const SortPass& a, const SortOut& o,
                               cudaStream_t st) {
  constexpr int TILE = WARPS * 32 * ITEMS;
  constexpr int kMost = std::max(kMaxBins, 1 << kPassBits) * (8 + 2 * WARPS) + TILE * 4;
  const auto hist = sort_hist_kernel<TL, FIRST, WARPS, ITEMS>;
  const auto scatter = sort_scatter_kernel<TL, FIRST, LAST, WARPS, ITEMS>;
  const size_t sm = static_cast<size_t>(a.bins) * (8 + 2 * WARPS) + TILE * 4;
  cudaError_t e = more_smem(reinterpret_cast<const void*>(scatter), sm, kMost);
  if (e != cudaSuccess) return e;
  const unsigned tiles = static_cast<unsigned>((a.n + TILE - 1) / TILE);
  // Each kernel may start while the one before it runs, if all their blocks fit beside one
  // another with little shared memory and few counts to pass on: 131072 slots of 128 labels
  // took 8.1 us so (in tiles of 2048) and 11.4 one after another, 16384 of 700 8.8 and 11.3,
  // but 30011 of 1000 23 and 14; in two passes, 40000 of 131072 23.1 and 26.0, but 131072 of
  // 131072 34 and 28.
  const int64_t counts = static_cast<int64_t>(a.bins) * tiles;
  const bool fits = FIRST && LAST ? a.bins <= 512 || (a.bins <= 1025 && counts <= 21000)
                                  : a.bins <= 512 && tiles <= 64;
  const bool early = fits && static_cast<int>(tiles) <= num_sms();
  e = launch_after(!FIRST && early, hist, tiles, WARPS * 32, static_cast<size_t>(a.bins) * 4, st, in, a);
  if (e == cudaSuccess)
    e = launch_after(early, sort_tiles_kernel, static_cast<unsigned>((a.bins + 7) / 8), 256, 0, st, a);
  if (e == cudaSuccess) e = launch_after(early, scatter, tiles, WARPS * 32, sm, st, in, in_slots, a, o);
  return e;
}

template <typename TL, bool FIRST, bool LAST>
static cudaError_t sort_pass(const SortPlan& p, const TL* in, const uint32_t* in_slots, const SortPass& a,
                             const SortOut& o, cudaStream_t st) {
  if (p.items == 8) return sort_pass_t<TL, FIRST, LAST, 16, 8>(in, in_slots, a, o, st);
  if (p.warps == 8) return sort_pass_t<TL, FIRST, LAST, 8, 4>(in, in_slots, a, o, st);
  return sort_pass_t<TL, FIRST, LAST, 16, 4>(in, in_slots, a, o, st);
}

template <typename TL>
static cudaError_t group_t(const TL* labels, int64_t n, int64_t k, int32_t* offsets, int32_t* order, int32_t* position,
                           int32_t* sorted, uint8_t* ws, cudaStream_t st) {
  const SortPlan p = sort_plan(n, k);
  SortOut o{};
  o.order = order;
  o.position = position;
  o.labels = sorted;
  o.offsets = p.passes == 1 ? offsets : nullptr;
  uint32_t* buf[4] = {nullptr, nullptr, nullptr, nullptr};
  for (int i = 0; i < 2 * std::min(p.passes - 1, 2); ++i) {
    buf[i] = reinterpret_cast<uint32_t*>(ws);
    ws += al(static_cast<size_t>(n) * 4);
  }
  cudaError_t e = cudaSuccess;
  if (p.block) {
    BlockSort a{};
    a.n = static_cast<int>(n);
    a.k = static_cast<uint32_t>(k);
    a.passes = p.passes;
    a.bits = p.bits;
    a.bins = p.bins;
    for (int i = 0; i < 2; ++i) {
      a.keys[i] = buf[2 * i];
      a.slots[i] = buf[2 * i + 1];
    }
    e = sort_block(labels, a, o, st);
  } else {
    SortPass a{};
    a.n = n;
    a.k = static_cast<uint32_t>(k);
    a.bins = p.bins;
    a.tiles = p.tiles;
    a.T = reinterpret_cast<uint32_t*>(ws);
    a.total = reinterpret_cast<uint32_t*>(ws + al(static_cast<size_t>(p.bins) * p.tiles * 4));
    if (p.passes == 1) {
      a.mask = 0xffffffffu;
      return sort_pass<TL, true, true>(p, labels, nullptr, a, o, st);
    }
    a.mask = static_cast<uint32_t>(p.bins - 1);
    o.keys = buf[0];
    o.slots = buf[1];
    e = sort_pass<TL, true, false>(p, labels, nullptr, a, o, st);
    const uint32_t *keys = buf[0], *slots = buf[1];
    if (e == cudaSuccess && p.passes == 3) {
      a.shift = p.bits;
      o.keys = buf[2];
      o.slots = buf[3];
      e = sort_pass<uint32_t, false, false>(p, keys, slots, a, o, st);
      keys = buf[2];
      slots = buf[3];
    }
    a.shift = p.bits * (p.passes - 1);
    if (e == cudaSuccess) e = sort_pass<uint32_t, false, true>(p, keys, slots, a, o, st);
  }
  if (e == cudaSuccess && p.passes > 1)
    e = launch_after(true, sort_offsets_kernel, static_cast<unsigned>((k + 1 + 255) / 256), 256, 0, st, sorted, n,
                     static_cast<int>(k), offsets);
  return e;
}

cudaError_t launch_group_rows(const void* labels, bool labels_i64, int64_t n, int64_t k, int32_t* offsets,
                              int32_t* order, int32_t* position, int32_t* sorted, void* ws, cudaStream_t st) {
  if (n == 0) return cudaMemsetAsync(offsets, 0, static_cast<size_t>(k + 1) * 4, st);
  uint8_t* w = static_cast<uint8_t*>(ws);
  if (labels_i64) return group_t(static_cast<const long long*>(labels), n, k, offsets, order, position, sorted, w, st);
  return group_t(static_cast<const int*>(labels), n, k, offsets, order, position, sorted, w, st);
}

// ------------------------------------------------------------------ rows there
// A vector of a row is read once and stored at each of the row's kept positions.  The output's
// rows behind the last kept slot are set to zero by the grid's last blocks.
template <typename R>
__device__ __forceinline__ void zero_rows(R* Y, int64_t filled, int64_t slots, int64_t nv, int64_t block, int64_t blocks) {
  const int64_t first = max(static_cast<int64_t>(0), min(filled, slots)) * nv, end = slots * nv;
  for (int64_t f = first + block * blockDim.x + threadIdx.x; f < end; f += blocks * blockDim.x)
    store_once(Y + f, raw_zero<R>());
}

template <typename R, int U, bool WIDE>
__global__ void __launch_bounds__(256) rows_to_groups_kernel(const R* __restrict__ X,
                                                             const int32_t* __restrict__ position,
                                                             const int32_t* __restrict__ kept, int64_t n, int p,
                                                             int64_t nv, int64_t chunks, int64_t copy_blocks,
                                                             R* __restrict__ Y) {
  const int64_t slots = n * p;
  if (static_cast<int64_t>(blockIdx.x) >= copy_blocks) {
    zero_rows(Y, *kept, slots, nv, blockIdx.x - copy_blocks, gridDim.x - copy_blocks);
    return;
  }
  R x[U];
  if constexpr (WIDE) {
    const WideRows<1, U> w(chunks);
    if (w.row >= n) return;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (w.v + 32 * u < nv) x[u] = load_once(X + w.row * nv + w.v + 32 * u);
    for (int j = 0; j < p; ++j) {
      const int64_t r = __ldg(position + w.row * p + j);
      if (r < 0 || r >= slots) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (w.v + 32 * u < nv) store_once(Y + r * nv + w.v + 32 * u, x[u]);
    }
  } else {
    const NarrowRows<U> w(nv);
    int64_t row[U];
    uint32_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w.at(u, row[u], v[u]);
      if (row[u] < n) x[u] = load_once(X + row[u] * nv + v[u]);
    }
    for (int j = 0; j < p; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = row[u] < n ? __ldg(position + row[u] * p + j) : -1;
        if (r >= 0 && r < slots) store_once(Y + r * nv + v[u], x[u]);
      }
  }
}

// ------------------------------------------------------------------ rows back
// A vector of an output row is the sum, in order of j, of the row's p vectors, J of them in
// flight for each of the lane's U output vectors; slots that were dropped (position -1) add
// nothing.
template <typename T, int N, int J, int U, bool WEIGHTED, bool WIDE>
__global__ void __launch_bounds__(256) rows_from_groups_kernel(const T* __restrict__ Z,
                                                               const int32_t* __restrict__ position,
                                                               const Acc<T>* __restrict__ weights, int64_t n, int p,
                                                               int64_t nv, int64_t chunks, T* __restrict__ out) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  static_assert(WIDE || U == 1, "a narrow row's vector has a row of its own");
  const Raw* Zr = reinterpret_cast<const Raw*>(Z);
  const int64_t slots = n * p;
  int64_t row, v;
  if constexpr (WIDE) {
    const WideRows<1, U> w(chunks);
    row = w.row;
    v = w.v;
  } else {
    uint32_t at;
    NarrowRows<1>(nv).at(0, row, at);
    v = at;
  }
  if (row >= n) return;
  const int32_t* pos = position + row * p;
  const A* wts = WEIGHTED ? weights + row * p : nullptr;
  A acc[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) acc[u][e] = A(0);
  for (int j0 = 0; j0 < p; j0 += J) {
    V z[J][U];
    A wt[J];
    bool ok[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t r = j0 + j < p ? __ldg(pos + j0 + j) : -1;
      ok[j] = r >= 0 && r < slots;
      wt[j] = WEIGHTED && j0 + j < p ? __ldg(wts + j0 + j) : A(1);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        z[j][u].raw = raw_zero<Raw>();
        if (ok[j] && v + 32 * u < nv) z[j][u].raw = load_once(Zr + r * nv + v + 32 * u);
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {  // (the weight is first looked at here, behind the rows' loads)
      const A w = ok[j] ? wt[j] : A(0);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[u][e] += w * to_acc(z[j][u].e[e]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (v + 32 * u >= nv) continue;
    V o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(acc[u][e]);
    store_once(reinterpret_cast<Raw*>(out) + row * nv + v + 32 * u, o.raw);
  }
}

// 16-bit rows of odd length: a thread takes the elements between two 16-byte boundaries of the
// output row, shifted out of the two aligned words of each of the row's vectors that hold them
// (12595 rows of 333 bf16, 8 picks: 28 us element by element, 22 so; 65536 of 33, 4 picks:
// 26 and 12; of 17 the same.  The way there, which would read a row once per pick, took 21
// us element by element and 34 so).
template <typename T, int J, bool WEIGHTED>
__global__ void __launch_bounds__(256) rows_from_groups_any_kernel(const T* __restrict__ Z,
                                                                   const int32_t* __restrict__ position,
                                                                   const float* __restrict__ weights, int64_t n,
                                                                   int p, int dim, int64_t nv, T* __restrict__ out) {
  const int64_t slots = n * p;
  int64_t row;
  uint32_t v;
  NarrowRows<1>(nv).at(0, row, v);
  if (row >= n) return;
  T* to = out + row * dim;
  const int at = static_cast<int>(v) * 8 - static_cast<int>((reinterpret_cast<uintptr_t>(to) & 15u) / 2);
  if (at >= dim) return;
  const int32_t* pos = position + row * p;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (int j0 = 0; j0 < p; j0 += J) {
    Words16 z[J];
    float wt[J];
    bool ok[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t r = j0 + j < p ? __ldg(pos + j0 + j) : -1;
      ok[j] = r >= 0 && r < slots;
      wt[j] = WEIGHTED && j0 + j < p ? __ldg(weights + row * p + j0 + j) : 1.f;
      z[j].clear();
      if (ok[j]) z[j].load(Z + r * dim + at, -at, dim - at, Z, Z + slots * dim);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float w = ok[j] ? wt[j] : 0.f;
      Vec<T, 8> x;
      x.raw = z[j].get();
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += w * to_acc(x.e[e]);
    }
  }
  Vec<T, 8> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o.e[e] = from_acc<T>(acc[e]);
  store_16(to + at, o, -at, dim - at);
}

// ------------------------------------------------------------------ the way back's gradient
// A team of 8, 32 or 256 threads per row, J picks at a time: dOut[i] is read once for all of
// them (and again, from L1, for the next J), each thread keeps its partial products of the J
// picks, and they are summed over the team in a fixed order.
template <int TEAM, typename A, int J> __device__ __forceinline__ void team_dots(A (&dot)[J], int lane) {
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int s = (TEAM < 32 ? TEAM : 32) / 2; s > 0; s >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], s);
}

template <typename T, int N, int TEAM, int J>
__global__ void __launch_bounds__(256) rows_from_groups_grad_kernel(
    const T* __restrict__ G, const T* __restrict__ Z, const int32_t* __restrict__ position,
    const Acc<T>* __restrict__ weights, const int32_t* __restrict__ kept, int64_t n, int p, int64_t nv,
    T* __restrict__ gZ, Acc<T>* __restrict__ gW) {
  using A = Acc<T>;
  using V = Vec<T, N>;
  using Raw = typename V::Raw;
  constexpr int TEAMS = 256 / TEAM;
  constexpr int BYTES = N * static_cast<int>(sizeof(T));
  constexpr int UV = BYTES >= 16 ? (J > 2 ? 1 : 2) : BYTES == 8 ? 2 : 4;  // vectors in flight, with each pick's
  __shared__ A part[8][J];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = static_cast<int>(threadIdx.x) / TEAM, in_team = static_cast<int>(threadIdx.x) % TEAM;
  const int64_t slots = n * p;
  const Raw* Gr = reinterpret_cast<const Raw*>(G);
  const Raw* Zr = reinterpret_cast<const Raw*>(Z);
  Raw* gZr = reinterpret_cast<Raw*>(gZ);
  // every team of a block takes the same number of turns, for the barriers below
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * TEAMS; i0 < n; i0 += static_cast<int64_t>(gridDim.x) * TEAMS) {
    const int64_t i = i0 + team;
    for (int j0 = 0; j0 < p; j0 += J) {
      A dot[J];
      int64_t r[J];
      A wt[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        dot[j] = A(0);
        r[j] = i < n && j0 + j < p ? __ldg(position + i * p + j0 + j) : -1;
        if (r[j] >= slots) r[j] = -1;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) wt[j] = weights && i < n && j0 + j < p ? __ldg(weights + i * p + j0 + j) : A(1);
      for (int64_t v0 = in_team; v0 < nv && i < n; v0 += UV * TEAM) {
        V g[UV], z[UV][J];
#pragma unroll
        for (int q = 0; q < UV; ++q) {
          const int64_t v = v0 + q * TEAM;
          g[q].raw = raw_zero<Raw>();
          if (v < nv) g[q].raw = load_keep(Gr + i * nv + v);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            z[q][j].raw = raw_zero<Raw>();
            if (gW && r[j] >= 0 && v < nv) z[q][j].raw = load_once(Zr + r[j] * nv + v);
          }
        }
#pragma unroll
        for (int q = 0; q < UV; ++q) {
          const int64_t v = v0 + q * TEAM;
          if (v >= nv) continue;
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (gW && r[j] >= 0) {
#pragma unroll
              for (int e = 0; e < N; ++e) dot[j] += to_acc(g[q].e[e]) * to_acc(z[q][j].e[e]);
            }
          if (gZ)
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (r[j] >= 0) {
              V o;
#pragma unroll
              for (int e = 0; e < N; ++e) o.e[e] = from_acc<T>(wt[j] * to_acc(g[q].e[e]));
              store_once(gZr + r[j] * nv + v, o.raw);
            }
        }
      }
      if (gW) {
        team_dots<TEAM>(dot, lane);
        if (TEAM <= 32) {
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (in_team == j % TEAM && i < n && j0 + j < p) gW[i * p + j0 + j] = dot[j];
        } else {
          if (lane == 0)
#pragma unroll
            for (int j = 0; j < J; ++j) part[warp][j] = dot[j];
          __syncthreads();
          if (in_team < J && i < n && j0 + in_team < p) {
            A s = A(0);
#pragma unroll
            for (int w = 0; w < 8; ++w) s += part[w][in_team];
            gW[i * p + j0 + in_team] = s;
          }
          __syncthreads();
        }
      }
    }
  }
  if (gZ) zero_rows(gZr, *kept, slots, nv, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------ launches
// Blocks that clear the rows behind the last kept slot (how many there are is known on the
// device alone): enough to write at HBM's rate, and gone at once where there are none.
static int64_t clear_blocks(int64_t vectors) {
  return std::min<int64_t>((vectors + 255) / 256, static_cast<int64_t>(num_sms()) * 4);
}

template <typename R, int U>
static cudaError_t to_groups_u(const R* X, const int32_t* position, const int32_t* kept, int64_t n, int p, int64_t nv,
                               R* Y, cudaStream_t st) {
  const bool wide = nv >= 32;
  const int64_t chunks = (nv + 32 * U - 1) / (32 * U);
  const int64_t copy = wide ? wide_blocks(n, nv, 1, U) : narrow_blocks(n, nv, U);
  const unsigned g = static_cast<unsigned>(copy + clear_blocks(n * p * nv));
  if (wide)
    rows_to_groups_kernel<R, U, true><<<g, 256, 0, st>>>(X, position, kept, n, p, nv, chunks, copy, Y);
  else
    rows_to_groups_kernel<R, U, false><<<g, 256, 0, st>>>(X, position, kept, n, p, nv, chunks, copy, Y);
  return cudaGetLastError();
}

// Four vectors a lane in flight, eight narrow ones; fewer where the row has no more.
template <typename R>
static cudaError_t to_groups_t(const void* X, const int32_t* position, const int32_t* kept, int64_t n, int p,
                               int64_t row_bytes, void* Y, cudaStream_t st) {
  const int64_t nv = row_bytes / static_cast<int64_t>(sizeof(R));
  const R* x = static_cast<const R*>(X);
  R* y = static_cast<R*>(Y);
  if (nv >= 32 && nv <= 64) return to_groups_u<R, 2>(x, position, kept, n, p, nv, y, st);
  if (sizeof(R) >= 8 || nv < 256) return to_groups_u<R, 4>(x, position, kept, n, p, nv, y, st);
  return to_groups_u<R, 8>(x, position, kept, n, p, nv, y, st);
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

template <typename T, int N, int J, bool WEIGHTED>
static cudaError_t from_groups_j(const T* Z, const int32_t* position, const Acc<T>* w, int64_t n, int p, int64_t nv,
                                 T* out, cudaStream_t st) {
  constexpr int U = N * sizeof(T) >= 8 ? 2 : 4;
  if (nv >= 32)
    rows_from_groups_kernel<T, N, J, U, WEIGHTED, true><<<static_cast<unsigned>(wide_blocks(n, nv, 1, U)), 256, 0, st>>>(
        Z, position, w, n, p, nv, (nv + 32 * U - 1) / (32 * U), out);
  else
    rows_from_groups_kernel<T, N, J, 1, WEIGHTED, false><<<static_cast<unsigned>(narrow_blocks(n, nv, 1)), 256, 0, st>>>(
        Z, position, w, n, p, nv, 1, out);
  return cudaGetLastError();
}

template <typename T, int N, bool WEIGHTED>
static cudaError_t from_groups_w(const T* Z, const int32_t* position, const Acc<T>* w, int64_t n, int p, int64_t nv,
                                 T* out, cudaStream_t st) {
  if (p <= 2) return from_groups_j<T, N, 2, WEIGHTED>(Z, position, w, n, p, nv, out, st);
  if (p <= 4) return from_groups_j<T, N, 4, WEIGHTED>(Z, position, w, n, p, nv, out, st);
  return from_groups_j<T, N, 8, WEIGHTED>(Z, position, w, n, p, nv, out, st);
}

template <typename T, int N>
static cudaError_t from_groups_n(const T* Z, const int32_t* position, const void* weights, int64_t n, int p,
                                 int64_t dim, T* out, cudaStream_t st) {
  const Acc<T>* w = static_cast<const Acc<T>*>(weights);
  return w ? from_groups_w<T, N, true>(Z, position, w, n, p, dim / N, out, st)
           : from_groups_w<T, N, false>(Z, position, w, n, p, dim / N, out, st);
}

template <typename T, int N, int TEAM>
static cudaError_t from_groups_grad_team(const T* G, const T* Z, const int32_t* position, const void* weights,
                                         const int32_t* kept, int64_t n, int p, int64_t nv, T* gZ, void* gW,
                                         cudaStream_t st) {
  const Acc<T>* w = static_cast<const Acc<T>*>(weights);
  Acc<T>* gw = static_cast<Acc<T>*>(gW);
  const unsigned g = static_cast<unsigned>(
      std::min<int64_t>((n * TEAM + 255) / 256, static_cast<int64_t>(num_sms()) * 64));
  if (p == 1)
    rows_from_groups_grad_kernel<T, N, TEAM, 1><<<g, 256, 0, st>>>(G, Z, position, w, kept, n, p, nv, gZ, gw);
  else if (p == 2)
    rows_from_groups_grad_kernel<T, N, TEAM, 2><<<g, 256, 0, st>>>(G, Z, position, w, kept, n, p, nv, gZ, gw);
  else
    rows_from_groups_grad_kernel<T, N, TEAM, 4><<<g, 256, 0, st>>>(G, Z, position, w, kept, n, p, nv, gZ, gw);
  return cudaGetLastError();
}

template <typename T, int N>
static cudaError_t from_groups_grad_n(const T* G, const T* Z, const int32_t* position, const void* weights,
                                      const int32_t* kept, int64_t n, int p, int64_t dim, T* gZ, void* gW,
                                      cudaStream_t st) {
  const int64_t nv = dim / N;
  // as many threads per row as it has vectors to give them; blocks of 256 where there are few rows
  if (nv <= 16) return from_groups_grad_team<T, N, 8>(G, Z, position, weights, kept, n, p, nv, gZ, gW, st);
  if (nv <= 64 || (nv <= 384 && n >= static_cast<int64_t>(num_sms()) * 32))
    return from_groups_grad_team<T, N, 32>(G, Z, position, weights, kept, n, p, nv, gZ, gW, st);
  return from_groups_grad_team<T, N, 256>(G, Z, position, weights, kept, n, p, nv, gZ, gW, st);
}

template <typename T, int J>
static cudaError_t from_groups_any(const T* Z, const int32_t* position, const float* w, int64_t n, int p, int64_t dim,
                                   T* out, cudaStream_t st) {
  const int64_t nv = (dim + 14) / 8;  // vectors that cover a row at any alignment
  const unsigned g = static_cast<unsigned>(narrow_blocks(n, nv, 1));
  if (w)
    rows_from_groups_any_kernel<T, J, true><<<g, 256, 0, st>>>(Z, position, w, n, p, static_cast<int>(dim), nv, out);
  else
    rows_from_groups_any_kernel<T, J, false><<<g, 256, 0, st>>>(Z, position, w, n, p, static_cast<int>(dim), nv, out);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t from_groups_t(const void* Z, const int32_t* position, const void* weights, int64_t n, int p,
                                 int64_t dim, void* out, cudaStream_t st) {
  const int b = row_vec_bytes(dim * static_cast<int64_t>(sizeof(T)),
                              reinterpret_cast<uintptr_t>(Z) | reinterpret_cast<uintptr_t>(out));
  if constexpr (sizeof(T) == 2)
    // (with fewer threads, latency counts: 1024 rows of 333, 4 picks, 2.6 us by elements and 3.0
    // so, 4096 rows 5.7 and 5.2)
    if (b == 2 && dim >= 32 && n * ((dim + 14) / 8) >= static_cast<int64_t>(num_sms()) * 384) {
      const T* z = static_cast<const T*>(Z);
      const float* w = static_cast<const float*>(weights);
      return p <= 2 ? from_groups_any<T, 2>(z, position, w, n, p, dim, static_cast<T*>(out), st)
                    : from_groups_any<T, 4>(z, position, w, n, p, dim, static_cast<T*>(out), st);
    }
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
