// Rows of any element type as vectors of up to 16 bytes, for the kernels that move and
// sum whole rows (k_groups.cu, k_codebook.cu) and read rows of scores (k_scores.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace euc {

// sums and weights: 32 bits for every type of 32 bits or fewer, 64 for fp64
template <typename T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
template <typename T> using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }

// one rounding, to nearest even
template <typename T> __device__ __forceinline__ T from_acc(Acc<T> v);
template <> __device__ __forceinline__ float from_acc<float>(float v) { return v; }
template <> __device__ __forceinline__ double from_acc<double>(double v) { return v; }
template <> __device__ __forceinline__ __half from_acc<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = unsigned short; };

// N elements of T in one machine word of N * sizeof(T) bytes
template <typename T, int N> struct Vec {
  using Raw = typename RawOf<N * static_cast<int>(sizeof(T))>::type;
  union {
    Raw raw;
    T e[N];
  };
  __device__ __forceinline__ Vec() {}
};

template <typename R> __device__ __forceinline__ R load_keep(const R* p) { return __ldg(p); }
// read once: the line is not kept ahead of data that is read again
template <typename R> __device__ __forceinline__ R load_once(const R* p) { return __ldcs(p); }
template <typename R> __device__ __forceinline__ void store_once(R* p, R v) { __stcs(p, v); }
template <typename R> __device__ __forceinline__ R raw_zero();
template <> __device__ __forceinline__ uint4 raw_zero<uint4>() { return make_uint4(0u, 0u, 0u, 0u); }
template <> __device__ __forceinline__ uint2 raw_zero<uint2>() { return make_uint2(0u, 0u); }
template <> __device__ __forceinline__ uint32_t raw_zero<uint32_t>() { return 0u; }
template <> __device__ __forceinline__ unsigned short raw_zero<unsigned short>() { return 0; }

template <int BYTES> struct BitsOf;
template <> struct BitsOf<2> { using type = unsigned short; };
template <> struct BitsOf<4> { using type = uint32_t; };
template <> struct BitsOf<8> { using type = unsigned long long; };

// the 16 bytes that begin `shift` (even, below 16) bytes behind the start of (a, b)
__device__ __forceinline__ uint4 shift_16(const uint4& a, const uint4& b, unsigned shift) {
  const unsigned bits = (shift & 3u) * 8u;
  auto pick = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4) {
    return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                      __funnelshift_r(w3, w4, bits));
  };
  switch (shift >> 2) {  // the same for all vectors of a row
    case 0: return pick(a.x, a.y, a.z, a.w, b.x);
    case 1: return pick(a.y, a.z, a.w, b.x, b.y);
    case 2: return pick(a.z, a.w, b.x, b.y, b.z);
    default: return pick(a.w, b.x, b.y, b.z, b.w);
  }
}

// The 16 bytes at any address that T's alignment allows, from the two aligned 16-byte words
// that hold them (neighbouring lanes share them, so the second comes from L1); element by
// element where one of the words is not inside [begin, end).
template <typename T>
__device__ __forceinline__ uint4 load_any_16(const T* p, const void* begin, const void* end) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), shift = at & 15u;
  const uint4* w = reinterpret_cast<const uint4*>(at - shift);
  if (shift == 0) return load_keep(w);
  if (static_cast<const void*>(w) < begin || static_cast<const void*>(w + 2) > end) {
    using Bits = typename BitsOf<sizeof(T)>::type;
    union {
      uint4 raw;
      Bits e[16 / sizeof(T)];
    } v;
#pragma unroll
    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) v.e[e] = reinterpret_cast<const Bits*>(p)[e];
    return v.raw;
  }
  return shift_16(load_keep(w), load_keep(w + 1), static_cast<unsigned>(shift));
}

// The same for elements [first, last) of the 8 at `from` (16-bit ones, those around them not
// looked at), as the two words and the shift, so that several such loads are in flight at once.
struct Words16 {
  uint4 lo, hi;
  unsigned shift;
  __device__ __forceinline__ void clear() {
    lo = hi = make_uint4(0u, 0u, 0u, 0u);
    shift = 0u;
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* from, int first, int last, const void* begin, const void* end) {
    static_assert(sizeof(T) == 2, "16-bit elements");
    shift = static_cast<unsigned>(reinterpret_cast<uintptr_t>(from) & 15u);
    const uint4* w = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(from) - shift);
    if (static_cast<const void*>(w) >= begin && static_cast<const void*>(w + 2) <= end) {
      lo = load_keep(w);
      hi = load_keep(w + 1);
      return;
    }
    Vec<T, 8> x;  // at the buffer's ends: element by element
    x.raw = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= first && e < last) x.e[e] = from[e];
    lo = x.raw;
    hi = make_uint4(0u, 0u, 0u, 0u);
    shift = 0u;
  }
  __device__ __forceinline__ uint4 get() const { return shift_16(lo, hi, shift); }
};

// 8 16-bit elements to a 16-byte boundary, but for those outside [first, last)
template <typename T> __device__ __forceinline__ void store_16(T* to, const Vec<T, 8>& x, int first, int last) {
  if (first <= 0 && last >= 8) {
    store_once(reinterpret_cast<uint4*>(to), x.raw);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e >= first && e < last) to[e] = x.e[e];
}

// Bytes of the widest vector that every row of `row_bytes` starts and ends on, given the
// OR of the buffers' addresses: 16, 8, 4 or 2 (elements are of 2 bytes at least).
inline int row_vec_bytes(int64_t row_bytes, uintptr_t addresses) {
  const uintptr_t a = addresses | static_cast<uintptr_t>(row_bytes);
  return (a & 15u) == 0 ? 16 : (a & 7u) == 0 ? 8 : (a & 3u) == 0 ? 4 : 2;
}

// Programmatic dependent launch: a kernel launched with `early` may start while the one before
// it on the stream still runs; what it does before wait_for_previous() reads nothing
// that kernel writes and writes nothing that it touches, and what that kernel writes is read
// behind it through L2 (ld.cg), past lines that an SM may hold from before.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... Q>
inline cudaError_t launch_after(bool early, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                                Q... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// How the row kernels cut rows of nv vectors into work (kUnit threads' worth a block).
//
// Wide rows (nv >= 32): a warp takes R neighbouring rows times a chunk of 32 U vectors, so a
// row's number and what goes with it (label, position) are the warp's own, and R U vectors a
// lane are in flight.  Narrow rows: a block takes 256 U consecutive vectors of the matrix,
// each thread those at a stride of 256, and finds every vector's row by a 32-bit division.
// Either way neighbouring lanes hold neighbouring vectors.
template <int R, int U> struct WideRows {
  int64_t row;  // the first of the warp's R rows
  int64_t v;    // this lane's first vector; the u-th is v + 32 u
  __device__ __forceinline__ WideRows(int64_t chunks) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    int64_t group;
    if (unit < 0x80000000ll && chunks < 0x80000000ll) {
      group = static_cast<uint32_t>(unit) / static_cast<uint32_t>(chunks);
    } else {
      group = unit / chunks;
    }
    row = group * R;
    v = (unit - group * chunks) * (32 * U) + (threadIdx.x & 31);
  }
};
template <int U> struct NarrowRows {
  int64_t row0;
  uint32_t rest, nv;
  __device__ __forceinline__ NarrowRows(int64_t nv_) : nv(static_cast<uint32_t>(nv_)) {
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 * U);
    row0 = first < 0x80000000ll ? static_cast<int64_t>(static_cast<uint32_t>(first) / nv) : first / nv_;
    rest = static_cast<uint32_t>(first - row0 * nv_) + threadIdx.x;
  }
  // row and vector of this thread's u-th
  __device__ __forceinline__ void at(int u, int64_t& row, uint32_t& v) const {
    const uint32_t f = rest + 256u * u, q = f / nv;
    row = row0 + q;
    v = f - q * nv;
  }
};

// blocks of 256 threads for `rows` rows of nv vectors
inline int64_t wide_blocks(int64_t rows, int64_t nv, int R, int U) {
  const int64_t chunks = (nv + 32 * U - 1) / (32 * U);
  return ((rows + R - 1) / R * chunks + 7) / 8;
}
inline int64_t narrow_blocks(int64_t rows, int64_t nv, int U) { return (rows * nv + 256 * U - 1) / (256 * U); }

// Calls F<T, N>(...) for the widest vector of N elements that `bytes` allows.
#define EUC_ROW_VEC(T, bytes, F, ...)                                                    \
  switch ((bytes) / static_cast<int>(sizeof(T))) {                                       \
    case 8: if constexpr (sizeof(T) == 2) return F<T, 8>(__VA_ARGS__); break;            \
    case 4: if constexpr (sizeof(T) <= 4) return F<T, 4>(__VA_ARGS__); break;            \
    case 2: return F<T, 2>(__VA_ARGS__);                                                 \
    default: return F<T, 1>(__VA_ARGS__);                                                \
  }                                                                                      \
  return cudaErrorInvalidValue

}  // namespace euc
