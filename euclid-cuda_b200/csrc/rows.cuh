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

// Bytes of the widest vector that every row of `row_bytes` starts and ends on, given the
// OR of the buffers' addresses: 16, 8, 4 or 2 (elements are of 2 bytes at least).
inline int row_vec_bytes(int64_t row_bytes, uintptr_t addresses) {
  const uintptr_t a = addresses | static_cast<uintptr_t>(row_bytes);
  return (a & 15u) == 0 ? 16 : (a & 7u) == 0 ? 8 : (a & 3u) == 0 ? 4 : 2;
}

// A walk over the vectors of consecutive rows, one vector of a row per thread: the flat
// index is split into (row, vector) by one division at the start, and a step of `step`
// vectors adds the step's own (rows, vectors) with a carry.
struct RowWalk {
  int64_t row;
  int64_t v;
  int64_t step_rows;
  int64_t step_v;
  int64_t nv;
  __device__ __forceinline__ RowWalk(int64_t first, int64_t step, int64_t nv_) : nv(nv_) {
    row = first / nv;
    v = first - row * nv;
    step_rows = step / nv;
    step_v = step - step_rows * nv;
  }
  __device__ __forceinline__ void next() {
    row += step_rows;
    v += step_v;
    if (v >= nv) {
      v -= nv;
      ++row;
    }
  }
};

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
