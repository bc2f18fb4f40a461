// Row kernels' shared parts (LayerNorm, the RMS norm, the embedding): rows of any alignment as 16-byte vectors,
// sums over the waves of a row, and the ordered sum of per-workgroup column sums.
#pragma once

#include "sparton_common.h"

namespace sparton {

constexpr int kSumWaves = 16;

// A 16-byte vector (or one element) at any address.
template <typename T, int VE> struct Vec {
  typedef __attribute__((ext_vector_type(VE))) T type;
  typedef type loose __attribute__((aligned(sizeof(T))));
};
template <typename T> struct Vec<T, 1> {
  struct type {
    T v;
    __device__ __forceinline__ T operator[](int) const { return v; }
    __device__ __forceinline__ T& operator[](int) { return v; }
  };
  typedef type loose;
};
template <typename T, int VE> using vec_t = typename Vec<T, VE>::type;
template <typename T, int VE> __device__ __forceinline__ vec_t<T, VE> load_any(const T* p) {
  return *(const typename Vec<T, VE>::loose*)p;
}
template <typename T, int VE> __device__ __forceinline__ void store_any(T* p, vec_t<T, VE> v) {
  *(typename Vec<T, VE>::loose*)p = v;
}

// Where a lane's vector lies in the row, and which of its elements are its own: from `own` on. Past
// the row end none are (own = VE), and the loads repeat the row's last vector.
template <int VE> struct Place {
  int at, own;
  __device__ __forceinline__ Place(int want, int D) {
    at = min(want, D - VE);
    own = want >= D ? VE : want - at;
  }
};

// A lane's elements of weight or bias, in fp32 or in the rows' type.
template <typename T, int VE> __device__ __forceinline__ void vec_param(float* out, const void* p, int dt, int at) {
  if (dt == SPARTON_F32) {  // uniform
    constexpr int N = VE < 4 ? VE : 4;
#pragma unroll
    for (int i = 0; i < VE; i += N) {
      const vec_t<float, N> v = load_any<float, N>((const float*)p + at + i);
#pragma unroll
      for (int e = 0; e < N; ++e) out[i + e] = v[e];
    }
  } else {
    const vec_t<T, VE> v = load_any<T, VE>((const T*)p + at);
#pragma unroll
    for (int e = 0; e < VE; ++e) out[e] = to_f32(v[e]);
  }
}

// Sum over the WPR waves of a row, in wave order; result in every lane. `slot` is the row group's
// [WPR] floats of LDS; consecutive sums alternate between two of them, so one barrier each will do.
template <int WPR> __device__ __forceinline__ float row_sum(float x, float* slot, int wave_in_row) {
  x = wave_sum(x);
  if constexpr (WPR == 1) return x;
  if ((threadIdx.x & 63) == 0) slot[wave_in_row] = x;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < WPR; ++w) s += slot[w];
  return s;
}

// The largest value over the WPR waves of a row; NaN is passed over.
template <int WPR> __device__ __forceinline__ float row_max(float x, float* slot, int wave_in_row) {
  x = wave_max(x);
  if constexpr (WPR == 1) return x;
  if ((threadIdx.x & 63) == 0) slot[wave_in_row] = x;
  __syncthreads();
  float s = slot[0];
#pragma unroll
  for (int w = 1; w < WPR; ++w) s = fmaxf(s, slot[w]);
  return s;
}

// part[blocks][ncol] summed in block order, columns [0, D) to `dgamma`, [D, 2 D) to `dbeta`: 64 columns a
// workgroup, one per lane; wave w adds blocks [w seg, (w + 1) seg), and wave 0 the waves' sums in wave order.
// 1.5 MB in 3.8 us at D = 768 and two vectors, most of it the launch.
static __global__ __launch_bounds__(64 * kSumWaves) void colsum_kernel(const float* __restrict__ part, int blocks, int D,
                                                                       int ncol, void* dgamma, void* dbeta,
                                                                       int vec_dtype) {
  __shared__ float wsum[kSumWaves][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = blockIdx.x * 64 + lane;
  const int seg = (blocks + kSumWaves - 1) / kSumWaves;
  float a = 0.0f;
  if (col < ncol) {
    const int b1 = min(blocks, (wave + 1) * seg);
#pragma unroll 8
    for (int b = wave * seg; b < b1; ++b) a += part[(int64_t)b * ncol + col];
  }
  wsum[wave][lane] = a;
  __syncthreads();
  if (wave > 0 || col >= ncol) return;
  a = 0.0f;
#pragma unroll
  for (int w = 0; w < kSumWaves; ++w) a += wsum[w][lane];
  void* to = col < D ? dgamma : dbeta;
  if (to == nullptr) return;
  const int c = col < D ? col : col - D;
  switch (vec_dtype) {
    case SPARTON_BF16: ((bf16*)to)[c] = from_f32<bf16>(a); break;
    case SPARTON_F16: ((f16*)to)[c] = from_f32<f16>(a); break;
    default: ((float*)to)[c] = a;
  }
}

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace sparton
