// Element types of the token operators: accumulation type, conversions and
// vector accesses (fp16, bf16 and fp32 accumulate in fp32, fp64 in fp64).
#pragma once

#include <cuda_bf16.h>

#include "tpo_common.cuh"

namespace tpo {

template <typename T>
struct AccOf { using type = float; };
template <>
struct AccOf<double> { using type = double; };
template <typename T>
using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T, typename A>
__device__ __forceinline__ T from_acc(A v) { return (T)v; }
template <>
__device__ __forceinline__ __half from_acc<__half, float>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16, float>(float v) { return __float2bfloat16_rn(v); }

// N elements at p (N * sizeof(T) a multiple of 16 and p 16-byte aligned, or N == 1).
template <typename T, int N>
struct alignas(N == 1 ? sizeof(T) : 16) Pack { T v[N]; };

template <int N, typename T, typename A>
__device__ __forceinline__ void load_vec(const T* p, A* out) {
  const Pack<T, N> k = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_acc(k.v[i]);
}
template <int N, typename T, typename A>
__device__ __forceinline__ void store_vec(T* p, const A* in) {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = from_acc<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = k;
}

}  // namespace tpo
