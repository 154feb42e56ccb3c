// Element types of the token operators: accumulation type, conversions and
// vector accesses (fp16, bf16 and fp32 accumulate in fp32, fp64 in fp64).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

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

// Two 16-bit values in a register, rounded together.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// x and y as the sum of two rounded pairs: returns the first, `rest` gets what it left.
template <typename T>
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& rest) {
  const uint32_t first = pack2<T>(x, y);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    rest = pack2<T>(x - __uint_as_float(first << 16), y - __uint_as_float(first & 0xffff0000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&first));
    rest = pack2<T>(x - f.x, y - f.y);
  }
  return first;
}

// N elements (a power of two) that move as one access, or several of 16 bytes.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T v[N]; };

// Elements 2i and 2i + 1 of a vector.
template <typename T, int N, typename A>
__device__ __forceinline__ void pair_of(const Pack<T, N>& p, int i, A& x, A& y) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t u = reinterpret_cast<const uint32_t*>(&p)[i];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x = __uint_as_float(u << 16);
      y = __uint_as_float(u & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
      x = f.x, y = f.y;
    }
  } else {
    x = to_acc(p.v[2 * i]), y = to_acc(p.v[2 * i + 1]);
  }
}
template <int N, typename T, typename A>
__device__ __forceinline__ void load_vec(const T* p, A* out) {
  const Pack<T, N> k = *reinterpret_cast<const Pack<T, N>*>(p);
  if constexpr (N == 1) {
    out[0] = to_acc(k.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) pair_of(k, i, out[2 * i], out[2 * i + 1]);
  }
}
template <int N, typename T, typename A>
__device__ __forceinline__ void store_vec(T* p, const A* in) {
  Pack<T, N> k;
  if constexpr (N > 1 && sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) reinterpret_cast<uint32_t*>(&k)[i] = pack2<T>(in[2 * i], in[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) k.v[i] = from_acc<T>(in[i]);
  }
  *reinterpret_cast<Pack<T, N>*>(p) = k;
}

}  // namespace tpo
