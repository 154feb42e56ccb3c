// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  rstd = 1 / sqrt(var + eps)
//   y  = xh * w + b                      with xh = (x - mean) * rstd
//   dx = rstd * (u - mean(u) - xh * mean(u * xh))      with u = dy * w
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// A few operations per element: HBM traffic is the bound (forward 2 passes over
// (R, C), backward 3).  So a row is read once and stays in registers for both
// moments and the result; the variance is the centred second pass over those
// registers.  That pass also sums the centred values: what the mean's rounding left
// (up to some 2^-20 |mean|, which 1 / std magnifies) is taken out of y, the
// variance and the mean that the backward reads.  All sums are fp32 (fp64 for fp64
// rows); outputs are rounded once.
//
// Measured (B200, GB/s of the passes above; a plain copy moves 6555), inputs where the last
// call left them: forward 65536 x 512 fp32 42.9 us (6260), 32768 x 1024 bf16 24.3 us (5520: issue
// slots, conversions), 10007 x 771 fp16 12.0 us (2580: one element per load); backward 65.0 us
// (6200), 38.7 us (5200), 16.2 us (2860).  With L2 flushed before each call: fp64 8192 x 1024
// forward 34.8 us (3860), backward 103 us (1950: registers, spills); rows wider than 8192
// loop over single elements: 4096 x 16384 bf16 forward 119 us (2260), backward 251 us
// (1600), 4096 x 9000 fp32 100 us (2930) and 174 us (2540).
#include "tpo_internal.h"
#include "tpo_types.cuh"

namespace tpo {
namespace {

constexpr int kMaxRegWidth = 8192;  // wider rows take the looping kernels

// Sum over the TPR threads of a row.  One warp: shuffles.  More: one word per
// warp through shared memory, added in warp order by every thread (the same
// order everywhere, so all threads hold the same bits).  `bar` is the row
// group's named barrier; `red` has room for two rounds used alternately, so one
// barrier per reduction is enough.
template <int TPR, typename A>
__device__ __forceinline__ A row_sum(A v, A* red, int bar) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (TPR > 32) {
    const int wid = (threadIdx.x % TPR) / 32;
    if (threadIdx.x % 32 == 0) red[wid] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(TPR) : "memory");
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) v += red[i];
  }
  return v;
}

// Two such sums with one barrier.
template <int TPR, typename A>
__device__ __forceinline__ void row_sums(A& v, A& w, A* red_v, A* red_w, int bar) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  if (TPR > 32) {
    const int wid = (threadIdx.x % TPR) / 32;
    if (threadIdx.x % 32 == 0) red_v[wid] = v, red_w[wid] = w;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(TPR) : "memory");
    v = red_v[0], w = red_w[0];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) v += red_v[i], w += red_w[i];
  }
}

template <typename A>
__device__ __forceinline__ A inv_std(A var, A eps);
template <>
__device__ __forceinline__ float inv_std<float>(float var, float eps) { return rsqrtf(var + eps); }  // within 2 ulp
template <>
__device__ __forceinline__ double inv_std<double>(double var, double eps) { return rsqrt(var + eps); }

// var - part where that is positive, else 0; a variance beyond the type's range stays infinite.
template <typename A>
__device__ __forceinline__ A without(A var, A part) {
  return part < var ? var - part : var < (A)INFINITY ? (A)0 : var;
}

// Two values at a time: fp32 has packed instructions, which take half of the issue slots.
struct Doubles { double x, y; };
using tpo::add2;
using tpo::fma2;
using tpo::sub2;
template <typename A>
using Two = std::conditional_t<std::is_same<A, float>::value, u64, Doubles>;
__device__ __forceinline__ u64 two(float x, float y) { return pk(x, y); }
__device__ __forceinline__ Doubles two(double x, double y) { return {x, y}; }
__device__ __forceinline__ void apart(u64 v, float& x, float& y) { upk(v, x, y); }
__device__ __forceinline__ void apart(Doubles v, double& x, double& y) { x = v.x, y = v.y; }
__device__ __forceinline__ Doubles add2(Doubles a, Doubles b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Doubles sub2(Doubles a, Doubles b) { return {a.x - b.x, a.y - b.y}; }
__device__ __forceinline__ Doubles fma2(Doubles a, Doubles b, Doubles c) { return {fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)}; }
template <typename A>
__device__ __forceinline__ A both(Two<A> v) {
  A x, y;
  apart(v, x, y);
  return x + y;
}

// A thread's vectors of a row (vector i: columns (i * TPR + t) * VEC on) as accumulators.
// Vectors beyond column C are zeros: they are cleared once and never loaded, so no
// element needs a test of its own.
template <int VEC, int N, typename T, typename A>
__device__ __forceinline__ void unpack(A (&v)[N * VEC], const Pack<T, VEC> (&raw)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (VEC == 1) {
      v[i] = to_acc(raw[i].v[0]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) pair_of(raw[i], j, v[i * VEC + 2 * j], v[i * VEC + 2 * j + 1]);
    }
  }
}
template <int VEC, int TPR, int EPT, typename T>
__device__ __forceinline__ void load_row(Pack<T, VEC> (&raw)[EPT / VEC], const T* row, int t, int C) {
#pragma unroll
  for (int i = 0; i < EPT / VEC; ++i) {
    const int c = (i * TPR + t) * VEC;
    if (c < C) raw[i] = *reinterpret_cast<const Pack<T, VEC>*>(row + c);
  }
}
template <int VEC, int N, typename T>
__device__ __forceinline__ void fill(Pack<T, VEC> (&raw)[N], Acc<T> value) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) raw[i].v[j] = from_acc<T>(value);
}
template <int VEC, int TPR, int EPT, typename T, typename A>
__device__ __forceinline__ void store_row(T* row, const A (&v)[EPT], int t, int C) {
#pragma unroll
  for (int i = 0; i < EPT / VEC; ++i) {
    const int c = (i * TPR + t) * VEC;
    if (c < C) store_vec<VEC>(row + c, v + i * VEC);
  }
}

// TPR threads per row, EPT elements per thread in vectors of VEC, RPB rows per block.
// Blocks stay resident and walk over the rows: weight and bias are read once into
// registers (with a block per row group they cost as many loads as the row itself).
template <typename T, typename W, int VEC, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR* RPB)
    ln_fwd_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ w,
                  const W* __restrict__ b, int64_t rows, int C, double eps_, T* __restrict__ y,
                  Acc<T>* __restrict__ mean_out, Acc<T>* __restrict__ rstd_out) {
  using A = Acc<T>;
  constexpr int NV = EPT / VEC;
  // 32 and 64 bits: the next row is on its way while this one is reduced and written.
  // 16 bits: conversions keep the issue slots busy, and the registers of a second
  // row cost more warps than it brings (measured, bf16, 32768 x 1024: 25.3 against 24.3 us).
  constexpr bool AHEAD = sizeof(T) != 2;
  __shared__ A red[RPB][6][TPR / 32];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const A eps = (A)eps_, inv_c = (A)1 / (A)C;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + g;
  // Whole vectors of 16-bit rows wider than 512: the parameters wait in shared memory, their registers
  // would cost a third of the warps (measured, bf16: 32768 x 1024 29.7 against 24.3 us, 32768 x
  // 2048 57.7 against 50.4; narrower rows have few: 32768 x 512 10.0 against 12.0 with shared memory).
  constexpr bool SHARED = sizeof(T) == 2 && VEC == 8 && TPR * EPT > 512 && 2 * NV * TPR * sizeof(Pack<W, VEC>) <= 40960;
  __shared__ Pack<W, VEC> ws[SHARED ? NV * TPR : 1], bs[SHARED ? NV * TPR : 1];
  Pack<T, VEC> cur[NV], nxt[NV];
  Pack<W, VEC> wv[NV], bv[NV];
  fill(cur, 0);
  fill(nxt, 0);
  fill(wv, 1);  // no weight, no bias: one and zero, so that the loop has no branches
  fill(bv, 0);
  if (SHARED) {
    if (g == 0) {
      if (w) load_row<VEC, TPR, EPT>(wv, w, t, C);
      if (b) load_row<VEC, TPR, EPT>(bv, b, t, C);
#pragma unroll
      for (int i = 0; i < NV; ++i) ws[i * TPR + t] = wv[i], bs[i * TPR + t] = bv[i];
    }
    __syncthreads();
  }
  if (row >= rows) return;  // a whole row group: its barrier is its own
  load_row<VEC, TPR, EPT>(cur, x + row * xs, t, C);
  if (!SHARED && w) load_row<VEC, TPR, EPT>(wv, w, t, C);
  if (!SHARED && b) load_row<VEC, TPR, EPT>(bv, b, t, C);
  int phase = 0;
  while (row < rows) {
    const int64_t next = row + step;
    if (AHEAD && next < rows) load_row<VEC, TPR, EPT>(nxt, x + next * xs, t, C);
    Two<A> v[EPT / 2], sum, squares;
    {
      A one[EPT];
      unpack(one, cur);
#pragma unroll
      for (int e = 0; e < EPT / 2; ++e) v[e] = two(one[2 * e], one[2 * e + 1]);
    }
    sum = v[0];
#pragma unroll
    for (int e = 1; e < EPT / 2; ++e) sum = add2(sum, v[e]);
    const A mean = row_sum<TPR>(both<A>(sum), red[g][phase], g + 1) * inv_c;
    sum = squares = two((A)0, (A)0);
#pragma unroll
    for (int e = 0; e < EPT / 2; ++e) {
      // vectors beyond C are no part of the variance
      const bool in0 = (2 * e / VEC * TPR + t) * VEC < C, in1 = ((2 * e + 1) / VEC * TPR + t) * VEC < C;
      v[e] = sub2(v[e], two(in0 ? mean : (A)0, in1 ? mean : (A)0));
      sum = add2(sum, v[e]);
      squares = fma2(v[e], v[e], squares);
    }
    A rest = both<A>(sum), var = both<A>(squares);
    row_sums<TPR>(rest, var, red[g][phase + 1], red[g][phase + 2], g + 1);
    rest *= inv_c;  // what the mean's rounding left
    const A rstd = inv_std<A>(without(var * inv_c, rest * rest), eps), shift = -rest * rstd;
    phase ^= 3;
    if (t == 0 && mean_out) {
      mean_out[row] = mean + rest;
      rstd_out[row] = rstd;
    }
    A o[EPT], wk[EPT], bk[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<VEC, 1>(reinterpret_cast<A(&)[VEC]>(wk[i * VEC]), reinterpret_cast<const Pack<W, VEC>(&)[1]>(SHARED ? ws[i * TPR + t] : wv[i]));
      unpack<VEC, 1>(reinterpret_cast<A(&)[VEC]>(bk[i * VEC]), reinterpret_cast<const Pack<W, VEC>(&)[1]>(SHARED ? bs[i * TPR + t] : bv[i]));
    }
#pragma unroll
    for (int e = 0; e < EPT / 2; ++e)
      apart(fma2(fma2(v[e], two(rstd, rstd), two(shift, shift)), two(wk[2 * e], wk[2 * e + 1]), two(bk[2 * e], bk[2 * e + 1])),
            o[2 * e], o[2 * e + 1]);
    store_row<VEC, TPR, EPT>(y + row * C, o, t, C);
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < NV; ++i) cur[i] = nxt[i];
    } else if (next < rows) {
      load_row<VEC, TPR, EPT>(cur, x + next * xs, t, C);
    }
    row = next;
  }
}

// Backward for rows that fit in registers.  Blocks stay resident and walk over
// the rows; a thread always owns the same columns, so the weight and bias
// gradients accumulate in its registers and every block writes one partial row
// of each (summed by ln_bwd_reduce_kernel in block order: no atomics, the same
// bits in every run).
template <typename T, typename W, int VEC, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR* RPB, TPR* RPB <= 256 ? 2 : 1)
    ln_bwd_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ dy, int64_t dys,
                  const W* __restrict__ w, const Acc<T>* __restrict__ mean_in,
                  const Acc<T>* __restrict__ rstd_in, int64_t rows, int C, T* __restrict__ dx,
                  Acc<T>* __restrict__ pw, Acc<T>* __restrict__ pb) {
  using A = Acc<T>;
  constexpr int NV = EPT / VEC;
  __shared__ A red[RPB][4][TPR / 32];
  __shared__ A comb[RPB > 1 ? 2 * TPR * EPT : 1];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const A inv_c = (A)1 / (A)C;
  A aw[EPT], ab[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) aw[e] = ab[e] = 0;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + g;
  Pack<T, VEC> cx[NV], cy[NV];
  Pack<W, VEC> wv[NV];
  fill(cx, 0);
  fill(cy, 0);
  fill(wv, 1);
  A mean = 0, rstd = 0;
  auto fetch = [&](int64_t r) {
    load_row<VEC, TPR, EPT>(cx, x + r * xs, t, C);
    load_row<VEC, TPR, EPT>(cy, dy + r * dys, t, C);
    mean = mean_in[r], rstd = rstd_in[r];
  };
  // 16-bit rows: the next one is on its way while this one is reduced and written.
  // Wider types have as many bytes in flight without it, and no registers for it.
  constexpr bool AHEAD = sizeof(T) == 2;
  if (AHEAD && row < rows) fetch(row);
  if (w) load_row<VEC, TPR, EPT>(wv, w, t, C);
  int phase = 0;
  for (; row < rows; row += step) {
    if (!AHEAD) fetch(row);
    const A m = mean, r = rstd;
    A xh[EPT], u[EPT], s1 = 0, s2 = 0;
    unpack(xh, cx);
    unpack(u, cy);
    if (AHEAD && row + step < rows) fetch(row + step);
    // Beyond column C dy is zero, but (0 - mean) * rstd has to be finite to add nothing.  A rare
    // branch, since a select per vector costs registers (65536 x 512 fp32: 72.8 against 85.0 us); fp64
    // rows spill either way, less with the select (8192 x 1024: 103 against 124 us).
    constexpr bool SELECT = sizeof(T) == 8;
    if (!SELECT && !(fabsf((float)(m * r)) < INFINITY)) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if ((i * TPR + t) * VEC >= C) xh[i * VEC + j] = m;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      A wk[VEC];
      unpack<VEC, 1>(wk, reinterpret_cast<const Pack<W, VEC>(&)[1]>(wv[i]));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = i * VEC + j;
        xh[e] = (xh[e] - (!SELECT || (i * TPR + t) * VEC < C ? m : (A)0)) * r;
        aw[e] += u[e] * xh[e];
        ab[e] += u[e];
        u[e] *= wk[j];
        s1 += u[e];
        s2 += u[e] * xh[e];
      }
    }
    if (dx) {
      s1 = row_sum<TPR>(s1, red[g][phase], g + 1) * inv_c;
      s2 = row_sum<TPR>(s2, red[g][phase + 1], g + 1) * inv_c;
      phase ^= 2;
#pragma unroll
      for (int e = 0; e < EPT; ++e) u[e] = r * (u[e] - s1 - xh[e] * s2);
      store_row<VEC, TPR, EPT>(dx + row * C, u, t, C);
    }
  }
  if (!pw && !pb) return;
  // row groups of the block added in group order
  for (int k = 1; k < RPB; ++k) {
    if (g == k) {
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        comb[e * TPR + t] = aw[e];
        comb[(EPT + e) * TPR + t] = ab[e];
      }
    }
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        aw[e] += comb[e * TPR + t];
        ab[e] += comb[(EPT + e) * TPR + t];
      }
    }
    __syncthreads();
  }
  if (g == 0) {
    if (pw) store_row<VEC, TPR, EPT>(pw + (int64_t)blockIdx.x * C, aw, t, C);
    if (pb) store_row<VEC, TPR, EPT>(pb + (int64_t)blockIdx.x * C, ab, t, C);
  }
}

// Column sums of the blocks' partial rows: 32 columns per block, STRANDS strands of
// rows each, strands added in order.  blockIdx.y 0: weight, 1: bias.
template <typename W, typename A, int STRANDS>
__global__ void __launch_bounds__(32 * STRANDS)
    ln_bwd_reduce_kernel(const A* __restrict__ pw, const A* __restrict__ pb, int parts, int C,
                         W* __restrict__ dw, W* __restrict__ db) {
  __shared__ A sm[STRANDS][33];
  pdl_wait();
  const A* p = blockIdx.y ? pb : pw;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  A s = 0;
  if (c < C) {
#pragma unroll 8
    for (int r = threadIdx.y; r < parts; r += STRANDS) s += p[(int64_t)r * C + c];
  }
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    s = 0;
#pragma unroll
    for (int i = 0; i < STRANDS; ++i) s += sm[i][threadIdx.x];
    out[c] = from_acc<W>(s);
  }
}

// ---- rows wider than kMaxRegWidth: a block of 512 threads loops over the row ----
template <typename T, typename W>
__global__ void __launch_bounds__(512)
    ln_fwd_wide_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ w,
                       const W* __restrict__ b, int64_t rows, int64_t C, double eps_,
                       T* __restrict__ y, Acc<T>* __restrict__ mean_out,
                       Acc<T>* __restrict__ rstd_out) {
  using A = Acc<T>;
  __shared__ A red[6][16];
  const A inv_c = (A)1 / (A)C;
  int phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    A s = 0;
    for (int64_t c = threadIdx.x; c < C; c += 512) s += to_acc(xr[c]);
    const A mean = row_sum<512>(s, red[phase], 1) * inv_c;
    A rest = 0;
    s = 0;
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A d = to_acc(xr[c]) - mean;
      rest += d;
      s += d * d;
    }
    row_sums<512>(rest, s, red[phase + 1], red[phase + 2], 1);
    rest *= inv_c;
    const A rstd = inv_std<A>(without(s * inv_c, rest * rest), (A)eps_), shift = -rest * rstd;
    phase ^= 3;
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = mean + rest;
      rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A wv = w ? to_acc(w[c]) : (A)1, bv = b ? to_acc(b[c]) : (A)0;
      y[row * C + c] = from_acc<T>(((to_acc(xr[c]) - mean) * rstd + shift) * wv + bv);
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(512)
    ln_bwd_wide_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ dy, int64_t dys,
                       const W* __restrict__ w, const Acc<T>* __restrict__ mean_in,
                       const Acc<T>* __restrict__ rstd_in, int64_t rows, int64_t C,
                       T* __restrict__ dx) {
  using A = Acc<T>;
  __shared__ A red[4][16];
  const A inv_c = (A)1 / (A)C;
  int phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const A mean = mean_in[row], rstd = rstd_in[row];
    A s1 = 0, s2 = 0;
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A u = to_acc(dy[row * dys + c]) * (w ? to_acc(w[c]) : (A)1);
      s1 += u;
      s2 += u * ((to_acc(x[row * xs + c]) - mean) * rstd);
    }
    s1 = row_sum<512>(s1, red[phase], 1) * inv_c;
    s2 = row_sum<512>(s2, red[phase + 1], 1) * inv_c;
    phase ^= 2;
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A u = to_acc(dy[row * dys + c]) * (w ? to_acc(w[c]) : (A)1);
      const A xh = (to_acc(x[row * xs + c]) - mean) * rstd;
      dx[row * C + c] = from_acc<T>(rstd * (u - s1 - xh * s2));
    }
  }
}

// Partial weight / bias gradients of wide rows: a thread per column, blockIdx.y
// walks over the rows.
template <typename T>
__global__ void __launch_bounds__(256)
    ln_bwd_wide_cols_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ dy,
                            int64_t dys, const Acc<T>* __restrict__ mean_in,
                            const Acc<T>* __restrict__ rstd_in, int64_t rows, int64_t C,
                            Acc<T>* __restrict__ pw, Acc<T>* __restrict__ pb) {
  using A = Acc<T>;
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  A aw = 0, ab = 0;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const A g = to_acc(dy[row * dys + c]);
    aw += g * ((to_acc(x[row * xs + c]) - mean_in[row]) * rstd_in[row]);
    ab += g;
  }
  if (pw) pw[(int64_t)blockIdx.y * C + c] = aw;
  if (pb) pb[(int64_t)blockIdx.y * C + c] = ab;
}

// Blocks of the backward kernel: two per SM.
constexpr int kBwdBlocks = 148 * 2;
constexpr int kWideParts = 32;

// Rows per block of the backward kernel.  Whole 16-byte vectors: 16 elements per
// thread; else 8, so that the narrow loads spread over more warps.
int bwd_rows_per_block(int64_t C, bool vec) {
  if (vec) return C <= 512 ? 8 : C <= 1024 ? 4 : C <= 2048 ? 2 : 1;
  return C <= 256 ? 8 : C <= 512 ? 4 : C <= 1024 ? 2 : 1;
}
int bwd_parts(int64_t rows, int64_t C, int rpb) {
  return (int)min64((rows + rpb - 1) / rpb, C > kMaxRegWidth ? kWideParts : kBwdBlocks);
}

template <typename K>
int resident_blocks(K kern, int threads) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != cudaSuccess || n < 1) n = 1;
  return 148 * n;
}

template <typename T, typename W, int VEC>
int fwd_launch(const T* x, int64_t xs, const W* w, const W* b, int64_t rows, int C, double eps, T* y,
               Acc<T>* mean, Acc<T>* rstd, cudaStream_t st) {
#define TPO_LN(TPR, EPT, RPB)                                                                          \
  do {                                                                                                 \
    auto kern = ln_fwd_kernel<T, W, VEC, TPR, EPT, RPB>;                                               \
    static const int most = resident_blocks(kern, TPR * RPB);                                          \
    kern<<<(unsigned)min64((rows + RPB - 1) / RPB, most), TPR * RPB, 0, st>>>(x, xs, w, b, rows, C,    \
                                                                              eps, y, mean, rstd);     \
    return check_launch();                                                                             \
  } while (0)
  if (C <= 256) TPO_LN(32, 8, 4);
  if constexpr (VEC * sizeof(T) == 16) {  // a warp per row up to 1024 columns: no barrier
    if (C <= 512) TPO_LN(32, 16, 4);
    if (C <= 1024) TPO_LN(32, 32, 4);
    if (C <= 2048) TPO_LN(128, 16, 1);
    if (C <= 4096) TPO_LN(128, 32, 1);
    TPO_LN(256, 32, 1);
  } else {  // narrow loads: 8 elements per thread, more warps
    if (C <= 512) TPO_LN(64, 8, 2);
    if (C <= 1024) TPO_LN(128, 8, 1);
    if (C <= 2048) TPO_LN(256, 8, 1);
    if (C <= 4096) TPO_LN(512, 8, 1);
    TPO_LN(512, 16, 1);
  }
#undef TPO_LN
}

template <typename T, typename W, int VEC>
int bwd_launch(const T* x, int64_t xs, const T* dy, int64_t dys, const W* w, const Acc<T>* mean,
               const Acc<T>* rstd, int64_t rows, int C, int grid, T* dx, Acc<T>* pw, Acc<T>* pb,
               cudaStream_t st) {
#define TPO_LN(TPR, EPT, RPB)                                                                   \
  do {                                                                                          \
    ln_bwd_kernel<T, W, VEC, TPR, EPT, RPB><<<grid, TPR * RPB, 0, st>>>(                        \
        x, xs, dy, dys, w, mean, rstd, rows, C, dx, pw, pb);                                    \
    return check_launch();                                                                      \
  } while (0)
  if (C <= 256) TPO_LN(32, 8, 8);
  if constexpr (VEC * sizeof(T) == 16) {
    if (C <= 512) TPO_LN(32, 16, 8);
    if (C <= 1024) TPO_LN(64, 16, 4);
    if (C <= 2048) TPO_LN(128, 16, 2);
    if (C <= 4096) TPO_LN(256, 16, 1);
  } else {
    if (C <= 512) TPO_LN(64, 8, 4);
    if (C <= 1024) TPO_LN(128, 8, 2);
    if (C <= 2048) TPO_LN(256, 8, 1);
    if (C <= 4096) TPO_LN(512, 8, 1);
  }
  TPO_LN(512, 16, 1);
#undef TPO_LN
}

// Whether vectors of V elements (at most 16 bytes of alignment) may be read from rows of p.
template <typename T, int V>
bool vec_ok(const void* p, int64_t stride) {
  constexpr size_t bytes = alignof(Pack<T, V>);
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride % V == 0;
}

template <typename T, typename W>
int fwd_typed(const void* x_, int64_t xs, const void* w_, const void* b_, int64_t rows, int64_t C,
              double eps, void* y_, void* mean_, void* rstd_, cudaStream_t st) {
  const T* x = (const T*)x_;
  const W *w = (const W*)w_, *b = (const W*)b_;
  T* y = (T*)y_;
  Acc<T>*mean = (Acc<T>*)mean_, *rstd = (Acc<T>*)rstd_;
  constexpr int V = 16 / sizeof(T);
  if (C > kMaxRegWidth) {
    ln_fwd_wide_kernel<T, W><<<(unsigned)min64(rows, 148 * 4), 512, 0, st>>>(x, xs, w, b, rows, C, eps, y,
                                                                          mean, rstd);
    return check_launch();
  }
  // 16-byte accesses where every row and the parameters start on 16 bytes; pairs of
  // 16-bit elements where they start on whole pairs; else single elements
  const bool vec = vec_ok<T, V>(x, xs) && vec_ok<T, V>(y, C) && vec_ok<W, V>(w, 0) && vec_ok<W, V>(b, 0) && C % V == 0;
  if constexpr (V == 8) {
    if (!vec && vec_ok<T, 2>(x, xs) && vec_ok<T, 2>(y, C) && vec_ok<W, 2>(w, 0) && vec_ok<W, 2>(b, 0) && C % 2 == 0)
      return fwd_launch<T, W, 2>(x, xs, w, b, rows, (int)C, eps, y, mean, rstd, st);
  }
  return vec ? fwd_launch<T, W, V>(x, xs, w, b, rows, (int)C, eps, y, mean, rstd, st)
             : fwd_launch<T, W, 1>(x, xs, w, b, rows, (int)C, eps, y, mean, rstd, st);
}

template <typename T, typename W>
int bwd_typed(const void* x_, int64_t xs, const void* dy_, int64_t dys, const void* w_,
              const void* mean_, const void* rstd_, int64_t rows, int64_t C, void* dx_, void* dw_,
              void* db_, void* ws, cudaStream_t st) {
  using A = Acc<T>;
  const T *x = (const T*)x_, *dy = (const T*)dy_;
  const W* w = (const W*)w_;
  const A *mean = (const A*)mean_, *rstd = (const A*)rstd_;
  T* dx = (T*)dx_;
  W *dw = (W*)dw_, *db = (W*)db_;
  constexpr int V = 16 / sizeof(T);
  const bool vec = vec_ok<T, V>(x, xs) && vec_ok<T, V>(dy, dys) && vec_ok<T, V>(dx, C) && vec_ok<W, V>(w, 0) && C % V == 0;
  const bool pairs = V == 8 && !vec && vec_ok<T, 2>(x, xs) && vec_ok<T, 2>(dy, dys) && vec_ok<T, 2>(dx, C) &&
                     vec_ok<W, 2>(w, 0) && C % 2 == 0;
  const int parts = bwd_parts(rows, C, C > kMaxRegWidth ? 1 : bwd_rows_per_block(C, vec));
  A* pw = dw ? (A*)ws : nullptr;
  A* pb = db ? (A*)ws + (int64_t)parts * C : nullptr;
  int s = TPO_OK;
  if (C > kMaxRegWidth) {
    if (dx) {
      ln_bwd_wide_kernel<T, W><<<(unsigned)min64(rows, 148 * 4), 512, 0, st>>>(x, xs, dy, dys, w, mean, rstd,
                                                                            rows, C, dx);
      if ((s = check_launch())) return s;
    }
    if (dw || db) {
      ln_bwd_wide_cols_kernel<T><<<dim3((unsigned)((C + 255) / 256), parts), 256, 0, st>>>(
          x, xs, dy, dys, mean, rstd, rows, C, pw, pb);
      if ((s = check_launch())) return s;
    }
  } else {
    if constexpr (V == 8) {
      if (pairs) s = bwd_launch<T, W, 2>(x, xs, dy, dys, w, mean, rstd, rows, (int)C, parts, dx, pw, pb, st);
    }
    if (!pairs) s = vec ? bwd_launch<T, W, V>(x, xs, dy, dys, w, mean, rstd, rows, (int)C, parts, dx, pw, pb, st)
                        : bwd_launch<T, W, 1>(x, xs, dy, dys, w, mean, rstd, rows, (int)C, parts, dx, pw, pb, st);
    if (s) return s;
  }
  if (!dw && !db) return TPO_OK;
  // many columns fill the GPU with short strands, few need the long ones' parallel loads
  const dim3 grid((unsigned)((C + 31) / 32), 2);
  if (parts <= 32 || C >= 2048)
    return launch_pdl(ln_bwd_reduce_kernel<W, A, 8>, grid, dim3(32, 8), 0, st, (const A*)pw, (const A*)pb, parts, (int)C, dw, db);
  return launch_pdl(ln_bwd_reduce_kernel<W, A, 32>, grid, dim3(32, 32), 0, st, (const A*)pw, (const A*)pb, parts, (int)C, dw, db);
}

}  // namespace

size_t layer_norm_bwd_workspace_size(int dtype, int64_t rows, int64_t C) {
  return (size_t)2 * bwd_parts(rows, C, 1) * (size_t)C * (dtype == TPO_F64 ? 8 : 4);
}

#define TPO_LN_TYPES(CALL)                                                                  \
  do {                                                                                      \
    if (dtype == TPO_F32 && wdtype == TPO_F32) return CALL(float, float);                   \
    if (dtype == TPO_F64 && wdtype == TPO_F64) return CALL(double, double);                 \
    if (dtype == TPO_F16 && wdtype == TPO_F16) return CALL(__half, __half);                 \
    if (dtype == TPO_F16 && wdtype == TPO_F32) return CALL(__half, float);                  \
    if (dtype == TPO_BF16 && wdtype == TPO_BF16) return CALL(__nv_bfloat16, __nv_bfloat16); \
    if (dtype == TPO_BF16 && wdtype == TPO_F32) return CALL(__nv_bfloat16, float);          \
    return set_error(TPO_ERR_INVALID_ARGUMENT, "layer_norm: unsupported dtypes");           \
  } while (0)

int layer_norm_forward(int dtype, int wdtype, const void* x, int64_t xs, const void* w, const void* b,
                       int64_t rows, int64_t C, double eps, void* y, void* mean, void* rstd,
                       cudaStream_t st) {
#define TPO_CALL(T, W) (fwd_typed<T, W>(x, xs, w, b, rows, C, eps, y, mean, rstd, st))
  TPO_LN_TYPES(TPO_CALL);
#undef TPO_CALL
}

int layer_norm_backward(int dtype, int wdtype, const void* x, int64_t xs, const void* dy, int64_t dys,
                        const void* w, const void* mean, const void* rstd, int64_t rows, int64_t C,
                        void* dx, void* dw, void* db, void* ws, cudaStream_t st) {
#define TPO_CALL(T, W) (bwd_typed<T, W>(x, xs, dy, dys, w, mean, rstd, rows, C, dx, dw, db, ws, st))
  TPO_LN_TYPES(TPO_CALL);
#undef TPO_CALL
}

}  // namespace tpo
