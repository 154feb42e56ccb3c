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
// registers, which loses nothing when |mean| >> std.  All sums are fp32 (fp64 for
// fp64 rows); outputs are rounded once.
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

template <typename A>
__device__ __forceinline__ A inv_std(A var, A eps);
template <>
__device__ __forceinline__ float inv_std<float>(float var, float eps) { return 1.0f / sqrtf(var + eps); }
template <>
__device__ __forceinline__ double inv_std<double>(double var, double eps) { return 1.0 / sqrt(var + eps); }

// TPR threads per row, EPT elements per thread in vectors of VEC, RPB rows per block.
template <typename T, typename W, int VEC, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR* RPB)
    ln_fwd_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ w,
                  const W* __restrict__ b, int64_t rows, int C, double eps_, T* __restrict__ y,
                  Acc<T>* __restrict__ mean_out, Acc<T>* __restrict__ rstd_out) {
  using A = Acc<T>;
  constexpr int NV = EPT / VEC;
  __shared__ A red[RPB][4][TPR / 32];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const A eps = (A)eps_, inv_c = (A)1 / (A)C;
  int phase = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPB + g; row < rows; row += (int64_t)gridDim.x * RPB) {
    const T* xr = x + row * xs;
    A v[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < C) {
        load_vec<VEC>(xr + c, v + i * VEC);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = 0;
      }
    }
    A s = 0;
#pragma unroll
    for (int e = 0; e < EPT; ++e) s += v[e];
    const A mean = row_sum<TPR>(s, red[g][phase], g + 1) * inv_c;
    s = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * TPR + t) * VEC < C) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const A d = v[i * VEC + j] - mean;
          s += d * d;
        }
      }
    }
    const A rstd = inv_std<A>(row_sum<TPR>(s, red[g][phase + 1], g + 1) * inv_c, eps);
    phase ^= 2;
    if (t == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    T* yr = y + row * C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < C) {
        A o[VEC], wv[VEC], bv[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) wv[j] = 1, bv[j] = 0;
        if (w) load_vec<VEC>(w + c, wv);
        if (b) load_vec<VEC>(b + c, bv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = (v[i * VEC + j] - mean) * rstd * wv[j] + bv[j];
        store_vec<VEC>(yr + c, o);
      }
    }
  }
}

// Backward for rows that fit in registers.  Blocks stay resident and walk over
// the rows; a thread always owns the same columns, so the weight and bias
// gradients accumulate in its registers and every block writes one partial row
// of each (summed by ln_bwd_reduce_kernel in block order: no atomics, the same
// bits in every run).
template <typename T, typename W, int VEC, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR* RPB)
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
  A wv[EPT], aw[EPT], ab[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) wv[e] = 1, aw[e] = 0, ab[e] = 0;
  if (w) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < C) load_vec<VEC>(w + c, wv + i * VEC);
    }
  }
  int phase = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPB + g; row < rows; row += (int64_t)gridDim.x * RPB) {
    A xh[EPT], gy[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < C) {
        load_vec<VEC>(x + row * xs + c, xh + i * VEC);
        load_vec<VEC>(dy + row * dys + c, gy + i * VEC);
      }
    }
    const A mean = mean_in[row], rstd = rstd_in[row];
    A s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = (i * TPR + t) * VEC < C;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = i * VEC + j;
        xh[e] = in ? (xh[e] - mean) * rstd : 0;
        gy[e] = in ? gy[e] : 0;
        aw[e] += gy[e] * xh[e];
        ab[e] += gy[e];
        const A u = gy[e] * wv[e];
        s1 += u;
        s2 += u * xh[e];
      }
    }
    if (dx) {
      s1 = row_sum<TPR>(s1, red[g][phase], g + 1) * inv_c;
      s2 = row_sum<TPR>(s2, red[g][phase + 1], g + 1) * inv_c;
      phase ^= 2;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c < C) {
          A o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int e = i * VEC + j;
            o[j] = rstd * (gy[e] * wv[e] - s1 - xh[e] * s2);
          }
          store_vec<VEC>(dx + row * C + c, o);
        }
      }
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
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (i * TPR + t) * VEC + j;
        if (c < C) {
          if (pw) pw[(int64_t)blockIdx.x * C + c] = aw[i * VEC + j];
          if (pb) pb[(int64_t)blockIdx.x * C + c] = ab[i * VEC + j];
        }
      }
    }
  }
}

// Column sums of the blocks' partial rows: 32 columns per block, 32 strands of
// rows each, strands added in order.  blockIdx.y 0: weight, 1: bias.
template <typename W, typename A>
__global__ void __launch_bounds__(1024)
    ln_bwd_reduce_kernel(const A* __restrict__ pw, const A* __restrict__ pb, int parts, int C,
                         W* __restrict__ dw, W* __restrict__ db) {
  __shared__ A sm[32][33];
  pdl_wait();
  const A* p = blockIdx.y ? pb : pw;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  A s = 0;
  if (c < C)
    for (int r = threadIdx.y; r < parts; r += 32) s += p[(int64_t)r * C + c];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    s = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sm[i][threadIdx.x];
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
  __shared__ A red[4][16];
  const A inv_c = (A)1 / (A)C;
  int phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    A s = 0;
    for (int64_t c = threadIdx.x; c < C; c += 512) s += to_acc(xr[c]);
    const A mean = row_sum<512>(s, red[phase], 1) * inv_c;
    s = 0;
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A d = to_acc(xr[c]) - mean;
      s += d * d;
    }
    const A rstd = inv_std<A>(row_sum<512>(s, red[phase + 1], 1) * inv_c, (A)eps_);
    phase ^= 2;
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < C; c += 512) {
      const A wv = w ? to_acc(w[c]) : (A)1, bv = b ? to_acc(b[c]) : (A)0;
      y[row * C + c] = from_acc<T>((to_acc(xr[c]) - mean) * rstd * wv + bv);
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

// Resident blocks of the backward kernel: two per SM.
constexpr int kBwdBlocks = 148 * 2;
constexpr int kWideParts = 32;

int bwd_parts(int64_t rows, int64_t C) {
  if (C > kMaxRegWidth) return (int)min64(rows, kWideParts);
  const int rpb = C <= 512 ? 8 : C <= 1024 ? 4 : C <= 2048 ? 2 : 1;
  return (int)min64((rows + rpb - 1) / rpb, kBwdBlocks);
}

template <typename T, typename W, int VEC>
int fwd_launch(const T* x, int64_t xs, const W* w, const W* b, int64_t rows, int C, double eps, T* y,
               Acc<T>* mean, Acc<T>* rstd, cudaStream_t st) {
  constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
#define TPO_LN(TPR, EPT, RPB)                                                                   \
  do {                                                                                          \
    const int64_t grid = min64((rows + RPB - 1) / RPB, kMaxGrid);                               \
    ln_fwd_kernel<T, W, VEC, TPR, EPT, RPB>                                                     \
        <<<(unsigned)grid, TPR * RPB, 0, st>>>(x, xs, w, b, rows, C, eps, y, mean, rstd);       \
    return check_launch();                                                                      \
  } while (0)
  // A warp per row up to 1024 columns (no block barrier), four rows per block;
  // one block per row beyond.
  if (C <= 256) TPO_LN(32, 8, 4);
  if (C <= 512) TPO_LN(32, 16, 4);
  if (C <= 1024) TPO_LN(32, 32, 4);
  if (C <= 2048) TPO_LN(128, 16, 1);
  if (C <= 4096) TPO_LN(128, 32, 1);
  TPO_LN(256, 32, 1);
#undef TPO_LN
}

template <typename T, typename W, int VEC>
int bwd_launch(const T* x, int64_t xs, const T* dy, int64_t dys, const W* w, const Acc<T>* mean,
               const Acc<T>* rstd, int64_t rows, int C, T* dx, Acc<T>* pw, Acc<T>* pb,
               cudaStream_t st) {
  const int grid = bwd_parts(rows, C);
#define TPO_LN(TPR, RPB)                                                                        \
  do {                                                                                          \
    ln_bwd_kernel<T, W, VEC, TPR, C16(TPR), RPB><<<grid, TPR * RPB, 0, st>>>(                   \
        x, xs, dy, dys, w, mean, rstd, rows, C, dx, pw, pb);                                    \
    return check_launch();                                                                      \
  } while (0)
#define C16(TPR) 16
  if (C <= 256) {
    ln_bwd_kernel<T, W, VEC, 32, 8, 8>
        <<<grid, 256, 0, st>>>(x, xs, dy, dys, w, mean, rstd, rows, C, dx, pw, pb);
    return check_launch();
  }
  if (C <= 512) TPO_LN(32, 8);
  if (C <= 1024) TPO_LN(64, 4);
  if (C <= 2048) TPO_LN(128, 2);
  if (C <= 4096) TPO_LN(256, 1);
  TPO_LN(512, 1);
#undef C16
#undef TPO_LN
}

template <typename T>
bool vec_ok(const void* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
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
  // 16-byte accesses where every row and the parameters start on 16 bytes
  const bool vec = vec_ok<T>(x, xs) && vec_ok<T>(y, C) && vec_ok<W>(w, 0) && vec_ok<W>(b, 0) && C % V == 0;
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
  const int parts = bwd_parts(rows, C);
  A* pw = dw ? (A*)ws : nullptr;
  A* pb = db ? (A*)ws + (int64_t)parts * C : nullptr;
  int s;
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
    constexpr int V = 16 / sizeof(T);
    const bool vec = vec_ok<T>(x, xs) && vec_ok<T>(dy, dys) && vec_ok<T>(dx, C) && vec_ok<W>(w, 0) && C % V == 0;
    s = vec ? bwd_launch<T, W, V>(x, xs, dy, dys, w, mean, rstd, rows, (int)C, dx, pw, pb, st)
            : bwd_launch<T, W, 1>(x, xs, dy, dys, w, mean, rstd, rows, (int)C, dx, pw, pb, st);
    if (s) return s;
  }
  if (!dw && !db) return TPO_OK;
  return launch_pdl(ln_bwd_reduce_kernel<W, A>, dim3((unsigned)((C + 31) / 32), 2), dim3(32, 32), 0, st,
                    (const A*)pw, (const A*)pb, parts, (int)C, dw, db);
}

}  // namespace

size_t layer_norm_bwd_workspace_size(int dtype, int64_t rows, int64_t C) {
  return (size_t)2 * bwd_parts(rows, C) * (size_t)C * (dtype == TPO_F64 ? 8 : 4);
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
