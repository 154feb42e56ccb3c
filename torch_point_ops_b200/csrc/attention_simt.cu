// Attention over packed clouds on the FP32 pipe: every dtype, width up to 256,
// any strides.  Exact fp32 products, so it is the path of fp32 inputs; 16-bit
// inputs come here only where the tensor-core kernels' alignment or width rules
// do not hold.
//
//   S = scale * Q K^T over the keys that a row sees,  P = softmax(S),  O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P * (dP - delta) * scale,  delta = dO . O
//   dQ = dS K,  dK = dS^T Q (dK and dV summed over the query heads of a group)
//
// Forward: one pass over the keys with the running maximum and sum of each row.
// Backward: P is rebuilt from the forward's log-sum-exp; one kernel owns key
// tiles (dK, dV), one owns query tiles (dQ), so nothing is added by atomics and
// every run gives the same bits, at 7 products in place of 5.
//
// 256 threads as TY x TX; thread (ty, tx) holds rows ty + TY r (r < RM) x columns
// tx + TX c (c < CN) of a score tile and the same rows x DP/TX columns of an output
// tile.  Scores are packed fp32 FMAs over neighbouring elements of the summed dimension
// (both operands come as pairs out of 16-byte loads): they hold the FP32 pipe for two
// cycles and leave every other issue slot to loads.  Outputs are single FMAs: pairs would
// need one operand doubled in registers, and the moves cost more than they save.  The
// probabilities are kept transposed, a thread's rows side by side.  A warp is
// 4 rows x 8 columns; rows of operand tiles have DP + 4 floats, so that neighbouring
// rows lie in different banks.
//
// Measured (B200, fp32, 8 clouds of 2048 tokens, 16 heads of width 64): forward 3.63 ms, 38
// TFLOP/s of the two products; dQ and dK dV 34 TFLOP/s.  16-bit inputs of width 256 (4 clouds of 4096,
// 8 heads): forward 28 TFLOP/s, backward 16 of the five.  The FP32 pipe is 50 to 56 % busy,
// the shared-memory pipe 65 to 75 %: operand loads are the bound (larger results per
// thread would need fewer of them, and more registers than there are).
#include "attention_common.cuh"

namespace tpo {
namespace {

constexpr int kThreads = 256;

// rows x DP tile from packed memory into fp32 shared memory (row pitch DP + 4);
// rows beyond `valid` and columns beyond D are zero, so that nothing from another
// cloud (a NaN would survive 0 * NaN) enters a product.
template <typename T, int VEC, int DP>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int rows,
                                          int valid, int D) {
  constexpr int PER_ROW = DP / VEC;
  for (int i = threadIdx.x; i < rows * PER_ROW; i += kThreads) {
    const int r = i / PER_ROW, c = (i % PER_ROW) * VEC;
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    if (r < valid && c < D) load_vec<VEC>(src + r * stride + c, v);
    float* d = dst + r * (DP + 4) + c;
    if (VEC % 4 == 0) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4)
        *reinterpret_cast<float4*>(d + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) d[j] = v[j];
    }
  }
}

// s[r][c] = sum_d a[ty + TY r][d] * b[tx + TX c][d]
template <int DP, int TY, int TX, int RM, int CN>
__device__ __forceinline__ void product_nt(float (&s)[RM][CN], const float* a, const float* b, int ty,
                                           int tx) {
  constexpr int LD = DP + 4;
  u64 acc[RM][CN];
#pragma unroll
  for (int r = 0; r < RM; ++r)
#pragma unroll
    for (int c = 0; c < CN; ++c) acc[r][c] = 0;  // two zeros
  const float* ar = a + ty * LD;
  const float* br = b + tx * LD;
#pragma unroll 2
  for (int d = 0; d < DP; d += 4) {
    ulonglong2 bv[CN];
#pragma unroll
    for (int c = 0; c < CN; ++c) bv[c] = *reinterpret_cast<const ulonglong2*>(br + c * TX * LD + d);
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const ulonglong2 av = *reinterpret_cast<const ulonglong2*>(ar + r * TY * LD + d);
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        acc[r][c] = fma2(av.x, bv[c].x, acc[r][c]);
        acc[r][c] = fma2(av.y, bv[c].y, acc[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RM; ++r)
#pragma unroll
    for (int c = 0; c < CN; ++c) {
      float x, y;
      upk(acc[r][c], x, y);
      s[r][c] = x + y;
    }
}

// A thread's column j of a score-shaped tile, rows side by side, into p[j][ty*RM...].
template <int BM, int RM>
__device__ __forceinline__ void put_rows(float* p, int j, int ty, const float (&v)[RM]) {
  float* at = p + j * (BM + 4) + ty * RM;
  if constexpr (RM % 4 == 0) {
#pragma unroll
    for (int r = 0; r < RM; r += 4) *reinterpret_cast<float4*>(at + r) = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
  } else {
#pragma unroll
    for (int r = 0; r < RM; r += 2) *reinterpret_cast<float2*>(at + r) = make_float2(v[r], v[r + 1]);
  }
}

// o[r][4g + i] += sum_j p[j][ty*RM + r] * v[j][tx*4 + 4 TX g + i]
template <int DP, int TY, int TX, int RM, int BN>
__device__ __forceinline__ void product_nn(float (&o)[RM][DP / TX], const float* p, const float* v,
                                           int ty, int tx) {
  constexpr int LDP = TY * RM + 4;
  const float* pr = p + ty * RM;
  const float* vr = v + tx * 4;
#pragma unroll 4
  for (int j = 0; j < BN; ++j) {
    float pv[RM];
    if constexpr (RM % 4 == 0) {
#pragma unroll
      for (int r = 0; r < RM; r += 4) {
        const float4 t = *reinterpret_cast<const float4*>(pr + j * LDP + r);
        pv[r] = t.x, pv[r + 1] = t.y, pv[r + 2] = t.z, pv[r + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int r = 0; r < RM; r += 2) {
        const float2 t = *reinterpret_cast<const float2*>(pr + j * LDP + r);
        pv[r] = t.x, pv[r + 1] = t.y;
      }
    }
#pragma unroll
    for (int g = 0; g < DP / TX / 4; ++g) {
      const float4 t = *reinterpret_cast<const float4*>(vr + j * (DP + 4) + g * 4 * TX);
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        o[r][g * 4 + 0] = fmaf(pv[r], t.x, o[r][g * 4 + 0]);
        o[r][g * 4 + 1] = fmaf(pv[r], t.y, o[r][g * 4 + 1]);
        o[r][g * 4 + 2] = fmaf(pv[r], t.z, o[r][g * 4 + 2]);
        o[r][g * 4 + 3] = fmaf(pv[r], t.w, o[r][g * 4 + 3]);
      }
    }
  }
}

// The thread's part of a tile on its way from global to shared memory: requested early
// (get), written where the buffer is free (put).
template <typename T, int VEC, int DP, int ROWS>
struct InFlight {
  static constexpr int PER_ROW = DP / VEC, N = ROWS * PER_ROW / kThreads;
  Pack<T, VEC> v[N];
  __device__ __forceinline__ void get(const T* src, int64_t stride, int64_t valid, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * kThreads, r = at / PER_ROW, c = (at % PER_ROW) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i].v[j] = from_acc<T>(0.f);
      if (r < valid && c < D) v[i] = *reinterpret_cast<const Pack<T, VEC>*>(src + r * stride + c);
    }
  }
  __device__ __forceinline__ void put(float* dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * kThreads, r = at / PER_ROW, c = (at % PER_ROW) * VEC;
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = to_acc(v[i].v[j]);
      float* d = dst + r * (DP + 4) + c;
      if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) *reinterpret_cast<float4*>(d + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[j] = f[j];
      }
    }
  }
};

template <int DP, int RM>
struct FwdShape {
  static constexpr int TY = 32, TX = 8, BM = TY * RM, BN = 64, CN = BN / TX;
  static constexpr int smem = ((BM + 2 * BN) * (DP + 4) + BN * (BM + 4)) * 4;
};

template <typename T, int VEC, int DP, int RM>
__global__ void __launch_bounds__(kThreads) packed_simt_fwd_kernel(const PackedArgs a) {
  using Sh = FwdShape<DP, RM>;
  constexpr int TY = Sh::TY, TX = Sh::TX, BM = Sh::BM, BN = Sh::BN, CN = Sh::CN;
  extern __shared__ float4 smem4[];
  float* qs = reinterpret_cast<float*>(smem4);
  float* ks = qs + BM * (DP + 4);
  float* vs = ks + BN * (DP + 4);
  float* ps = vs + BN * (DP + 4);
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int head = blockIdx.x % a.H, kvh = head / (a.H / a.Hk);
  const Tile t = find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, BM, blockIdx.x / a.H, gridDim.x / a.H, a.causal);
  if (t.rows <= 0) return;
  const int64_t shift = t.nb - t.na;            // a row sees keys up to its place + shift
  const int64_t first = t.row0 - t.a0;          // place of the tile's first row in its cloud
  int64_t nk = t.nb;
  if (a.causal) nk = min64(nk, max64(first + t.rows + shift, 0));
  const float qscale = a.scale * kLog2e;

  const T* kp = (const T*)a.k + t.b0 * a.k_st + kvh * a.k_sh;
  const T* vp = (const T*)a.v + t.b0 * a.v_st + kvh * a.v_sh;
  InFlight<T, VEC, DP, BN> next;
  if (nk > 0) next.get(kp, a.k_st, nk, a.D);
  load_tile<T, VEC, DP>(qs, (const T*)a.q + t.row0 * a.q_st + head * a.q_sh, a.q_st, BM, t.rows, a.D);
  float o[RM][DP / TX];
  float m[RM], l[RM];
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / TX; ++c) o[r][c] = 0.f;
  }
  for (int64_t j0 = 0; j0 < nk; j0 += BN) {
    const int valid = (int)min64(nk - j0, BN);
    next.put(ks);  // the last readers of ks have passed the barrier before this step's P V
    next.get(vp + j0 * a.v_st, a.v_st, nk - j0, a.D);
    __syncthreads();
    float s[RM][CN];
    product_nt<DP, TY, TX, RM, CN>(s, qs, ks, ty, tx);
    next.put(vs);  // the last P V is over: every thread has passed the barrier above since
    if (j0 + BN < nk) next.get(kp + (j0 + BN) * a.k_st, a.k_st, nk - j0 - BN, a.D);
    float corr[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      int64_t lim = valid;
      if (a.causal) lim = min64(lim, first + ty + TY * r + shift + 1 - j0);
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        s[r][c] = tx + TX * c < lim ? s[r][c] * qscale : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
#pragma unroll
      for (int x = TX / 2; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float base = mx == -INFINITY ? 0.f : mx;  // a row that has seen nothing yet
      corr[r] = exp2f(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        s[r][c] = exp2f(s[r][c] - base);
        sum += s[r][c];
      }
      m[r] = mx;
      l[r] = l[r] * corr[r] + sum;
    }
#pragma unroll
    for (int c = 0; c < CN; ++c) {
      float col[RM];
#pragma unroll
      for (int r = 0; r < RM; ++r) col[r] = s[r][c];
      put_rows<BM, RM>(ps, tx + TX * c, ty, col);
    }
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int c = 0; c < DP / TX; ++c) o[r][c] *= corr[r];
    __syncthreads();
    product_nn<DP, TY, TX, RM, BN>(o, ps, vs, ty, tx);
  }
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    float sum = l[r];
#pragma unroll
    for (int x = TX / 2; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const int row = ty + TY * r;
    if (row >= t.rows) continue;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // NaN stays NaN
    const int64_t tok = t.row0 + row;
    if (tx == 0 && a.lse) a.lse[(int64_t)head * a.Tq + tok] = sum == 0.f ? -INFINITY : (m[r] + log2f(sum)) * kLn2;
    T* op = (T*)a.o + (tok * a.H + head) * a.D;
#pragma unroll
    for (int g = 0; g < DP / TX / 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = tx * 4 + g * 4 * TX + i;
        if (c < a.D) op[c] = from_acc<T>(o[r][g * 4 + i] * inv);
      }
  }
}

// Backward.  DKV: rows are keys (X1 = K, X2 = V), columns queries (Y1 = Q,
// Y2 = dO), summed over the group's query heads; else rows are queries and
// columns keys.  In both, s = X1 Y1^T and dp = X2 Y2^T.
template <int DP, int RM>
struct BwdShape {
  static constexpr int TY = 16, TX = 16, BM = TY * RM, BN = TX * RM, CN = RM;
  static constexpr int smem = (2 * (BM + BN) * (DP + 4) + 2 * BN * (BM + 4)) * 4 + 2 * BN * 4;
};

template <typename T, int VEC, int DP, int RM, bool DKV>
__global__ void __launch_bounds__(kThreads) packed_simt_bwd_kernel(const PackedArgs a) {
  using Sh = BwdShape<DP, RM>;
  constexpr int TY = Sh::TY, TX = Sh::TX, BM = Sh::BM, BN = Sh::BN, CN = Sh::CN, LD = DP + 4;
  extern __shared__ float4 smem4[];
  float* x1 = reinterpret_cast<float*>(smem4);
  float* x2 = x1 + BM * LD;
  float* y1 = x2 + BM * LD;
  float* y2 = y1 + BN * LD;
  float* ps = y2 + BN * LD;            // P^T (DKV only)
  float* ds = ps + BN * (BM + 4);      // dS or dS^T
  float* cl = ds + BN * (BM + 4);      // log-sum-exp and delta of the columns (DKV)
  float* cd = cl + BN;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int tx = lane % 8 + 8 * (warp % 2), ty = lane / 8 + 4 * (warp / 2);
  const int group = a.H / a.Hk;
  const int nheads = DKV ? a.Hk : a.H, slot = blockIdx.x / nheads, slots = gridDim.x / nheads;
  const Tile t = DKV ? find_tile(a.off_k, a.Tk, a.off_q, a.Tq, a.B, BM, slot, slots, false)
                     : find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, BM, slot, slots, a.causal);
  if (t.rows <= 0) return;
  const int64_t nq = DKV ? t.nb : t.na, nkeys = DKV ? t.na : t.nb, shift = nkeys - nq;
  const int64_t first = t.row0 - t.a0;
  // columns that any row of the tile meets
  int64_t c_begin = 0, c_end = t.nb;
  if (a.causal) {
    if (DKV) c_begin = max64(0, first - shift) / BN * BN;
    else c_end = min64(c_end, max64(first + t.rows + shift, 0));
  }
  const float qscale = a.scale * kLog2e;
  const int block_head = blockIdx.x % nheads, kvh = DKV ? block_head : block_head / group;
  const int head0 = DKV ? kvh * group : block_head, heads = DKV ? group : 1;
  const T* kp = (const T*)a.k + kvh * a.k_sh;
  const T* vp = (const T*)a.v + kvh * a.v_sh;
  float acc1[RM][DP / TX], acc2[DKV ? RM : 1][DKV ? DP / TX : 1];
#pragma unroll
  for (int r = 0; r < RM; ++r)
#pragma unroll
    for (int c = 0; c < DP / TX; ++c) {
      acc1[r][c] = 0.f;
      if (DKV) acc2[r][c] = 0.f;
    }
  float row_lse[RM], row_delta[RM];
  if (DKV) {
    load_tile<T, VEC, DP>(x1, kp + t.row0 * a.k_st, a.k_st, BM, t.rows, a.D);
    load_tile<T, VEC, DP>(x2, vp + t.row0 * a.v_st, a.v_st, BM, t.rows, a.D);
  } else {
    load_tile<T, VEC, DP>(x1, (const T*)a.q + t.row0 * a.q_st + head0 * a.q_sh, a.q_st, BM, t.rows, a.D);
    load_tile<T, VEC, DP>(x2, (const T*)a.go + t.row0 * a.go_st + head0 * a.go_sh, a.go_st, BM, t.rows, a.D);
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const int row = ty + TY * r;
      const bool in = row < t.rows;
      row_lse[r] = in ? a.lse[(int64_t)head0 * a.Tq + t.row0 + row] * kLog2e : 0.f;
      row_delta[r] = in ? a.delta[(int64_t)head0 * a.Tq + t.row0 + row] : 0.f;
    }
  }
  for (int h = 0; h < heads; ++h) {
    const int head = head0 + h;
    for (int64_t c0 = c_begin; c0 < c_end; c0 += BN) {
      const int valid = (int)min64(c_end - c0, BN);
      __syncthreads();
      if (DKV) {
        const int64_t tok = t.b0 + c0;
        load_tile<T, VEC, DP>(y1, (const T*)a.q + tok * a.q_st + head * a.q_sh, a.q_st, BN, valid, a.D);
        load_tile<T, VEC, DP>(y2, (const T*)a.go + tok * a.go_st + head * a.go_sh, a.go_st, BN, valid, a.D);
        if (threadIdx.x < BN) {
          const bool in = threadIdx.x < valid;
          cl[threadIdx.x] = in ? a.lse[(int64_t)head * a.Tq + tok + threadIdx.x] * kLog2e : 0.f;
          cd[threadIdx.x] = in ? a.delta[(int64_t)head * a.Tq + tok + threadIdx.x] : 0.f;
        }
      } else {
        load_tile<T, VEC, DP>(y1, kp + (t.b0 + c0) * a.k_st, a.k_st, BN, valid, a.D);
        load_tile<T, VEC, DP>(y2, vp + (t.b0 + c0) * a.v_st, a.v_st, BN, valid, a.D);
      }
      __syncthreads();
      float s[RM][CN], dp[RM][CN];
      product_nt<DP, TY, TX, RM, CN>(s, x1, y1, ty, tx);
      product_nt<DP, TY, TX, RM, CN>(dp, x2, y2, ty, tx);
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        const int row = ty + TY * r;
        int64_t lo = 0, hi = row < t.rows ? valid : 0;  // columns that this row meets
        if (a.causal) {
          if (DKV) lo = first + row - shift - c0;       // queries from the key's place - shift on
          else hi = min64(hi, first + row + shift + 1 - c0);
        }
#pragma unroll
        for (int c = 0; c < CN; ++c) {
          const int col = tx + TX * c;
          const float lse = DKV ? cl[col] : row_lse[r], delta = DKV ? cd[col] : row_delta[r];
          const bool in = col >= lo && col < hi;
          s[r][c] = in ? exp2f(fmaf(s[r][c], qscale, -lse)) : 0.f;
          dp[r][c] = in ? s[r][c] * (dp[r][c] - delta) : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        float x[RM], y[RM];
#pragma unroll
        for (int r = 0; r < RM; ++r) x[r] = s[r][c], y[r] = dp[r][c];
        if (DKV) put_rows<BM, RM>(ps, tx + TX * c, ty, x);
        put_rows<BM, RM>(ds, tx + TX * c, ty, y);
      }
      __syncthreads();
      product_nn<DP, TY, TX, RM, BN>(acc1, ds, y1, ty, tx);
      if constexpr (DKV) product_nn<DP, TY, TX, RM, BN>(acc2, ps, y2, ty, tx);
    }
  }
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int row = ty + TY * r;
    if (row >= t.rows) continue;
    const int64_t at = ((int64_t)(t.row0 + row) * (DKV ? a.Hk : a.H) + (DKV ? kvh : head0)) * a.D;
    T* d1 = (T*)(DKV ? a.dk : a.dq) + at;
    T* d2 = DKV ? (T*)a.dv + at : nullptr;
#pragma unroll
    for (int g = 0; g < DP / TX / 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = tx * 4 + g * 4 * TX + i;
        if (c < a.D) {
          d1[c] = from_acc<T>(acc1[r][g * 4 + i] * a.scale);
          if (DKV) d2[c] = from_acc<T>(acc2[r][g * 4 + i]);
        }
      }
  }
}

// delta = dO . O per (head, token), and where asked for the row's |dO| (with a zero for the
// largest |v|^2, which the next kernel raises) and its log-sum-exp in base 2; lpr lanes per
// row, vectors of VEC.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) packed_delta_kernel(const PackedArgs a, int lpr) {
  const int64_t rows = a.Tq * a.H;
  const int rpb = 256 / lpr, l = threadIdx.x % lpr;
  for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < rows; r0 += (int64_t)gridDim.x * rpb) {
    const int64_t r = r0 + threadIdx.x / lpr;
    float s = 0.f, square = 0.f;
    int64_t tok = 0;
    int head = 0;
    if (r < rows) {
      // a 64-bit division costs more than the row itself
      tok = rows <= 0xffffffffll ? (int64_t)((uint32_t)r / (uint32_t)a.H) : r / a.H;
      head = (int)(r - tok * a.H);
      const T* o = (const T*)a.o + r * a.D;
      const T* g = (const T*)a.go + tok * a.go_st + head * a.go_sh;
      for (int c = l * VEC; c < a.D; c += lpr * VEC) {
        float x[VEC], y[VEC];
        load_vec<VEC>(o + c, x);
        load_vec<VEC>(g + c, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s += x[i] * y[i];
          square += y[i] * y[i];
        }
      }
    }
    for (int x = lpr / 2; x > 0; x >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, x);
      square += __shfl_xor_sync(0xffffffffu, square, x);
    }
    if (r < rows && l == 0) {
      a.delta[(int64_t)head * a.Tq + tok] = s;
      if (a.ds_bound) {
        a.ds_bound[(int64_t)head * a.Tq + tok] = sqrtf(square);
        a.v_max[(int64_t)head * a.Tq + tok] = 0.f;
      }
      if (a.lse2) a.lse2[(int64_t)head * a.Tq + tok] = fmaf(a.lse[(int64_t)head * a.Tq + tok], kLog2e, a.ds_bound ? -(float)kHalfLift : 0.f);
    }
  }
}

template <typename K>
int set_smem(K kern, int bytes) {
  return cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

template <typename T, int VEC, int DP, int RM>
int fwd(const PackedArgs& a, cudaStream_t st) {
  using Sh = FwdShape<DP, RM>;
  auto kern = packed_simt_fwd_kernel<T, VEC, DP, RM>;
  int s = set_smem(kern, Sh::smem);
  if (s) return s;
  unsigned blocks;
  if ((s = packed_grid(a.Tq, a.B, Sh::BM, a.H, &blocks))) return s;
  kern<<<blocks, kThreads, Sh::smem, st>>>(a);
  return check_launch();
}

template <typename T, int VEC, int DP, int RM>
int bwd(const PackedArgs& a, cudaStream_t st) {
  using Sh = BwdShape<DP, RM>;
  if (a.dk && a.Tk > 0) {
    auto kern = packed_simt_bwd_kernel<T, VEC, DP, RM, true>;
    int s = set_smem(kern, Sh::smem);
    if (s) return s;
    unsigned blocks;
    if ((s = packed_grid(a.Tk, a.B, Sh::BM, a.Hk, &blocks))) return s;
    kern<<<blocks, kThreads, Sh::smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  if (a.dq && a.Tq > 0) {
    auto kern = packed_simt_bwd_kernel<T, VEC, DP, RM, false>;
    int s = set_smem(kern, Sh::smem);
    if (s) return s;
    unsigned blocks;
    if ((s = packed_grid(a.Tq, a.B, Sh::BM, a.H, &blocks))) return s;
    kern<<<blocks, kThreads, Sh::smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  return TPO_OK;
}

// 16-byte loads where every row of every input starts on 16 bytes and the width
// is whole vectors.
template <typename T>
bool vec_ok(const PackedArgs& a, bool backward) {
  constexpr int V = 16 / sizeof(T);
  auto ok = [](const void* p, int64_t s1, int64_t s2) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s1 % V == 0 && s2 % V == 0;
  };
  return a.D % V == 0 && ok(a.q, a.q_st, a.q_sh) && ok(a.k, a.k_st, a.k_sh) && ok(a.v, a.v_st, a.v_sh) &&
         (!backward || ok(a.go, a.go_st, a.go_sh));
}

template <typename T, int VEC>
int fwd_width(const PackedArgs& a, cudaStream_t st) {
  if (a.D <= 64) return fwd<T, VEC, 64, 4>(a, st);
  if (a.D <= 128) return fwd<T, VEC, 128, 4>(a, st);
  return fwd<T, VEC, 256, 2>(a, st);
}
template <typename T, int VEC>
int bwd_width(const PackedArgs& a, cudaStream_t st) {
  if (a.D <= 64) return bwd<T, VEC, 64, 4>(a, st);
  if (a.D <= 128) return bwd<T, VEC, 128, 4>(a, st);
  return bwd<T, VEC, 256, 2>(a, st);
}

template <typename T>
int fwd_typed(const PackedArgs& a, cudaStream_t st) {
  return vec_ok<T>(a, false) ? fwd_width<T, 16 / sizeof(T)>(a, st) : fwd_width<T, 1>(a, st);
}
template <typename T>
int bwd_typed(const PackedArgs& a, cudaStream_t st) {
  return vec_ok<T>(a, true) ? bwd_width<T, 16 / sizeof(T)>(a, st) : bwd_width<T, 1>(a, st);
}

template <typename T, int VEC>
int delta_launch(const PackedArgs& a, cudaStream_t st) {
  int lpr = 32;
  while (lpr > 1 && (lpr / 2) * VEC >= a.D) lpr /= 2;
  const int rpb = 256 / lpr;
  packed_delta_kernel<T, VEC><<<(unsigned)min64((a.Tq * a.H + rpb - 1) / rpb, 148 * 16), 256, 0, st>>>(a, lpr);
  return check_launch();
}
template <typename T>
int delta_typed(const PackedArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = a.D % V == 0 && (reinterpret_cast<uintptr_t>(a.go) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.o) & 15) == 0 && a.go_st % V == 0 && a.go_sh % V == 0;
  return vec ? delta_launch<T, V>(a, st) : delta_launch<T, 1>(a, st);
}

}  // namespace

#define TPO_DISPATCH(F)                                              \
  switch (dtype) {                                                   \
    case TPO_F32: return F<float>(a, st);                            \
    case TPO_F16: return F<__half>(a, st);                           \
    case TPO_BF16: return F<__nv_bfloat16>(a, st);                   \
    default: return set_error(TPO_ERR_INVALID_ARGUMENT, "packed_attention: dtype must be f32, f16 or bf16"); \
  }

int packed_simt_forward(int dtype, const PackedArgs& a, cudaStream_t st) { TPO_DISPATCH(fwd_typed) }
int packed_simt_backward(int dtype, const PackedArgs& a, cudaStream_t st) { TPO_DISPATCH(bwd_typed) }
int packed_delta(int dtype, const PackedArgs& a, cudaStream_t st) { TPO_DISPATCH(delta_typed) }

int attention_simt_error_word(unsigned** word) { return attention_error_word(word); }

}  // namespace tpo
