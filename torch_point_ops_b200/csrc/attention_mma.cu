// Attention over packed clouds on the tensor cores: 16-bit inputs, width a
// multiple of 8 up to 128, rows on 16-byte boundaries.
//
// All products are tcgen05 with fp32 accumulators in tensor memory (TMEM).  A block has
// row warps (a thread owns a row of the score tile), two copy warps and a warp that issues
// products (two warps in the backward), one elected lane of it; tiles travel through a ring in
// shared memory.
//
// The tensor cores take no wider operand beside 16-bit ones.  P is rounded to 16 bits
// before it multiplies V (and dO): that adds about as much error as the rounding of the
// result.  dS is a difference of large terms that the gradients sum up.  With delta from
// the rounded O and one rounding, dQ and dK of causal clouds come out 1.5 to 1.6 times as
// far from the exact ones as their own rounding puts them.  So for dQ it travels as two 16-bit
// values (its rounding and what that left: 1.1 times); the dQ kernel also sums delta = P dP
// without O's rounding, and with that one rounding does for dK (1.4 times).
// Every sum, maximum, P and dS themselves are fp32.
//
// Measured (B200, bf16, 4 causal clouds of 4096 tokens, 16 heads; of the products that the
// formulas need): width 128 forward 270 to 280 us (1.0 PFLOP/s; two clouds without causal: 1.1),
// dQ and dK dV together 1.24 ms (0.55); width 64 forward 240 to 275 us, backward 0.76 to
// 0.81 ms.  Width 128: the tensor pipe is 47 to 49 % busy, P V and the next S follow one another
// on the tile that waits for them.  Width 64: the exponentials (special-function unit 57 %
// busy) and the row threads' issue slots.  The clock falls to 1.4 to 1.6 GHz under the power
// limit in long runs.
#include <type_traits>

#include "attention_common.cuh"
#include "tcgen05.cuh"

namespace tpo {
namespace {

constexpr int kTile = 128;  // rows of a block's own tiles
constexpr int kCopyThreads = 64;

// ROWS rows of a packed tensor into a swizzled tile, by THREADS threads (t = index).
// Rows at or beyond `valid` and columns at or beyond D become zeros: nothing from
// another cloud enters a product (0 * NaN would).  A whole tile takes an address
// addition and a copy per 16 bytes: two warps have to keep up with the tensor core.
template <typename T, int DP, int ROWS, int THREADS = kCopyThreads>
__device__ __forceinline__ void copy_tile(uint32_t dst, const T* src, int64_t stride, int valid, int D, int t) {
  constexpr int CH = DP / 8;               // 16-byte chunks per row
  constexpr int STEP = THREADS / CH;       // rows per pass: 4, 8 or 16
  const int c = t % CH, r0 = t / CH;
  const bool col = c * 8 < D;
  const uint32_t at = dst + (c >> 3) * ROWS * kPanelRow + r0 * kPanelRow;
  // the swizzle depends on the row modulo 8: the same in every second pass
  const uint32_t even = at + (((c & 7) ^ (r0 & 7)) << 4), odd = at + (((c & 7) ^ ((r0 + STEP) & 7)) << 4);
  const T* p = src + (int64_t)r0 * stride + (col ? c * 8 : 0);
  const int64_t hop = STEP * stride;
  if (valid >= ROWS) {
#pragma unroll
    for (int i = 0; i < ROWS / STEP; ++i) {
      cp_async16((i & 1 ? odd : even) + i * STEP * kPanelRow, p, col);
      p += hop;
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < ROWS / STEP; ++i) {
      const bool in = r0 + i * STEP < valid;
      cp_async16((i & 1 ? odd : even) + i * STEP * kPanelRow, in ? p : src, in && col);
      p += hop;
    }
  }
}

// d (+)= x y^T over the width: x 128 rows, y NY rows, both K-major.
template <typename T, int DP, int NY>
__device__ __forceinline__ void mma_nt(uint32_t lane, uint32_t d, uint32_t x, uint32_t y) {
  constexpr uint32_t id = mma_desc<T>(kTile, NY, false);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks)
    mma_ss(lane, d, smem_desc(x + (ks / 4) * kTile * kPanelRow + (ks % 4) * 32, 16),
           smem_desc(y + (ks / 4) * NY * kPanelRow + (ks % 4) * 32, 16), id, ks > 0);
}
// d (+)= p y over y's NY rows: p 128 rows of 16-bit values in TMEM, y MN-major.
template <typename T, int DP, int NY>
__device__ __forceinline__ void mma_nn(uint32_t lane, uint32_t d, uint32_t p, uint32_t y, bool more) {
  constexpr uint32_t id = mma_desc<T>(kTile, DP, true);
#pragma unroll
  for (int ks = 0; ks < NY / 16; ++ks)
    mma_ts(lane, d, p + ks * 8, smem_desc(y + ks * 16 * kPanelRow, NY * kPanelRow), id, more || ks > 0);
}

// 32 accumulator columns times f as 16-bit values to global memory, whole chunks of 8.
template <typename T>
__device__ __forceinline__ void store32(T* out, const uint32_t (&v)[32], float f, int col, int D) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (col + i >= D) continue;
    uint4 o;
    uint32_t* ov = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      ov[e] = pack2<T>(__uint_as_float(v[i + 2 * e]) * f, __uint_as_float(v[i + 2 * e + 1]) * f);
    *reinterpret_cast<uint4*>(out + col + i) = o;
  }
}

// The ring of copied tiles.  A tile is announced by the copies themselves (each copy
// thread's arrival follows its last copy); the reader orders them before the tensor
// core's reads with a proxy fence.  A stage is handed back only where another tile will
// fill it, so that no arrival is still on its way when the block ends.
template <int ST>
struct Ring {
  uint32_t full, empty;  // barrier arrays
  int tiles;
  volatile int* abort;
  __device__ __forceinline__ void wait_empty(int i) const {
    if (i >= ST) bar_wait(empty + 8 * (i % ST), (i / ST - 1) & 1, abort, &g_attention_error);
  }
  __device__ __forceinline__ void announce(int i) const { cp_async_arrive(full + 8 * (i % ST)); }
  __device__ __forceinline__ void wait_full(int i) const {
    bar_wait(full + 8 * (i % ST), (i / ST) & 1, abort, &g_attention_error);
  }
  __device__ __forceinline__ void wait_operand(int i) const {
    wait_full(i);
    fence_async_smem();
  }
  __device__ __forceinline__ void release(uint32_t lane, int i) const {
    if (i + ST < tiles) mma_commit(lane, empty + 8 * (i % ST));
  }
};

// ---------------------------------------------------------------- forward
// TILES tiles of 128 query rows pass once over the keys in tiles of 128.
//
// Width above 64: two query tiles per block (one block per SM), which share every key
// and value tile; while one tile's softmax runs, the tensor core works for the
// other.  TMEM is full (two S, two O), so P lies over the S that it was made from and
// the next S waits for P V.
//
// Width up to 64: one tile per block and two blocks per SM, which hide each other's
// start and end, and half the waste on short clouds; P has columns of its own, so the next
// S is computed as soon as this one is read.
template <int DP>
struct Fwd {
  static constexpr int TILES = DP == 128 ? 2 : 1;
  static constexpr bool APART = DP == 64;  // P apart from S
  static constexpr int threads = TILES * 128 + 128;
  static constexpr int row_regs = 200, other_regs = TILES == 2 ? 104 : 56;
  static constexpr int launch_regs = TILES == 2 ? 168 : 128;
  static_assert(TILES * 128 * row_regs + 128 * other_regs <= threads * launch_regs, "register split");
  static constexpr int tile = kTile * DP * 2;
  static constexpr int stages = 5;
  static constexpr int bars = (TILES + stages) * tile;
  static constexpr int smem = bars + 256 + 1024;  // + alignment of the base
  static constexpr int tmem = TILES * 256;
  static constexpr int s = 0, p = APART ? 128 : 0, o = APART ? 192 : TILES * 128;  // columns
};

template <typename T, int DP>
__global__ void __launch_bounds__(Fwd<DP>::threads, Fwd<DP>::TILES == 2 ? 1 : 2)
    packed_mma_fwd_kernel(const PackedArgs a) {
  using F = Fwd<DP>;
  constexpr int ST = F::stages, TILES = F::TILES;
  constexpr int kCopyWarp = TILES * 4, kMmaWarp = kCopyWarp + 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  const uint32_t sq = base, skv = base + TILES * F::tile, bars = base + F::bars;
  const uint32_t b_q = bars, b_full = bars + 16, b_empty = b_full + 8 * ST, b_s = b_empty + 8 * ST, b_p = b_s + 16,
                 b_o = b_p + 16, b_read = b_o + 16, s_tmem = b_read + 16, s_abort = s_tmem + 4;
  volatile int* abort = reinterpret_cast<volatile int*>(smem_raw + (s_abort - raw));
  unsigned* err = &g_attention_error;

  const int warp = threadIdx.x / 32, head = blockIdx.x % a.H, kvh = head / (a.H / a.Hk);
  const Tile t = find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, TILES * kTile, blockIdx.x / a.H, gridDim.x / a.H, a.causal);
  if (t.rows <= 0) return;
  const int first = t.row0 - t.a0;
  int steps[TILES], n = 0;  // key tiles that each query tile meets
#pragma unroll
  for (int w = 0; w < TILES; ++w) {
    const int rows = max(0, min(kTile, t.rows - w * kTile));
    const int nk = rows == 0 ? 0 : a.causal ? max(t.edge(first + w * kTile + rows), 0) : t.nb;
    steps[w] = (nk + kTile - 1) / kTile;
    n = max(n, steps[w]);
  }

  if (warp == kMmaWarp) {
    if (threadIdx.x % 32 == 0) {
      for (int i = 0; i < ST; ++i) {
        bar_init(b_full + 8 * i, kCopyThreads);
        bar_init(b_empty + 8 * i, 1);
      }
      for (int w = 0; w < TILES; ++w) {
        bar_init(b_q + 8 * w, 128);
        bar_init(b_s + 8 * w, 1);
        bar_init(b_p + 8 * w, 128);
        bar_init(b_o + 8 * w, 1);
        bar_init(b_read + 8 * w, 128);
      }
      *abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tmem_alloc(s_tmem, F::tmem);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(s_tmem));
  const uint32_t t_s = tmem + F::s, t_p = tmem + F::p, t_o = tmem + F::o;
  const Ring<ST> ring = {b_full, b_empty, 2 * n, abort};

  if (warp >= kCopyWarp) {
    give_registers<F::other_regs>();
    if (warp < kMmaWarp) {
      // ---- copies: K0 V0 K1 V1 ... ----
      const int tid = threadIdx.x - 32 * kCopyWarp;
      if (n > 0) {
        const T* kp = (const T*)a.k + t.b0 * a.k_st + kvh * a.k_sh;
        const T* vp = (const T*)a.v + t.b0 * a.v_st + kvh * a.v_sh;
        for (int i = 0; i < 2 * n; ++i) {
          ring.wait_empty(i);
          const int j = (i >> 1) * kTile;
          const uint32_t dst = skv + (i % ST) * F::tile;
          if (i & 1) copy_tile<T, DP, kTile>(dst, vp + j * a.v_st, a.v_st, t.nb - j, a.D, tid);
          else copy_tile<T, DP, kTile>(dst, kp + j * a.k_st, a.k_st, t.nb - j, a.D, tid);
          ring.announce(i);
        }
        cp_async_wait_all();
      }
    } else if (warp == kMmaWarp && n > 0) {
      // ---- products: the warp stays together, one lane issues ----
      const uint32_t one = elect_lane();
      const uint32_t u_tmem = uniform(tmem), u_base = uniform(base);
      const uint32_t u_s = u_tmem + F::s, u_p = u_tmem + F::p, u_o = u_tmem + F::o, u_q = u_base, u_kv = u_base + TILES * F::tile;
      const int un = (int)uniform(n);  // loops and stages count in uniform registers too
      auto score = [&](int w, int j) {  // S_w = Q_w K_j^T
        mma_nt<T, DP, kTile>(one, u_s + w * kTile, u_q + w * F::tile, u_kv + ((2 * j) % ST) * F::tile);
        mma_commit(one, b_s + 8 * w);
      };
      ring.wait_full(0);
#pragma unroll
      for (int w = 0; w < TILES; ++w)
        if (steps[w] > 0) {
          bar_wait(b_q + 8 * w, 0, abort, err);
          fence_async_smem();
          score(w, 0);
        }
      ring.release(one, 0);
      for (int j = 0; j < un; ++j) {
        const int iv = 2 * j + 1, ik = 2 * j + 2;
        const uint32_t v = u_kv + (iv % ST) * F::tile;
        if (F::APART && j + 1 < un) {
          bar_wait(b_read, j & 1, abort, err);
          tc_fence_after();
          ring.wait_operand(ik);
          score(0, j + 1);
          ring.release(one, ik);
        }
        ring.wait_operand(iv);
        if (!F::APART && j + 1 < un) ring.wait_operand(ik);
#pragma unroll
        for (int w = 0; w < TILES; ++w) {
          if (j >= steps[w]) continue;
          bar_wait(b_p + 8 * w, j & 1, abort, err);
          tc_fence_after();
          mma_nn<T, DP, kTile>(one, u_o + w * DP, u_p + w * kTile, v, j > 0);
          if (F::APART || j + 1 == steps[w]) mma_commit(one, b_o + 8 * w);
          else score(w, j + 1);
        }
        ring.release(one, iv);
        if (!F::APART) ring.release(one, ik);
      }
    }
  } else {
    // ---- softmax: a thread owns a row ----
    draw_registers<F::row_regs>();
    const int w = warp / 4, row = threadIdx.x % kTile;
    if (t.rows > w * kTile) {  // its queries
      copy_tile<T, DP, kTile, 128>(sq + w * F::tile, (const T*)a.q + (int64_t)(t.row0 + w * kTile) * a.q_st + head * a.q_sh, a.q_st,
                                   t.rows - w * kTile, a.D, row);
      cp_async_arrive(b_q + 8 * w);
    }
    const uint32_t lane = (uint32_t)(warp % 4) * 32 << 16;
    const uint32_t ts = t_s + w * kTile + lane, tp = t_p + w * kTile + lane, to = t_o + w * DP + lane;
    const bool live = w * kTile + row < t.rows;
    const float qscale = a.scale * kLog2e;
    const int my_steps = w == 0 ? steps[0] : steps[TILES - 1];
    // this row sees keys below `sees`
    const int sees = a.causal ? min(t.nb, max(0, t.edge(first + w * kTile + row + 1))) : t.nb;
    float m = -INFINITY, l = 0.f;
    // one step's row: masked columns count as -inf
    auto step = [&](int j, int lim, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, v[c]);
      tmem_wait_ld();
      if (F::APART) {
        tc_fence_before();
        bar_arrive(b_read);
      }
      if (MASK) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[c][i] = c * 32 + i < lim ? v[c][i] : 0xff800000u;
      }
      float mx[4];  // four chains: a maximum waits for the one before it
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = m;
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx[c] = max3(mx[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
      }
      const float top = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
      if (F::APART && j > 0) {  // O and P are free: P V of the step before is done
        bar_wait(b_o, (j - 1) & 1, abort, err);
        tc_fence_after();
      }
      // The base of the exponentials moves only when a maximum outgrows it by
      // more than 2^8: P stays below 256 (exact scaling by a power of the base is
      // undone by the division), and O is seldom rescaled.
      const bool grow = (top - m) * qscale > 8.f;  // also the first finite maximum: m = -inf
      if (__any_sync(0xffffffffu, grow)) {
        const float corr = grow ? ex2((m - top) * qscale) : 1.f;
        if (grow) m = top;
        l *= corr;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            uint32_t o[16];
            tmem_ld16(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(to + c, o);
          }
        }
      }
      const float mb = m == -INFINITY ? 0.f : m * qscale;
      const u64 q2 = pk(qscale, qscale), m2 = pk(-mb, -mb);
      u64 sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x, y;
          upk(fma2(pku(v[c][2 * i], v[c][2 * i + 1]), q2, m2), x, y);
          x = ex2(x), y = ex2(y);
          sum[i & 1] = add2(sum[i & 1], pk(x, y));
          p[i] = pack2<T>(x, y);
        }
        tmem_st16(tp + c * 16, p);
      }
      float x, y;
      upk(add2(sum[0], sum[1]), x, y);
      l += x + y;
      tmem_wait_st();
      tc_fence_before();
      bar_arrive(b_p + 8 * w);
    };
    for (int j = 0; j < my_steps; ++j) {
      const int lim = min(kTile, max(0, sees - j * kTile));
      const bool whole = __all_sync(0xffffffffu, lim == kTile);
      bar_wait(b_s + 8 * w, j & 1, abort, err);
      tc_fence_after();
      if (whole) step(j, lim, std::false_type{});
      else step(j, lim, std::true_type{});
    }
    const int64_t tok = t.row0 + w * kTile + row;
    if (live && a.lse) a.lse[(int64_t)head * a.Tq + tok] = l == 0.f ? -INFINITY : (m * qscale + log2f(l)) * kLn2;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    T* op = (T*)a.o + (tok * a.H + head) * a.D;
    if (my_steps > 0) {
      bar_wait(b_o + 8 * w, F::APART ? (my_steps - 1) & 1 : 0, abort, err);
      tc_fence_after();
    }
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
      uint32_t v[32];
      if (my_steps > 0) {
        tmem_ld32(to + c, v);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
      if (live) store32<T>(op, v, inv, c, a.D);
    }
    cp_async_wait_all();
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, F::tmem);
  }
}

// ---------------------------------------------------------------- backward
// P = exp(S - lse) and dS = P * (dP - delta) are rebuilt tile by tile from S and dP,
// which are recomputed.  DKV: rows are the block's 128 keys (x1 = K, x2 = V), the
// streamed columns are queries (y1 = Q, y2 = dO) of every head of the group;
// acc1 = dK += dS^T Q, acc2 = dV += P^T dO.  Otherwise rows are 128 queries
// (x1 = Q, x2 = dO), columns keys (y1 = K, y2 = V), acc1 = dQ += dS K.  In both,
// S = x1 y1^T, dP = x2 y2^T, and P and dS go back to TMEM as A operands, over S and dP.
// Each sum has one owner: no atomics, the same bits in every run.
//
// Columns come in tiles of 64.  Width above 64: two groups of row warps with their own S
// and dP take tiles in turn, so the tensor core works for one while the other
// computes.  Width up to 64: one group per block, two blocks per SM.
constexpr int kCols = 64;
template <int DP>
struct Bwd {
  static constexpr int GROUPS = DP == 128 ? 2 : 1;
  static constexpr int threads = GROUPS * 128 + 128;
  static constexpr int row_regs = 200, other_regs = GROUPS == 2 ? 104 : 56;
  static constexpr int launch_regs = GROUPS == 2 ? 168 : 128;
  static_assert(GROUPS * 128 * row_regs + 128 * other_regs <= threads * launch_regs, "register split");
  static constexpr int own = kTile * DP * 2, tile = kCols * DP * 2;
  static constexpr int stages = 8;
  static constexpr int stats = 2 * own + stages * tile;  // 64 floats per stage: base-2 lse with y1, delta with y2 (DKV)
  static constexpr int bars = stats + stages * kCols * 4;
  static constexpr int smem = bars + 256 + 1024;
  static constexpr int tmem = GROUPS * 256;
  static constexpr int acc1 = GROUPS * 128, acc2 = acc1 + DP;  // columns; S and dP of group g at 128 g and 128 g + 64
};

// P of the backward is normalised, about one over the number of keys: fp16 holds it as 2^12 P (the
// statistics bring the exponent along), or a few 10^4 keys would take it into the subnormal numbers
// (50000 keys: 1.4e-3 off in dV, against 4.9e-4 that a rounding costs).  2^12 leaves a
// factor of 16 to the largest fp16.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? (float)(1 << kHalfLift) : 1.f;

// dS of fp16 needs a power of two beside it, or it leaves the type's range at either end.
// By |dP| <= |dO| |v|, and since P (1 - P) <= 1/4 of the spread of dP is the most that a dS
// can be, |dS| <= |dO| max |v| / 2 over the keys that the row's tile meets.  2^(15 - e) with 2^e the
// power of two at or below that product (without the half) brings |dS| to 2^15 at most: a
// factor of two from the largest fp16 for what P and delta are off, and all of the range below
// for small P (undone when acc1 leaves).
__device__ __forceinline__ float grad_scale(float bound) {
  const unsigned e = __float_as_uint(bound) >> 23;
  return e < 15 || e >= 0xfe ? 1.f : __uint_as_float((269 - e) << 23);
}

// The largest |v|^2 of each tile of keys and kv head, in the slots of its cloud's queries (the last
// one has all further tiles); rows that are not finite
// are left out: what they spoil is spoilt whatever the scale is.  A maximum is the same in any
// order.  Four lanes share a row, and every load of a tile is in flight at once: 9.5 us for two
// clouds of 4096 to 8192 tokens, 8 heads of width 128 (0.4 % of the backward), 3 us for small ones.
template <int DP>
__global__ void __launch_bounds__(128) packed_value_max_kernel(const PackedArgs a) {
  constexpr int PASSES = kTile / 32, VECS = DP / 32;
  __shared__ unsigned best[4];
  const int kvh = blockIdx.x % a.Hk, l = threadIdx.x % 4, r = threadIdx.x / 4;
  const Tile t = find_tile(a.off_k, a.Tk, a.off_q, a.Tq, a.B, kTile, blockIdx.x / a.Hk, gridDim.x / a.Hk, false);
  if (t.rows <= 0 || t.nb <= 0) return;
  const __half* vp = (const __half*)a.v + t.row0 * a.v_st + kvh * a.v_sh;
  Pack<__half, 8> raw[PASSES][VECS];
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int x = 0; x < VECS; ++x) {
      const int row = i * 32 + r, c = (x * 4 + l) * 8;
      *reinterpret_cast<uint4*>(&raw[i][x]) = make_uint4(0, 0, 0, 0);
      if (row < t.rows && c < a.D) raw[i][x] = *reinterpret_cast<const Pack<__half, 8>*>(vp + row * a.v_st + c);
    }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < VECS; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float lo, hi;
        pair_of(raw[i][x], e, lo, hi);
        s = fmaf(lo, lo, fmaf(hi, hi, s));
      }
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    if (s < INFINITY) top = fmaxf(top, s);
  }
  const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // not negative: ordered as integers
  if (threadIdx.x % 32 == 0) best[threadIdx.x / 32] = bits;
  __syncthreads();
  if (threadIdx.x == 0)
    atomicMax(reinterpret_cast<unsigned*>(a.v_max) + (int64_t)kvh * (a.H / a.Hk) * a.Tq + t.b0 +
                  min((t.row0 - t.a0) / kTile, t.nb - 1),
              max(max(best[0], best[1]), max(best[2], best[3])));
}

template <typename T, int DP, bool DKV>
__global__ void __launch_bounds__(Bwd<DP>::threads, Bwd<DP>::GROUPS == 2 ? 1 : 2)
    packed_mma_bwd_kernel(const PackedArgs a) {
  using W = Bwd<DP>;
  constexpr int ST = W::stages, GROUPS = W::GROUPS;
  constexpr int kCopyWarp = GROUPS * 4, kMmaWarp = kCopyWarp + 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  const uint32_t sx1 = base, sx2 = base + W::own, sy = base + 2 * W::own, bars = base + W::bars;
  const float* stats = reinterpret_cast<const float*>(smem_raw + (base + W::stats - raw));
  const uint32_t b_x = bars, b_full = bars + 8, b_empty = b_full + 8 * ST, b_s = b_empty + 8 * ST, b_dp = b_s + 16,
                 b_p = b_dp + 16, b_ds = b_p + 16, b_used1 = b_ds + 16, b_used2 = b_used1 + 16, b_done = b_used2 + 16, s_tmem = b_done + 8, s_abort = s_tmem + 4;
  volatile int* abort = reinterpret_cast<volatile int*>(smem_raw + (s_abort - raw));
  unsigned* err = &g_attention_error;

  const int warp = threadIdx.x / 32, group = a.H / a.Hk;
  const int heads = DKV ? a.Hk : a.H, slot = blockIdx.x / heads, slots = gridDim.x / heads;
  const Tile t = DKV ? find_tile(a.off_k, a.Tk, a.off_q, a.Tq, a.B, kTile, slot, slots, false)
                     : find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, kTile, slot, slots, a.causal);
  if (t.rows <= 0) return;
  const int first = t.row0 - t.a0;
  int c_begin = 0, c_end = t.nb;  // columns that any row of the tile meets
  if (a.causal) {
    if (DKV) c_begin = max(0, t.edge(first)) / kCols * kCols;
    else c_end = max(t.edge(first + t.rows), 0);
  }
  const int per_head = max(0, (c_end - c_begin + kCols - 1) / kCols);
  const int block_head = blockIdx.x % heads;
  const int kvh = DKV ? block_head : block_head / group;
  const int head0 = DKV ? kvh * group : block_head;
  const int n = per_head * (DKV ? group : 1);

  if (warp == kMmaWarp) {
    if (threadIdx.x % 32 == 0) {
      bar_init(b_x, kCopyThreads);
      for (int i = 0; i < ST; ++i) {
        bar_init(b_full + 8 * i, kCopyThreads);
        bar_init(b_empty + 8 * i, 1);
      }
      for (int g = 0; g < GROUPS; ++g) {
        bar_init(b_s + 8 * g, 1);
        bar_init(b_dp + 8 * g, 1);
        bar_init(b_p + 8 * g, 128);
        bar_init(b_ds + 8 * g, 128);
        bar_init(b_used1 + 8 * g, 1);
        bar_init(b_used2 + 8 * g, 1);
      }
      bar_init(b_done, 1);
      *abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tmem_alloc(s_tmem, W::tmem);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(s_tmem));
  const uint32_t t_1 = tmem + W::acc1, t_2 = tmem + W::acc2;
  const Ring<ST> ring = {b_full, b_empty, 2 * n, abort};

  if (warp >= kCopyWarp) {
    give_registers<W::other_regs>();
    if (warp < kMmaWarp) {
      // ---- copies: x1 x2, then y1 y2 of column tile 0, 1, ... (DKV: head after head) ----
      const int tid = threadIdx.x - 32 * kCopyWarp;
      const T* kp = (const T*)a.k + kvh * a.k_sh;
      const T* vp = (const T*)a.v + kvh * a.v_sh;
      if (n > 0) {
        if (DKV) {
          copy_tile<T, DP, kTile>(sx1, kp + t.row0 * a.k_st, a.k_st, t.rows, a.D, tid);
          copy_tile<T, DP, kTile>(sx2, vp + t.row0 * a.v_st, a.v_st, t.rows, a.D, tid);
        } else {
          copy_tile<T, DP, kTile>(sx1, (const T*)a.q + t.row0 * a.q_st + head0 * a.q_sh, a.q_st, t.rows, a.D, tid);
          copy_tile<T, DP, kTile>(sx2, (const T*)a.go + t.row0 * a.go_st + head0 * a.go_sh, a.go_st, t.rows, a.D, tid);
        }
        cp_async_arrive(b_x);
        int h = 0, step = 0;
        for (int i = 0; i < 2 * n; ++i) {
          ring.wait_empty(i);
          const int s = i % ST;
          const int c0 = c_begin + step * kCols;
          const int64_t tok = t.b0 + c0;
          const uint32_t dst = sy + s * W::tile;
          if (DKV) {
            const int head = head0 + h;
            if (i & 1) copy_tile<T, DP, kCols>(dst, (const T*)a.go + tok * a.go_st + head * a.go_sh, a.go_st, t.nb - c0, a.D, tid);
            else copy_tile<T, DP, kCols>(dst, (const T*)a.q + tok * a.q_st + head * a.q_sh, a.q_st, t.nb - c0, a.D, tid);
            const float* from = (i & 1 ? a.delta : a.lse2) + (int64_t)head * a.Tq + tok;
            static_assert(kCols == kCopyThreads, "one statistic per copy thread");
            cp_async4(base + W::stats + (s * kCols + tid) * 4, c0 + tid < t.nb ? from + tid : a.lse2, c0 + tid < t.nb);
          } else {
            if (i & 1) copy_tile<T, DP, kCols>(dst, vp + tok * a.v_st, a.v_st, t.nb - c0, a.D, tid);
            else copy_tile<T, DP, kCols>(dst, kp + tok * a.k_st, a.k_st, t.nb - c0, a.D, tid);
          }
          if (i & 1) {
            if (++step == per_head) step = 0, ++h;
          }
          ring.announce(i);
        }
        cp_async_wait_all();
      }
    } else if (n > 0) {
      // ---- products: a warp stays together, one lane issues.  One warp computes S and dP, the other
      // dK and dV or dQ: waiting on a barrier costs some 130 clocks even when it is open,
      // and one warp alone would spend more on its four waits per tile than the products take.
      const uint32_t one = elect_lane();
      const uint32_t u_tmem = uniform(tmem), u_x1 = uniform(base), u_x2 = u_x1 + W::own, u_y = u_x1 + 2 * W::own;
      const int un = (int)uniform(n);  // loops and stages count in uniform registers too
      auto y_of = [&](int i) { return u_y + (i % ST) * W::tile; };
      auto s_of = [&](int j) { return u_tmem + (j % GROUPS) * 128; };
      if (warp == kMmaWarp) {
        bar_wait(b_x, 0, abort, err);
        fence_async_smem();
        for (int j = 0; j < un; ++j) {
          const int g = j % GROUPS, parity = (j / GROUPS - 1) & 1;
          ring.wait_operand(2 * j);
          if (j >= GROUPS) {  // S of the tile before is read (DKV: and its P has been multiplied)
            bar_wait((DKV ? b_used2 : b_p) + 8 * g, parity, abort, err);
            tc_fence_after();
          }
          mma_nt<T, DP, kCols>(one, s_of(j), u_x1, y_of(2 * j));
          mma_commit(one, b_s + 8 * g);
          ring.wait_operand(2 * j + 1);
          if (j >= GROUPS) {  // dS of the tile before has been multiplied
            bar_wait(b_used1 + 8 * g, parity, abort, err);
            tc_fence_after();
          }
          mma_nt<T, DP, kCols>(one, s_of(j) + 64, u_x2, y_of(2 * j + 1));
          mma_commit(one, b_dp + 8 * g);
          if (!DKV) ring.release(one, 2 * j + 1);
        }
      } else {
        for (int j = 0; j < un; ++j) {
          const int g = j % GROUPS, parity = (j / GROUPS) & 1;
          if (DKV) {
            bar_wait(b_p + 8 * g, parity, abort, err);
            tc_fence_after();
            ring.wait_operand(2 * j + 1);
            mma_nn<T, DP, kCols>(one, u_tmem + W::acc2, s_of(j), y_of(2 * j + 1), j > 0);
            if (j + GROUPS < un) mma_commit(one, b_used2 + 8 * g);
          }
          bar_wait(b_ds + 8 * g, parity, abort, err);
          tc_fence_after();
          fence_async_smem();  // y1 has landed: the other warp waited for it before S, and dS came after S
          mma_nn<T, DP, kCols>(one, u_tmem + W::acc1, s_of(j) + 64, y_of(2 * j), j > 0);
          if (!DKV) mma_nn<T, DP, kCols>(one, u_tmem + W::acc1, s_of(j) + 96, y_of(2 * j), true);
          if (j + GROUPS < un) mma_commit(one, b_used1 + 8 * g);
          ring.release(one, 2 * j);
          if (DKV) ring.release(one, 2 * j + 1);  // not before: the threads read delta from it
        }
        mma_commit(one, b_done);
      }
    }
  } else {
    draw_registers<W::row_regs>();
    const int g = warp / 4, row = threadIdx.x % kTile;
    const uint32_t lane = (uint32_t)(warp % 4) * 32 << 16;
    const uint32_t ts = tmem + g * 128 + lane, tdp = ts + 64;
    const bool live = row < t.rows;
    const float qscale = a.scale * kLog2e;
    float c = 1.f, big = 0.f;
    if (std::is_same<T, __half>::value) {
      // a row of dQ: its own bound; dK: every row's that the block meets
      if (!DKV) {
        const float* tiles = a.v_max + (int64_t)kvh * group * a.Tq + t.a0;
        for (int i = threadIdx.x % 32; i <= min((c_end - 1) / kTile, t.na - 1); i += 32) big = fmaxf(big, tiles[i]);
        big = sqrtf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big))));
        big *= live && n > 0 ? a.ds_bound[(int64_t)head0 * a.Tq + t.row0 + row] : 0.f;
        if (!(big < INFINITY)) big = 0.f;  // such a row's gradients are not finite whatever the scale is
      } else {
        for (int h = 0; h < group; ++h)
          for (int i = c_begin + threadIdx.x % 32; i < c_end; i += 32)
            big = fmaxf(big, a.ds_bound[(int64_t)(head0 + h) * a.Tq + t.b0 + i]);
        big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
      }
      c = grad_scale(big) / kLift<T>;
    }
    float row_lse = 0.f, row_delta = 0.f;
    if (!DKV && live) {
      row_lse = a.lse2[(int64_t)head0 * a.Tq + t.row0 + row];
      row_delta = a.delta[(int64_t)head0 * a.Tq + t.row0 + row];
    }
    u64 exact[2] = {0, 0};  // this row's sum of P dP over the group's tiles: delta without O's rounding (not DKV)
    // one step's row: P from S, then dS from dP
    auto step_rows = [&](int j, int lo, int hi, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      const int parity = (j / GROUPS) & 1;
      const u64 q2 = pk(qscale, qscale);
      u64 p[32];
      {
        const float* lse = stats + ((2 * j) % ST) * kCols;
        uint32_t v[2][32];
        bar_wait(b_s + 8 * g, parity, abort, err);
        if (DKV) ring.wait_full(2 * j);
        tc_fence_after();
        tmem_ld32(ts, v[0]);
        tmem_ld32(ts + 32, v[1]);
        tmem_wait_ld();
        if (!DKV) {  // S is read: the next product may overwrite it
          tc_fence_before();
          bar_arrive(b_p + 8 * g);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          u64 l0, l1;
          if (DKV) {
            const float4 f = *reinterpret_cast<const float4*>(lse + 2 * i);
            l0 = pk(-f.x, -f.y), l1 = pk(-f.z, -f.w);
          } else {
            l0 = l1 = pk(-row_lse, -row_lse);
          }
          const uint32_t* s = &v[i / 16][(2 * i) % 32];
          float x[4];
          upk(fma2(pku(s[0], s[1]), q2, l0), x[0], x[1]);
          upk(fma2(pku(s[2], s[3]), q2, l1), x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = ex2(x[e]);
            if (MASK) x[e] = 2 * i + e >= lo && 2 * i + e < hi ? x[e] : 0.f;
          }
          p[i] = pk(x[0], x[1]), p[i + 1] = pk(x[2], x[3]);
        }
      }
      if (DKV) {
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float x, y;
          upk(p[i], x, y);
          o[i] = pack2<T>(x, y);
        }
        tmem_st32(ts, o);
        tmem_wait_st();
        tc_fence_before();
        bar_arrive(b_p + 8 * g);
      }
      const float* delta = stats + ((2 * j + 1) % ST) * kCols;
      bar_wait(b_dp + 8 * g, parity, abort, err);
      if (DKV) ring.wait_full(2 * j + 1);
      tc_fence_after();
      uint32_t v[2][32];
      tmem_ld32(tdp, v[0]);
      tmem_ld32(tdp + 32, v[1]);
      tmem_wait_ld();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi16[16], lo16[16];
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const int i = 16 * h + k;
          u64 d0, d1;
          if (DKV) {
            const float4 f = *reinterpret_cast<const float4*>(delta + 2 * i);
            d0 = pk(f.x, f.y), d1 = pk(f.z, f.w);
          } else {
            d0 = d1 = pk(row_delta, row_delta);
          }
          const uint32_t* s = &v[h][2 * k];
          if (!DKV) {
            exact[0] = fma2(p[i], pku(s[0], s[1]), exact[0]);
            exact[1] = fma2(p[i + 1], pku(s[2], s[3]), exact[1]);
          }
          u64 a0 = mul2(p[i], sub2(pku(s[0], s[1]), d0)), a1 = mul2(p[i + 1], sub2(pku(s[2], s[3]), d1));
          if (std::is_same<T, __half>::value) a0 = mul2(a0, pk(c, c)), a1 = mul2(a1, pk(c, c));
          float x[4];
          upk(a0, x[0], x[1]);
          upk(a1, x[2], x[3]);
          if (MASK) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = 2 * i + e >= lo && 2 * i + e < hi ? x[e] : 0.f;
          }
          if (DKV) {
            hi16[k] = pack2<T>(x[0], x[1]);
            hi16[k + 1] = pack2<T>(x[2], x[3]);
          } else {
            hi16[k] = split2<T>(x[0], x[1], lo16[k]);
            hi16[k + 1] = split2<T>(x[2], x[3], lo16[k + 1]);
          }
        }
        tmem_st16(tdp + 16 * h, hi16);
        if (!DKV) tmem_st16(tdp + 32 + 16 * h, lo16);
      }
      tmem_wait_st();
      tc_fence_before();
      bar_arrive(b_ds + 8 * g);
    };
    // Columns [lo, hi) of a tile that the row meets.  Keys beyond the cloud's end must not
    // reach dS (their P is unbounded); queries beyond it have zero rows of Q and dO and
    // lse 0, so they add nothing.  Counted from c_begin.
    const int from = DKV && a.causal ? max(0, t.edge(first + row) - c_begin) : 0;
    const int to = DKV ? 0 : a.causal ? min(t.nb, max(0, t.edge(first + row + 1))) : t.nb;
    int step = per_head > 0 ? g % per_head : 0;
    for (int j = g; j < n; j += GROUPS) {
      const int lo = DKV ? min(kCols, max(0, from - step * kCols)) : 0;
      const int hi = DKV ? kCols : min(kCols, max(0, to - step * kCols));
      for (step += GROUPS; step >= per_head;) step -= per_head;
      if (__all_sync(0xffffffffu, lo == 0 && hi == kCols)) step_rows(j, lo, hi, std::false_type{});
      else step_rows(j, lo, hi, std::true_type{});
    }
    if (!DKV && n > 0) {  // for the kernel of dK and dV, which runs next
      float x, y;
      upk(add2(exact[0], exact[1]), x, y);
      x = (x + y) / kLift<T>;
      if (GROUPS == 2) {
        float* other = const_cast<float*>(stats);  // no statistics travel with keys: the space is free
        if (g == 1) other[row] = x;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (g == 0) x += other[row];
      }
      if (g == 0 && live) {  // both groups have read their rows' bounds: the barrier above
        a.delta[(int64_t)head0 * a.Tq + t.row0 + row] = x;
        if (std::is_same<T, __half>::value) a.ds_bound[(int64_t)head0 * a.Tq + t.row0 + row] = big;
      }
    } else if (!DKV && std::is_same<T, __half>::value && g == 0 && live) {
      a.ds_bound[(int64_t)head0 * a.Tq + t.row0 + row] = 0.f;  // these rows see nothing
    }
    if (n > 0) {
      bar_wait(b_done, 0, abort, err);
      tc_fence_after();
    }
    // two groups: DKV: the first stores dK, the second dV; else half of the columns each
    const int64_t at = ((int64_t)(t.row0 + row) * (DKV ? a.Hk : a.H) + (DKV ? kvh : head0)) * a.D;
#pragma unroll
    for (int which = 0; which < (DKV ? 2 : 1); ++which) {
      if (DKV && GROUPS == 2 && which != g) continue;
      T* op = (T*)(DKV ? (which ? a.dv : a.dk) : a.dq) + at;
      const float f = which ? 1.f / kLift<T> : a.scale / (c * kLift<T>);
      const uint32_t acc = (which ? t_2 : t_1) + lane;
#pragma unroll
      for (int x = 0; x < DP; x += 32) {
        if (!DKV && GROUPS == 2 && (x / 32) % 2 != g) continue;
        uint32_t v[32];
        if (n > 0) {
          tmem_ld32(acc + x, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (live && (DKV || a.dq)) store32<T>(op, v, f, x, a.D);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, W::tmem);
  }
}

template <typename K>
int set_smem(K kern, int bytes) {
  return cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

template <typename T, int DP>
int fwd(const PackedArgs& a, cudaStream_t st) {
  using F = Fwd<DP>;
  auto kern = packed_mma_fwd_kernel<T, DP>;
  int s = set_smem(kern, F::smem);
  if (s) return s;
  unsigned blocks;
  if ((s = packed_grid(a.Tq, a.B, F::TILES * kTile, a.H, &blocks))) return s;
  kern<<<blocks, F::threads, F::smem, st>>>(a);
  return check_launch();
}

template <typename T, int DP>
int bwd(const PackedArgs& a, cudaStream_t st) {
  using W = Bwd<DP>;
  if (std::is_same<T, __half>::value && (a.dq || a.dk) && a.Tq > 0 && a.Tk > 0) {
    unsigned blocks;
    int s = packed_grid(a.Tk, a.B, kTile, a.Hk, &blocks);
    if (s) return s;
    packed_value_max_kernel<DP><<<blocks, 128, 0, st>>>(a);
    if ((s = check_launch())) return s;
  }
  // dQ first, wanted or not: it leaves an exact delta
  if ((a.dq || a.dk) && a.Tq > 0) {
    auto kern = packed_mma_bwd_kernel<T, DP, false>;
    int s = set_smem(kern, W::smem);
    if (s) return s;
    unsigned blocks;
    if ((s = packed_grid(a.Tq, a.B, kTile, a.H, &blocks))) return s;
    kern<<<blocks, W::threads, W::smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  if (a.dk && a.Tk > 0) {
    auto kern = packed_mma_bwd_kernel<T, DP, true>;
    int s = set_smem(kern, W::smem);
    if (s) return s;
    unsigned blocks;
    if ((s = packed_grid(a.Tk, a.B, kTile, a.Hk, &blocks))) return s;
    kern<<<blocks, W::threads, W::smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  return TPO_OK;
}

bool rows16(const void* p, int64_t s1, int64_t s2) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s1 % 8 == 0 && s2 % 8 == 0;
}

}  // namespace

bool packed_mma_takes(int dtype, const PackedArgs& a, bool backward) {
  // every row of inputs and outputs starts on 16 bytes (outputs are contiguous; null ones are not written)
  const bool out = backward ? rows16(a.dq, 0, 0) && rows16(a.dk, 0, 0) && rows16(a.dv, 0, 0) : rows16(a.o, 0, 0);
  return (dtype == TPO_F16 || dtype == TPO_BF16) && a.D % 8 == 0 && a.D <= 128 && rows16(a.q, a.q_st, a.q_sh) &&
         rows16(a.k, a.k_st, a.k_sh) && rows16(a.v, a.v_st, a.v_sh) && out && (!backward || rows16(a.go, a.go_st, a.go_sh));
}

int packed_mma_forward(int dtype, const PackedArgs& a, cudaStream_t st) {
  if (dtype == TPO_F16) return a.D <= 64 ? fwd<__half, 64>(a, st) : fwd<__half, 128>(a, st);
  return a.D <= 64 ? fwd<__nv_bfloat16, 64>(a, st) : fwd<__nv_bfloat16, 128>(a, st);
}

int packed_mma_backward(int dtype, const PackedArgs& a, cudaStream_t st) {
  if (dtype == TPO_F16) return a.D <= 64 ? bwd<__half, 64>(a, st) : bwd<__half, 128>(a, st);
  return a.D <= 64 ? bwd<__nv_bfloat16, 64>(a, st) : bwd<__nv_bfloat16, 128>(a, st);
}

int attention_mma_error_word(unsigned** word) { return attention_error_word(word); }

}  // namespace tpo
