// Attention over packed clouds on the tensor cores: 16-bit inputs, width a
// multiple of 8 up to 128, rows on 16-byte boundaries.
//
// Forward: a block owns 256 query rows of one (cloud, head) as two tiles of 128
// and passes once over the keys in tiles of 128.  S = Q K^T and O += P V are
// tcgen05 products with fp32 accumulators in tensor memory; P returns to tensor
// memory as the A operand, over the columns of S that it was made from.  While
// one tile's softmax runs, the tensor core works for the other tile.
#include <type_traits>

#include "attention_common.cuh"
#include "tcgen05.cuh"

namespace tpo {
namespace {

constexpr int kTile = 128;                        // rows of Q per softmax group, keys per step
constexpr int kPanel = kTile * kPanelRow;         // 16 KB: 128 rows x 64 elements

// 128 rows of a packed tensor into a swizzled tile, by the kCopyThreads threads of
// the copy warps (t = index).  Rows at or beyond `valid` and columns at or beyond D
// become zeros: nothing from another cloud enters a product (0 * NaN would).
constexpr int kCopyThreads = 64;
template <typename T, int DP>
__device__ __forceinline__ void copy_tile(uint32_t dst, const T* src, int64_t stride, int64_t valid, int D, int t) {
  constexpr int CH = DP / 8;                 // 16-byte chunks per row
  constexpr int STEP = kCopyThreads / CH;    // rows per pass
  const int c = t % CH, r0 = t / CH;
  const uint32_t at = dst + (c >> 3) * kPanel;
  const bool col = c * 8 < D;
  const T* p = src + (int64_t)r0 * stride + c * 8;
#pragma unroll 8
  for (int r = r0; r < kTile; r += STEP) {
    const bool in = col && r < valid;
    cp_async16(at + r * kPanelRow + (((c & 7) ^ (r & 7)) << 4), in ? (const void*)p : (const void*)src, in);
    p += STEP * stride;
  }
}

// ---------------------------------------------------------------- forward
template <int DP>
struct FwdSmem {
  static constexpr int q = kTile * DP * 2;          // one query tile
  static constexpr int kv = kTile * DP * 2;         // one key or value tile
  static constexpr int stages = DP == 128 ? 5 : 8;  // tiles in flight
  static constexpr int bars = 2 * q + stages * kv;
  static constexpr int total = bars + 256 + 1024;   // + alignment of the base
};
// 8 warps with a row per thread, 2 copy warps, 1 warp that issues products, and one
// idle (registers are handed out per four warps anyway)
constexpr int kThreads = 32 * 12, kCopyWarp = 8, kMmaWarp = 10;
// 384 threads are launched with 168 registers each; the row warps draw what the others give
constexpr int kRowRegs = 200, kOtherRegs = 104;
static_assert(256 * kRowRegs + 128 * kOtherRegs <= kThreads * 168, "register split");

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) packed_mma_fwd_kernel(const PackedArgs a) {
  using Sm = FwdSmem<DP>;
  constexpr int ST = Sm::stages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  const uint32_t sq = base, skv = base + 2 * Sm::q, bars = base + Sm::bars;
  // barriers: queries full, stages full, stages empty, S full x 2, P full x 2, O done x 2
  const uint32_t b_q = bars, b_full = bars + 8, b_empty = b_full + 8 * ST, b_s = b_empty + 8 * ST, b_p = b_s + 16,
                 b_o = b_p + 16, s_tmem = b_o + 16, s_abort = s_tmem + 4;
  volatile int* abort = reinterpret_cast<volatile int*>(smem_raw + (s_abort - raw));
  unsigned* err = &g_attention_error;

  const int warp = threadIdx.x / 32, head = blockIdx.y, kvh = head / (a.H / a.Hk);
  const int64_t slot = a.causal ? (int64_t)gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const Tile t = find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, 2 * kTile, slot);
  if (t.rows <= 0) return;
  const int64_t shift = t.nb - t.na, first = t.row0 - t.a0;
  // keys that tile w meets, and its steps
  int64_t nk[2];
  int steps[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int rows = max(0, min(kTile, t.rows - w * kTile));
    nk[w] = rows == 0 ? 0 : a.causal ? min64(t.nb, max64(first + w * kTile + rows + shift, 0)) : t.nb;
    steps[w] = (int)((nk[w] + kTile - 1) / kTile);
  }
  const int n = max(steps[0], steps[1]);

  if (warp == kMmaWarp) {
    if (threadIdx.x % 32 == 0) {
      bar_init(b_q, kCopyThreads);
      for (int i = 0; i < ST; ++i) {
        bar_init(b_full + 8 * i, kCopyThreads);
        bar_init(b_empty + 8 * i, 1);
      }
      for (int w = 0; w < 2; ++w) {
        bar_init(b_s + 8 * w, 1);
        bar_init(b_p + 8 * w, 128);
        bar_init(b_o + 8 * w, 1);
      }
      *abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tmem_alloc(s_tmem, 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(s_tmem));
  // columns: S0 | S1 | O0 | O1; P over the first half of its S
  const uint32_t t_s = tmem, t_o = tmem + 256;

  if (warp >= kCopyWarp) {
  give_registers<kOtherRegs>();
  if (warp == kCopyWarp || warp == kCopyWarp + 1) {
    // ---- copies: Q, then K0 V0 K1 V1 ... through the ring ----
    const int tid = threadIdx.x - 32 * kCopyWarp;
    const T* qp = (const T*)a.q + t.row0 * a.q_st + head * a.q_sh;
    const T* kp = (const T*)a.k + t.b0 * a.k_st + kvh * a.k_sh;
    const T* vp = (const T*)a.v + t.b0 * a.v_st + kvh * a.v_sh;
    if (n > 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
        copy_tile<T, DP>(sq + w * Sm::q, qp + (int64_t)w * kTile * a.q_st, a.q_st, t.rows - w * kTile, a.D, tid);
      cp_async_commit();
      int told = -1;  // tiles below this one are announced; -1: Q is not yet
      auto announce = [&](int upto) {  // all copies of tiles < upto have landed
        fence_async_smem();
        if (told < 0) bar_arrive(b_q), told = 0;
        for (; told < upto; ++told) bar_arrive(b_full + 8 * (told % ST));
      };
      for (int i = 0; i < 2 * n; ++i) {
        const int s = i % ST;
        if (i >= ST) {
          const uint32_t parity = (i / ST - 1) & 1;
          if (!bar_try(b_empty + 8 * s, parity)) {
            cp_async_wait<0>();
            announce(i);
            bar_wait(b_empty + 8 * s, parity, abort, err);
          }
        }
        const int64_t j = (int64_t)(i >> 1) * kTile;
        if (i & 1) copy_tile<T, DP>(skv + s * Sm::kv, vp + j * a.v_st, a.v_st, t.nb - j, a.D, tid);
        else copy_tile<T, DP>(skv + s * Sm::kv, kp + j * a.k_st, a.k_st, t.nb - j, a.D, tid);
        cp_async_commit();
        cp_async_wait<1>();
        announce(i);
      }
      cp_async_wait<0>();
      announce(2 * n);
    }
  } else if (warp == kMmaWarp) {
    // ---- products, issued by one thread ----
    if (threadIdx.x % 32 == 0 && n > 0) {
      constexpr uint32_t id_s = mma_desc<T>(kTile, kTile, false), id_o = mma_desc<T>(kTile, DP, true);
      auto score = [&](int w, int j) {  // S_w = Q_w K_j^T
        const uint32_t k = skv + ((2 * j) % ST) * Sm::kv, q = sq + w * Sm::q;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const uint32_t at = (ks / 4) * kPanel + (ks % 4) * 32;
          mma_ss(t_s + w * kTile, smem_desc(q + at, 16), smem_desc(k + at, 16), id_s, ks > 0);
        }
      };
      auto wait_tile = [&](int i) { bar_wait(b_full + 8 * (i % ST), (i / ST) & 1, abort, err); };
      bar_wait(b_q, 0, abort, err);
      wait_tile(0);
      for (int w = 0; w < 2; ++w)
        if (steps[w] > 0) {
          score(w, 0);
          mma_commit(b_s + 8 * w);
        }
      // a stage is handed back only where another tile will fill it, so that no
      // arrival is still on its way when the block ends
      auto release = [&](int i) {
        if (i + ST < 2 * n) mma_commit(b_empty + 8 * (i % ST));
      };
      release(0);
      for (int j = 0; j < n; ++j) {
        const int iv = 2 * j + 1, ik = 2 * j + 2;
        wait_tile(iv);
        if (j + 1 < n) wait_tile(ik);
        const uint32_t v = skv + (iv % ST) * Sm::kv;
        for (int w = 0; w < 2; ++w) {
          if (j >= steps[w]) continue;
          bar_wait(b_p + 8 * w, j & 1, abort, err);
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            mma_ts(t_o + w * DP, t_s + w * kTile + ks * 8, smem_desc(v + ks * 16 * kPanelRow, kPanel), id_o,
                   j > 0 || ks > 0);
          if (j + 1 < steps[w]) {
            score(w, j + 1);
            mma_commit(b_s + 8 * w);
          } else {
            mma_commit(b_o + 8 * w);
          }
        }
        release(iv);
        release(ik);
      }
    }
    __syncwarp();
  }
  } else {
    // ---- softmax: a thread owns a row ----
    draw_registers<kRowRegs>();
    const int w = warp / 4, row = threadIdx.x % kTile;
    const uint32_t lane = (uint32_t)(warp % 4) * 32 << 16;
    const uint32_t ts = t_s + w * kTile + lane, to = t_o + w * DP + lane;
    const bool live = w * kTile + row < t.rows;
    const float qscale = a.scale * kLog2e;
    // this row sees keys below `sees`
    const int64_t sees = a.causal ? min64(t.nb, first + w * kTile + row + shift + 1) : t.nb;
    float m = -INFINITY, l = 0.f;
    // one step's row: masked columns count as -inf
    auto step = [&](int j, int lim, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, v[c]);
      tmem_wait_ld();
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
        tmem_st16(ts + c * 16, p);
      }
      float x, y;
      upk(add2(sum[0], sum[1]), x, y);
      l += x + y;
      tmem_wait_st();
      tc_fence_before();
      bar_arrive(b_p + 8 * w);
    };
    for (int j = 0; j < steps[w]; ++j) {
      const int64_t left = sees - (int64_t)j * kTile;
      const int lim = left >= kTile ? kTile : left > 0 ? (int)left : 0;
      const bool whole = __all_sync(0xffffffffu, lim == kTile);
      bar_wait(b_s + 8 * w, j & 1, abort, err);
      tc_fence_after();
      if (whole) step(j, lim, std::false_type{});
      else step(j, lim, std::true_type{});
    }
    if (live && a.lse) a.lse[(int64_t)head * a.Tq + t.row0 + w * kTile + row] =
        l == 0.f ? -INFINITY : (m * qscale + log2f(l)) * kLn2;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    T* op = (T*)a.o + ((t.row0 + w * kTile + row) * a.H + head) * a.D;
    if (steps[w] > 0) {
      bar_wait(b_o + 8 * w, 0, abort, err);
      tc_fence_after();
    }
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
      uint32_t v[32];
      if (steps[w] > 0) {
        tmem_ld32(to + c, v);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
      if (live) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          if (c + i >= a.D) continue;
          uint4 o;
          uint32_t* ov = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            ov[e] = pack2<T>(__uint_as_float(v[i + 2 * e]) * inv, __uint_as_float(v[i + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(op + c + i) = o;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// ---------------------------------------------------------------- backward
// P = exp(S - lse) and dS = P * (dP - delta) are rebuilt tile by tile from S and dP,
// which are recomputed.  DKV: rows are the block's 128 keys (x1 = K, x2 = V), the
// streamed columns are queries (y1 = Q, y2 = dO) of every head of the group;
// acc1 = dK += dS^T Q, acc2 = dV += P^T dO.  Otherwise rows are 128 queries
// (x1 = Q, x2 = dO), columns keys (y1 = K, y2 = V), acc1 = dQ += dS K.  In both,
// S = x1 y1^T, dP = x2 y2^T, and P and dS go back to tensor memory as A operands.
// Each sum has one owner: no atomics, the same bits in every run.
//
// Two phases alternate on single buffers: while the 256 threads turn S into P the
// tensor core runs acc1 of the step before and dP; while they turn dP into dS it
// runs acc2 and the next S.  A row's columns are shared by two threads (halves of
// 64), so the fp32 P stay in registers from one phase to the other.
template <int DP>
struct BwdSmem {
  static constexpr int tile = kTile * DP * 2;
  static constexpr int stages = DP == 128 ? 4 : 8;
  static constexpr int stats = 2 * tile + stages * tile;  // 128 floats per stage: base-2 lse with y1, delta with y2 (DKV)
  static constexpr int bars = stats + stages * kTile * 4;
  static constexpr int total = bars + 256 + 1024;
};

// 2^-e for the power of two 2^e at or below the largest |dO| that a sum meets: brings
// dS of fp16 away from the type's smallest step (undone when acc1 leaves).
__device__ __forceinline__ float grad_scale(float largest) {
  const unsigned e = __float_as_uint(largest) >> 23;
  return e == 0 || e >= 0xfe ? 1.f : __uint_as_float((254 - e) << 23);
}

template <typename T, int DP, bool DKV>
__global__ void __launch_bounds__(kThreads, 1) packed_mma_bwd_kernel(const PackedArgs a) {
  using Sm = BwdSmem<DP>;
  constexpr int ST = Sm::stages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  const uint32_t sx = base, sy = base + 2 * Sm::tile, bars = base + Sm::bars;
  const float* stats = reinterpret_cast<const float*>(smem_raw + (base + Sm::stats - raw));
  const uint32_t b_x = bars, b_full = bars + 8, b_empty = b_full + 8 * ST, b_s = b_empty + 8 * ST, b_dp = b_s + 8,
                 b_p = b_dp + 8, b_ds = b_p + 8, b_done = b_ds + 8, s_tmem = b_done + 8, s_abort = s_tmem + 4;
  volatile int* abort = reinterpret_cast<volatile int*>(smem_raw + (s_abort - raw));
  unsigned* err = &g_attention_error;

  const int warp = threadIdx.x / 32, group = a.H / a.Hk;
  const int64_t slot = !DKV && a.causal ? (int64_t)gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const Tile t = DKV ? find_tile(a.off_k, a.Tk, a.off_q, a.Tq, a.B, kTile, slot)
                     : find_tile(a.off_q, a.Tq, a.off_k, a.Tk, a.B, kTile, slot);
  if (t.rows <= 0) return;
  const int64_t nq = DKV ? t.nb : t.na, nkeys = DKV ? t.na : t.nb, shift = nkeys - nq, first = t.row0 - t.a0;
  int64_t c_begin = 0, c_end = t.nb;  // columns that any row of the tile meets
  if (a.causal) {
    if (DKV) c_begin = max64(0, first - shift) / kTile * kTile;
    else c_end = min64(c_end, max64(first + t.rows + shift, 0));
  }
  const int per_head = (int)max64(0, (c_end - c_begin + kTile - 1) / kTile);
  const int kvh = DKV ? blockIdx.y : blockIdx.y / group;
  const int head0 = DKV ? kvh * group : blockIdx.y;
  const int n = per_head * (DKV ? group : 1);

  if (warp == kMmaWarp) {
    if (threadIdx.x % 32 == 0) {
      bar_init(b_x, kCopyThreads);
      for (int i = 0; i < ST; ++i) {
        bar_init(b_full + 8 * i, kCopyThreads);
        bar_init(b_empty + 8 * i, 1);
      }
      bar_init(b_s, 1);
      bar_init(b_dp, 1);
      bar_init(b_p, 256);
      bar_init(b_ds, 256);
      bar_init(b_done, 1);
      *abort = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tmem_alloc(s_tmem, 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(s_tmem));
  // columns: S | dP | acc1 | acc2.  P lies over S and dS over dP: the 64 columns of a
  // half become 32 at the half's start, so neither half overwrites the other's input.
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_1 = tmem + 256, t_2 = tmem + 384;

  if (warp >= kCopyWarp) {
  give_registers<kOtherRegs>();
  if (warp == kCopyWarp || warp == kCopyWarp + 1) {
    const int tid = threadIdx.x - 32 * kCopyWarp;
    const T* kp = (const T*)a.k + kvh * a.k_sh;
    const T* vp = (const T*)a.v + kvh * a.v_sh;
    if (n > 0) {
      if (DKV) {
        copy_tile<T, DP>(sx, kp + t.row0 * a.k_st, a.k_st, t.rows, a.D, tid);
        copy_tile<T, DP>(sx + Sm::tile, vp + t.row0 * a.v_st, a.v_st, t.rows, a.D, tid);
      } else {
        copy_tile<T, DP>(sx, (const T*)a.q + t.row0 * a.q_st + head0 * a.q_sh, a.q_st, t.rows, a.D, tid);
        copy_tile<T, DP>(sx + Sm::tile, (const T*)a.go + t.row0 * a.go_st + head0 * a.go_sh, a.go_st, t.rows, a.D, tid);
      }
      cp_async_commit();
      int told = -1;
      auto announce = [&](int upto) {
        fence_async_smem();
        if (told < 0) bar_arrive(b_x), told = 0;
        for (; told < upto; ++told) bar_arrive(b_full + 8 * (told % ST));
      };
      int h = 0, step = 0;
      for (int i = 0; i < 2 * n; ++i) {
        const int s = i % ST;
        if (i >= ST) {
          const uint32_t parity = (i / ST - 1) & 1;
          if (!bar_try(b_empty + 8 * s, parity)) {
            cp_async_wait<0>();
            announce(i);
            bar_wait(b_empty + 8 * s, parity, abort, err);
          }
        }
        const int64_t c0 = c_begin + (int64_t)step * kTile, tok = t.b0 + c0;
        const uint32_t dst = sy + s * Sm::tile;
        if (DKV) {
          const int head = head0 + h;
          if (i & 1) copy_tile<T, DP>(dst, (const T*)a.go + tok * a.go_st + head * a.go_sh, a.go_st, t.nb - c0, a.D, tid);
          else copy_tile<T, DP>(dst, (const T*)a.q + tok * a.q_st + head * a.q_sh, a.q_st, t.nb - c0, a.D, tid);
          const float* from = (i & 1 ? a.delta : a.lse2) + (int64_t)head * a.Tq + tok;
#pragma unroll
          for (int r = tid; r < kTile; r += kCopyThreads) {
            const bool in = c0 + r < t.nb;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(base + Sm::stats + (s * kTile + r) * 4),
                         "l"(in ? from + r : a.lse2), "r"(in ? 4 : 0)
                         : "memory");
          }
        } else {
          if (i & 1) copy_tile<T, DP>(dst, vp + tok * a.v_st, a.v_st, t.nb - c0, a.D, tid);
          else copy_tile<T, DP>(dst, kp + tok * a.k_st, a.k_st, t.nb - c0, a.D, tid);
        }
        if (i & 1) {
          if (++step == per_head) step = 0, ++h;
        }
        cp_async_commit();
        cp_async_wait<1>();
        announce(i);
      }
      cp_async_wait<0>();
      announce(2 * n);
    }
  } else if (warp == kMmaWarp) {
    if (threadIdx.x % 32 == 0 && n > 0) {
      constexpr uint32_t id_s = mma_desc<T>(kTile, kTile, false), id_o = mma_desc<T>(kTile, DP, true);
      auto wait_tile = [&](int i) { bar_wait(b_full + 8 * (i % ST), (i / ST) & 1, abort, err); };
      auto release = [&](int i) {
        if (i + ST < 2 * n) mma_commit(b_empty + 8 * (i % ST));
      };
      auto nt = [&](uint32_t d, uint32_t x, int i) {  // d = x y_i^T
        const uint32_t y = sy + (i % ST) * Sm::tile;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const uint32_t at = (ks / 4) * kPanel + (ks % 4) * 32;
          mma_ss(d, smem_desc(x + at, 16), smem_desc(y + at, 16), id_s, ks > 0);
        }
      };
      auto add = [&](uint32_t d, uint32_t p, int i, bool more) {  // d (+)= p y_i
        const uint32_t y = sy + (i % ST) * Sm::tile;
#pragma unroll
        for (int ks = 0; ks < kTile / 16; ++ks)
          mma_ts(d, p + (ks / 4) * 64 + (ks % 4) * 8, smem_desc(y + ks * 16 * kPanelRow, kPanel), id_o, more || ks > 0);
      };
      bar_wait(b_x, 0, abort, err);
      wait_tile(0);
      nt(t_s, sx, 0);
      mma_commit(b_s);
      wait_tile(1);
      nt(t_dp, sx + Sm::tile, 1);
      mma_commit(b_dp);
      if (!DKV) release(1);
      for (int j = 0; j < n; ++j) {
        const int i1 = 2 * j, i2 = 2 * j + 1;
        bar_wait(b_p, j & 1, abort, err);
        tc_fence_after();
        if (DKV) add(t_2, t_s, i2, j > 0);
        if (j + 1 < n) {
          wait_tile(i1 + 2);
          nt(t_s, sx, i1 + 2);
          mma_commit(b_s);
        }
        bar_wait(b_ds, j & 1, abort, err);
        tc_fence_after();
        add(t_1, t_dp, i1, j > 0);
        release(i1);
        if (DKV) release(i2);  // not before: the threads read delta from it
        if (j + 1 < n) {
          wait_tile(i2 + 2);
          nt(t_dp, sx + Sm::tile, i2 + 2);
          mma_commit(b_dp);
          if (!DKV) release(i2 + 2);
        }
      }
      mma_commit(b_done);
    }
    __syncwarp();
  }
  } else {
    draw_registers<kRowRegs>();
    const int half = warp / 4, row = threadIdx.x % kTile;
    const uint32_t lane = (uint32_t)(warp % 4) * 32 << 16;
    const uint32_t ts = t_s + half * 64 + lane, tdp = t_dp + half * 64 + lane;
    const bool live = row < t.rows;
    const float qscale = a.scale * kLog2e;
    float c = 1.f;
    if (std::is_same<T, __half>::value) {
      // a row of dQ: its own dO; dK: every dO row that the block meets
      float big = 0.f;
      if (!DKV) {
        if (live) big = a.go_max[(int64_t)head0 * a.Tq + t.row0 + row];
      } else {
        for (int h = 0; h < group; ++h)
          for (int64_t i = c_begin + threadIdx.x % 32; i < c_end; i += 32)
            big = fmaxf(big, a.go_max[(int64_t)(head0 + h) * a.Tq + t.b0 + i]);
        big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
      }
      c = grad_scale(big);
    }
    float row_lse = 0.f, row_delta = 0.f;
    if (!DKV && live) {
      row_lse = a.lse2[(int64_t)head0 * a.Tq + t.row0 + row];
      row_delta = a.delta[(int64_t)head0 * a.Tq + t.row0 + row];
    }
    // one step's half row: P from S, then dS from dP
    auto step_rows = [&](int j, int lo, int hi, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      const u64 q2 = pk(qscale, qscale);
      u64 p[32];
      {
        const float* lse = stats + ((2 * j) % ST) * kTile + half * 64;  // base 2, negated below
        uint32_t v[2][32];
        bar_wait(b_s, j & 1, abort, err);
        if (DKV) bar_wait(b_full + 8 * ((2 * j) % ST), (2 * j / ST) & 1, abort, err);
        tc_fence_after();
        tmem_ld32(ts, v[0]);
        tmem_ld32(ts + 32, v[1]);
        tmem_wait_ld();
        if (!DKV) {  // S is read: the next product may overwrite it
          tc_fence_before();
          bar_arrive(b_p);
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
        bar_arrive(b_p);
      }
      const float* delta = stats + ((2 * j + 1) % ST) * kTile + half * 64;
      bar_wait(b_dp, j & 1, abort, err);
      if (DKV) bar_wait(b_full + 8 * ((2 * j + 1) % ST), ((2 * j + 1) / ST) & 1, abort, err);
      tc_fence_after();
      uint32_t v[2][32], o[32];
      tmem_ld32(tdp, v[0]);
      tmem_ld32(tdp + 32, v[1]);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        u64 d0, d1;
        if (DKV) {
          const float4 f = *reinterpret_cast<const float4*>(delta + 2 * i);
          d0 = pk(f.x, f.y), d1 = pk(f.z, f.w);
        } else {
          d0 = d1 = pk(row_delta, row_delta);
        }
        const uint32_t* s = &v[i / 16][(2 * i) % 32];
        u64 a0 = mul2(p[i], sub2(pku(s[0], s[1]), d0)), a1 = mul2(p[i + 1], sub2(pku(s[2], s[3]), d1));
        if (std::is_same<T, __half>::value) a0 = mul2(a0, pk(c, c)), a1 = mul2(a1, pk(c, c));
        float x[4];
        upk(a0, x[0], x[1]);
        upk(a1, x[2], x[3]);
        if (MASK) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = 2 * i + e >= lo && 2 * i + e < hi ? x[e] : 0.f;
        }
        o[i] = pack2<T>(x[0], x[1]);
        o[i + 1] = pack2<T>(x[2], x[3]);
      }
      tmem_st32(tdp, o);
      tmem_wait_st();
      tc_fence_before();
      bar_arrive(b_ds);
    };
    int step = 0;
    for (int j = 0; j < n; ++j) {
      const int64_t c0 = c_begin + (int64_t)step * kTile + half * 64;
      if (++step == per_head) step = 0;
      // columns [lo, hi) of this half that the row meets.  Keys beyond the cloud's end
      // must not reach dS (their P is unbounded); queries beyond it have zero rows
      // of Q and dO and lse 0, so they add nothing.
      int lo = 0, hi = 64;
      if (DKV) {
        if (a.causal) lo = (int)min64(64, max64(0, first + row - shift - c0));
      } else {
        int64_t end = t.nb;
        if (a.causal) end = min64(end, first + row + shift + 1);
        hi = (int)min64(64, max64(0, end - c0));
      }
      const bool whole = __all_sync(0xffffffffu, lo == 0 && hi == 64);
      if (whole) step_rows(j, lo, hi, std::false_type{});
      else step_rows(j, lo, hi, std::true_type{});
    }
    if (n > 0) {
      bar_wait(b_done, 0, abort, err);
      tc_fence_after();
    }
    // DKV: the first four warps store dK, the others dV; else each half of the columns
    const int64_t at = DKV ? ((t.row0 + row) * a.Hk + kvh) * a.D : ((t.row0 + row) * a.H + head0) * a.D;
    T* op = (T*)(DKV ? (half ? a.dv : a.dk) : a.dq) + at;
    const float f = DKV && half ? 1.f : a.scale / c;
    const uint32_t from = (DKV && half ? t_2 : t_1) + lane;
#pragma unroll
    for (int x = 0; x < DP; x += 32) {
      if (!DKV && (x / 32) % 2 != half) continue;
      uint32_t v[32];
      if (n > 0) {
        tmem_ld32(from + x, v);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
      if (live) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          if (x + i >= a.D) continue;
          uint4 o;
          uint32_t* ov = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            ov[e] = pack2<T>(__uint_as_float(v[i + 2 * e]) * f, __uint_as_float(v[i + 2 * e + 1]) * f);
          *reinterpret_cast<uint4*>(op + x + i) = o;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

template <typename K>
int set_smem(K kern, int bytes) {
  return cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

template <typename T, int DP>
int fwd(const PackedArgs& a, cudaStream_t st) {
  auto kern = packed_mma_fwd_kernel<T, DP>;
  int s = set_smem(kern, FwdSmem<DP>::total);
  if (s) return s;
  kern<<<dim3((unsigned)packed_slots(a.Tq, a.B, 2 * kTile), a.H), kThreads, FwdSmem<DP>::total, st>>>(a);
  return check_launch();
}

template <typename T, int DP>
int bwd(const PackedArgs& a, cudaStream_t st) {
  constexpr int smem = BwdSmem<DP>::total;
  if (a.dk && a.Tk > 0) {
    auto kern = packed_mma_bwd_kernel<T, DP, true>;
    int s = set_smem(kern, smem);
    if (s) return s;
    kern<<<dim3((unsigned)packed_slots(a.Tk, a.B, kTile), a.Hk), kThreads, smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  if (a.dq && a.Tq > 0) {
    auto kern = packed_mma_bwd_kernel<T, DP, false>;
    int s = set_smem(kern, smem);
    if (s) return s;
    kern<<<dim3((unsigned)packed_slots(a.Tq, a.B, kTile), a.H), kThreads, smem, st>>>(a);
    if ((s = check_launch())) return s;
  }
  return TPO_OK;
}

bool rows16(const void* p, int64_t s1, int64_t s2) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s1 % 8 == 0 && s2 % 8 == 0;
}

}  // namespace

bool packed_mma_takes(int dtype, const PackedArgs& a, bool backward) {
  return (dtype == TPO_F16 || dtype == TPO_BF16) && a.D % 8 == 0 && a.D <= 128 && rows16(a.q, a.q_st, a.q_sh) &&
         rows16(a.k, a.k_st, a.k_sh) && rows16(a.v, a.v_st, a.v_sh) && (!backward || rows16(a.go, a.go_st, a.go_sh));
}

int packed_mma_forward(int dtype, const PackedArgs& a, cudaStream_t st) {
  if (dtype == TPO_F16) return a.D <= 64 ? fwd<__half, 64>(a, st) : fwd<__half, 128>(a, st);
  return a.D <= 64 ? fwd<__nv_bfloat16, 64>(a, st) : fwd<__nv_bfloat16, 128>(a, st);
}

int packed_mma_backward(int dtype, const PackedArgs& a, cudaStream_t st) {
  if (dtype == TPO_F16) return a.D <= 64 ? bwd<__half, 64>(a, st) : bwd<__half, 128>(a, st);
  return a.D <= 64 ? bwd<__nv_bfloat16, 64>(a, st) : bwd<__nv_bfloat16, 128>(a, st);
}

int attention_mma_error_flags(unsigned* out, bool clear) { return read_attention_error(out, clear); }

}  // namespace tpo
