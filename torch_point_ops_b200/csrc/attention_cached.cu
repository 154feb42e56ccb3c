// Attention of one token per cloud over a padded cache: q (N, H, D) against
// k, v (N, P, Hk, D) of which the first lengths[n] tokens count.
//
//   s_j = scale * q . k_j (j < length),  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)
//
// Two to four operations per byte of cache: HBM is the bound, so a cached token is read
// once for all query heads of its group, up to 16 of them in the matrix kernel and 4 in the
// other; larger groups read it ceil(group / 16) or ceil(group / 4) times.  The key axis is cut into chunks
// of a fixed number of tokens (chosen by the host from N, Hk and P, so no length is copied
// to the host); a block takes one chunk of one (cloud, kv head).  Up to 8 short chunks are a
// thread-block cluster, which joins them through its shared memory in chunk order.  More
// or longer ones: blocks beyond a cloud's length leave at once, and the unnormalised
// partials are joined in chunk order by a second small kernel.
//
// Slots at or beyond lengths[n] are never read: they may hold anything.
//
// Measured (B200, bf16, width 128): 64 clouds of 4096 tokens, 32 heads over 8: 180 us, 5.97
// TB/s of cache; one cloud of 131072 tokens, 16 heads over 4: 50 us, 5.4 TB/s (a plain copy
// moves 6.56); fp32, 32 clouds of 4096 tokens: 32 heads over 8 256 us, 4.2 TB/s, 32 over 32
// 644 us, 6.7 TB/s (grouped heads: scores and sums per loaded byte); bf16 width 256 (the FP32
// pipe): 496 us, 2.2 TB/s.  What is left is the start of the blocks and the join (4 us).  One cloud of 256 tokens,
// 8 heads of width 64: 4.8 us, a chain of latencies.
#include "attention_common.cuh"
#include "tcgen05.cuh"  // asynchronous copies

namespace tpo {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

struct CachedArgs {
  const void *q, *k, *v;
  int64_t q_sn, q_sh, k_sn, k_sp, k_sh, v_sn, v_sp, v_sh;
  const int64_t* lengths;
  void* o;
  float* part;  // (N*H, chunks, pitch) sums, then (N*H, chunks, 2) maxima (base 2) and weights
  int64_t P, chunk;
  int N, H, Hk, D, chunks;
  int cluster;  // the chunks of a (cloud, kv head) are one thread-block cluster, which joins them itself
  float qscale;  // scale * log2(e)
};

__device__ __forceinline__ int64_t length_of(const CachedArgs& a, int n) {
  return min64(max64(a.lengths[n], 0), a.P);
}
__host__ __device__ __forceinline__ int part_pitch(int D) { return (D + 3) & ~3; }  // rows on 16 bytes
__device__ __forceinline__ float* part_stats(const CachedArgs& a) {
  return a.part + (int64_t)a.N * a.H * a.chunks * part_pitch(a.D);
}

// Writes one head's row: the result itself when the key axis is one chunk, else
// the partial.  `sum` is unnormalised, m the maximum (-inf: nothing seen).
template <typename T>
__device__ __forceinline__ void put(const CachedArgs& a, int64_t row, int chunk, int c, float sum, float l) {
  if (a.chunks == 1)
    ((T*)a.o)[row * a.D + c] = from_acc<T>(l > 0.f ? sum / l : l == 0.f ? 0.f : l);
  else
    a.part[(row * a.chunks + chunk) * part_pitch(a.D) + c] = sum;
}

// The chunks' sums of `rows` heads (res[row * pitch + c], {maximum, weight} in rs[row], in every
// block's shared memory at the same place) joined by the cluster in chunk order; the
// blocks share the columns.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float remote(uint32_t addr, int rank) {
  float v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
               : "=f"(v)
               : "r"(addr), "r"(rank)
               : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void cluster_join(const CachedArgs& a, int chunk, int64_t row0, int rows, const float* res,
                                             int pitch, const float2* rs) {
  cluster_sync();
  const uint32_t r = smem_addr(res), st = smem_addr(rs);
  for (int i = chunk * kThreads + threadIdx.x; i < rows * a.D; i += a.chunks * kThreads) {
    const int row = i / a.D, c = i - row * a.D;
    float m[8], mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = k < a.chunks ? remote(st + row * 8, k) : -INFINITY;
      mx = fmaxf(mx, m[k]);
    }
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, l = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= a.chunks) continue;
      const float f = exp2f(m[k] - base);
      sum = fmaf(f, remote(r + (row * pitch + c) * 4, k), sum);
      l = fmaf(f, remote(st + row * 8 + 4, k), l);
    }
    ((T*)a.o)[(row0 + row) * a.D + c] = from_acc<T>(l > 0.f ? sum / l : l == 0.f ? 0.f : l);
  }
  cluster_sync();  // nobody leaves while its shared memory is read
}

// ---------------------------------------------------------------------------
// Any dtype, any strides, D <= 256.  A warp takes 32 keys at a time: LPK lanes
// share a key's row (NVL vectors of VEC elements each), so 32 / LPK keys are read
// per instruction; scores meet in shared memory, where a lane owns a key for the
// softmax; the values are read with the lanes laid out as for the keys.  GB query
// heads of the group per block.
// ---------------------------------------------------------------------------
template <typename T, int VEC, int LPK, int NVL, int GB, bool CLUSTER>  // one kernel for both: 192 -> 260 us, by registers
__global__ void __launch_bounds__(kThreads) cached_simt_kernel(CachedArgs a) {
  constexpr int UNR = GB <= 2 ? 8 : 4;
  constexpr int KPI = 32 / LPK, W = LPK * NVL * VEC;
  __shared__ float sc[kWarps][GB][32];
  __shared__ float jm[kWarps][GB], jl[kWarps][GB];
  __shared__ float jo[kWarps][GB][W];
  __shared__ float res[CLUSTER ? GB * W : 1];
  __shared__ float2 rs[CLUSTER ? GB : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int kl = lane % LPK, kr = lane / LPK;
  const int group = a.H / a.Hk, gblocks = (group + GB - 1) / GB;
  const int n = blockIdx.z, kvh = blockIdx.x / gblocks, g0 = (blockIdx.x % gblocks) * GB, chunk = blockIdx.y;
  const int gn = min(GB, group - g0);
  const int64_t len = length_of(a, n);
  const int64_t j_begin = (int64_t)chunk * a.chunk, j_end = min64(len, j_begin + a.chunk);
  if (!CLUSTER && chunk > 0 && j_begin >= len) return;  // the join skips this chunk too
  const int64_t row0 = (int64_t)n * a.H + kvh * group + g0;
  float q[GB][NVL][VEC], acc[GB][NVL][VEC], m[GB], l[GB];
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < NVL; ++i) {
      const int c = (i * LPK + kl) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[g][i][j] = 0.f, acc[g][i][j] = 0.f;
      if (g < gn && c < a.D)
        load_vec<VEC>((const T*)a.q + n * a.q_sn + (kvh * group + g0 + g) * a.q_sh + c, q[g][i]);
    }
  }
  const T* kp = (const T*)a.k + n * a.k_sn + kvh * a.k_sh;
  const T* vp = (const T*)a.v + n * a.v_sn + kvh * a.v_sh;
  for (int64_t j0 = j_begin + warp * 32; j0 < j_end; j0 += kWarps * 32) {
#pragma unroll(UNR)
    for (int i = 0; i < 32; i += KPI) {
      // unconditional, so that the loads of several steps are in flight together; a key
      // beyond the end repeats the last one and is masked below
      const T* row = kp + min64(j0 + i + kr, j_end - 1) * a.k_sp;
      float s[GB];
#pragma unroll
      for (int g = 0; g < GB; ++g) s[g] = 0.f;
#pragma unroll
      for (int x = 0; x < NVL; ++x) {
        const int c = (x * LPK + kl) * VEC;
        float kv[VEC];
        load_vec<VEC>(row + (c < a.D ? c : 0), kv);
#pragma unroll
        for (int g = 0; g < GB; ++g)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[g] = fmaf(q[g][x][e], c < a.D ? kv[e] : 0.f, s[g]);
      }
#pragma unroll
      for (int g = 0; g < GB; ++g) {
#pragma unroll
        for (int x = LPK / 2; x > 0; x >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], x);
        if (kl == 0) sc[warp][g][i + kr] = s[g];
      }
    }
    __syncwarp();
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      const float s = j0 + lane < j_end ? sc[warp][g][lane] * a.qscale : -INFINITY;
      float mx = fmaxf(s, m[g]);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float base = mx == -INFINITY ? 0.f : mx;
      const float corr = exp2f(m[g] - base), p = exp2f(s - base);
      m[g] = mx;
      l[g] = l[g] * corr + p;  // this lane's keys; summed over lanes at the end
      sc[warp][g][lane] = p;
#pragma unroll
      for (int x = 0; x < NVL; ++x)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[g][x][e] *= corr;
    }
    __syncwarp();
#pragma unroll(UNR)
    for (int i = 0; i < 32; i += KPI) {
      // as above; the repeated last key has probability 0 in the repeats (a value that is
      // not finite there is in the result anyway), columns beyond D are never written
      const T* row = vp + min64(j0 + i + kr, j_end - 1) * a.v_sp;
#pragma unroll
      for (int x = 0; x < NVL; ++x) {
        const int c = (x * LPK + kl) * VEC;
        float vv[VEC];
        load_vec<VEC>(row + (c < a.D ? c : 0), vv);
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          const float p = sc[warp][g][i + kr];
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[g][x][e] = fmaf(p, vv[e], acc[g][x][e]);
        }
      }
    }
    __syncwarp();
  }
  // join: keys of a warp's rows, then the warps in order
#pragma unroll
  for (int g = 0; g < GB; ++g) {
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], x);
#pragma unroll
    for (int i = 0; i < NVL; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = acc[g][i][e];
#pragma unroll
        for (int x = 16; x >= LPK; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        if (kr == 0) jo[warp][g][(i * LPK + kl) * VEC + e] = v;
      }
    if (lane == 0) {
      jm[warp][g] = m[g];
      jl[warp][g] = l[g];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gn * a.D; i += kThreads) {
    const int g = i / a.D, c = i - g * a.D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, jm[w][g]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, ls = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(jm[w][g] - base);
      sum += f * jo[w][g][c];
      ls += f * jl[w][g];
    }
    if (CLUSTER) {
      res[g * W + c] = sum;
      if (c == 0) rs[g] = make_float2(mx, ls);
      continue;
    }
    put<T>(a, row0 + g, chunk, c, sum, ls);
    if (a.chunks > 1 && c == 0) {
      float* st = part_stats(a) + ((row0 + g) * a.chunks + chunk) * 2;
      st[0] = mx;
      st[1] = ls;
    }
  }
  if (CLUSTER) cluster_join<T>(a, chunk, row0, gn, res, W, rs);
}

// ---------------------------------------------------------------------------
// 16-bit types, D a multiple of 8 up to 128, rows on 16-byte boundaries: the heads
// of a group (16 to a block) are the M rows of m16n8k16 products, so the work per
// cached byte stays small for any group.  A warp takes 16 keys at a time.
//
// A warp owns a queue of kStages tiles in shared memory: each lane fetches one row of
// a tile (16 keys, 16 values) with one bulk copy, so the copies cost a handful of
// instructions per 8 KB and are not bound by the load unit's outstanding misses.  The
// row pitches (256 + 64 and 256 + 16 bytes) keep both products' 128-bit reads free of
// bank conflicts.  What the fragments want is met by permuting the summed or the
// free index:
//   S = Q K^T: lane (g = lane/4, c = lane%4) loads chunks 4i + c (8 elements each) of
//     key g; a chunk's register pairs serve as two k-steps, with Q's chunks loaded in
//     the same order.
//   O = P V: the score fragment is the A fragment (keys 2c, 2c+1, 2c+8, 2c+9 of lane
//     c); lane (g, c) loads chunk 8h + g of those four keys, and product t of half h takes
//     element t of every chunk as its column, so a lane ends with whole chunks 8h + 2c
//     and 8h + 2c + 1 of rows g and g + 8.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int DP>
struct MmaShape {
  static constexpr int KC = DP / 32, VC = DP / 64;
  static constexpr int kp = DP * 2 + 64, vp = DP * 2 + 16;  // row pitches, bytes
  static constexpr int tile = 16 * (kp + vp);
  static constexpr int stages = DP == 128 ? 2 : 3;  // three blocks per SM: measured against two blocks with a longer queue
  static constexpr int smem = kWarps * stages * tile;  // also holds the join: 16 rows of DP + 4 floats per warp
  static_assert(smem >= kWarps * 16 * (DP + 4) * 4 + 16 * DP * 4, "join buffers");
};

template <typename T, int DP, bool TALL, bool CLUSTER>  // TALL: the block has more than 8 heads
__global__ void __launch_bounds__(kThreads, 3) cached_mma_kernel(CachedArgs a) {
  using Sh = MmaShape<DP>;
  constexpr int KC = Sh::KC, VC = Sh::VC, ST = Sh::stages;
  __shared__ float jm[kWarps][16], jl[kWarps][16];
  __shared__ unsigned long long full[kWarps][ST];
  __shared__ float2 rs[16];
  extern __shared__ uint4 ring[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, c = lane % 4;
  const int group = a.H / a.Hk, gblocks = (group + 15) / 16;
  const int n = blockIdx.z, kvh = blockIdx.x / gblocks, g0 = (blockIdx.x % gblocks) * 16, chunk = blockIdx.y;
  const int gn = min(16, group - g0);
  const int64_t len = length_of(a, n);
  const int64_t j_begin = (int64_t)chunk * a.chunk, j_end = min64(len, j_begin + a.chunk);
  if (!CLUSTER && chunk > 0 && j_begin >= len) return;  // the join skips this chunk too
  pdl_trigger();
  const T* kp = (const T*)a.k + n * a.k_sn + kvh * a.k_sh;
  const T* vp = (const T*)a.v + n * a.v_sn + kvh * a.v_sh;
  uint8_t* mine = reinterpret_cast<uint8_t*>(ring) + warp * ST * Sh::tile;  // this warp's queue
  const int64_t j_first = j_begin + warp * 16;
  if (lane < ST) mbar_init(&full[warp][lane], 1);
  if (a.D < DP) {  // no copy writes the columns beyond D: zeros, once
    for (int i = lane; i < ST * Sh::tile / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  __syncwarp();
  // Lane 0-15: key of the tile, 16-31: value.  Beyond the end: keys are masked
  // whatever they hold, values become zeros (0 * NaN).
  const int r = lane & 15;
  const T* src = lane < 16 ? kp + r * a.k_sp : vp + r * a.v_sp;
  const int64_t src_step = lane < 16 ? a.k_sp : a.v_sp;
  const int dst_row = lane < 16 ? r * Sh::kp : 16 * Sh::kp + r * Sh::vp;
  const unsigned row_bytes = a.D * 2;
  auto fetch = [&](int64_t j0, int slot) {
    const int left = (int)min64(16, j_end - j0);
    uint8_t* dst = mine + slot * Sh::tile + dst_row;
    if (lane == 0) mbar_expect_tx(&full[warp][slot], 2 * left * row_bytes);
    __syncwarp();
    if (r < left) {
      bulk_g2s(dst, src + j0 * src_step, row_bytes, &full[warp][slot]);
    } else if (lane >= 16) {  // the warp's last tile: nothing is copied here afterwards
#pragma unroll
      for (int i = 0; i < DP * 2; i += 16) *reinterpret_cast<uint4*>(dst + i) = make_uint4(0, 0, 0, 0);
    }
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (j_first + s * kWarps * 16 < j_end) fetch(j_first + s * kWarps * 16, s);
  uint4 q[TALL ? 2 : 1][KC];
#pragma unroll
  for (int r = 0; r < (TALL ? 2 : 1); ++r)
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int ch = 4 * i + c, row = g + 8 * r;
      q[r][i] = make_uint4(0, 0, 0, 0);
      if (row < gn && ch * 8 < a.D)
        q[r][i] = *reinterpret_cast<const uint4*>((const T*)a.q + n * a.q_sn + (kvh * group + g0 + row) * a.q_sh + ch * 8);
    }
  float acc[VC][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < VC; ++h)
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h][t][e] = 0.f;

  int slot = 0;
  unsigned parity = 0;
  for (int64_t j0 = j_first; j0 < j_end; j0 += kWarps * 16) {
    const int left = (int)min64(16, j_end - j0);
    const int64_t ahead = j0 + (ST - 1) * kWarps * 16;
    __syncwarp();  // every lane has read the slot that is filled next
    if (ahead < j_end) fetch(ahead, slot == 0 ? ST - 1 : slot - 1);
    mbar_wait(&full[warp][slot], parity, &g_attention_error);
    __syncwarp();
    const uint8_t* keys = mine + slot * Sh::tile + g * Sh::kp + c * 16;
    const uint8_t* vals = mine + slot * Sh::tile + 16 * Sh::kp + 2 * c * Sh::vp + g * 16;
    if (++slot == ST) slot = 0, parity ^= 1;
    float s[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[b][e] = 0.f;
      float s2[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products: each waits for its predecessor
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint4 x = q[0][i], y = TALL ? q[TALL ? 1 : 0][i] : make_uint4(0, 0, 0, 0);
        const uint4 kk = *reinterpret_cast<const uint4*>(keys + b * 8 * Sh::kp + i * 64);
        mma16816<T>(s[b], x.x, y.x, x.y, y.y, kk.x, kk.y);
        mma16816<T>(s2, x.z, y.z, x.w, y.w, kk.z, kk.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[b][e] += s2[e];
    }
    // rows g (e = 0, 1) and g + 8 (e = 2, 3); keys 8 b + 2 c + (e & 1)
    float p[2][4];
    bool moved = false;
    float corr[2] = {1.f, 1.f};
#pragma unroll
    for (int r = 0; r < (TALL ? 2 : 1); ++r) {
      float mx = m[r];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[b][2 * r + e];
          x = 8 * b + 2 * c + e < left ? x * a.qscale : -INFINITY;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float base = mx == -INFINITY ? 0.f : mx;
      if (mx != m[r]) {
        corr[r] = exp2f(m[r] - base);
        moved = true;
      }
      m[r] = mx;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) sum += p[b][2 * r + e] = exp2f(s[b][2 * r + e] - base);
      l[r] = l[r] * corr[r] + sum;  // this lane's keys
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < VC; ++h)
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          acc[h][t][0] *= corr[0], acc[h][t][1] *= corr[0];
          if (TALL) acc[h][t][2] *= corr[1], acc[h][t][3] *= corr[1];
        }
    }
    // P is rounded to the cache's type here; its sum is not
    const uint32_t a0 = pack2<T>(p[0][0], p[0][1]), a2 = pack2<T>(p[1][0], p[1][1]);
    const uint32_t a1 = TALL ? pack2<T>(p[0][2], p[0][3]) : 0u, a3 = TALL ? pack2<T>(p[1][2], p[1][3]) : 0u;
#pragma unroll
    for (int h = 0; h < VC; ++h) {
      uint4 vv[4];
#pragma unroll
      for (int b = 0; b < 4; ++b)
        vv[b] = *reinterpret_cast<const uint4*>(vals + ((b & 1) + 8 * (b >> 1)) * Sh::vp + h * 128);
      const uint32_t *v0 = reinterpret_cast<const uint32_t*>(&vv[0]), *v1 = reinterpret_cast<const uint32_t*>(&vv[1]);
      const uint32_t *v2 = reinterpret_cast<const uint32_t*>(&vv[2]), *v3 = reinterpret_cast<const uint32_t*>(&vv[3]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        mma16816<T>(acc[h][2 * x], a0, a1, a2, a3, __byte_perm(v0[x], v1[x], 0x5410), __byte_perm(v2[x], v3[x], 0x5410));
        mma16816<T>(acc[h][2 * x + 1], a0, a1, a2, a3, __byte_perm(v0[x], v1[x], 0x7632), __byte_perm(v2[x], v3[x], 0x7632));
      }
    }
  }
  // the warps' rows, joined in order (every copy has been waited for)
  __syncthreads();
  float* jo = reinterpret_cast<float*>(ring);  // [warp][row][DP + 4]
  float* res = jo + kWarps * 16 * (DP + 4);    // [row][DP]
#pragma unroll
  for (int r = 0; r < (TALL ? 2 : 1); ++r) {
    float x = l[r];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    if (c == 0) {
      jm[warp][g + 8 * r] = m[r];
      jl[warp][g + 8 * r] = x;
    }
#pragma unroll
    for (int h = 0; h < VC; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* o = jo + (warp * 16 + g + 8 * r) * (DP + 4) + (8 * h + 2 * c + e) * 8;
#pragma unroll
        for (int t = 0; t < 8; t += 4)
          *reinterpret_cast<float4*>(o + t) = make_float4(acc[h][t][2 * r + e], acc[h][t + 1][2 * r + e],
                                                          acc[h][t + 2][2 * r + e], acc[h][t + 3][2 * r + e]);
      }
  }
  __syncthreads();
  const int64_t row0 = (int64_t)n * a.H + kvh * group + g0;
  for (int i = threadIdx.x; i < gn * (DP / 4); i += kThreads) {
    const int row = i / (DP / 4), col = (i % (DP / 4)) * 4;
    if (col >= a.D) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, jm[w][row]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(jm[w][row] - base);
      const float4 o = *reinterpret_cast<const float4*>(jo + (w * 16 + row) * (DP + 4) + col);
      sum[0] += f * o.x, sum[1] += f * o.y, sum[2] += f * o.z, sum[3] += f * o.w;
      ls += f * jl[w][row];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (CLUSTER) res[row * DP + col + e] = sum[e];
      else put<T>(a, row0 + row, chunk, col + e, sum[e], ls);
    }
    if (CLUSTER) {
      if (col == 0) rs[row] = make_float2(mx, ls);
      continue;
    }
    if (a.chunks > 1 && col == 0) {
      float* st = part_stats(a) + ((row0 + row) * a.chunks + chunk) * 2;
      st[0] = mx;
      st[1] = ls;
    }
  }
  if (CLUSTER) cluster_join<T>(a, chunk, row0, gn, res, DP, rs);
}

// Joins the chunks of a head's row: o = sum_c 2^(m_c - m) sum_c / sum_c 2^(m_c - m) l_c.
// CL lanes of four columns, STRANDS of chunks per row (joined in order); what is left of
// the block's 256 threads are further rows.  Few chunks: a warp per row.  Many: 32
// strands for 32 columns, so that even one row keeps many loads in flight.
template <typename T, int CL, int STRANDS>
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedArgs a) {
  constexpr int TPR = CL * STRANDS, ROWS = 256 / TPR;
  static_assert(TPR == 32 || TPR == 256, "a row is a warp or the block");
  __shared__ float4 so[STRANDS > 1 ? STRANDS : 1][CL];
  __shared__ float red[2][8];
  pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  if (row >= (int64_t)a.N * a.H) return;  // whole warps; with one row per block, none
  const int64_t len = length_of(a, (int)(row / a.H));
  const int used = (int)max64(1, (len + a.chunk - 1) / a.chunk);
  const float2* st = reinterpret_cast<const float2*>(part_stats(a) + row * a.chunks * 2);
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  float mx = -INFINITY;
  for (int c = t; c < used; c += TPR) mx = fmaxf(mx, st[c].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  if (TPR > 32) {
    if (lane == 0) red[0][warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[0][w]);
  }
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  for (int c = t; c < used; c += TPR) l += exp2f(st[c].x - base) * st[c].y;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if (TPR > 32) {
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) l += red[1][w];
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  const int pitch = part_pitch(a.D), strand = t / CL;
  for (int col = ((int)blockIdx.y * CL + t % CL) * 4; col - (t % CL) * 4 < a.D; col += (int)gridDim.y * CL * 4) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < a.D) {
      const float* p = a.part + row * a.chunks * pitch + col;
#pragma unroll 8
      for (int c = strand; c < used; c += STRANDS) {
        const float f = exp2f(st[c].x - base);
        const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)c * pitch);
        s.x = fmaf(f, v.x, s.x), s.y = fmaf(f, v.y, s.y), s.z = fmaf(f, v.z, s.z), s.w = fmaf(f, v.w, s.w);
      }
    }
    if (STRANDS > 1) {
      __syncthreads();
      so[strand][t % CL] = s;
      __syncthreads();
      if (strand == 0) {
#pragma unroll 8
        for (int i = 1; i < STRANDS; ++i) {
          const float4 v = so[i][t];
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
      }
    }
    if (strand == 0) {
      T* o = (T*)a.o + row * a.D + col;
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < a.D) o[e] = from_acc<T>(v[e] * inv);
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Blocks that an SM holds: of the matrix kernel by its shared memory, of the other
// by its registers (for the common widths).
constexpr int kMmaBlocks = 3, kSimtBlocks = 8;

// Chunks of a short axis that one cluster joins, with no second launch and no workspace: 8, 4 or
// 2, of 33 to 128 tokens, while two blocks per SM hold them all; else 1.  Measured against
// chunks and a join: 300 tokens, 8 heads of 64, bf16: 4.8 against 7.0 us; 1024 tokens: 6.4 and
// 6.4 us, the whole call 8.2 against 9.8.  Longer chunks lose, since a cluster ends at 8:
// 2048 tokens 9.1 against 6.6 us.
int cluster_chunks(int64_t N, int64_t Hk, int64_t P) {
  for (int c = 8; c > 1; c /= 2)
    if (N * Hk * c <= 148 * 2 && P > 32 * c) return P <= 128 * c ? c : 1;
  return 1;
}

// Tokens per chunk.  One cloud: as many chunks as blocks fit on the GPU at once.
// Several: two such waves and at least five chunks each, since their lengths are not
// known here and differ.  Splitting a short axis costs a join (about 4 us): with enough
// blocks without it, not below 512 tokens.
int64_t chunk_tokens(int64_t N, int64_t Hk, int64_t P, int per_sm) {
  if (const int c = cluster_chunks(N, Hk, P); c > 1) return (P + c - 1) / c;
  const int64_t pairs = max64(1, N * Hk), waves = 148 * per_sm, least = pairs < 148 ? 64 : 512;
  const int64_t wish = N == 1 ? waves / pairs : max64(2 * waves / pairs, 5);
  const int64_t chunks = max64(1, min64((P + least - 1) / least, wish));
  return max64(64, ((P + chunks - 1) / chunks + 63) / 64 * 64);
}
int64_t chunk_count(int64_t N, int64_t Hk, int64_t P, int per_sm) {
  const int64_t c = chunk_tokens(N, Hk, P, per_sm);
  return max64(1, (P + c - 1) / c);
}

int chunk_launch(void (*kern)(CachedArgs), dim3 grid, int smem, const CachedArgs& a, cudaStream_t st) {
  if (!a.cluster) {
    kern<<<grid, kThreads, smem, st>>>(a);
    return check_launch();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1;
  at[0].val.clusterDim.y = a.chunks;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
}

template <typename T, int VEC, int LPK, int NVL, int GB>
int simt_launch(const CachedArgs& a, cudaStream_t st) {
  const int gblocks = (a.H / a.Hk + GB - 1) / GB;
  const auto kern =
      a.cluster ? cached_simt_kernel<T, VEC, LPK, NVL, GB, true> : cached_simt_kernel<T, VEC, LPK, NVL, GB, false>;
  return chunk_launch(kern, dim3(a.Hk * gblocks, a.chunks, a.N), 0, a, st);
}
template <typename T, int VEC, int LPK, int NVL>
int simt_group(const CachedArgs& a, cudaStream_t st) {
  const int g = a.H / a.Hk;
  if (g == 1) return simt_launch<T, VEC, LPK, NVL, 1>(a, st);
  if (g == 2) return simt_launch<T, VEC, LPK, NVL, 2>(a, st);
  return simt_launch<T, VEC, LPK, NVL, 4>(a, st);
}

template <typename T>
bool aligned16(const CachedArgs& a) {
  constexpr int V = 16 / sizeof(T);
  auto ok = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  return a.D % V == 0 && ok(a.q) && ok(a.k) && ok(a.v) &&
         (a.q_sn | a.q_sh | a.k_sn | a.k_sp | a.k_sh | a.v_sn | a.v_sp | a.v_sh) % V == 0;
}

// A warp per row while that leaves no long chain of chunks.
template <typename T>
int join_launch(const CachedArgs& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.N * a.H;
  if (a.chunks <= 8)
    return launch_pdl(cached_join_kernel<T, 32, 1>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, a);
  return launch_pdl(cached_join_kernel<T, 8, 32>, dim3((unsigned)rows, (a.D + 31) / 32), dim3(256), 0, st, a);
}

template <typename T, int DP>
int mma_launch(const CachedArgs& a, cudaStream_t st) {
  const int group = a.H / a.Hk;
  const dim3 grid(a.Hk * ((group + 15) / 16), a.chunks, a.N);  // neighbours read the same tokens' heads
  const auto kern = a.cluster ? group > 8 ? cached_mma_kernel<T, DP, true, true> : cached_mma_kernel<T, DP, false, true>
                    : group > 8 ? cached_mma_kernel<T, DP, true, false>
                                : cached_mma_kernel<T, DP, false, false>;
  constexpr int smem = MmaShape<DP>::smem;
  const int s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (s) return s;
  return chunk_launch(kern, grid, smem, a, st);
}

template <typename T>
int cached_typed(CachedArgs a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool mma = sizeof(T) == 2 && a.D <= 128 && aligned16<T>(a);
  const int per_sm = mma ? kMmaBlocks : kSimtBlocks;
  a.chunk = chunk_tokens(a.N, a.Hk, a.P, per_sm);
  a.cluster = cluster_chunks(a.N, a.Hk, a.P) > 1;
  a.chunks = (int)chunk_count(a.N, a.Hk, a.P, per_sm);
  const bool joined = a.cluster || a.chunks == 1;
  int s;
  if constexpr (sizeof(T) == 2) {
    if (mma) {
      s = a.D <= 64 ? mma_launch<T, 64>(a, st) : mma_launch<T, 128>(a, st);
      if (s || joined) return s;
      return join_launch<T>(a, st);
    }
  }
  if (aligned16<T>(a)) {
    if constexpr (sizeof(T) == 2) {  // wider than 128, or the matrix kernel had it
      s = simt_group<T, V, 32, 1>(a, st);
    } else {
      if (a.D <= 16 * V) s = simt_group<T, V, 16, 1>(a, st);
      else if (a.D <= 32 * V) s = simt_group<T, V, 32, 1>(a, st);
      else s = simt_group<T, V, 32, 2>(a, st);
    }
  } else {
    if (a.D <= 64) s = simt_group<T, 1, 32, 2>(a, st);
    else if (a.D <= 128) s = simt_group<T, 1, 32, 4>(a, st);
    else s = simt_group<T, 1, 32, 8>(a, st);
  }
  if (s || joined) return s;
  return join_launch<T>(a, st);
}

}  // namespace

size_t cached_workspace_size(int64_t N, int64_t H, int64_t Hk, int64_t P, int64_t D) {
  if (cluster_chunks(N, Hk, P) > 1) return 0;
  const int64_t chunks = max64(chunk_count(N, Hk, P, kMmaBlocks), chunk_count(N, Hk, P, kSimtBlocks));
  return chunks == 1 ? 0 : (size_t)(N * H) * chunks * (part_pitch((int)D) + 2) * sizeof(float);
}

int cached_attention(int dtype, const void* q, const int64_t* q_stride, const void* k,
                     const int64_t* k_stride, const void* v, const int64_t* v_stride,
                     const int64_t* lengths, int64_t N, int64_t P, int64_t H, int64_t Hk, int64_t D,
                     float scale, void* o, void* ws, cudaStream_t st) {
  CachedArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_sn = q_stride[0], a.q_sh = q_stride[1];
  a.k_sn = k_stride[0], a.k_sp = k_stride[1], a.k_sh = k_stride[2];
  a.v_sn = v_stride[0], a.v_sp = v_stride[1], a.v_sh = v_stride[2];
  a.lengths = lengths;
  a.o = o, a.part = (float*)ws;
  a.P = P;
  a.N = (int)N, a.H = (int)H, a.Hk = (int)Hk, a.D = (int)D;
  a.qscale = scale * kLog2e;
  switch (dtype) {
    case TPO_F32: return cached_typed<float>(a, st);
    case TPO_F16: return cached_typed<__half>(a, st);
    case TPO_BF16: return cached_typed<__nv_bfloat16>(a, st);
    default: return set_error(TPO_ERR_INVALID_ARGUMENT, "cached_attention: dtype must be f32, f16 or bf16");
  }
}

int attention_cached_error_word(unsigned** word) { return attention_error_word(word); }

}  // namespace tpo
