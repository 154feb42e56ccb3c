// Attention of one token per cloud over a padded cache: q (N, H, D) against
// k, v (N, P, Hk, D) of which the first lengths[n] tokens count.
//
//   s_j = scale * q . k_j (j < length),  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)
//
// Two to four operations per byte of cache: HBM is the bound, so every cached
// token is read once for all query heads of its group and never staged anywhere
// but in registers.  The key axis is cut into chunks of a fixed number of tokens
// (chosen by the host from N, Hk and P, so no length is copied to the host); a
// block takes one chunk of one (cloud, kv head), blocks beyond a cloud's length
// leave at once, and with more than one chunk the unnormalised partials are
// joined in chunk order by a second small kernel.
//
// Slots at or beyond lengths[n] are never read: they may hold anything.
#include "attention_common.cuh"
#include "tcgen05.cuh"  // pack2

namespace tpo {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

struct CachedArgs {
  const void *q, *k, *v;
  int64_t q_sn, q_sh, k_sn, k_sp, k_sh, v_sn, v_sp, v_sh;
  const int64_t* lengths;
  void* o;
  float* part;  // (N*H, chunks, D) sums, then (N*H, chunks, 2) maxima (base 2) and weights
  int64_t P, chunk;
  int N, H, Hk, D, chunks;
  float qscale;  // scale * log2(e)
};

__device__ __forceinline__ int64_t length_of(const CachedArgs& a, int n) {
  return min64(max64(a.lengths[n], 0), a.P);
}
__device__ __forceinline__ float* part_stats(const CachedArgs& a) {
  return a.part + (int64_t)a.N * a.H * a.chunks * a.D;
}

// Writes one head's row: the result itself when the key axis is one chunk, else
// the partial.  `sum` is unnormalised, m the maximum (-inf: nothing seen).
template <typename T>
__device__ __forceinline__ void put(const CachedArgs& a, int64_t row, int chunk, int c, float sum, float l) {
  if (a.chunks == 1)
    ((T*)a.o)[row * a.D + c] = from_acc<T>(l > 0.f ? sum / l : l == 0.f ? 0.f : l);
  else
    a.part[(row * a.chunks + chunk) * a.D + c] = sum;
}

// ---------------------------------------------------------------------------
// Any dtype, any strides, D <= 256.  A warp takes 32 keys at a time: LPK lanes
// share a key's row (NVL vectors of VEC elements each), so 32 / LPK keys are read
// per instruction; scores meet in shared memory, where a lane owns a key for the
// softmax; the values are read with the lanes laid out as for the keys.  GB query
// heads of the group per block.
// ---------------------------------------------------------------------------
template <typename T, int VEC, int LPK, int NVL, int GB>
__global__ void __launch_bounds__(kThreads) cached_simt_kernel(const CachedArgs a) {
  constexpr int KPI = 32 / LPK, W = LPK * NVL * VEC;
  __shared__ float sc[kWarps][GB][32];
  __shared__ float jm[kWarps][GB], jl[kWarps][GB];
  __shared__ float jo[kWarps][GB][W];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int kl = lane % LPK, kr = lane / LPK;
  const int group = a.H / a.Hk, gblocks = (group + GB - 1) / GB;
  const int n = blockIdx.y, kvh = blockIdx.z / gblocks, g0 = (blockIdx.z % gblocks) * GB;
  const int gn = min(GB, group - g0);
  const int64_t len = length_of(a, n);
  const int64_t j_begin = (int64_t)blockIdx.x * a.chunk, j_end = min64(len, j_begin + a.chunk);
  if (blockIdx.x > 0 && j_begin >= len) return;  // the join skips this chunk too
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
#pragma unroll 4
    for (int i = 0; i < 32; i += KPI) {
      const int64_t j = j0 + i + kr;
      float s[GB];
#pragma unroll
      for (int g = 0; g < GB; ++g) s[g] = 0.f;
      if (j < j_end) {
#pragma unroll
        for (int x = 0; x < NVL; ++x) {
          const int c = (x * LPK + kl) * VEC;
          float kv[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) kv[e] = 0.f;
          if (c < a.D) load_vec<VEC>(kp + j * a.k_sp + c, kv);
#pragma unroll
          for (int g = 0; g < GB; ++g)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[g] = fmaf(q[g][x][e], kv[e], s[g]);
        }
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
#pragma unroll 4
    for (int i = 0; i < 32; i += KPI) {
      const int64_t j = j0 + i + kr;
      if (j < j_end) {
#pragma unroll
        for (int x = 0; x < NVL; ++x) {
          const int c = (x * LPK + kl) * VEC;
          float vv[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) vv[e] = 0.f;
          if (c < a.D) load_vec<VEC>(vp + j * a.v_sp + c, vv);
#pragma unroll
          for (int g = 0; g < GB; ++g) {
            const float p = sc[warp][g][i + kr];
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[g][x][e] = fmaf(p, vv[e], acc[g][x][e]);
          }
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
    put<T>(a, row0 + g, blockIdx.x, c, sum, ls);
    if (a.chunks > 1 && c == 0) {
      float* st = part_stats(a) + ((row0 + g) * a.chunks + blockIdx.x) * 2;
      st[0] = mx;
      st[1] = ls;
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit types, D a multiple of 8 up to 128, rows on 16-byte boundaries: the heads
// of a group (16 to a block) are the M rows of m16n8k16 products, so the work per
// cached byte stays small for any group.  A warp takes 16 keys at a time.
//
// Both products take their cache operand straight from 16-byte global loads; what
// the fragments want is met by permuting the summed or the free index:
//   S = Q K^T: lane (g = lane/4, c = lane%4) loads chunks 4i + c (8 elements each) of
//     key g; a chunk's register pairs serve as two k-steps, with Q's chunks loaded in
//     the same order.
//   O = P V: the score fragment is the A fragment (keys 2c, 2c+1, 2c+8, 2c+9 of lane
//     c); lane (g, c) loads chunk 8h + g of those four keys, and product t of half h takes
//     element t of every chunk as its column, so a lane ends with whole chunks 8h + 2c
//     and 8h + 2c + 1 of rows g and g + 8.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint4 load16(const void* p, bool in) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (in)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}
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

template <typename T, int DP, bool TALL>  // TALL: the block has more than 8 heads
__global__ void __launch_bounds__(kThreads) cached_mma_kernel(const CachedArgs a) {
  constexpr int KC = DP / 32, VC = DP / 64;
  __shared__ float jm[kWarps][16], jl[kWarps][16];
  __shared__ float jo[kWarps][TALL ? 16 : 8][DP + 4];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, c = lane % 4;
  const int group = a.H / a.Hk, gblocks = (group + 15) / 16;
  const int n = blockIdx.y, kvh = blockIdx.z / gblocks, g0 = (blockIdx.z % gblocks) * 16;
  const int gn = min(16, group - g0);
  const int64_t len = length_of(a, n);
  const int64_t j_begin = (int64_t)blockIdx.x * a.chunk, j_end = min64(len, j_begin + a.chunk);
  if (blockIdx.x > 0 && j_begin >= len) return;  // the join skips this chunk too
  const T* kp = (const T*)a.k + n * a.k_sn + kvh * a.k_sh;
  const T* vp = (const T*)a.v + n * a.v_sn + kvh * a.v_sh;
  uint4 q[TALL ? 2 : 1][KC];
#pragma unroll
  for (int r = 0; r < (TALL ? 2 : 1); ++r)
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int ch = 4 * i + c, row = g + 8 * r;
      q[r][i] = load16((const T*)a.q + n * a.q_sn + (kvh * group + g0 + row) * a.q_sh + ch * 8, row < gn && ch * 8 < a.D);
    }
  float acc[VC][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < VC; ++h)
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h][t][e] = 0.f;

  for (int64_t j0 = j_begin + warp * 16; j0 < j_end; j0 += kWarps * 16) {
    const int left = (int)min64(16, j_end - j0);
    uint4 kk[2][KC], vv[4][VC];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const int key = 8 * b + g, ch = 4 * i + c;
        kk[b][i] = load16(kp + (j0 + key) * a.k_sp + ch * 8, key < left && ch * 8 < a.D);
      }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int h = 0; h < VC; ++h) {
        const int key = 2 * c + (b & 1) + 8 * (b >> 1), ch = 8 * h + g;
        vv[b][h] = load16(vp + (j0 + key) * a.v_sp + ch * 8, key < left && ch * 8 < a.D);
      }
    float s[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[b][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint4 x = q[0][i], y = TALL ? q[TALL ? 1 : 0][i] : make_uint4(0, 0, 0, 0);
        mma16816<T>(s[b], x.x, y.x, x.y, y.y, kk[b][i].x, kk[b][i].y);
        mma16816<T>(s[b], x.z, y.z, x.w, y.w, kk[b][i].z, kk[b][i].w);
      }
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
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vv[0][h]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vv[1][h]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vv[2][h]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vv[3][h]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        mma16816<T>(acc[h][2 * x], a0, a1, a2, a3, __byte_perm(v0[x], v1[x], 0x5410), __byte_perm(v2[x], v3[x], 0x5410));
        mma16816<T>(acc[h][2 * x + 1], a0, a1, a2, a3, __byte_perm(v0[x], v1[x], 0x7632), __byte_perm(v2[x], v3[x], 0x7632));
      }
    }
  }
  // the warps' rows, joined in order
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
        float* o = &jo[warp][g + 8 * r][(8 * h + 2 * c + e) * 8];
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
      const float4 o = *reinterpret_cast<const float4*>(&jo[w][row][col]);
      sum[0] += f * o.x, sum[1] += f * o.y, sum[2] += f * o.z, sum[3] += f * o.w;
      ls += f * jl[w][row];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) put<T>(a, row0 + row, blockIdx.x, col + e, sum[e], ls);
    if (a.chunks > 1 && col == 0) {
      float* st = part_stats(a) + ((row0 + row) * a.chunks + blockIdx.x) * 2;
      st[0] = mx;
      st[1] = ls;
    }
  }
}

// Joins the chunks of a head's row: o = sum_c 2^(m_c - m) sum_c / sum_c 2^(m_c - m) l_c.
// A block per row; eight strands of chunks, joined in order.
template <typename T>
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedArgs a) {
  __shared__ float so[8][256 + 1];
  __shared__ float red[8];
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int n = (int)(row / a.H);
  const int64_t len = length_of(a, n);
  const int used = (int)max64(1, (len + a.chunk - 1) / a.chunk);
  const float* st = part_stats(a) + row * a.chunks * 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  float mx = -INFINITY;
  for (int c = threadIdx.x; c < used; c += 256) mx = fmaxf(mx, st[2 * c]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  if (lane == 0) red[warp] = mx;
  __syncthreads();
  mx = red[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) mx = fmaxf(mx, red[w]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (int c = warp; c < used; c += 8) {
    const float f = exp2f(st[2 * c] - base);
    l += f * st[2 * c + 1];
    const float* p = a.part + (row * a.chunks + c) * a.D;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.D) acc[i] = fmaf(f, p[lane + 32 * i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = acc[i];
  if (lane == 0) so[warp][256] = l;
  __syncthreads();
  const int c = threadIdx.x;
  if (c < a.D) {
    float s = 0.f, ls = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      s += so[w][c];
      ls += so[w][256];
    }
    ((T*)a.o)[row * a.D + c] = from_acc<T>(ls > 0.f ? s / ls : ls == 0.f ? 0.f : ls);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Tokens per chunk: a whole number of block steps (128 tokens), few enough that
// the grid holds about eight blocks per SM, at least 128.
int64_t chunk_tokens(int64_t N, int64_t Hk, int64_t P) {
  const int64_t pairs = max64(1, N * Hk), target = 148 * 8;
  const int64_t chunks = max64(1, min64((P + 127) / 128, (target + pairs - 1) / pairs));
  return max64(128, ((P + chunks - 1) / chunks + 127) / 128 * 128);
}
int64_t chunk_count(int64_t N, int64_t Hk, int64_t P) {
  const int64_t c = chunk_tokens(N, Hk, P);
  return max64(1, (P + c - 1) / c);
}

template <typename T, int VEC, int LPK, int NVL, int GB>
int simt_launch(const CachedArgs& a, cudaStream_t st) {
  const int gblocks = (a.H / a.Hk + GB - 1) / GB;
  cached_simt_kernel<T, VEC, LPK, NVL, GB>
      <<<dim3(a.chunks, a.N, a.Hk * gblocks), kThreads, 0, st>>>(a);
  return check_launch();
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

template <typename T, int DP>
int mma_launch(const CachedArgs& a, cudaStream_t st) {
  const int group = a.H / a.Hk;
  const dim3 grid(a.chunks, a.N, a.Hk * ((group + 15) / 16));
  if (group > 8) cached_mma_kernel<T, DP, true><<<grid, kThreads, 0, st>>>(a);
  else cached_mma_kernel<T, DP, false><<<grid, kThreads, 0, st>>>(a);
  return check_launch();
}

template <typename T>
int cached_typed(const CachedArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  int s;
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 128 && aligned16<T>(a)) {
      s = a.D <= 64 ? mma_launch<T, 64>(a, st) : mma_launch<T, 128>(a, st);
      if (s || a.chunks == 1) return s;
      return launch_pdl(cached_join_kernel<T>, dim3((unsigned)(a.N * a.H)), dim3(256), 0, st, a);
    }
  }
  if (aligned16<T>(a)) {
    if (a.D <= 16 * V) s = simt_group<T, V, 16, 1>(a, st);
    else if (a.D <= 32 * V) s = simt_group<T, V, 32, 1>(a, st);
    else s = simt_group<T, V, 32, 256 / (32 * V)>(a, st);
  } else {
    if (a.D <= 64) s = simt_group<T, 1, 32, 2>(a, st);
    else if (a.D <= 128) s = simt_group<T, 1, 32, 4>(a, st);
    else s = simt_group<T, 1, 32, 8>(a, st);
  }
  if (s || a.chunks == 1) return s;
  return launch_pdl(cached_join_kernel<T>, dim3((unsigned)(a.N * a.H)), dim3(256), 0, st, a);
}

}  // namespace

size_t cached_workspace_size(int64_t N, int64_t H, int64_t Hk, int64_t P, int64_t D) {
  const int64_t chunks = chunk_count(N, Hk, P);
  return chunks == 1 ? 0 : (size_t)(N * H) * chunks * (D + 2) * sizeof(float);
}

int cached_attention(int dtype, const void* q, const int64_t* q_stride, const void* k,
                     const int64_t* k_stride, const void* v, const int64_t* v_stride,
                     const int64_t* lengths, int64_t N, int64_t P, int64_t H, int64_t Hk, int64_t D,
                     float scale, void* o, void* ws, cudaStream_t st) {
  CachedArgs a;
  a.q = q, a.k = k, a.v = v;
  a.q_sn = q_stride[0], a.q_sh = q_stride[1];
  a.k_sn = k_stride[0], a.k_sp = k_stride[1], a.k_sh = k_stride[2];
  a.v_sn = v_stride[0], a.v_sp = v_stride[1], a.v_sh = v_stride[2];
  a.lengths = lengths;
  a.o = o, a.part = (float*)ws;
  a.P = P, a.chunk = chunk_tokens(N, Hk, P);
  a.N = (int)N, a.H = (int)H, a.Hk = (int)Hk, a.D = (int)D, a.chunks = (int)chunk_count(N, Hk, P);
  a.qscale = scale * kLog2e;
  switch (dtype) {
    case TPO_F32: return cached_typed<float>(a, st);
    case TPO_F16: return cached_typed<__half>(a, st);
    case TPO_BF16: return cached_typed<__nv_bfloat16>(a, st);
    default: return set_error(TPO_ERR_INVALID_ARGUMENT, "cached_attention: dtype must be f32, f16 or bf16");
  }
}

}  // namespace tpo
