// Shared by the attention kernels: the problem's description and the map from
// blocks to tiles of packed clouds.
#pragma once

#include "tpo_internal.h"
#include "tpo_types.cuh"

namespace tpo {

// Set by a kernel that met offsets that decrease or leave [0, tokens]
// (TPO_DEVERR_BAD_OFFSETS); what it reads and writes stays clamped.
constexpr unsigned kErrBadOffsets = 4u;
static __device__ unsigned g_attention_error = 0;  // one per translation unit: each is in capi.cu's table
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kHalfLift = 12;  // exponent that lifts P of the fp16 backward on the tensor cores

// One packed problem, by value to every kernel.  Strides in elements; the width
// dimension has stride 1.  o, dq are (Tq, H, D), dk, dv (Tk, Hk, D), lse and
// delta (H, Tq), all contiguous.
struct PackedArgs {
  const void *q, *k, *v, *go;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, go_st, go_sh;  // token and head strides
  const int64_t *off_q, *off_k;
  void *o, *dq, *dk, *dv;
  float *lse, *delta, *lse2;  // lse2: lse in base 2 (backward on the tensor cores; fp16: less kHalfLift), or null
  // fp16 on the tensor cores, else null, each (H, Tq): the length of each row of go, which the dQ
  // kernel replaces by a bound of the row's |dS|; and the largest |v|^2 of each tile of keys, in
  // the row of a group's first head: tile i of a cloud at its query i, those beyond the last query
  // there too (a cloud without queries has no dS).
  float *ds_bound, *v_max;
  int64_t Tq, Tk;
  int B, H, Hk, D, causal;
  float scale;
};

// A tile of one cloud: rows [row0, row0 + rows) of the packed tensor that was
// tiled; [a0, a0 + na) and [b0, b0 + nb) are the cloud's rows there and in the
// other tensor.  rows == 0: nothing to do.  Tokens fit 31 bits (the host checks), and these
// live in every warp of a block: 32-bit fields save it registers.
struct Tile {
  int row0, rows, a0, na, b0, nb;
  // Causal: a row at place x of the tiled side (from the cloud's start) sees keys below
  // edge(x) + 1, or is seen by queries from edge(x) on.  Fits 32 bits in this order.
  __device__ __forceinline__ int edge(int x) const { return (x - na) + nb; }
};

// Blocks per head for tiles of BM rows: with e(i) the start of cloud i, cloud i
// gets the slots from e(i)/BM + i on.  The next cloud's first slot is at least
// ceil(length / BM) further, so every tile has a slot, at most one slot per cloud
// stays empty, and the host needs no lengths.  Two more "clouds" cover the tokens
// before the first and after the last offset; nobody attends there.
inline int64_t packed_slots(int64_t tokens, int64_t clouds, int BM) { return tokens / BM + clouds + 2; }
// The grid: heads within slots, so that the slots' order is the blocks' order.
inline int packed_grid(int64_t tokens, int64_t clouds, int BM, int64_t heads, unsigned* blocks) {
  const int64_t n = packed_slots(tokens, clouds, BM) * heads;
  if (n >= (int64_t(1) << 31)) return set_error(TPO_ERR_UNSUPPORTED, "packed_attention: too many tokens times heads");
  *blocks = (unsigned)n;
  return TPO_OK;
}

// All 32 lanes of a warp call this with the same slot.
//
// With at most 30 clouds every lane holds one of them after one round of loads, and the
// slots go to the clouds by falling length, so that no long tile starts last (late_first:
// a cloud's last tile first, where causal rows see most keys).  With more, a search with
// 32 probes a round finds the cloud, in the clouds' own order.
__device__ __forceinline__ Tile find_tile(const int64_t* off, int64_t T, const int64_t* other,
                                          int64_t To, int B, int BM, int64_t slot, int64_t slots,
                                          bool late_first) {
  const int lane = threadIdx.x & 31;
  // clamped start of extended cloud i in [0, B + 2], from its raw offset
  auto start = [&](int i, int64_t raw) -> int64_t { return i == 0 ? 0 : i >= B + 2 ? T : min64(max64(raw, 0), T); };
  int lo = 0, lo0 = 0;  // lane k holds the offsets of cloud lo0 + k
  int64_t raw = 0, raw_other = 0, tile;
  if (B + 2 <= 31) {
    const bool in = lane >= 1 && lane <= B + 1;
    raw = in ? off[lane - 1] : 0;
    raw_other = in ? other[lane - 1] : 0;
    const int64_t s = start(lane, raw), e = __shfl_down_sync(0xffffffffu, s, 1);
    const int64_t next = __shfl_down_sync(0xffffffffu, raw, 1), next_other = __shfl_down_sync(0xffffffffu, raw_other, 1);
    if (lane >= 1 && lane <= B && (raw < 0 || next < raw || next > T || raw_other < 0 || next_other < raw_other || next_other > To))
      atomicOr(&g_attention_error, kErrBadOffsets);
    const int len = lane < B + 2 ? (int)max64(e - s, 0) : 0;  // tokens fit 31 bits
    int before = 0;  // tiles of longer clouds
    for (int i = 0; i < B + 2; ++i) {
      const int l = __shfl_sync(0xffffffffu, len, i);
      if (l > len || (l == len && i < lane)) before += (l + BM - 1) / BM;
    }
    const int mine = (len + BM - 1) / BM;
    const unsigned m = __ballot_sync(0xffffffffu, slot >= before && slot < before + mine);
    lo = m ? __ffs(m) - 1 : 0;
    tile = m ? slot - __shfl_sync(0xffffffffu, before, lo) : T;  // no tile left: behind every row
    if (late_first && m) tile = __shfl_sync(0xffffffffu, mine, lo) - 1 - tile;
  } else {
    if (slot == 0) {  // the first block of a head looks all offsets over
      for (int i = lane; i < B; i += 32) {
        const int64_t r0 = off[i], r1 = off[i + 1], o0 = other[i], o1 = other[i + 1];
        if (r0 < 0 || r1 < r0 || r1 > T || o0 < 0 || o1 < o0 || o1 > To) atomicOr(&g_attention_error, kErrBadOffsets);
      }
    }
    if (late_first) slot = slots - 1 - slot;
    int hi = B + 2;
    while (hi - lo > 1) {  // greatest i in [lo, hi) with start(i)/BM + i <= slot
      const int width = (hi - lo + 31) / 32;
      const int i = lo + lane * width;
      const bool le = i < hi && (lane == 0 || start(i, i >= 1 && i <= B + 1 ? off[i - 1] : 0) / BM + i <= slot);
      const unsigned m = __ballot_sync(0xffffffffu, le);
      const int last = 31 - __clz(m);
      hi = min(hi, lo + (last + 1) * width);
      lo += last * width;
    }
    lo0 = lo;
    const int i = lo + lane;
    const bool in = lane < 2 && i >= 1 && i <= B + 1;
    raw = in ? off[i - 1] : 0;
    raw_other = in ? other[i - 1] : 0;
    tile = slot - (start(lo, __shfl_sync(0xffffffffu, raw, 0)) / BM + lo);
  }
  const int64_t r0 = __shfl_sync(0xffffffffu, raw, lo - lo0), r1 = __shfl_sync(0xffffffffu, raw, lo - lo0 + 1);
  const int64_t o0 = __shfl_sync(0xffffffffu, raw_other, lo - lo0), o1 = __shfl_sync(0xffffffffu, raw_other, lo - lo0 + 1);
  const int64_t a0 = start(lo, r0), end = start(lo + 1, r1), row0 = a0 + tile * BM;
  Tile t;
  t.a0 = (int)a0;
  t.na = (int)max64(end - a0, 0);
  t.rows = row0 < a0 ? 0 : (int)max64(0, min64(end - row0, BM));
  t.row0 = t.rows ? (int)row0 : 0;
  t.b0 = t.nb = 0;
  if (lo >= 1 && lo <= B) {
    const int64_t b0 = min64(max64(o0, 0), To);
    t.b0 = (int)b0;
    t.nb = (int)max64(min64(max64(o1, 0), To) - b0, 0);
  }
  return t;
}

static inline int attention_error_word(unsigned** word) {  // of this translation unit
  return cuda_status(cudaGetSymbolAddress((void**)word, g_attention_error));
}

int packed_simt_forward(int dtype, const PackedArgs& a, cudaStream_t st);
int packed_simt_backward(int dtype, const PackedArgs& a, cudaStream_t st);
// Whether the tensor-core kernels take the problem, and those kernels.
bool packed_mma_takes(int dtype, const PackedArgs& a, bool backward);
int packed_mma_forward(int dtype, const PackedArgs& a, cudaStream_t st);
int packed_mma_backward(int dtype, const PackedArgs& a, cudaStream_t st);
int packed_delta(int dtype, const PackedArgs& a, cudaStream_t st);

}  // namespace tpo
