// Host side of attention over packed clouds: which kernels a problem takes.
#include "attention_common.cuh"

namespace tpo {
namespace {

PackedArgs args_of(const tpo_packed_attention* p) {
  PackedArgs a = {};
  a.q = p->q, a.k = p->k, a.v = p->v;
  a.q_st = p->q_token_stride, a.q_sh = p->q_head_stride;
  a.k_st = p->k_token_stride, a.k_sh = p->k_head_stride;
  a.v_st = p->v_token_stride, a.v_sh = p->v_head_stride;
  a.off_q = p->offsets_q, a.off_k = p->offsets_k;
  a.Tq = p->tokens_q, a.Tk = p->tokens_k;
  a.B = (int)p->clouds, a.H = (int)p->heads, a.Hk = (int)p->kv_heads, a.D = (int)p->width;
  a.causal = p->causal != 0;
  a.scale = p->scale;
  return a;
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

// [delta][lse in base 2][bound of |dS|][largest |v|^2], each (heads, tokens_q)
static size_t packed_stat_bytes(int64_t tokens_q, int64_t heads) {
  return align256((size_t)tokens_q * heads * sizeof(float)) + 256;
}
size_t packed_bwd_workspace_size(int64_t tokens_q, int64_t heads) { return 4 * packed_stat_bytes(tokens_q, heads); }

int packed_forward(const tpo_packed_attention* p, void* o, float* lse, cudaStream_t st) {
  PackedArgs a = args_of(p);
  a.o = o, a.lse = lse;
  return packed_mma_takes(p->dtype, a, false) ? packed_mma_forward(p->dtype, a, st)
                                              : packed_simt_forward(p->dtype, a, st);
}

int packed_backward(const tpo_packed_attention* p, const void* o, const float* lse, const void* grad_o,
                    int64_t go_token_stride, int64_t go_head_stride, void* dq, void* dk, void* dv,
                    void* ws, cudaStream_t st) {
  PackedArgs a = args_of(p);
  a.o = const_cast<void*>(o), a.lse = const_cast<float*>(lse), a.go = grad_o;
  a.go_st = go_token_stride, a.go_sh = go_head_stride;
  a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = (float*)ws;
  const bool mma = packed_mma_takes(p->dtype, a, true);
  if (mma) a.lse2 = (float*)((char*)ws + packed_stat_bytes(a.Tq, a.H));
  if (mma && p->dtype == TPO_F16) {
    a.ds_bound = (float*)((char*)ws + 2 * packed_stat_bytes(a.Tq, a.H));
    a.v_max = (float*)((char*)ws + 3 * packed_stat_bytes(a.Tq, a.H));
  }
  int s;
  if (a.Tq > 0 && (s = packed_delta(p->dtype, a, st))) return s;
  return mma ? packed_mma_backward(p->dtype, a, st) : packed_simt_backward(p->dtype, a, st);
}

}  // namespace tpo
