// extern "C" boundary of libtpo_b200 (declared in include/tpo_b200.h).
// Validates arguments, never aborts, returns tpo_status codes.
#include <cstdio>
#include <cstring>

#include "tpo_internal.h"

namespace tpo {

static thread_local char g_msg[256] = "";

int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return TPO_OK;
  snprintf(g_msg, sizeof(g_msg), "CUDA error: %s", cudaGetErrorString(e));
  return TPO_ERR_CUDA;
}
int check_launch() { return cuda_status(cudaGetLastError()); }

static bool valid_dtype(int dt) { return dt == TPO_F32 || dt == TPO_F16 || dt == TPO_F64; }

static int fail(int code, const char* what) {
  snprintf(g_msg, sizeof(g_msg), "%s", what);
  return code;
}

int set_error(int code, const char* msg) { return fail(code, msg); }

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace tpo

using namespace tpo;

extern "C" {

int tpo_abi_version(void) { return TPO_B200_ABI_VERSION; }

const char* tpo_status_string(int status) {
  switch (status) {
    case TPO_OK: return "ok";
    case TPO_ERR_INVALID_ARGUMENT: return g_msg[0] ? g_msg : "invalid argument";
    case TPO_ERR_UNSUPPORTED: return g_msg[0] ? g_msg : "unsupported";
    case TPO_ERR_WORKSPACE: return g_msg[0] ? g_msg : "workspace too small";
    case TPO_ERR_CUDA: return g_msg[0] ? g_msg : "CUDA error";
    case TPO_ERR_DEVICE: return g_msg[0] ? g_msg : "no usable device";
  }
  return "unknown status";
}

// Every file whose kernels set error flags.
static int (*const kErrorWords[])(unsigned**) = {chamfer_error_word,        fps_error_word,           knn_error_word,
                                                 attention_simt_error_word, attention_mma_error_word, attention_cached_error_word};

int tpo_device_error_flags(unsigned* flags, int clear) {
  if (!flags) return fail(TPO_ERR_INVALID_ARGUMENT, "device_error_flags: null output");
  *flags = 0;
  for (auto word_of : kErrorWords) {
    unsigned *word = nullptr, value = 0;
    const unsigned zero = 0;
    int s = word_of(&word);
    if (!s) s = cuda_status(cudaMemcpy(&value, word, sizeof value, cudaMemcpyDeviceToHost));
    if (!s && clear) s = cuda_status(cudaMemcpy(word, &zero, sizeof zero, cudaMemcpyHostToDevice));
    if (s) return s;
    *flags |= value;
  }
  return TPO_OK;
}

int tpo_device_error_raise(int unit, unsigned flags) {
  if (unit < 0 || unit >= (int)(sizeof kErrorWords / sizeof *kErrorWords))
    return fail(TPO_ERR_INVALID_ARGUMENT, "device_error_raise: no such unit");
  unsigned *word = nullptr, value = 0;
  int s = kErrorWords[unit](&word);
  if (!s) s = cuda_status(cudaMemcpy(&value, word, sizeof value, cudaMemcpyDeviceToHost));
  value |= flags;
  return s ? s : cuda_status(cudaMemcpy(word, &value, sizeof value, cudaMemcpyHostToDevice));
}

int tpo_chamfer_key_bytes(int dtype) {
  if (!valid_dtype(dtype)) return 0;
  return dtype == TPO_F64 ? 16 : 8;
}

size_t tpo_chamfer_fwd_workspace_size(int dtype, int64_t B, int64_t N, int64_t M) {
  if (!valid_dtype(dtype) || B < 0 || N < 0 || M < 0) return 0;
  const size_t kb = (size_t)tpo_chamfer_key_bytes(dtype);
  return align256(kb * (size_t)B * (size_t)N) + align256(kb * (size_t)B * (size_t)M);
}

int tpo_chamfer_keys_init(int dtype, void* keys, int64_t n, void* stream) {
  if (!valid_dtype(dtype) || n < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "keys_init: bad dtype or size");
  if (n == 0) return TPO_OK;
  if (!keys) return fail(TPO_ERR_INVALID_ARGUMENT, "keys_init: null keys");
  return cuda_status(cudaMemsetAsync(keys, 0xff, (size_t)n * tpo_chamfer_key_bytes(dtype),
                                     (cudaStream_t)stream));
}

static int check_chamfer_shape(int dtype, const void* x1, const void* x2, int64_t B, int64_t N,
                               int64_t M) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: dtype must be f32, f16 or f64");
  if (B < 0 || N < 0 || M < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: negative size");
  if (N >= (int64_t(1) << 31) || M >= (int64_t(1) << 31))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: clouds are limited to 2^31-1 points (int32 indices)");
  if ((B * N > 0 && !x1) || (B * M > 0 && !x2)) return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: null input");
  return TPO_OK;
}

int tpo_chamfer_fwd_keys(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                         int64_t N, int64_t M, int64_t row_begin, int64_t row_end, void* keys1,
                         void* keys2, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (row_begin < 0 || row_end > N || row_begin > row_end)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: bad row range");
  if (B * (row_end - row_begin) > 0 && M > 0 && (!keys1 || !keys2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: null keys");
  return chamfer_fwd_keys(dtype, flags, xyz1, xyz2, B, N, M, row_begin, row_end, keys1, keys2,
                          (cudaStream_t)stream);
}

int tpo_chamfer_finalize(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                         int64_t N, int64_t M, int64_t row_begin, int64_t row_end,
                         const void* keys1, const void* keys2, void* dist1, int32_t* idx1,
                         void* dist2, int32_t* idx2, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (row_begin < 0 || row_end > N || row_begin > row_end)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: bad row range");
  if (B * (row_end - row_begin) > 0 && (!dist1 || !idx1 || (M > 0 && !keys1)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: null row outputs");
  if (dist2 && B * M > 0 && (!idx2 || (N > 0 && !keys2)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: null column outputs");
  return chamfer_finalize(dtype, flags, xyz1, xyz2, B, N, M, row_begin, row_end, keys1, keys2,
                          dist1, idx1, dist2, idx2, dist2 != nullptr, nullptr, 0, nullptr,
                          (cudaStream_t)stream);
}

int tpo_chamfer_fwd(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                    int64_t N, int64_t M, void* dist1, void* dist2, int32_t* idx1, int32_t* idx2,
                    void* workspace, size_t workspace_bytes, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if ((B * N > 0 && (!dist1 || !idx1)) || (B * M > 0 && (!dist2 || !idx2)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer: null output");
  const size_t need = tpo_chamfer_fwd_workspace_size(dtype, B, N, M);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(TPO_ERR_WORKSPACE, "chamfer: workspace missing or smaller than tpo_chamfer_fwd_workspace_size()");
  if ((uintptr_t)workspace % 256) return fail(TPO_ERR_WORKSPACE, "chamfer: workspace must be 256-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  const size_t kb = (size_t)tpo_chamfer_key_bytes(dtype);
  char* k1 = (char*)workspace;
  char* k2 = k1 + align256(kb * (size_t)B * (size_t)N);
  if (B > 0 && N > 0 && M > 0) {
    const size_t es = (size_t)dtype_size(dtype);
    if ((s = fill_prefetch(workspace, need, nullptr, 0, 0xff, xyz1, es * 3 * B * N, xyz2,
                           es * 3 * B * M, st)))
      return s;
    if ((s = chamfer_fwd_keys(dtype, flags, xyz1, xyz2, B, N, M, 0, N, k1, k2, st))) return s;
  }
  return chamfer_finalize(dtype, flags, xyz1, xyz2, B, N, M, 0, N, k1, k2, dist1, idx1, dist2, idx2,
                          true, nullptr, 0, nullptr, st);
}

int tpo_chamfer_bwd(int dtype, const void* xyz1, const void* xyz2, int64_t B, int64_t N,
                    int64_t M, const int32_t* idx1, const int32_t* idx2, const void* grad_dist1,
                    const void* grad_dist2, void* grad_xyz1, void* grad_xyz2, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if ((B * N > 0 && !grad_xyz1) || (B * M > 0 && !grad_xyz2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_bwd: null gradient output");
  if ((grad_dist1 && B * N > 0 && !idx1) || (grad_dist2 && B * M > 0 && !idx2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_bwd: null index");
  cudaStream_t st = (cudaStream_t)stream;
  const size_t es = (size_t)dtype_size(dtype);
  if (B * N > 0 && (s = cuda_status(cudaMemsetAsync(grad_xyz1, 0, es * 3 * B * N, st)))) return s;
  if (B * M > 0 && (s = cuda_status(cudaMemsetAsync(grad_xyz2, 0, es * 3 * B * M, st)))) return s;
  return chamfer_bwd_accumulate(dtype, xyz1, xyz2, B, N, M, 0, N, 0, M, idx1, idx2, grad_dist1,
                                grad_dist2, nullptr, 0, grad_xyz1, grad_xyz2, st);
}

int tpo_chamfer_bwd_partial(int dtype, const void* xyz1, const void* xyz2, int64_t B, int64_t N,
                            int64_t M, int64_t row_begin, int64_t row_end, int64_t col_begin,
                            int64_t col_end, const int32_t* idx1, const int32_t* idx2,
                            const void* grad_dist1, const void* grad_dist2, void* grad_xyz1,
                            void* grad_xyz2, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (row_begin < 0 || row_end > N || row_begin > row_end || col_begin < 0 || col_end > M ||
      col_begin > col_end)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_bwd_partial: bad range");
  if ((B * N > 0 && !grad_xyz1) || (B * M > 0 && !grad_xyz2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_bwd_partial: null gradient output");
  return chamfer_bwd_accumulate(dtype, xyz1, xyz2, B, N, M, row_begin, row_end, col_begin, col_end,
                                idx1, idx2, grad_dist1, grad_dist2, nullptr, 0, grad_xyz1,
                                grad_xyz2, (cudaStream_t)stream);
}

// Fused-loss workspace: everything the backward needs stays in it.
//   [keys1|keys2][keys-loss counters|batch partials][finalize partials|counter][idx1][idx2]
// fp32 with a non-empty problem uses the keys kernel's fused reduction and the
// backward re-derives the neighbours from the keys; other cases finalize into
// idx1/idx2 and reduce there.
struct LossLayout {
  size_t keys, kl, fin, idx1, idx2, g1, g2, total;
};
static LossLayout loss_layout(int dtype, int64_t B, int64_t N, int64_t M) {
  LossLayout L;
  L.keys = 0;
  L.kl = tpo_chamfer_fwd_workspace_size(dtype, B, N, M);
  L.fin = L.kl + keys_loss_bytes(B);
  L.idx1 = L.fin + align256(kFinLossWorkspace);
  L.idx2 = L.idx1 + align256(4 * (size_t)B * (size_t)N);
  // gradient region, zero-filled by the forward (tpo_chamfer_loss_bwd_workspace)
  const size_t es = (size_t)dtype_size(dtype);
  L.g1 = L.idx2 + align256(4 * (size_t)B * (size_t)M);
  L.g2 = L.g1 + align256(es * 3 * (size_t)B * (size_t)N);
  L.total = L.g2 + align256(es * 3 * (size_t)B * (size_t)M);
  return L;
}
static bool loss_uses_keys_kernel(int dtype, int64_t B, int64_t N, int64_t M) {
  return (dtype == TPO_F32 || dtype == TPO_F16) && B > 0 && N > 0 && M > 0;
}

size_t tpo_chamfer_loss_workspace_size(int dtype, int64_t B, int64_t N, int64_t M) {
  if (!valid_dtype(dtype) || B < 0 || N < 0 || M < 0) return 0;
  return loss_layout(dtype, B, N, M).total;
}

int tpo_chamfer_loss_fwd(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                         int64_t N, int64_t M, int reduction, void* loss, void* workspace,
                         size_t workspace_bytes, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (reduction != TPO_REDUCE_MEAN && reduction != TPO_REDUCE_SUM)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss: reduction must be TPO_REDUCE_MEAN or TPO_REDUCE_SUM");
  if (!loss) return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss: null loss");
  const LossLayout L = loss_layout(dtype, B, N, M);
  if (!workspace || workspace_bytes < L.total || (uintptr_t)workspace % 256)
    return fail(TPO_ERR_WORKSPACE, "chamfer_loss: workspace missing, unaligned or smaller than tpo_chamfer_loss_workspace_size()");
  cudaStream_t st = (cudaStream_t)stream;
  char* w = (char*)workspace;
  const size_t kb = (size_t)tpo_chamfer_key_bytes(dtype);
  char* k1 = w;
  char* k2 = k1 + align256(kb * (size_t)B * (size_t)N);
  if (loss_uses_keys_kernel(dtype, B, N, M)) {
    // keys to the empty key and the reduction counters to 0xffffffff: one fill
    const size_t es = (size_t)dtype_size(dtype);
    // ... and the gradient region to zero, in the same launch
    if ((s = fill_prefetch(w, L.kl + keys_loss_counter_bytes(B), w + L.g1, L.total - L.g1, 0xff,
                           xyz1, es * 3 * B * N, xyz2, es * 3 * B * M, st, 0)))
      return s;
    return chamfer_loss_keys(dtype, flags, xyz1, xyz2, B, N, M, reduction, k1, k2, w + L.kl, loss,
                             w + L.fin, st);
  }
  if (L.kl && (s = cuda_status(cudaMemsetAsync(w, 0xff, L.kl, st)))) return s;
  if ((s = cuda_status(cudaMemsetAsync(w + L.fin + kFinPartialBytes, 0xff, 256, st)))) return s;
  if (L.total > L.g1 && (s = cuda_status(cudaMemsetAsync(w + L.g1, 0, L.total - L.g1, st)))) return s;
  if (B > 0 && N > 0 && M > 0 &&
      (s = chamfer_fwd_keys(dtype, flags, xyz1, xyz2, B, N, M, 0, N, k1, k2, st)))
    return s;
  return chamfer_finalize(dtype, flags, xyz1, xyz2, B, N, M, 0, N, k1, k2, nullptr,
                          (int32_t*)(w + L.idx1), nullptr, (int32_t*)(w + L.idx2), true, loss,
                          reduction, w + L.fin, st);
}

// The gradient scatter of the fused loss into (already zeroed) gradient buffers.
static int loss_bwd_scatter(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                            int64_t N, int64_t M, int reduction, const char* w,
                            const void* grad_loss, void* grad_xyz1, void* grad_xyz2, cudaStream_t st) {
  const LossLayout L = loss_layout(dtype, B, N, M);
  if (loss_uses_keys_kernel(dtype, B, N, M)) {
    const size_t kb = (size_t)tpo_chamfer_key_bytes(dtype);
    return chamfer_bwd_from_keys(dtype, flags, xyz1, xyz2, B, N, M, w,
                                 w + align256(kb * (size_t)B * (size_t)N), grad_loss, reduction,
                                 grad_xyz1, grad_xyz2, st);
  }
  return chamfer_bwd_accumulate(dtype, xyz1, xyz2, B, N, M, 0, N, 0, M,
                                (const int32_t*)(w + L.idx1), (const int32_t*)(w + L.idx2),
                                nullptr, nullptr, grad_loss,
                                reduction == TPO_REDUCE_MEAN ? 1 : 2, grad_xyz1, grad_xyz2, st);
}

int tpo_chamfer_loss_bwd(int dtype, int flags, const void* xyz1, const void* xyz2, int64_t B,
                         int64_t N, int64_t M, int reduction, const void* workspace,
                         const void* grad_loss, void* grad_xyz1, void* grad_xyz2, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (reduction != TPO_REDUCE_MEAN && reduction != TPO_REDUCE_SUM)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss_bwd: bad reduction");
  if (!grad_loss || !workspace || (B * N > 0 && !grad_xyz1) || (B * M > 0 && !grad_xyz2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss_bwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const size_t es = (size_t)dtype_size(dtype);
  if ((s = fill_prefetch(grad_xyz1, es * 3 * B * N, grad_xyz2, es * 3 * B * M, 0, nullptr, 0,
                         nullptr, 0, st)))
    return s;
  return loss_bwd_scatter(dtype, flags, xyz1, xyz2, B, N, M, reduction, (const char*)workspace,
                          grad_loss, grad_xyz1, grad_xyz2, st);
}

size_t tpo_chamfer_loss_grad_offset(int dtype, int64_t B, int64_t N, int64_t M, int which) {
  if (!valid_dtype(dtype) || B < 0 || N < 0 || M < 0 || (which != 1 && which != 2)) return 0;
  const LossLayout L = loss_layout(dtype, B, N, M);
  return which == 1 ? L.g1 : L.g2;
}

int tpo_chamfer_loss_bwd_workspace(int dtype, int flags, const void* xyz1, const void* xyz2,
                                   int64_t B, int64_t N, int64_t M, int reduction,
                                   void* workspace, const void* grad_loss, void* stream) {
  int s = check_chamfer_shape(dtype, xyz1, xyz2, B, N, M);
  if (s) return s;
  if (reduction != TPO_REDUCE_MEAN && reduction != TPO_REDUCE_SUM)
    return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss_bwd_workspace: bad reduction");
  if (!grad_loss || !workspace) return fail(TPO_ERR_INVALID_ARGUMENT, "chamfer_loss_bwd_workspace: null pointer");
  const LossLayout L = loss_layout(dtype, B, N, M);
  char* w = (char*)workspace;
  return loss_bwd_scatter(dtype, flags, xyz1, xyz2, B, N, M, reduction, w, grad_loss, w + L.g1,
                          w + L.g2, (cudaStream_t)stream);
}

static int check_knn(int dtype, const void* p1, const void* p2, int64_t N, int64_t P1, int64_t P2,
                     int64_t D, int64_t norm, int64_t K) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: dtype must be f32, f16 or f64");
  if (N < 0 || P1 < 0 || P2 < 0 || D < 1) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: bad shape");
  if (norm != 1 && norm != 2) return fail(TPO_ERR_INVALID_ARGUMENT, "Norm must be 1 or 2.");
  if (K < 1) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: K must be >= 1");
  if (K > kKnnMaxK) return fail(TPO_ERR_UNSUPPORTED, "knn: this build supports K <= 1024");
  if (P2 >= (int64_t(1) << 31)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: P2 limited to 2^31-1");
  if ((N * P1 > 0 && !p1) || (N * P2 > 0 && !p2)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: null input");
  return TPO_OK;
}

int tpo_knn_fwd(int dtype, int flags, const void* p1, const void* p2, const int64_t* lengths1,
                const int64_t* lengths2, int64_t N, int64_t P1, int64_t P2, int64_t D,
                int64_t norm, int64_t K, void* dists, int64_t* idxs, void* stream) {
  int s = check_knn(dtype, p1, p2, N, P1, P2, D, norm, K);
  if (s) return s;
  if (N * P1 > 0 && (!dists || !idxs)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn: null output");
  return knn_forward(dtype, flags, p1, p2, lengths1, lengths2, N, P1, P2, D, norm, K, dists, idxs,
                     (cudaStream_t)stream);
}

int tpo_knn_bwd(int dtype, const void* p1, const void* p2, const int64_t* lengths1,
                const int64_t* lengths2, const int64_t* idxs, int64_t N, int64_t P1, int64_t P2,
                int64_t D, int64_t K, int64_t norm, const void* grad_dists, void* grad_p1,
                void* grad_p2, void* stream) {
  int s = check_knn(dtype, p1, p2, N, P1, P2, D, norm, K);
  if (s) return s;
  if ((N * P1 > 0 && (!grad_p1 || !idxs || !grad_dists)) || (N * P2 > 0 && !grad_p2))
    return fail(TPO_ERR_INVALID_ARGUMENT, "knn_bwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  if (N * P2 > 0 &&
      (s = cuda_status(cudaMemsetAsync(grad_p2, 0, (size_t)dtype_size(dtype) * N * P2 * D, st))))
    return s;
  return knn_backward(dtype, p1, p2, lengths1, lengths2, idxs, N, P1, P2, D, K, norm, grad_dists,
                      grad_p1, grad_p2, st);
}

int tpo_knn_gather_fwd(int dtype, const void* x, const int64_t* idx, const int64_t* lengths,
                       int64_t N, int64_t M, int64_t U, int64_t L, int64_t K, void* out,
                       void* stream) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather: bad dtype");
  if (N < 0 || M < 0 || U < 0 || L < 0 || K < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather: bad shape");
  if (N * L * K * U > 0 && (!idx || !out || (M * U > 0 && !x)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather: null pointer");
  return knn_gather_forward(dtype, x, idx, lengths, N, M, U, L, K, out, (cudaStream_t)stream);
}

int tpo_knn_gather_bwd(int dtype, const void* grad_out, const int64_t* idx, const int64_t* lengths,
                       int64_t N, int64_t M, int64_t U, int64_t L, int64_t K, void* grad_x,
                       void* stream) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather_bwd: bad dtype");
  if (N < 0 || M < 0 || U < 0 || L < 0 || K < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather_bwd: bad shape");
  if (N * M * U > 0 && !grad_x) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather_bwd: null grad_x");
  if (N * L * K * U > 0 && (!idx || !grad_out)) return fail(TPO_ERR_INVALID_ARGUMENT, "knn_gather_bwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  int s;
  if (N * M * U > 0 &&
      (s = cuda_status(cudaMemsetAsync(grad_x, 0, (size_t)dtype_size(dtype) * N * M * U, st))))
    return s;
  return knn_gather_backward(dtype, grad_out, idx, lengths, N, M, U, L, K, grad_x, st);
}

size_t tpo_fps_workspace_size(int dtype, int64_t B, int64_t P) {
  if (!valid_dtype(dtype) || B < 0 || P <= 0) return 0;
  return fps_workspace_size(dtype, B, P);
}

int tpo_fps_fwd(int dtype, const void* points, int64_t B, int64_t P, int64_t S, int64_t* idx,
                void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "fps: dtype must be f32, f16 or f64");
  if (B < 0 || P < 0 || P > INT32_MAX) return fail(TPO_ERR_INVALID_ARGUMENT, "fps: bad shape");
  if (S <= 0) return fail(TPO_ERR_INVALID_ARGUMENT, "fps: nsamples must be positive");
  if (S > P) return fail(TPO_ERR_INVALID_ARGUMENT, "fps: nsamples cannot exceed number of points");
  if (B > 0 && (!points || !idx)) return fail(TPO_ERR_INVALID_ARGUMENT, "fps: null pointer");
  return fps_forward(dtype, points, B, P, S, idx, workspace, workspace_bytes, (cudaStream_t)stream);
}

int tpo_gather_points_fwd(int dtype, const void* points, const int64_t* idx, int64_t N, int64_t C,
                          int64_t P, int64_t M, void* out, void* stream) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points: bad dtype");
  if (N < 0 || C < 0 || P < 0 || M < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points: bad shape");
  if (N * C * M > 0 && (!points || !idx || !out)) return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points: null pointer");
  return gather_points_forward(dtype, points, idx, N, C, P, M, out, (cudaStream_t)stream);
}

int tpo_gather_points_bwd(int dtype, const void* grad_out, const int64_t* idx, int64_t N, int64_t C,
                          int64_t P, int64_t M, void* grad_points, void* stream) {
  if (!valid_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points_bwd: bad dtype");
  if (N < 0 || C < 0 || P < 0 || M < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points_bwd: bad shape");
  if ((N * C * P > 0 && !grad_points) || (N * C * M > 0 && (!grad_out || !idx)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "gather_points_bwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  int s;
  if (N * C * P > 0 &&
      (s = cuda_status(cudaMemsetAsync(grad_points, 0, (size_t)dtype_size(dtype) * N * C * P, st))))
    return s;
  return gather_points_backward(dtype, grad_out, idx, N, C, P, M, grad_points, st);
}

// ---- token operators: layer norm, attention ----

static int check_layer_norm(int dtype, int wdtype, const void* x, int64_t x_stride, int64_t rows,
                            int64_t width) {
  const bool half = dtype == TPO_F16 || dtype == TPO_BF16;
  if (dtype < TPO_F32 || dtype > TPO_BF16)
    return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: dtype must be f32, f16, bf16 or f64");
  if (wdtype != dtype && !(half && wdtype == TPO_F32))
    return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: weight and bias must have the rows' dtype, or f32 with 16-bit rows");
  if (rows < 0 || width < 0 || width > INT32_MAX)
    return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: bad shape");
  if (x_stride < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: negative row stride");
  if (rows * width > 0 && !x) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: null input");
  return TPO_OK;
}

int tpo_layer_norm_fwd(int dtype, int wdtype, const void* x, int64_t x_stride, const void* weight,
                       const void* bias, int64_t rows, int64_t width, double eps, void* y, void* mean,
                       void* rstd, void* stream) {
  int s = check_layer_norm(dtype, wdtype, x, x_stride, rows, width);
  if (s) return s;
  if (!(eps >= 0)) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: eps must not be negative");
  if (!mean != !rstd) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: mean and rstd go together");
  if (rows == 0 || width == 0) return TPO_OK;
  if (!y) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm: null output");
  return layer_norm_forward(dtype, wdtype, x, x_stride, weight, bias, rows, width, eps, y, mean, rstd,
                            (cudaStream_t)stream);
}

size_t tpo_layer_norm_bwd_workspace_size(int dtype, int64_t rows, int64_t width) {
  if (dtype < TPO_F32 || dtype > TPO_BF16 || rows <= 0 || width <= 0) return 0;
  return layer_norm_bwd_workspace_size(dtype, rows, width);
}

int tpo_layer_norm_bwd(int dtype, int wdtype, const void* x, int64_t x_stride, const void* dy,
                       int64_t dy_stride, const void* weight, const void* mean, const void* rstd,
                       int64_t rows, int64_t width, void* dx, void* dweight, void* dbias,
                       void* workspace, size_t workspace_bytes, void* stream) {
  int s = check_layer_norm(dtype, wdtype, x, x_stride, rows, width);
  if (s) return s;
  if (dy_stride < 0) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm_bwd: negative row stride");
  if (width == 0) return TPO_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {  // sums over no rows
    const size_t n = (size_t)dtype_size(wdtype) * width;
    if (dweight && (s = cuda_status(cudaMemsetAsync(dweight, 0, n, st)))) return s;
    return dbias ? cuda_status(cudaMemsetAsync(dbias, 0, n, st)) : TPO_OK;
  }
  if (!dy || !mean || !rstd) return fail(TPO_ERR_INVALID_ARGUMENT, "layer_norm_bwd: null pointer");
  if (!dx && !dweight && !dbias) return TPO_OK;
  if ((dweight || dbias) &&
      (!workspace || workspace_bytes < layer_norm_bwd_workspace_size(dtype, rows, width)))
    return fail(TPO_ERR_WORKSPACE, "layer_norm_bwd: workspace missing or smaller than tpo_layer_norm_bwd_workspace_size()");
  if ((uintptr_t)workspace % 16) return fail(TPO_ERR_WORKSPACE, "layer_norm_bwd: workspace must be 16-byte aligned");
  return layer_norm_backward(dtype, wdtype, x, x_stride, dy, dy_stride, weight, mean, rstd, rows, width,
                             dx, dweight, dbias, workspace, st);
}

static bool attention_dtype(int dt) { return dt == TPO_F32 || dt == TPO_F16 || dt == TPO_BF16; }

static int check_packed(const tpo_packed_attention* p) {
  if (!p) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: null problem");
  if (!attention_dtype(p->dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: dtype must be f32, f16 or bf16");
  if (p->clouds < 0 || p->clouds > (1 << 24) || p->tokens_q < 0 || p->tokens_k < 0 ||
      p->tokens_q > INT32_MAX - 1024 || p->tokens_k > INT32_MAX - 1024)
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: bad shape");
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0 || p->heads > 65535)
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: heads must be a multiple of kv_heads (at most 65535)");
  if (p->width < 1) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: width must be positive");
  if (p->width > kAttentionMaxWidth) return fail(TPO_ERR_UNSUPPORTED, "packed_attention: width is limited to 256");
  if (!(p->scale > 0) || p->scale > 1e30f)
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: scale must be positive and finite");
  if (p->q_token_stride < 0 || p->q_head_stride < 0 || p->k_token_stride < 0 || p->k_head_stride < 0 ||
      p->v_token_stride < 0 || p->v_head_stride < 0)
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: negative stride");
  if (!p->offsets_q || !p->offsets_k) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: null offsets");
  if ((p->tokens_q > 0 && !p->q) || (p->tokens_k > 0 && (!p->k || !p->v)))
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: null input");
  return TPO_OK;
}

int tpo_packed_attention_fwd(const tpo_packed_attention* p, void* o, float* lse, void* stream) {
  int s = check_packed(p);
  if (s) return s;
  if (p->tokens_q == 0) return TPO_OK;
  if (!o) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention: null output");
  return packed_forward(p, o, lse, (cudaStream_t)stream);
}

size_t tpo_packed_attention_bwd_workspace_size(int64_t tokens_q, int64_t heads) {
  if (tokens_q < 0 || heads < 0) return 0;
  return packed_bwd_workspace_size(tokens_q, heads);
}

int tpo_packed_attention_bwd(const tpo_packed_attention* p, const void* o, const float* lse,
                             const void* grad_o, int64_t grad_o_token_stride,
                             int64_t grad_o_head_stride, void* dq, void* dk, void* dv, void* workspace,
                             size_t workspace_bytes, void* stream) {
  int s = check_packed(p);
  if (s) return s;
  if (!dk != !dv) return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention_bwd: dk and dv go together");
  if (grad_o_token_stride < 0 || grad_o_head_stride < 0)
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention_bwd: negative stride");
  if (p->tokens_q > 0 && (!o || !lse || !grad_o))
    return fail(TPO_ERR_INVALID_ARGUMENT, "packed_attention_bwd: null pointer");
  if (workspace_bytes < packed_bwd_workspace_size(p->tokens_q, p->heads) || !workspace)
    return fail(TPO_ERR_WORKSPACE, "packed_attention_bwd: workspace missing or smaller than tpo_packed_attention_bwd_workspace_size()");
  if ((uintptr_t)workspace % 256) return fail(TPO_ERR_WORKSPACE, "packed_attention_bwd: workspace must be 256-byte aligned");
  return packed_backward(p, o, lse, grad_o, grad_o_token_stride, grad_o_head_stride, dq, dk, dv,
                         workspace, (cudaStream_t)stream);
}

size_t tpo_cached_attention_workspace_size(int64_t N, int64_t H, int64_t Hk, int64_t P, int64_t D) {
  if (N <= 0 || H <= 0 || Hk <= 0 || P < 0 || D <= 0) return 0;
  return cached_workspace_size(N, H, Hk, P, D);
}

int tpo_cached_attention(int dtype, const void* q, const int64_t* q_stride, const void* k,
                         const int64_t* k_stride, const void* v, const int64_t* v_stride,
                         const int64_t* lengths, int64_t N, int64_t P, int64_t H, int64_t Hk, int64_t D,
                         float scale, void* o, void* workspace, size_t workspace_bytes, void* stream) {
  if (!attention_dtype(dtype)) return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: dtype must be f32, f16 or bf16");
  if (N < 0 || N > 65535 || P < 0 || P >= (int64_t(1) << 31))
    return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: bad shape (at most 65535 clouds)");
  if (H < 1 || Hk < 1 || H % Hk != 0 || H > 65535)
    return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: heads must be a multiple of kv_heads (at most 65535)");
  if (D < 1) return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: width must be positive");
  if (D > kAttentionMaxWidth) return fail(TPO_ERR_UNSUPPORTED, "cached_attention: width is limited to 256");
  if (!(scale > 0) || scale > 1e30f)
    return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: scale must be positive and finite");
  if (N == 0) return TPO_OK;
  if (!q_stride || !k_stride || !v_stride) return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: null strides");
  for (int i = 0; i < 3; ++i)
    if ((i < 2 && q_stride[i] < 0) || k_stride[i] < 0 || v_stride[i] < 0)
      return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: negative stride");
  if (!q || !o || !lengths || (P > 0 && (!k || !v))) return fail(TPO_ERR_INVALID_ARGUMENT, "cached_attention: null pointer");
  const size_t need = cached_workspace_size(N, H, Hk, P, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(TPO_ERR_WORKSPACE, "cached_attention: workspace missing or smaller than tpo_cached_attention_workspace_size()");
  if ((uintptr_t)workspace % 16) return fail(TPO_ERR_WORKSPACE, "cached_attention: workspace must be 16-byte aligned");
  return cached_attention(dtype, q, q_stride, k, k_stride, v, v_stride, lengths, N, P, H, Hk, D, scale, o,
                          workspace, (cudaStream_t)stream);
}

}  // extern "C"
