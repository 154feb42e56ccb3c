// torch.library binding of the token operators (layer norm, attention over packed
// clouds, attention over a cache) over the tpo_b200 C ABI.
//
// layer_norm and packed_attention are the differentiable entry points: their
// Autograd kernels run the *_forward op, keep what the *_backward op needs, and
// raise on a second differentiation and on a forward-mode derivative.  Only CUDA
// implementations are registered: a CPU tensor raises.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/all.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <cmath>

#include "../../include/tpo_b200.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

int to_dtype(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return TPO_F32;
    case at::kHalf: return TPO_F16;
    case at::kDouble: return TPO_F64;
    case at::kBFloat16: return TPO_BF16;
    default: TORCH_CHECK(false, what, ": unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void ok(int status, const char* where) { TORCH_CHECK(status == TPO_OK, where, ": ", tpo_status_string(status)); }

void* stream_of(const at::Tensor& t) { return (void*)at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// A dual tensor need not require a gradient: without this check its tangent would be dropped below autograd.
template <typename... Tensors>
void no_tangents(const char* what, const Tensors&... inputs) {
  TORCH_CHECK(!(... || (inputs.defined() && inputs._fw_grad(0).defined())), what,
              ": forward-mode derivatives are not implemented");
}

// Raises when a gradient that this library computed is differentiated again.
class FirstOrderOnly : public torch::autograd::Function<FirstOrderOnly> {
 public:
  // `inputs`: the tensors that the gradients depend on, the gradients themselves first
  static variable_list forward(AutogradContext*, at::TensorList inputs, int64_t grads) {
    variable_list out;
    for (int64_t i = 0; i < grads; ++i) out.push_back(inputs[i].detach());
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "torch_point_ops_b200: a second differentiation of this operator is not implemented");
    return {};
  }
};

// With create_graph=True, hangs the gradients under a node that raises when it is
// reached, instead of passing them on as constants.
variable_list first_order(variable_list grads, variable_list inputs) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) defined.push_back(g);
  variable_list all = defined;
  for (auto& t : inputs)
    if (t.defined()) all.push_back(t);
  auto out = FirstOrderOnly::apply(at::TensorList(all), (int64_t)defined.size());
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ---------------------------------------------------------------- layer norm
// x as (rows, C) with unit stride along a row; copies only where no such view exists.
at::Tensor as_rows(const at::Tensor& x) {
  const int64_t C = x.size(-1);
  if (x.dim() == 2 && x.stride(1) == 1) return x;
  if (x.is_contiguous()) return x.view({C ? x.numel() / C : 0, C});
  return x.contiguous().view({C ? x.numel() / C : 0, C});
}

int check_layer_norm(const at::Tensor& x, const OptTensor& w, const OptTensor& b) {
  TORCH_CHECK(x.is_cuda(), "layer_norm: x must be a CUDA tensor");
  TORCH_CHECK(x.dim() >= 1, "layer_norm: x must have at least one dimension");
  int wd = to_dtype(x, "layer_norm");
  for (const OptTensor* t : {&w, &b}) {
    if (!has(*t)) continue;
    TORCH_CHECK((*t)->device() == x.device(), "layer_norm: weight and bias must be on x's device");
    TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == x.size(-1), "layer_norm: weight and bias must have shape (",
                x.size(-1), ",)");
    wd = to_dtype(**t, "layer_norm");
  }
  TORCH_CHECK(!has(w) || !has(b) || w->scalar_type() == b->scalar_type(), "layer_norm: weight and bias dtypes differ");
  return wd;
}

at::Tensor layer_norm_run(const at::Tensor& x_, const OptTensor& w_, const OptTensor& b_, double eps,
                          at::Tensor* mean, at::Tensor* rstd) {
  const int wd = check_layer_norm(x_, w_, b_);
  const c10::cuda::CUDAGuard g(x_.device());
  const at::Tensor x = as_rows(x_);
  const at::Tensor w = has(w_) ? w_->contiguous() : at::Tensor(), b = has(b_) ? b_->contiguous() : at::Tensor();
  auto y = at::empty(x_.sizes(), x_.options().memory_format(at::MemoryFormat::Contiguous));
  if (mean) {
    const auto o = x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
    *mean = at::empty({x.size(0)}, o);
    *rstd = at::empty({x.size(0)}, o);
  }
  ok(tpo_layer_norm_fwd(to_dtype(x, "layer_norm"), wd, x.data_ptr(), x.stride(0), w.defined() ? w.data_ptr() : nullptr,
                        b.defined() ? b.data_ptr() : nullptr, x.size(0), x.size(1), eps, y.data_ptr(),
                        mean ? mean->data_ptr() : nullptr, mean ? rstd->data_ptr() : nullptr, stream_of(x)),
     "layer_norm");
  return y;
}

at::Tensor layer_norm_cuda(const at::Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  return layer_norm_run(x, w, b, eps, nullptr, nullptr);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_forward(const at::Tensor& x, const OptTensor& w,
                                                                  const OptTensor& b, double eps) {
  at::Tensor mean, rstd;
  auto y = layer_norm_run(x, w, b, eps, &mean, &rstd);
  return {y, mean, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward(const at::Tensor& dy_, const at::Tensor& x_,
                                                                   const OptTensor& w_, const OptTensor& b_,
                                                                   const at::Tensor& mean, const at::Tensor& rstd,
                                                                   bool need_x, bool need_w, bool need_b) {
  const int wd = check_layer_norm(x_, w_, b_);
  TORCH_CHECK(dy_.sizes() == x_.sizes(), "layer_norm_backward: grad must have x's shape");
  TORCH_CHECK(dy_.device() == x_.device(), "layer_norm_backward: grad must be on x's device");
  TORCH_CHECK((!need_w || has(w_)) && (!need_b || has(b_)), "layer_norm_backward: no such parameter");
  const c10::cuda::CUDAGuard g(x_.device());
  const at::Tensor x = as_rows(x_), dy = as_rows(dy_.to(x_.scalar_type()));
  const at::Tensor w = has(w_) ? w_->contiguous() : at::Tensor();
  const int64_t rows = x.size(0), C = x.size(1);
  const int dt = to_dtype(x, "layer_norm");
  const auto stat = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
  TORCH_CHECK(mean.numel() == rows && rstd.numel() == rows && mean.scalar_type() == stat &&
                  rstd.scalar_type() == stat && mean.is_contiguous() && rstd.is_contiguous() &&
                  mean.device() == x.device() && rstd.device() == x.device(),
              "layer_norm_backward: mean and rstd do not belong to x");
  auto dx = at::empty(need_x ? x_.sizes() : at::IntArrayRef{0}, x_.options().memory_format(at::MemoryFormat::Contiguous));
  auto dw = at::empty({need_w ? C : 0}, (has(w_) ? *w_ : x).options());
  auto db = at::empty({need_b ? C : 0}, (has(b_) ? *b_ : x).options());
  at::Tensor ws;
  size_t wsn = 0;
  if (need_w || need_b) {
    wsn = tpo_layer_norm_bwd_workspace_size(dt, rows, C);
    ws = at::empty({(int64_t)wsn}, x.options().dtype(at::kByte));
  }
  ok(tpo_layer_norm_bwd(dt, wd, x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0),
                        w.defined() ? w.data_ptr() : nullptr, mean.data_ptr(), rstd.data_ptr(), rows, C,
                        need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
                        need_b ? db.data_ptr() : nullptr, wsn ? ws.data_ptr() : nullptr, wsn, stream_of(x)),
     "layer_norm_backward");
  return {dx, dw, db};
}

class LayerNormFn : public torch::autograd::Function<LayerNormFn> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& w_, const OptTensor& b_,
                            double eps) {
    const at::Tensor w = has(w_) ? *w_ : at::Tensor(), b = has(b_) ? *b_ : at::Tensor();
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torch_point_ops_b200_norm::layer_norm_forward", "")
                         .typed<std::tuple<at::Tensor, at::Tensor, at::Tensor>(const at::Tensor&, const OptTensor&,
                                                                               const OptTensor&, double)>();
    auto out = op.call(x, w_, b_, eps);
    ctx->save_for_backward({x, w, b, std::get<1>(out), std::get<2>(out)});
    ctx->saved_data["x"] = x.requires_grad();
    ctx->saved_data["w"] = w.defined() && w.requires_grad();
    ctx->saved_data["b"] = b.defined() && b.requires_grad();
    ctx->set_materialize_grads(false);
    return std::get<0>(out);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool nx = ctx->saved_data["x"].toBool(), nw = ctx->saved_data["w"].toBool(), nb = ctx->saved_data["b"].toBool();
    std::tuple<at::Tensor, at::Tensor, at::Tensor> g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      static auto op =
          c10::Dispatcher::singleton()
              .findSchemaOrThrow("torch_point_ops_b200_norm::layer_norm_backward", "")
              .typed<std::tuple<at::Tensor, at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&,
                                                                    const OptTensor&, const OptTensor&,
                                                                    const at::Tensor&, const at::Tensor&, bool, bool,
                                                                    bool)>();
      g = op.call(grads[0], s[0], s[1].defined() ? OptTensor(s[1]) : OptTensor(),
                  s[2].defined() ? OptTensor(s[2]) : OptTensor(), s[3], s[4], nx, nw, nb);
    }
    auto out = first_order({nx ? std::get<0>(g) : at::Tensor(), nw ? std::get<1>(g) : at::Tensor(),
                            nb ? std::get<2>(g) : at::Tensor()},
                           {grads[0], s[0], s[1]});
    out.push_back(at::Tensor());
    return out;
  }
};

at::Tensor layer_norm_autograd(const at::Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  no_tangents("layer_norm", x, has(w) ? *w : at::Tensor(), has(b) ? *b : at::Tensor());
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || (has(w) && w->requires_grad()) ||
                                                   (has(b) && b->requires_grad()));
  if (!grad) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torch_point_ops_b200_norm::layer_norm", "")
                         .typed<at::Tensor(const at::Tensor&, const OptTensor&, const OptTensor&, double)>();
    return op.call(x, w, b, eps);
  }
  return LayerNormFn::apply(x, w, b, eps);
}

// ---------------------------------------------------------------- attention
at::Tensor unit_last(const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

at::Tensor offsets_of(const at::Tensor& o, const at::Tensor& like, const char* name) {
  TORCH_CHECK(o.dim() == 1 && o.numel() >= 1, "packed_attention: ", name, " must have shape (clouds + 1,)");
  TORCH_CHECK(o.scalar_type() == at::kLong || o.scalar_type() == at::kInt, "packed_attention: ", name,
              " must be int64 or int32");
  return o.to(like.device(), at::kLong).contiguous();
}

struct Packed {
  at::Tensor q, k, v, off_q, off_k;
  tpo_packed_attention p;
};

Packed packed_problem(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
                      const OptTensor& offsets_k, bool causal, double scale) {
  TORCH_CHECK(q.is_cuda(), "packed_attention: q must be a CUDA tensor");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "packed_attention: q, k, v must have shape (tokens, heads, width)");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "packed_attention: devices differ");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "packed_attention: dtypes differ");
  TORCH_CHECK(k.sizes() == v.sizes(), "packed_attention: k and v must have the same shape");
  TORCH_CHECK(q.size(2) == k.size(2), "packed_attention: q and k must have the same width");
  TORCH_CHECK(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0,
              "packed_attention: the heads of q must be a multiple of the heads of k");
  TORCH_CHECK(has(offsets_k) || q.size(0) == k.size(0),
              "packed_attention: without offsets_k, q and k must hold the same tokens");
  TORCH_CHECK(!has(offsets_k) || offsets_k->numel() == offsets.numel(),
              "packed_attention: offsets and offsets_k must have the same length");
  Packed r;
  r.q = unit_last(q), r.k = unit_last(k), r.v = unit_last(v);
  r.off_q = offsets_of(offsets, q, "offsets");
  r.off_k = has(offsets_k) ? offsets_of(*offsets_k, q, "offsets_k") : r.off_q;
  tpo_packed_attention& p = r.p;
  p.dtype = to_dtype(q, "packed_attention");
  p.causal = causal;
  p.clouds = r.off_q.numel() - 1;
  p.heads = q.size(1), p.kv_heads = k.size(1), p.width = q.size(2);
  p.tokens_q = q.size(0), p.tokens_k = k.size(0);
  p.offsets_q = r.off_q.data_ptr<int64_t>(), p.offsets_k = r.off_k.data_ptr<int64_t>();
  p.scale = (float)scale;
  p.q = r.q.data_ptr(), p.k = r.k.data_ptr(), p.v = r.v.data_ptr();
  p.q_token_stride = r.q.stride(0), p.q_head_stride = r.q.stride(1);
  p.k_token_stride = r.k.stride(0), p.k_head_stride = r.k.stride(1);
  p.v_token_stride = r.v.stride(0), p.v_head_stride = r.v.stride(1);
  return r;
}

at::Tensor packed_run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
                      const OptTensor& offsets_k, bool causal, double scale, at::Tensor* lse) {
  TORCH_CHECK(q.is_cuda(), "packed_attention: q must be a CUDA tensor");
  const c10::cuda::CUDAGuard g(q.device());
  const Packed r = packed_problem(q, k, v, offsets, offsets_k, causal, scale);
  auto o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (lse) *lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  ok(tpo_packed_attention_fwd(&r.p, o.data_ptr(), lse ? lse->data_ptr<float>() : nullptr, stream_of(q)),
     "packed_attention");
  return o;
}

at::Tensor packed_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
                       const OptTensor& offsets_k, bool causal, double scale) {
  return packed_run(q, k, v, offsets, offsets_k, causal, scale, nullptr);
}

std::tuple<at::Tensor, at::Tensor> packed_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                  const at::Tensor& offsets, const OptTensor& offsets_k, bool causal,
                                                  double scale) {
  at::Tensor lse;
  auto o = packed_run(q, k, v, offsets, offsets_k, causal, scale, &lse);
  return {o, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_backward(const at::Tensor& go_, const at::Tensor& q,
                                                               const at::Tensor& k, const at::Tensor& v,
                                                               const at::Tensor& o, const at::Tensor& lse,
                                                               const at::Tensor& offsets, const OptTensor& offsets_k,
                                                               bool causal, double scale, bool need_q, bool need_kv) {
  TORCH_CHECK(q.is_cuda(), "packed_attention_backward: q must be a CUDA tensor");
  const c10::cuda::CUDAGuard g(q.device());
  const Packed r = packed_problem(q, k, v, offsets, offsets_k, causal, scale);
  TORCH_CHECK(go_.sizes() == q.sizes() && go_.device() == q.device(), "packed_attention_backward: grad must have q's shape and device");
  TORCH_CHECK(o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type() && o.is_contiguous() &&
                  lse.dim() == 2 && lse.size(0) == q.size(1) && lse.size(1) == q.size(0) &&
                  lse.scalar_type() == at::kFloat && lse.is_contiguous() && o.device() == q.device() &&
                  lse.device() == q.device(),
              "packed_attention_backward: o and lse do not belong to q");
  const at::Tensor go = unit_last(go_.to(q.scalar_type()));
  const auto c = at::MemoryFormat::Contiguous;
  auto dq = at::empty(need_q ? q.sizes() : at::IntArrayRef{0}, q.options().memory_format(c));
  auto dk = at::empty(need_kv ? k.sizes() : at::IntArrayRef{0}, k.options().memory_format(c));
  auto dv = at::empty(need_kv ? v.sizes() : at::IntArrayRef{0}, v.options().memory_format(c));
  const size_t wsn = tpo_packed_attention_bwd_workspace_size(q.size(0), q.size(1));
  auto ws = at::empty({(int64_t)wsn}, q.options().dtype(at::kByte).memory_format(c));
  ok(tpo_packed_attention_bwd(&r.p, o.data_ptr(), lse.data_ptr<float>(), go.data_ptr(), go.stride(0), go.stride(1),
                              need_q ? dq.data_ptr() : nullptr, need_kv ? dk.data_ptr() : nullptr,
                              need_kv ? dv.data_ptr() : nullptr, ws.data_ptr(), wsn, stream_of(q)),
     "packed_attention_backward");
  return {dq, dk, dv};
}

class PackedFn : public torch::autograd::Function<PackedFn> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& offsets, const OptTensor& offsets_k, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torch_point_ops_b200_attention::packed_attention_forward", "")
                         .typed<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&,
                                                                   const at::Tensor&, const at::Tensor&,
                                                                   const OptTensor&, bool, double)>();
    auto out = op.call(q, k, v, offsets, offsets_k, causal, scale);
    ctx->save_for_backward({q, k, v, std::get<0>(out), std::get<1>(out), offsets,
                            has(offsets_k) ? *offsets_k : at::Tensor()});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["q"] = q.requires_grad();
    ctx->saved_data["k"] = k.requires_grad();
    ctx->saved_data["v"] = v.requires_grad();
    ctx->set_materialize_grads(false);
    return std::get<0>(out);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor none;
    if (!grads[0].defined()) return {none, none, none, none, none, none, none};
    const auto s = ctx->get_saved_variables();
    const bool nq = ctx->saved_data["q"].toBool(), nk = ctx->saved_data["k"].toBool(), nv = ctx->saved_data["v"].toBool();
    std::tuple<at::Tensor, at::Tensor, at::Tensor> g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      static auto op =
          c10::Dispatcher::singleton()
              .findSchemaOrThrow("torch_point_ops_b200_attention::packed_attention_backward", "")
              .typed<std::tuple<at::Tensor, at::Tensor, at::Tensor>(
                  const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                  const at::Tensor&, const at::Tensor&, const OptTensor&, bool, double, bool, bool)>();
      g = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6].defined() ? OptTensor(s[6]) : OptTensor(),
                  ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), nq, nk || nv);
    }
    auto out = first_order({nq ? std::get<0>(g) : none, nk ? std::get<1>(g) : none, nv ? std::get<2>(g) : none},
                           {grads[0], s[0], s[1], s[2]});
    out.insert(out.end(), 4, none);
    return out;
  }
};

at::Tensor packed_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
                           const OptTensor& offsets_k, bool causal, double scale) {
  no_tangents("packed_attention", q, k, v);
  if (!(at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torch_point_ops_b200_attention::packed_attention", "")
                         .typed<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                           const OptTensor&, bool, double)>();
    return op.call(q, k, v, offsets, offsets_k, causal, scale);
  }
  return PackedFn::apply(q, k, v, offsets, offsets_k, causal, scale);
}

at::Tensor cached_cuda(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& lengths,
                       double scale) {
  TORCH_CHECK(q_.is_cuda(), "cached_attention: q must be a CUDA tensor");
  TORCH_CHECK(q_.dim() == 3 && k_.dim() == 4 && v_.dim() == 4,
              "cached_attention: q must have shape (N, heads, width), k and v (N, P, heads, width)");
  TORCH_CHECK(q_.device() == k_.device() && q_.device() == v_.device(), "cached_attention: devices differ");
  TORCH_CHECK(q_.scalar_type() == k_.scalar_type() && q_.scalar_type() == v_.scalar_type(), "cached_attention: dtypes differ");
  TORCH_CHECK(k_.sizes() == v_.sizes(), "cached_attention: k and v must have the same shape");
  TORCH_CHECK(q_.size(0) == k_.size(0) && q_.size(2) == k_.size(3), "cached_attention: q and k do not match");
  TORCH_CHECK(q_.size(1) > 0 && k_.size(2) > 0 && q_.size(1) % k_.size(2) == 0,
              "cached_attention: the heads of q must be a multiple of the heads of k");
  TORCH_CHECK(lengths.dim() == 1 && lengths.numel() == q_.size(0), "cached_attention: lengths must have shape (N,)");
  TORCH_CHECK(lengths.scalar_type() == at::kLong || lengths.scalar_type() == at::kInt,
              "cached_attention: lengths must be int64 or int32");
  const c10::cuda::CUDAGuard g(q_.device());
  const at::Tensor q = unit_last(q_), k = unit_last(k_), v = unit_last(v_);
  const at::Tensor len = lengths.to(q.device(), at::kLong).contiguous();
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2), P = k.size(1), Hk = k.size(2);
  auto o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  const size_t wsn = tpo_cached_attention_workspace_size(N, H, Hk, P, D);
  at::Tensor ws;
  if (wsn) ws = at::empty({(int64_t)wsn}, q.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
  const int64_t qs[2] = {q.stride(0), q.stride(1)}, ks[3] = {k.stride(0), k.stride(1), k.stride(2)},
                vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  ok(tpo_cached_attention(to_dtype(q, "cached_attention"), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                          len.data_ptr<int64_t>(), N, P, H, Hk, D, (float)scale, o.data_ptr(),
                          wsn ? ws.data_ptr() : nullptr, wsn, stream_of(q)),
     "cached_attention");
  return o;
}

at::Tensor cached_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lengths,
                           double scale) {
  no_tangents("cached_attention", q, k, v);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad()),
              "cached_attention has no backward pass: call it under torch.no_grad(), or train with packed_attention");
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("torch_point_ops_b200_attention::cached_attention", "")
                       .typed<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, double)>();
  return op.call(q, k, v, lengths, scale);
}

}  // namespace

TORCH_LIBRARY(torch_point_ops_b200_norm, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, Tensor rstd, "
        "bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(torch_point_ops_b200_norm, CUDA, m) {
  m.impl("layer_norm", &layer_norm_cuda);
  m.impl("layer_norm_forward", &layer_norm_forward);
  m.impl("layer_norm_backward", &layer_norm_backward);
}
TORCH_LIBRARY_IMPL(torch_point_ops_b200_norm, Autograd, m) { m.impl("layer_norm", &layer_norm_autograd); }

TORCH_LIBRARY(torch_point_ops_b200_attention, m) {
  m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor offsets, Tensor? offsets_k, bool causal, float scale) "
        "-> Tensor");
  m.def("packed_attention_forward(Tensor q, Tensor k, Tensor v, Tensor offsets, Tensor? offsets_k, bool causal, "
        "float scale) -> (Tensor, Tensor)");
  m.def("packed_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor offsets, "
        "Tensor? offsets_k, bool causal, float scale, bool need_q, bool need_kv) -> (Tensor, Tensor, Tensor)");
  m.def("cached_attention(Tensor q, Tensor k, Tensor v, Tensor lengths, float scale) -> Tensor");
}
TORCH_LIBRARY_IMPL(torch_point_ops_b200_attention, CUDA, m) {
  m.impl("packed_attention", &packed_cuda);
  m.impl("packed_attention_forward", &packed_forward);
  m.impl("packed_attention_backward", &packed_backward);
  m.impl("cached_attention", &cached_cuda);
}
TORCH_LIBRARY_IMPL(torch_point_ops_b200_attention, Autograd, m) {
  m.impl("packed_attention", &packed_autograd);
  m.impl("cached_attention", &cached_autograd);
}
