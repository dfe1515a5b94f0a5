// Autograd functions of the layer, of the experts on given picks, of the conv router, of the group top-k, of the router losses, of
// the block-scaled 8-bit products, of the root-mean-square norm and of the low-rank adapters as compiled code: the host side of the Python
// Functions of the same name (layer.py, moe.py, router.py, fp8_block.py, norm.py, lora.py) for plain calls.  Each function returns None for a call
// that is not plain (a tensor that would have to be cast or made contiguous, autocast, functorch transforms, forward-mode
// gradients, dispatch modes, tensor subclasses, a shape that is an error), and the caller then takes the Python Function, which
// casts, refuses or raises as it always did.
//
// Why: between two small passes the host was the bound.  A Python Function costs the caller 8 us to enter, its allocations and
// argument checks 15 to 30 more each way, and in the backward the autograd engine's thread waits for the interpreter lock before
// it can call it.  us a pass, Python / compiled: one token through 64 experts of 2048 x 1408 62 / 39; forward and backward of 512 tokens
// at width 256 237 / 148; conv router of 16 384 tokens 145 / 118.
// Of the operators below, host time of a call of 512 tokens, forward and backward: top-k 118 / 75, losses 141 / 84, an 8-bit product 154 / 89.
//
// Nothing is kept between calls but what autograd saves (saved-tensor hooks see it); the workspace of a forward is a saved tensor.
#include <limits>
#include <ATen/autocast_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>
#include <torch/version.h>

#include "../../include/b200moe.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc) {
  if (rc == 0) return;
  const std::string msg = "b200moe error " + std::to_string(rc) + ": " + b200moe_last_error_string();
  if (rc == B200MOE_E_CUDA) TORCH_CHECK(false, msg);
  TORCH_CHECK_VALUE(false, msg);
}

// a contiguous CUDA tensor of its own memory that nothing wraps
bool plain(const Tensor& t, at::ScalarType type, c10::Device dev) {
  if (!t.defined() || t.scalar_type() != type || t.device() != dev || t.layout() != at::kStrided) return false;
  const auto ks = t.key_set();
  if (ks.has(c10::DispatchKey::Python) || ks.has(c10::DispatchKey::FuncTorchBatched) ||
      ks.has(c10::DispatchKey::FuncTorchGradWrapper) || ks.has(c10::DispatchKey::Functionalize))
    return false;
  return t.is_contiguous() && !t._fw_grad(0).defined();
}
bool plain_or_none(const optional<Tensor>& t, at::ScalarType type, c10::Device dev) { return !t.has_value() || plain(*t, type, dev); }

// no mode or transform that has to see the operations of this call
bool plain_call(const Tensor& x) {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  return x.is_cuda() && !tls.included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::autocast::is_autocast_enabled(at::kCUDA);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }
b200moe_stream_t stream_of(const Tensor& t) { return reinterpret_cast<b200moe_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()); }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)); }
Tensor grad_like(bool want, const Tensor& t) { return want ? at::empty(t.sizes(), t.options().dtype(at::kBFloat16)) : Tensor(); }
int32_t* status_ptr(const Tensor& t) { return t.data_ptr<int32_t>(); }

// ---------------------------------------------------------------------------- router and experts
struct LayerArgs {
  optional<Tensor> bias, codes, load;
  Tensor status;
  int64_t k, norm;
  double scale;
};

std::tuple<Tensor, Tensor, Tensor> layer_forward(const Tensor& x, const Tensor& gate, const Tensor& gate_up, const Tensor& down,
                                                 const LayerArgs& a, int keep) {
  const int64_t T = x.size(0), H = x.size(1), E = gate_up.size(0), I = down.size(2);
  Tensor ws = bytes(b200moe_layer_fwd_ws_bytes(T, H, I, E, a.k, keep), x);
  Tensor out = at::empty({T, H}, x.options()), counts = at::empty({E}, x.options().dtype(at::kInt));
  check(b200moe_layer_forward(ptr(x), ptr(gate), static_cast<const float*>(ptr(a.bias)), ptr(gate_up), ptr(down),
                              static_cast<const int32_t*>(ptr(a.codes)), T, H, I, E, a.k, a.norm, static_cast<float>(a.scale), keep, ptr(ws),
                              counts.data_ptr<int32_t>(), static_cast<int64_t*>(ptr(a.load)), ptr(out), status_ptr(a.status), stream_of(x)));
  return {out, counts, ws};
}

struct Layer : torch::autograd::Function<Layer> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& gate_up, const Tensor& down,
                               const LayerArgs& a) {
    auto [out, counts, ws] = layer_forward(x, gate, gate_up, down, a, 1);
    variable_list saved{x, gate, gate_up, down, ws};
    if (a.codes.has_value()) saved.push_back(*a.codes);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["status"] = a.status;
    ctx->saved_data["k"] = a.k;
    ctx->saved_data["norm"] = a.norm;
    ctx->saved_data["scale"] = a.scale;
    ctx->mark_non_differentiable({counts});
    ctx->set_materialize_grads(false);   // no zero-filled gradient for the counts
    return {out, counts};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(5);
    if (!grads[0].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &gate = s[1], &gate_up = s[2], &down = s[3], &ws = s[4];
    const Tensor codes = s.size() > 5 ? s[5] : Tensor(), status = ctx->saved_data["status"].toTensor();
    const int64_t T = x.size(0), H = x.size(1), E = gate_up.size(0), I = down.size(2), k = ctx->saved_data["k"].toInt();
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor go = grads[0].to(at::kBFloat16).contiguous();
    for (int i = 0; i < 4; ++i) res[i] = grad_like(ctx->needs_input_grad(i), s[i]);
    Tensor tmp = bytes(b200moe_layer_bwd_ws_bytes(T, H, I, E, k), x);
    check(b200moe_layer_backward(ptr(go), ptr(x), ptr(gate), ptr(gate_up), ptr(down), static_cast<const int32_t*>(ptr(codes)), T, H, I, E, k,
                                 ctx->saved_data["norm"].toInt(), static_cast<float>(ctx->saved_data["scale"].toDouble()), ptr(ws),
                                 ptr(tmp), ptr(res[0]), ptr(res[1]), ptr(res[2]), ptr(res[3]), status_ptr(status), stream_of(x)));
    return res;
  }
};

// (out (T,H), counts (E,) int32), or None
optional<std::tuple<Tensor, Tensor>> layer(const Tensor& x, const Tensor& gate, const optional<Tensor>& bias, const Tensor& gate_up,
                                           const Tensor& down, const optional<Tensor>& codes, const optional<Tensor>& load,
                                           const Tensor& status, int64_t k, int64_t norm, double scale) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  for (const Tensor* t : {&x, &gate, &gate_up, &down})
    if (!plain(*t, at::kBFloat16, dev)) return std::nullopt;
  if (!plain_or_none(bias, at::kFloat, dev) || !plain_or_none(codes, at::kInt, dev) || !plain_or_none(load, at::kLong, dev)) return std::nullopt;
  if (x.dim() != 2 || gate.dim() != 2 || gate_up.dim() != 3 || down.dim() != 3) return std::nullopt;
  const int64_t H = x.size(1), E = gate_up.size(0), I = down.size(2);
  if (x.size(0) == 0 || gate_up.size(1) != 2 * I || gate_up.size(2) != H || down.size(0) != E || down.size(1) != H || gate.size(0) != E ||
      gate.size(1) != H || (bias.has_value() && bias->numel() != E))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const LayerArgs a{bias, codes, load, status, k, norm, scale};
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || gate_up.requires_grad() || down.requires_grad())) {
    variable_list r = Layer::apply(x, gate, gate_up, down, a);
    return std::make_tuple(r[0], r[1]);
  }
  auto [out, counts, ws] = layer_forward(x, gate, gate_up, down, a, 0);
  return std::make_tuple(out, counts);
}

// ---------------------------------------------------------------------------- experts on given picks
struct ExpertsArgs {
  Tensor idx;
  optional<Tensor> codes;
  Tensor status;
  int64_t E, row_kernels;
};

std::tuple<Tensor, Tensor> experts_forward(const Tensor& x, const Tensor& w, const Tensor& gate_up, const Tensor& down,
                                           const optional<Tensor>& params, const ExpertsArgs& a, int keep) {
  const int64_t T = x.size(0), H = x.size(1), n = gate_up.size(0), I = down.size(2), k = a.idx.size(1);
  Tensor ws = bytes(b200moe_moe_fwd_ws_bytes(T, H, I, a.E, n, k, keep, a.row_kernels), x), out = at::empty({T, H}, x.options());
  check(b200moe_moe_forward(ptr(x), a.idx.data_ptr<int64_t>(), w.data_ptr<float>(), ptr(gate_up), ptr(down),
                            static_cast<const int32_t*>(ptr(a.codes)), static_cast<const float*>(ptr(params)), T, H, I, a.E, n, k, keep,
                            a.row_kernels, ptr(ws), ptr(out), status_ptr(a.status), stream_of(x)));
  return {out, ws};
}

struct Experts : torch::autograd::Function<Experts> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& gate_up, const Tensor& down,
                        const optional<Tensor>& params, const ExpertsArgs& a) {
    auto [out, ws] = experts_forward(x, w, gate_up, down, params, a, 1);
    variable_list saved{ws, w, gate_up, down};
    if (a.codes.has_value()) saved.push_back(*a.codes);
    if (params.has_value()) saved.push_back(*params);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["status"] = a.status;
    ctx->saved_data["has"] = static_cast<int64_t>((a.codes.has_value() ? 1 : 0) | (params.has_value() ? 2 : 0));
    ctx->saved_data["E"] = a.E;
    ctx->saved_data["rows"] = a.row_kernels;
    ctx->saved_data["H"] = x.size(1);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &ws = s[0], &w = s[1], &gate_up = s[2], &down = s[3];
    const int64_t has = ctx->saved_data["has"].toInt(), E = ctx->saved_data["E"].toInt(), rows = ctx->saved_data["rows"].toInt();
    const Tensor codes = (has & 1) ? s[4] : Tensor(), params = (has & 2) ? s.back() : Tensor(), status = ctx->saved_data["status"].toTensor();
    const int64_t T = w.size(0), k = w.size(1), H = ctx->saved_data["H"].toInt(), n = gate_up.size(0), I = down.size(2);
    const c10::cuda::CUDAGuard guard(ws.device());
    const Tensor go = grads[0].to(at::kBFloat16).contiguous();
    const Tensor gw = at::empty_like(w);
    const Tensor gx = ctx->needs_input_grad(0) ? at::empty({T, H}, gate_up.options()) : Tensor();
    const Tensor ggu = grad_like(ctx->needs_input_grad(2), gate_up), gdn = grad_like(ctx->needs_input_grad(3), down);
    const Tensor gp = params.defined() && ctx->needs_input_grad(4) ? at::empty_like(params) : Tensor();
    Tensor tmp = bytes(b200moe_moe_bwd_ws_bytes(T, H, I, E, n, k, rows), ws);
    check(b200moe_moe_backward(ptr(go), w.data_ptr<float>(), ptr(gate_up), ptr(down), static_cast<const int32_t*>(ptr(codes)),
                               static_cast<const float*>(ptr(params)), T, H, I, E, n, k, rows, ptr(ws), ptr(tmp), ptr(gx), gw.data_ptr<float>(),
                               ptr(ggu), ptr(gdn), static_cast<float*>(ptr(gp)), status_ptr(status), stream_of(ws)));
    return {gx, ctx->needs_input_grad(1) ? gw : Tensor(), ggu, gdn, gp, Tensor()};
  }
};

// out (T,H), or None.  codes and params as the native call wants them: on the device, int32 and fp32
optional<Tensor> experts(const Tensor& x, const Tensor& idx, const Tensor& w, const Tensor& gate_up, const Tensor& down,
                         const optional<Tensor>& codes, const optional<Tensor>& params, const Tensor& status, int64_t E, int64_t n_glu,
                         int64_t row_kernels) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  for (const Tensor* t : {&x, &gate_up, &down})
    if (!plain(*t, at::kBFloat16, dev)) return std::nullopt;
  if (!plain(idx, at::kLong, dev) || !plain(w, at::kFloat, dev) || !plain_or_none(codes, at::kInt, dev) || !plain_or_none(params, at::kFloat, dev))
    return std::nullopt;
  if (x.dim() != 2 || idx.dim() != 2 || gate_up.dim() != 3 || down.dim() != 3 || x.size(0) == 0) return std::nullopt;
  const int64_t T = x.size(0), H = x.size(1), I = down.size(2);
  if (gate_up.size(0) != n_glu || gate_up.size(1) != 2 * I || gate_up.size(2) != H || down.size(0) != n_glu || down.size(1) != H ||
      idx.size(0) != T || w.sizes() != idx.sizes() || (codes.has_value() && codes->numel() != E) ||
      (params.has_value() && (params->dim() != 2 || params->size(0) != E || params->size(1) != 2)))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const ExpertsArgs a{idx, codes, status, E, row_kernels};
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || gate_up.requires_grad() || down.requires_grad() ||
                                     (params.has_value() && params->requires_grad())))
    return Experts::apply(x, w, gate_up, down, params, a);
  return std::get<0>(experts_forward(x, w, gate_up, down, params, a, row_kernels ? 1 : 0));
}

// ---------------------------------------------------------------------------- conv router
struct ConvArgs {
  optional<Tensor> bias;
  Tensor status;
  int64_t k, norm;
  double scale;
};

struct ConvRouter : torch::autograd::Function<ConvRouter> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const ConvArgs& a) {
    const int64_t B = x.size(0), S = x.size(1), H = x.size(2), E = weight.size(0), taps = weight.size(2);
    Tensor wt = at::empty({taps * E, H}, x.options()), logits = at::empty({B * S, E}, x.options());
    Tensor idx = at::empty({B, S, a.k}, x.options().dtype(at::kLong)), w = at::empty({B, S, a.k}, x.options().dtype(at::kFloat));
    Tensor counts = at::empty({E}, x.options().dtype(at::kInt)), ws = bytes(b200moe_conv_router_fwd_ws_bytes(B, S, H, E, taps), x);
    check(b200moe_conv_router_forward(ptr(x), ptr(weight), static_cast<const float*>(ptr(a.bias)), B, S, H, E, taps, a.k, a.norm,
                                      static_cast<float>(a.scale), ptr(ws), ptr(wt), ptr(logits), idx.data_ptr<int64_t>(),
                                      w.data_ptr<float>(), counts.data_ptr<int32_t>(), status_ptr(a.status), stream_of(x)));
    ctx->save_for_backward({x, wt, logits, idx});
    ctx->saved_data["status"] = a.status;
    ctx->saved_data["taps"] = taps;
    ctx->saved_data["norm"] = a.norm;
    ctx->saved_data["scale"] = a.scale;
    ctx->mark_non_differentiable({idx, counts});
    ctx->set_materialize_grads(false);
    return {idx, w, counts};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(3);
    if (!grads[1].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wt = s[1], &logits = s[2], &idx = s[3];
    const Tensor status = ctx->saved_data["status"].toTensor();
    const int64_t taps = ctx->saved_data["taps"].toInt(), B = x.size(0), S = x.size(1), H = x.size(2), E = logits.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor gw = grads[1].contiguous().to(at::kFloat);
    res[0] = grad_like(ctx->needs_input_grad(0), x);
    res[1] = ctx->needs_input_grad(1) ? at::empty({E, H, taps}, x.options()) : Tensor();
    Tensor ws = bytes(b200moe_conv_router_bwd_ws_bytes(B, S, H, E, taps), x);
    check(b200moe_conv_router_backward(ptr(x), ptr(wt), ptr(logits), idx.data_ptr<int64_t>(), gw.data_ptr<float>(), B, S, H, E, taps,
                                       idx.size(2), ctx->saved_data["norm"].toInt(), static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                       ptr(ws), ptr(res[0]), ptr(res[1]), status_ptr(status), stream_of(x)));
    return res;
  }
};

// (idx (B,S,k) int64, weights (B,S,k) fp32, counts (E,) int32), or None
optional<std::tuple<Tensor, Tensor, Tensor>> conv_router(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                                                         const Tensor& status, int64_t k, int64_t experts, int64_t norm, double scale) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  if (!plain(x, at::kBFloat16, dev) || !plain(weight, at::kBFloat16, dev) || !plain_or_none(bias, at::kFloat, dev)) return std::nullopt;
  if (x.dim() != 3 || weight.dim() != 3 || weight.size(1) != x.size(2) || weight.size(0) != experts || x.numel() == 0 || k < 1 ||
      (bias.has_value() && bias->numel() != experts))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  variable_list r = ConvRouter::apply(x, weight, ConvArgs{bias, status, k, norm, scale});
  return std::make_tuple(r[0], r[1], r[2]);
}

// Gradients that are not differentiable themselves: where a graph of the backward is being made, going through them is an error, as with the
// Python Functions' once_differentiable
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int>(grads.size()));
  variable_list in(grads.size());
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) in[i] = grads[i].detach().requires_grad_(true);
  return (*error)(std::move(in));
}

// ---------------------------------------------------------------------------- group-limited top-k
// of the logits' types
optional<int> logits_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return B200MOE_LOGITS_BF16;
    case at::kFloat: return B200MOE_LOGITS_F32;
    case at::kHalf: return B200MOE_LOGITS_F16;
    default: return std::nullopt;
  }
}

struct GroupArgs {
  optional<Tensor> bias;
  int type;
  int64_t k, groups, open, scoring, top2, norm;
  double scale;
  bool counts;
};

variable_list group_forward(const Tensor& z, const GroupArgs& a) {
  const int64_t E = z.size(-1), T = z.numel() / E;
  std::vector<int64_t> shape(z.sizes().begin(), z.sizes().end());
  shape.back() = a.k;
  Tensor idx = at::empty(shape, z.options().dtype(at::kLong)), w = at::empty(shape, z.options().dtype(at::kFloat));
  Tensor counts = a.counts ? at::empty({E}, z.options().dtype(at::kInt)) : Tensor();
  check(b200moe_group_topk_fwd(ptr(z), a.type, static_cast<const float*>(ptr(a.bias)), T, E, a.k, a.groups, a.open, a.scoring, a.top2, a.norm,
                               static_cast<float>(a.scale), idx.data_ptr<int64_t>(), w.data_ptr<float>(), static_cast<int32_t*>(ptr(counts)),
                               stream_of(z)));
  return {idx, w, counts};
}

struct GroupTopk : torch::autograd::Function<GroupTopk> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const GroupArgs& a) {
    variable_list r = group_forward(z, a);
    ctx->save_for_backward({z, r[0]});
    ctx->saved_data["scoring"] = a.scoring;
    ctx->saved_data["norm"] = a.norm;
    ctx->saved_data["scale"] = a.scale;
    ctx->mark_non_differentiable({r[0], r[2]});
    ctx->set_materialize_grads(false);
    return r;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(2);
    if (!grads[1].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &z = s[0], &idx = s[1];
    const c10::cuda::CUDAGuard guard(z.device());
    const Tensor gw = grads[1].contiguous().to(at::kFloat);
    const int64_t E = z.size(-1);
    res[0] = at::empty_like(z);
    check(b200moe_group_topk_bwd(ptr(z), *logits_type(z), idx.data_ptr<int64_t>(), gw.data_ptr<float>(), z.numel() / E, E, idx.size(-1),
                                 ctx->saved_data["scoring"].toInt(), ctx->saved_data["norm"].toInt(),
                                 static_cast<float>(ctx->saved_data["scale"].toDouble()), ptr(res[0]), stream_of(z)));
    return once(std::move(res));
  }
};

// (idx (...,k) int64, weights (...,k) fp32, counts (E,) int32 or None), or None
optional<std::tuple<Tensor, Tensor, optional<Tensor>>> group_topk(const Tensor& z, const optional<Tensor>& bias, int64_t k, int64_t groups,
                                                                  int64_t open, int64_t scoring, int64_t top2, bool norm, double scale,
                                                                  bool counts) {
  if (!plain_call(z)) return std::nullopt;
  const auto dev = z.device();
  const auto type = logits_type(z);
  if (!type.has_value() || !plain(z, z.scalar_type(), dev) || !plain_or_none(bias, at::kFloat, dev)) return std::nullopt;
  if (z.dim() < 2 || z.dim() > 3 || z.numel() == 0 || k < 1 || k > B200MOE_MAX_TOPK || (bias.has_value() && bias->numel() != z.size(-1)))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const bool grad = at::GradMode::is_enabled() && z.requires_grad();
  const GroupArgs a{bias, *type, k, groups, open, scoring, top2, norm, scale, counts || grad};
  variable_list r = grad ? GroupTopk::apply(z, a) : group_forward(z, a);
  return std::make_tuple(r[0], r[1], r[2].defined() ? optional<Tensor>(r[2]) : std::nullopt);
}

// ---------------------------------------------------------------------------- router losses
struct LossArgs {
  Tensor idx, status;
  optional<Tensor> mask;
  int type;
  int64_t segs, scoring;
};

variable_list losses_forward(const Tensor& z, const LossArgs& a) {
  const int64_t E = z.size(-1), S = z.numel() / E / a.segs;
  Tensor balance = at::empty({}, z.options().dtype(at::kFloat)), zl = at::empty({}, z.options().dtype(at::kFloat));
  Tensor coef = at::empty({a.segs * E + 2}, z.options().dtype(at::kFloat)), ws = bytes(b200moe_router_losses_ws_bytes(S, a.segs, E), z);
  check(b200moe_router_losses_fwd(ptr(z), a.type, a.idx.data_ptr<int64_t>(), static_cast<const uint8_t*>(ptr(a.mask)), S, a.segs, E, a.idx.size(-1),
                                  a.scoring, ptr(ws), coef.data_ptr<float>(), balance.data_ptr<float>(), zl.data_ptr<float>(),
                                  status_ptr(a.status), stream_of(z)));
  return {balance, zl, coef};
}

struct RouterLosses : torch::autograd::Function<RouterLosses> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const LossArgs& a) {
    variable_list r = losses_forward(z, a);
    variable_list saved{z, r[2]};
    if (a.mask.has_value()) saved.push_back(*a.mask);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["segs"] = a.segs;
    ctx->saved_data["scoring"] = a.scoring;
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(2);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &z = s[0], &coef = s[1];
    const c10::cuda::CUDAGuard guard(z.device());
    Tensor g[2];
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) g[i] = grads[i].to(at::kFloat);
    const int64_t E = z.size(-1), segs = ctx->saved_data["segs"].toInt();
    res[0] = at::empty_like(z);
    check(b200moe_router_losses_bwd(ptr(z), *logits_type(z), s.size() > 2 ? static_cast<const uint8_t*>(ptr(s[2])) : nullptr,
                                    coef.data_ptr<float>(), static_cast<const float*>(ptr(g[0])), static_cast<const float*>(ptr(g[1])),
                                    z.numel() / E / segs, segs, E, ctx->saved_data["scoring"].toInt(), ptr(res[0]), stream_of(z)));
    return once(std::move(res));
  }
};

// (balance, z), or None
optional<std::tuple<Tensor, Tensor>> router_losses(const Tensor& z, const Tensor& idx, const optional<Tensor>& mask, const Tensor& status,
                                                   int64_t scoring, bool per_sequence) {
  if (!plain_call(z)) return std::nullopt;
  const auto dev = z.device();
  const auto type = logits_type(z);
  if (!type.has_value() || !plain(z, z.scalar_type(), dev) || !plain(idx, at::kLong, dev) || !plain_or_none(mask, at::kBool, dev))
    return std::nullopt;
  if (z.dim() < 2 || z.dim() > 3 || z.numel() == 0 || idx.dim() != z.dim() || (per_sequence && z.dim() != 3)) return std::nullopt;
  const auto rows = z.sizes().slice(0, z.dim() - 1);
  if (idx.sizes().slice(0, z.dim() - 1) != rows || (mask.has_value() && mask->sizes() != rows)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const LossArgs a{idx, status, mask, *type, per_sequence ? z.size(0) : 1, scoring};
  variable_list r = at::GradMode::is_enabled() && z.requires_grad() ? RouterLosses::apply(z, a) : losses_forward(z, a);
  return std::make_tuple(r[0], r[1]);
}

// ---------------------------------------------------------------------------- e4m3 weights with block scales
bool codes(const Tensor& w, const Tensor& scale, int64_t dim, c10::Device dev) {
  if (!plain(w, at::kFloat8_e4m3fn, dev) || !plain(scale, at::kFloat, dev) || w.dim() != dim || scale.dim() != dim || w.numel() == 0) return false;
  if (at::GradMode::is_enabled() && (w.requires_grad() || scale.requires_grad())) return false;      // refused
  if (dim == 3 && scale.size(0) != w.size(0)) return false;
  return scale.size(-2) == (w.size(-2) + 127) / 128 && scale.size(-1) == (w.size(-1) + 127) / 128;
}
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Rows that are codes already, their scales at a pitch of whole 128 rows
struct RowCodes {
  Tensor q, scale;
  int64_t pitch = 0;
};
Tensor rows_product(const RowCodes& r, const Tensor& w, const Tensor& scale, const Tensor& status) {
  const int64_t N = w.size(0), K = w.size(1), M = r.q.numel() / K;
  std::vector<int64_t> shape(r.q.sizes().begin(), r.q.sizes().end());
  shape.back() = N;
  Tensor out = at::empty(shape, r.q.options().dtype(at::kBFloat16));
  check(b200moe_fp8_block_linear_rows(ptr(r.q), r.scale.data_ptr<float>(), r.pitch, ptr(w), scale.data_ptr<float>(), M, N, K, ptr(out),
                                      status_ptr(status), stream_of(r.q)));
  return out;
}

Tensor block_product(const Tensor& x, const Tensor& w, const Tensor& scale, const Tensor& status, bool transposed) {
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / (transposed ? N : K);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = transposed ? K : N;
  Tensor out = at::empty(shape, x.options()), ws = bytes(b200moe_fp8_block_linear_ws_bytes(M, transposed ? N : K), x);
  check(b200moe_fp8_block_linear(ptr(x), ptr(w), scale.data_ptr<float>(), M, N, K, transposed, ptr(ws), ptr(out), status_ptr(status), stream_of(x)));
  return out;
}

struct BlockLinear : torch::autograd::Function<BlockLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& scale, const Tensor& status, const RowCodes& rows) {
    ctx->save_for_backward({w, scale});
    ctx->saved_data["status"] = status;
    return rows.q.defined() ? rows_product(rows, w, scale, status) : block_product(x, w, scale, status, false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    Tensor g = grads[0].to(at::kBFloat16).contiguous();
    if (!aligned(g)) g = g.clone();
    return once({block_product(g, s[0], s[1], ctx->saved_data["status"].toTensor(), true), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (..., N) bf16, or None
optional<Tensor> fp8_block_linear(const Tensor& x, const Tensor& w, const Tensor& scale, const Tensor& status) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  if (!plain(x, at::kBFloat16, dev) || !codes(w, scale, 2, dev) || x.dim() < 1 || x.numel() == 0 || x.size(-1) != w.size(1)) return std::nullopt;
  if (w.size(0) % 8 != 0 || w.size(1) % 16 != 0 || !aligned(x) || !aligned(w)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  if (at::GradMode::is_enabled() && x.requires_grad()) return BlockLinear::apply(x, w, scale, status, RowCodes());
  return block_product(x, w, scale, status, false);
}

// The same of rows that are codes; x: what the gradient goes to, if any
optional<Tensor> fp8_block_linear_rows(const optional<Tensor>& x, const Tensor& q, const Tensor& q_scale, const Tensor& w, const Tensor& scale,
                                       const Tensor& status) {
  if (!plain_call(q)) return std::nullopt;
  const auto dev = q.device();
  if (!plain(q, at::kFloat8_e4m3fn, dev) || !codes(w, scale, 2, dev) || q.dim() < 1 || q.numel() == 0 || q.size(-1) != w.size(1)) return std::nullopt;
  if (x.has_value() && (!plain(*x, at::kBFloat16, dev) || x->sizes() != q.sizes())) return std::nullopt;
  if (w.size(0) % 8 != 0 || w.size(1) % 16 != 0 || !aligned(q) || !aligned(w) || q.requires_grad()) return std::nullopt;
  // the scales as rms_norm_fp8_block left them: rows next to one another, blocks at a pitch
  if (q_scale.scalar_type() != at::kFloat || q_scale.device() != dev || q_scale.layout() != at::kStrided || q_scale.dim() != q.dim() ||
      q_scale.requires_grad() || q_scale._fw_grad(0).defined() || q_scale.key_set().has(c10::DispatchKey::Python))
    return std::nullopt;
  const int64_t blocks = (w.size(1) + 127) / 128, M = q.numel() / w.size(1), rows = (M + 127) / 128 * 128;
  const int64_t pitch = blocks == 1 ? rows : q_scale.stride(-1);
  if (q_scale.size(-1) != blocks || pitch % 4 != 0 || pitch < rows || !aligned(q_scale)) return std::nullopt;
  int64_t stride = 1;
  for (int64_t i = q.dim() - 2; i >= 0; --i) {
    if (q_scale.size(i) != q.size(i) || (q.size(i) > 1 && q_scale.stride(i) != stride)) return std::nullopt;
    stride *= q.size(i);
  }
  if (static_cast<int64_t>(q_scale.storage().nbytes()) < 4 * (q_scale.storage_offset() + (blocks - 1) * pitch + rows)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const RowCodes r{q, q_scale, pitch};
  if (x.has_value() && at::GradMode::is_enabled() && x->requires_grad()) return BlockLinear::apply(*x, w, scale, status, r);
  return rows_product(r, w, scale, status);
}

// (N,H) bf16, or None
optional<Tensor> moe_fp8_block(const Tensor& x, const Tensor& idx, const Tensor& w, const Tensor& gate_up, const Tensor& gate_up_scale,
                               const Tensor& down, const Tensor& down_scale, const Tensor& status) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  if (!plain(x, at::kBFloat16, dev) || !plain(idx, at::kLong, dev) || !plain(w, at::kFloat, dev) || !codes(gate_up, gate_up_scale, 3, dev) ||
      !codes(down, down_scale, 3, dev))
    return std::nullopt;
  if (x.dim() != 2 || idx.dim() != 2 || x.size(0) == 0 || (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad()))) return std::nullopt;
  const int64_t T = x.size(0), H = x.size(1), E = gate_up.size(0), I = down.size(2), k = idx.size(1);
  if (gate_up.size(1) != 2 * I || gate_up.size(2) != H || down.size(0) != E || down.size(1) != H || idx.size(0) != T || w.sizes() != idx.sizes() ||
      H % 128 != 0 || I % 128 != 0 || k < 1 || !aligned(x) || !aligned(gate_up) || !aligned(down))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = at::empty({T, H}, x.options()), ws = bytes(b200moe_moe_fp8_block_ws_bytes(T, H, I, E, k), x);
  check(b200moe_moe_fp8_block_forward(ptr(x), idx.data_ptr<int64_t>(), w.data_ptr<float>(), ptr(gate_up), gate_up_scale.data_ptr<float>(),
                                      ptr(down), down_scale.data_ptr<float>(), T, H, I, E, k, ptr(ws), ptr(out), status_ptr(status), stream_of(x)));
  return out;
}

// ---------------------------------------------------------------------------- root-mean-square norm
struct NormArgs {
  optional<Tensor> residual;
  Tensor status;
  Tensor q, scale;      // codes and [block][row] scales to be filled, or undefined
  int type, w_type;
  double eps;
  bool want_y;
};

// y where it is wanted, then h where there is a residual
variable_list norm_forward(const Tensor& x, const Tensor& w, const NormArgs& a) {
  const int64_t K = x.size(-1), N = x.numel() / K;
  Tensor y = a.want_y ? at::empty(x.sizes(), x.options()) : Tensor();
  Tensor h = a.residual.has_value() ? at::empty(x.sizes(), x.options()) : Tensor();
  check(b200moe_rms_norm_fwd(ptr(x), K, ptr(a.residual), K, a.type, ptr(w), a.w_type, N, K, static_cast<float>(a.eps), ptr(y), ptr(h), ptr(a.q),
                             static_cast<float*>(ptr(a.scale)), a.scale.defined() ? a.scale.size(1) : 0, status_ptr(a.status), stream_of(x)));
  variable_list r;
  if (y.defined()) r.push_back(y);
  if (h.defined()) r.push_back(h);
  return r;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const optional<Tensor>& residual, const NormArgs& a) {
    ctx->saved_data["residual"] = residual.has_value();      // an input only where there is one
    variable_list r = norm_forward(x, w, a);
    ctx->save_for_backward({residual.has_value() ? r.back() : x, w});
    ctx->saved_data["y"] = a.want_y;
    ctx->saved_data["status"] = a.status;
    ctx->saved_data["type"] = a.type;
    ctx->saved_data["w_type"] = a.w_type;
    ctx->saved_data["eps"] = a.eps;
    ctx->set_materialize_grads(false);
    return r;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(4);
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(2);
    const bool has_y = ctx->saved_data["y"].toBool(), has_h = ctx->saved_data["residual"].toBool();
    const Tensor grad_y = has_y ? grads[0] : Tensor(), grad_h = has_h ? grads[has_y] : Tensor();
    if (!grad_y.defined()) {      // the stream alone was used
      if (need_x) res[0] = grad_h;
      if (need_r) res[2] = grad_h;
      return res;
    }
    const variable_list s = ctx->get_saved_variables();
    const Tensor &h = s[0], &w = s[1];
    const int64_t K = h.size(-1), N = h.numel() / K;
    const c10::cuda::CUDAGuard guard(h.device());
    const Tensor gy = grad_y.contiguous(), gh = grad_h.defined() ? grad_h.contiguous() : Tensor();
    Tensor gx = need_x || need_r ? at::empty(h.sizes(), h.options()) : Tensor(), gw = need_w ? at::empty(w.sizes(), w.options()) : Tensor();
    Tensor ws = need_w ? bytes(b200moe_rms_norm_bwd_ws_bytes(N, K), h) : Tensor();
    check(b200moe_rms_norm_bwd(ptr(gy), ptr(gh), ptr(h), K, ctx->saved_data["type"].toInt(), ptr(w), ctx->saved_data["w_type"].toInt(), N, K,
                               static_cast<float>(ctx->saved_data["eps"].toDouble()), ptr(ws), ptr(gx), ptr(gw),
                               status_ptr(ctx->saved_data["status"].toTensor()), stream_of(h)));
    if (need_x) res[0] = gx;
    if (need_r) res[2] = gx;
    res[1] = gw;
    return once(res);
  }
};

// (y, h, codes, scales): those that were asked for; or None
optional<std::tuple<optional<Tensor>, optional<Tensor>, optional<Tensor>, optional<Tensor>>> rms_norm(const Tensor& x, const Tensor& w,
                                                                                                      const optional<Tensor>& residual, double eps,
                                                                                                      bool want_y, bool want_codes, const Tensor& status) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  const auto type = logits_type(x), w_type = logits_type(w);
  if (!type.has_value() || !w_type.has_value() || (*w_type != *type && *w_type != B200MOE_F32)) return std::nullopt;
  if (!plain(x, x.scalar_type(), dev) || !plain(w, w.scalar_type(), dev) || !plain_or_none(residual, x.scalar_type(), dev)) return std::nullopt;
  if (x.dim() < 1 || x.numel() == 0 || w.dim() != 1 || w.size(0) != x.size(-1) || (residual.has_value() && residual->sizes() != x.sizes())) return std::nullopt;
  const int64_t K = x.size(-1), N = x.numel() / K;
  if (K > 16384 || (want_codes && K % 8 != 0) || !(eps >= 0.0 && eps <= std::numeric_limits<float>::max()) || N >= (1LL << 31) - 256) return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  NormArgs a{residual, status, Tensor(), Tensor(), *type, *w_type, eps, want_y};
  if (want_codes) {
    a.q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    a.scale = at::empty({(K + 127) / 128, (N + 127) / 128 * 128}, x.options().dtype(at::kFloat));
  }
  const bool grad = at::GradMode::is_enabled() && (want_y || residual.has_value()) && (x.requires_grad() || w.requires_grad() || (residual.has_value() && residual->requires_grad()));
  const variable_list r = grad ? RmsNorm::apply(x, w, residual, a) : norm_forward(x, w, a);
  std::tuple<optional<Tensor>, optional<Tensor>, optional<Tensor>, optional<Tensor>> out;
  if (want_y) std::get<0>(out) = r[0];
  if (residual.has_value()) std::get<1>(out) = r.back();
  if (want_codes) {      // (..., blocks), rows next to one another
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end()), strides(sizes.size());
    sizes.back() = a.scale.size(0);
    strides.back() = a.scale.size(1);
    int64_t stride = 1;
    for (int64_t i = x.dim() - 2; i >= 0; --i) {
      strides[i] = stride;
      stride *= sizes[i];
    }
    std::get<2>(out) = a.q;
    std::get<3>(out) = a.scale.as_strided(sizes, strides);
  }
  return out;
}

// ---------------------------------------------------------------------------- low-rank adapters
struct LoraArgs {
  optional<Tensor> index, scales;
  Tensor status;
  double scale;
};

Tensor lora_forward(const Tensor& x, const Tensor& a, const Tensor& b, const optional<Tensor>& base, const LoraArgs& p, const Tensor& ws, bool keep) {
  const int64_t L = a.size(0), R = a.size(1), K = a.size(2), N = b.size(1), T = x.numel() / K;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  Tensor out = at::empty(shape, x.options());
  check(b200moe_lora_forward(ptr(x), K, ptr(a), ptr(b), ptr(p.index), p.index.has_value() ? p.index->element_size() : 0,
                             static_cast<const float*>(ptr(p.scales)), static_cast<float>(p.scale), ptr(base), N, T, K, N, R, L, keep, ptr(ws),
                             ptr(out), status_ptr(p.status), stream_of(x)));
  return out;
}

struct Lora : torch::autograd::Function<Lora> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& a, const Tensor& b, const optional<Tensor>& base,
                        const LoraArgs& p) {
    const bool keep = x.requires_grad() || a.requires_grad() || b.requires_grad();
    const Tensor ws = bytes(b200moe_lora_fwd_ws_bytes(x.numel() / a.size(2), a.size(1), a.size(0), keep), x);
    Tensor out = lora_forward(x, a, b, base, p, ws, keep);
    if (keep) ctx->save_for_backward({x, a, b, ws, p.scales.value_or(Tensor())});
    ctx->saved_data["status"] = p.status;
    ctx->saved_data["scale"] = p.scale;
    ctx->saved_data["index"] = p.index.has_value();
    ctx->saved_data["base"] = base.has_value();      // an input only where there is one
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(5);
    if (ctx->saved_data["base"].toBool() && ctx->needs_input_grad(3)) res[3] = grads[0];
    if (!ctx->needs_input_grad(0) && !ctx->needs_input_grad(1) && !ctx->needs_input_grad(2)) return once(res);
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &a = s[1], &b = s[2], &ws = s[3], &scales = s[4];
    const int64_t L = a.size(0), R = a.size(1), K = a.size(2), N = b.size(1), T = x.numel() / K;
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor g = grads[0].to(at::kBFloat16).contiguous();
    if (!aligned(g)) g = g.clone();
    for (int i = 0; i < 3; ++i) res[i] = grad_like(ctx->needs_input_grad(i), s[i]);
    Tensor tmp = bytes(b200moe_lora_bwd_ws_bytes(T, K, N, R, L), x);
    check(b200moe_lora_backward(ptr(g), ptr(x), K, ptr(a), ptr(b), ctx->saved_data["index"].toBool(), static_cast<const float*>(ptr(scales)),
                                static_cast<float>(ctx->saved_data["scale"].toDouble()), T, K, N, R, L, ptr(ws), ptr(tmp), ptr(res[0]), ptr(res[1]),
                                ptr(res[2]), 0, status_ptr(ctx->saved_data["status"].toTensor()), stream_of(x)));
    return once(res);
  }
};

// (..., N) bf16, or None
optional<Tensor> lora_linear(const Tensor& x, const Tensor& a, const Tensor& b, const optional<Tensor>& index, const optional<Tensor>& scales,
                             double scale, const optional<Tensor>& base, const Tensor& status) {
  if (!plain_call(x)) return std::nullopt;
  const auto dev = x.device();
  if (!plain(x, at::kBFloat16, dev) || !plain(a, at::kBFloat16, dev) || !plain(b, at::kBFloat16, dev) || !plain_or_none(base, at::kBFloat16, dev) ||
      !plain_or_none(scales, at::kFloat, dev))
    return std::nullopt;
  if (x.dim() < 1 || a.dim() != 3 || b.dim() != 3 || x.numel() == 0 || a.numel() == 0 || b.numel() == 0) return std::nullopt;
  const int64_t L = a.size(0), R = a.size(1), K = a.size(2), N = b.size(1);
  if (b.size(0) != L || b.size(2) != R || x.size(-1) != K || K % 8 != 0 || N % 8 != 0 || R % 8 != 0 || R > 128 || L > 65536) return std::nullopt;
  const auto rows = x.sizes().slice(0, x.dim() - 1);
  if (index.has_value()) {
    const auto type = index->scalar_type();
    if ((type != at::kInt && type != at::kLong) || !plain(*index, type, dev) || index->sizes() != rows) return std::nullopt;
  } else if (L != 1) {
    return std::nullopt;
  }
  if (scales.has_value() && (scales->dim() != 1 || scales->size(0) != L || (at::GradMode::is_enabled() && scales->requires_grad()))) return std::nullopt;
  if (base.has_value() && (base->dim() != x.dim() || base->sizes().slice(0, x.dim() - 1) != rows || base->size(-1) != N || !aligned(*base))) return std::nullopt;
  if (!aligned(x) || !aligned(a) || !aligned(b)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(dev);
  const LoraArgs p{index, scales, status, scale};
  if (at::GradMode::is_enabled() && (x.requires_grad() || a.requires_grad() || b.requires_grad() || (base.has_value() && base->requires_grad())))
    return Lora::apply(x, a, b, base, p);
  return lora_forward(x, a, b, base, p, bytes(b200moe_lora_fwd_ws_bytes(x.numel() / K, R, L, 0), x), false);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("torch_version") = TORCH_VERSION;
  m.def("layer", torch::wrap_pybind_function_no_gil(layer));
  m.def("experts", torch::wrap_pybind_function_no_gil(experts));
  m.def("conv_router", torch::wrap_pybind_function_no_gil(conv_router));
  m.def("group_topk", torch::wrap_pybind_function_no_gil(group_topk));
  m.def("router_losses", torch::wrap_pybind_function_no_gil(router_losses));
  m.def("fp8_block_linear", torch::wrap_pybind_function_no_gil(fp8_block_linear));
  m.def("fp8_block_linear_rows", torch::wrap_pybind_function_no_gil(fp8_block_linear_rows));
  m.def("rms_norm", torch::wrap_pybind_function_no_gil(rms_norm));
  m.def("lora_linear", torch::wrap_pybind_function_no_gil(lora_linear));
  m.def("moe_fp8_block", torch::wrap_pybind_function_no_gil(moe_fp8_block));
}
