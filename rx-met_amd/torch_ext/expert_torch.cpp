// expert_torch.cpp — the expert layers' operators (include/rxmet_experts.h) without the interpreter
// between their checks, allocations and launches.
//
// As in decoder_torch.cpp these functions take the calls that need no copy and refuse nothing; they return
// None for everything else, and expert_ops.py then goes its own way, which copies or raises.  A token's
// routing or sum takes some 5 us of kernel; the same calls take the host 14 to 18 us through ctypes, 110 with
// a Python autograd function.
#include "operator_calls.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include "rxmet_decoder.h"
#include "rxmet_experts.h"

namespace rxmet_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The entry points of the librxmet.so that rxmet_lib.py has loaded (bind_experts()).
decltype(&rxmet_route_forward) route_forward = nullptr;
decltype(&rxmet_route_backward) route_backward = nullptr;
decltype(&rxmet_group_experts) group = nullptr;
decltype(&rxmet_group_experts_workspace_bytes) group_bytes = nullptr;
decltype(&rxmet_experts_linear_int8) linear = nullptr;
decltype(&rxmet_experts_combine) combine = nullptr;
decltype(&rxmet_experts_combine_backward) combine_backward = nullptr;

bool saved_is(const Tensor &t, at::ScalarType type, at::Device device, at::IntArrayRef sizes) {
  return t.defined() && t.is_cuda() && t.scalar_type() == type && t.device() == device &&
         t.sizes() == sizes;
}

// Gradients that raise when they are differentiated: under create_graph they have no graph.
variable_list once(const char *name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto &g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  return std::make_shared<torch::autograd::DelayedError>(
             std::string(name) + " cannot be differentiated twice", static_cast<int64_t>(grads.size()))
      ->apply(std::move(grads));
}

// ---------------------------------------------------------------------------------------------
// Routing

struct Routed {
  Tensor experts, weights;
};

Routed run_route(const Tensor &logits, const OptTensor &bias, const rxmet_router &r) {
  int64_t tokens, cols, stride;
  TORCH_CHECK(as_rows(logits, tokens, cols, stride), "route_experts: the logits changed during the call");
  const c10::DeviceGuard guard(logits.device());
  auto shape = logits.sizes().vec();
  shape.back() = r.top_k;
  const auto o = logits.options().requires_grad(false);
  Routed out{at::empty(shape, o.dtype(at::kInt)), at::empty(shape, o.dtype(at::kFloat))};
  check(route_forward(&r, logits.const_data_ptr(), stride,
                      bias ? bias->const_data_ptr<float>() : nullptr,
                      out.experts.mutable_data_ptr<int32_t>(), out.weights.mutable_data_ptr<float>(),
                      tokens, type_code(logits.scalar_type()), stream_of(logits)),
        "rxmet_route_forward");
  return out;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const OptTensor &bias,
                               const rxmet_router &r) {
    const Routed out = run_route(logits, bias, r);
    ctx->save_for_backward({logits, out.experts});
    ctx->mark_non_differentiable({out.experts});
    ctx->set_materialize_grads(false);
    ctx->saved_data["router"] = std::vector<int64_t>{r.experts, r.top_k, r.score, r.renormalize};
    ctx->saved_data["scale"] = static_cast<double>(r.scale);
    return {out.experts, out.weights};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto p = ctx->saved_data["router"].toIntVector();
    const rxmet_router r{static_cast<int32_t>(p[0]), static_cast<int32_t>(p[1]),
                         static_cast<int32_t>(p[2]), static_cast<int32_t>(p[3]), 1, 1, 1,
                         static_cast<float>(ctx->saved_data["scale"].toDouble())};
    // Unpack hooks may hand back other tensors than were packed.  The engine has held the gradient
    // against the weights.
    const Tensor &g = grads[1];
    auto shape = g.sizes().vec();
    shape.back() = r.experts;
    TORCH_CHECK(g.is_cuda() && g.scalar_type() == at::kFloat && g.size(-1) == r.top_k &&
                    saved[0].defined() && type_code(saved[0].scalar_type()) >= 0 &&
                    saved_is(saved[0], saved[0].scalar_type(), g.device(), shape) &&
                    saved_is(saved[1], at::kInt, g.device(), g.sizes()),
                "route_experts: the saved tensors are not those of the forward pass");
    const c10::DeviceGuard guard(g.device());
    int64_t tokens, cols, stride;
    const Tensor logits = as_rows(saved[0], tokens, cols, stride) ? saved[0] : saved[0].contiguous();
    TORCH_CHECK(as_rows(logits, tokens, cols, stride), "route_experts: no rows");
    const Tensor experts = saved[1].contiguous(), dw = g.contiguous();
    const Tensor out = at::empty(shape, logits.options().requires_grad(false));
    check(route_backward(&r, logits.const_data_ptr(), stride, experts.const_data_ptr<int32_t>(),
                         dw.const_data_ptr<float>(), out.mutable_data_ptr(), tokens,
                         type_code(logits.scalar_type()), stream_of(g)),
          "rxmet_route_backward");
    return {once("route_experts", {out})[0], Tensor(), Tensor()};
  }
};

py::object route_experts(const Tensor &logits, int64_t top_k, int score, const OptTensor &bias,
                         int64_t groups, std::optional<int64_t> top_groups, int64_t group_best,
                         bool renormalize, double scale) {
  int64_t tokens, E, stride;
  if (!route_forward || type_code(logits.scalar_type()) < 0 || !plain(logits) || dual(logits) ||
      !as_rows(logits, tokens, E, stride) || E > RXMET_EXPERTS_MAX || groups < 1 ||
      groups > RXMET_EXPERT_GROUPS_MAX || E % groups != 0 || top_k < 1 || top_k > RXMET_TOP_K_MAX ||
      (group_best != 1 && group_best != 2))
    return py::none();
  const int64_t top = top_groups ? *top_groups : groups;
  if (top < 1 || top > groups || top_k > top * (E / groups)) return py::none();
  if (bias && !(is(*bias, at::kFloat, logits) && vector_of(*bias, E))) return py::none();
  const rxmet_router r{static_cast<int32_t>(E), static_cast<int32_t>(top_k), score, renormalize,
                       static_cast<int32_t>(groups), static_cast<int32_t>(top),
                       static_cast<int32_t>(group_best), static_cast<float>(scale)};
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const auto out = Route::apply(logits, bias ? OptTensor(bias->detach()) : bias, r);
    return py::make_tuple(out[0], out[1]);
  }
  const Routed out = run_route(logits, bias, r);
  return py::make_tuple(out.experts, out.weights);
}

// ---------------------------------------------------------------------------------------------
// Order by expert

py::object group_experts(const Tensor &experts, int64_t num_experts) {
  if (!group || !plain(experts) || experts.scalar_type() != at::kInt || experts.dim() < 1 ||
      !experts.is_contiguous() || experts.size(-1) < 1 || experts.size(-1) > RXMET_TOP_K_MAX ||
      num_experts < 1 || num_experts > RXMET_EXPERTS_MAX)
    return py::none();
  const c10::DeviceGuard guard(experts.device());
  const int64_t n = experts.numel(), bytes = group_bytes(n, static_cast<int32_t>(num_experts));
  const auto o = experts.options();
  const Tensor offsets = at::empty({num_experts + 1}, o), entries = at::empty({n}, o),
               places = at::empty(experts.sizes(), o);
  Tensor work;
  if (bytes > 0) work = at::empty({bytes}, o.dtype(at::kByte));
  check(group(experts.const_data_ptr<int32_t>(), n, static_cast<int32_t>(num_experts),
              offsets.mutable_data_ptr<int32_t>(), entries.mutable_data_ptr<int32_t>(),
              places.mutable_data_ptr<int32_t>(), bytes > 0 ? work.mutable_data_ptr() : nullptr,
              stream_of(experts)),
        "rxmet_group_experts");
  return py::make_tuple(offsets, entries, places);
}

// The groups as the library takes them; false where expert_ops.py has to look.
bool groups_of(const Tensor &offsets, const Tensor &entries, const Tensor &places,
               const Tensor &like, rxmet_expert_groups &g) {
  if (!is(places, at::kInt, like) || places.dim() < 1 || !places.is_contiguous() ||
      places.size(-1) < 1 || places.size(-1) > RXMET_TOP_K_MAX || !is(entries, at::kInt, like) ||
      !vector_of(entries, places.numel()) || !is(offsets, at::kInt, like) || offsets.dim() != 1 ||
      offsets.size(0) < 2 || offsets.size(0) > RXMET_EXPERTS_MAX + 1 || !offsets.is_contiguous())
    return false;
  const int64_t k = places.size(-1);
  g = {offsets.const_data_ptr<int32_t>(), entries.const_data_ptr<int32_t>(),
       places.const_data_ptr<int32_t>(), places.numel() / k, static_cast<int32_t>(k),
       static_cast<int32_t>(offsets.size(0) - 1)};
  return true;
}

// ---------------------------------------------------------------------------------------------
// Product

py::object experts_linear_int8(const Tensor &codes, const Tensor &scales, const Tensor &weight,
                               const Tensor &weight_scales, const Tensor &offsets,
                               const Tensor &entries, const Tensor &places, const OptTensor &bias,
                               int act, bool gated, bool grouped, at::ScalarType type) {
  rxmet_expert_groups g;
  int64_t n, K, xs;
  if (!linear || type_code(type) < 0 || !plain(codes) || codes.scalar_type() != at::kChar ||
      codes.dim() != 2 || !as_rows(codes, n, K, xs) || !groups_of(offsets, entries, places, codes, g) ||
      n != (grouped ? g.tokens * g.top_k : g.tokens) || !is(weight, at::kChar, codes) ||
      weight.dim() != 3 || weight.size(0) != g.experts || weight.size(1) < 1 || weight.size(2) != K ||
      K > RXMET_LINEAR_INT8_K_MAX || weight.stride(2) != 1 || (gated && weight.size(1) % 2 != 0) ||
      !is(scales, at::kFloat, codes) || !vector_of(scales, n) ||
      !is(weight_scales, at::kFloat, codes) || !weight_scales.is_contiguous() ||
      weight_scales.sizes() != weight.sizes().slice(0, 2))
    return py::none();
  if (bias && !(is(*bias, type, codes) && bias->is_contiguous() &&
                bias->sizes() == weight_scales.sizes()))
    return py::none();
  const int64_t N = gated ? weight.size(1) / 2 : weight.size(1);
  const c10::DeviceGuard guard(codes.device());
  const Tensor y = at::empty({g.tokens * g.top_k, N}, codes.options().dtype(type));
  check(linear(&g, grouped, codes.const_data_ptr<int8_t>(), xs, scales.const_data_ptr<float>(),
               weight.const_data_ptr<int8_t>(), weight.stride(1), weight.stride(0),
               weight_scales.const_data_ptr<float>(), ptr(bias), y.mutable_data_ptr(), N, K, gated,
               act, type_code(type), stream_of(codes)),
        "rxmet_experts_linear_int8");
  return py::cast(y);
}

// ---------------------------------------------------------------------------------------------
// Rows added up

struct Combine : torch::autograd::Function<Combine> {
  static Tensor run(const Tensor &y, const Tensor &weights, const OptTensor &residual,
                    const Tensor &offsets, const Tensor &entries, const Tensor &places) {
    rxmet_expert_groups g;
    int64_t rows, N, ys, rr, rc, rs = 0;
    TORCH_CHECK(as_rows(y, rows, N, ys) && groups_of(offsets, entries, places, y, g) &&
                    (!residual || as_rows(*residual, rr, rc, rs)),
                "experts_combine: the tensors changed during the call");
    auto shape = places.sizes().vec();
    shape.back() = N;
    const c10::DeviceGuard guard(y.device());
    const Tensor out = at::empty(shape, y.options().requires_grad(false));
    check(combine(&g, y.const_data_ptr(), ys, weights.const_data_ptr<float>(), ptr(residual), rs,
                  out.mutable_data_ptr(), N, type_code(y.scalar_type()), stream_of(y)),
          "rxmet_experts_combine");
    return out;
  }

  static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &weights,
                        const OptTensor &residual, const Tensor &offsets, const Tensor &entries,
                        const Tensor &places) {
    ctx->save_for_backward({y, weights, offsets, entries, places});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["experts"] = offsets.size(0);
    return run(y, weights, residual, offsets, entries, places);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &d = grads[0];
    const bool residual = ctx->saved_data["residual"].toBool();
    const bool need_y = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const int64_t N = d.size(-1);
    auto shape = d.sizes().vec();
    // Unpack hooks may hand back other tensors than were packed.  The engine has held the gradient
    // against the output, which has y's type.
    const char *what = "experts_combine: the saved tensors are not those of the forward pass";
    TORCH_CHECK(saved[4].defined() && saved[4].dim() == d.dim(), what);
    shape.back() = saved[4].size(-1);
    rxmet_expert_groups g;
    const c10::DeviceGuard guard(d.device());
    for (const auto &t : saved) TORCH_CHECK(t.defined(), what);
    const Tensor offsets = saved[2].contiguous(), entries = saved[3].contiguous(),
                 places = saved[4].contiguous();
    TORCH_CHECK(d.is_cuda() && saved_is(places, at::kInt, d.device(), shape) &&
                    saved_is(saved[1], at::kFloat, d.device(), shape) &&
                    saved_is(saved[0], d.scalar_type(), d.device(), {places.numel(), N}) &&
                    offsets.dim() == 1 && offsets.size(0) == ctx->saved_data["experts"].toInt() &&
                    groups_of(offsets, entries, places, d, g),
                what);
    int64_t rows, cols, ys, ds;
    const Tensor y = as_rows(saved[0], rows, cols, ys) ? saved[0] : saved[0].contiguous();
    const Tensor g_out = as_rows(d, rows, cols, ds) ? d : d.contiguous();
    TORCH_CHECK(as_rows(y, rows, cols, ys) && as_rows(g_out, rows, cols, ds), what);
    const Tensor weights = saved[1].contiguous();
    Tensor dy, dw;
    const auto o = y.options().requires_grad(false);
    if (need_y) dy = at::empty({places.numel(), N}, o);
    if (need_w) dw = at::empty(shape, o.dtype(at::kFloat));
    check(combine_backward(&g, g_out.const_data_ptr(), ds, y.const_data_ptr(), ys,
                           weights.const_data_ptr<float>(), need_y ? dy.mutable_data_ptr() : nullptr,
                           need_w ? dw.mutable_data_ptr<float>() : nullptr, N,
                           type_code(y.scalar_type()), stream_of(d)),
          "rxmet_experts_combine_backward");
    const auto out = once("experts_combine", {dy, dw});
    return {out[0], out[1], residual && ctx->needs_input_grad(2) ? d : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::object experts_combine(const Tensor &y, const Tensor &weights, const OptTensor &residual,
                           const Tensor &offsets, const Tensor &entries, const Tensor &places) {
  rxmet_expert_groups g;
  int64_t rows, N, ys, rr, rc, rs;
  if (!combine || type_code(y.scalar_type()) < 0 || !plain(y) || y.dim() != 2 ||
      !as_rows(y, rows, N, ys) || !groups_of(offsets, entries, places, y, g) ||
      rows != places.numel() || !is(weights, at::kFloat, y) || !weights.is_contiguous() ||
      weights.sizes() != places.sizes() || dual(y) || dual(weights))
    return py::none();
  if (residual) {
    auto shape = places.sizes().vec();
    shape.back() = N;
    if (!is(*residual, y.scalar_type(), y) || residual->sizes() != at::IntArrayRef(shape) ||
        !as_rows(*residual, rr, rc, rs) || dual(*residual))
      return py::none();
  }
  if (at::GradMode::is_enabled() && (y.requires_grad() || weights.requires_grad() ||
                                     (residual && residual->requires_grad())))
    return py::cast(Combine::apply(y, weights, residual, offsets, entries, places));
  return py::cast(Combine::run(y, weights, residual, offsets, entries, places));
}

void bind(const std::vector<uintptr_t> &p) {
  TORCH_CHECK(p.size() == 8, "bind_experts takes eight entry points");
  size_t i = 0;
  auto take = [&](auto &f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(p[i++]); };
  take(route_forward);
  take(route_backward);
  take(group);
  take(group_bytes);
  take(linear);
  take(combine);
  take(combine_backward);
  take(last_error);
}

}  // namespace

void add_experts(py::module_ &m) {
  m.def("bind_experts", &bind);
  m.def("route_experts", &route_experts);
  m.def("group_experts", &group_experts);
  m.def("experts_linear_int8", &experts_linear_int8);
  m.def("experts_combine", &experts_combine);
}

}  // namespace rxmet_torch
