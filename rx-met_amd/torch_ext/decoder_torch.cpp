// decoder_torch.cpp — the 8-bit decoder operators (include/rxmet_decoder.h) without the interpreter
// between their checks, allocations and launches.
//
// A single token's norm or projection takes 5 - 7 us of kernel; decoder_ops.py's checks and its
// call through ctypes take the host 14 - 18 us.  These functions take the calls that need no copy
// and refuse nothing: they return None for everything else (a wrong type, shape, device or stride, a tensor
// subclass, a trace, which would record the allocations without the kernels), and decoder_ops.py then
// goes its own way, which copies or raises.
#include "operator_calls.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>

#include "rxmet_decoder.h"

namespace rxmet_torch {
namespace {

// The entry points of the librxmet.so that rxmet_lib.py has loaded (bind_decoder()).
decltype(&rxmet_rms_quantize_forward) rms_forward = nullptr;
decltype(&rxmet_rms_quantize_backward) rms_backward = nullptr;
decltype(&rxmet_rms_quantize_backward_workspace_bytes) rms_backward_bytes = nullptr;
decltype(&rxmet_linear_int8) linear = nullptr;
decltype(&rxmet_linear_int8_workspace_bytes) linear_bytes = nullptr;
decltype(&rxmet_kv_append) append = nullptr;
decltype(&rxmet_kv_read) read = nullptr;
decltype(&rxmet_kv_attention) attention = nullptr;
decltype(&rxmet_kv_attention_workspace_bytes) attention_bytes = nullptr;

struct Rows {
  Tensor codes, y, scales, rstd, h;
};

// As decoder_ops._row_forward; false where it has to take over.
bool row_forward(const Tensor &x, const OptTensor &weight, const OptTensor &residual, double eps,
                 bool want_codes, bool training, Rows &out) {
  const int type = type_code(x.scalar_type());
  int64_t rows, cols, xs, rr, rc, rs = 0;
  if (!rms_forward || type < 0 || !plain(x) || !as_rows(x, rows, cols, xs) || cols > RXMET_ROW_MAX)
    return false;
  if (weight && !((weight->scalar_type() == x.scalar_type() ||
                   weight->scalar_type() == at::kFloat) &&
                  is(*weight, weight->scalar_type(), x) && vector_of(*weight, cols)))
    return false;
  if (residual && !(weight && is(*residual, x.scalar_type(), x) &&
                    residual->sizes() == x.sizes() && as_rows(*residual, rr, rc, rs)))
    return false;
  const c10::DeviceGuard guard(x.device());
  const auto o = x.options().requires_grad(false);
  out.scales = at::empty(x.sizes().slice(0, x.dim() - 1), o.dtype(at::kFloat));
  if (want_codes) out.codes = at::empty(x.sizes(), o.dtype(at::kChar));
  if (training) {
    out.y = at::empty(x.sizes(), o);
    out.rstd = at::empty({rows}, o.dtype(at::kFloat));
  }
  out.h = residual ? at::empty(x.sizes(), o) : x;
  check(rms_forward(x.const_data_ptr(), xs, ptr(residual), rs, ptr(weight),
                    weight && weight->scalar_type() == at::kFloat,
                    residual ? out.h.mutable_data_ptr() : nullptr,
                    want_codes ? out.codes.mutable_data_ptr<int8_t>() : nullptr,
                    training ? out.y.mutable_data_ptr() : nullptr,
                    out.scales.mutable_data_ptr<float>(),
                    training ? out.rstd.mutable_data_ptr<float>() : nullptr, rows, cols, type,
                    static_cast<float>(eps), stream_of(x)),
        "rxmet_rms_quantize_forward");
  return true;
}

py::object rms_norm_quantize(const Tensor &x, const Tensor &weight, const OptTensor &residual,
                             double eps) {
  Rows r;
  if (!row_forward(x, weight, residual, eps, true, false, r)) return py::none();
  return py::make_tuple(r.codes, r.scales, r.h.requires_grad() ? r.h.detach() : r.h);
}

py::object quantize_rows(const Tensor &x) {
  Rows r;
  if (!row_forward(x, std::nullopt, std::nullopt, 0.0, true, false, r)) return py::none();
  return py::make_tuple(r.codes, r.scales);
}

struct RmsQuantDequant : torch::autograd::Function<RmsQuantDequant> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx,
                                                const Tensor &x, const Tensor &weight,
                                                const OptTensor &residual, double eps) {
    Rows r;
    TORCH_CHECK(row_forward(x, weight, residual, eps, false, true, r),
                "rms_norm_quantize_dequantize: the tensors changed during the call");
    if (!residual) r.h = x.view_as(x);
    ctx->save_for_backward({r.h, weight, r.rstd});
    ctx->set_materialize_grads(false);
    ctx->saved_data["residual"] = residual.has_value();
    return {r.y, r.h};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    // Unpack hooks may hand back other tensors than were packed.  The engine has held the gradients
    // against the outputs, which are like x.
    const Tensor &like = grads[0].defined() ? grads[0] : grads[1];
    if (!like.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const at::ScalarType type = like.scalar_type();
    const at::Device device = like.device();
    const int64_t cols = like.size(-1), rows = like.numel() / cols;
    auto fits = [&](const Tensor &t, at::ScalarType want, at::IntArrayRef sizes) {
      return t.defined() && t.device() == device && t.scalar_type() == want && t.sizes() == sizes;
    };
    TORCH_CHECK(type_code(type) >= 0 && like.is_cuda() && fits(saved[0], type, like.sizes()) &&
                    (fits(saved[1], type, {cols}) || fits(saved[1], at::kFloat, {cols})) &&
                    fits(saved[2], at::kFloat, {rows}),
                "rms_norm_quantize_dequantize: the saved tensors are not those of the forward pass");
    const c10::DeviceGuard guard(device);
    const Tensor h = saved[0].contiguous(), weight = saved[1].contiguous(), rstd = saved[2].contiguous();
    auto gradient = [&](const Tensor &g) {
      TORCH_CHECK(fits(g, type, like.sizes()),
                  "rms_norm_quantize_dequantize: a gradient has another shape, type or device");
      return g.contiguous();
    };
    const Tensor dy = grads[0].defined() ? gradient(grads[0]) : at::zeros_like(h);
    Tensor dh;
    if (grads[1].defined()) dh = gradient(grads[1]);
    const bool need_w = ctx->needs_input_grad(1);
    Tensor dx = at::empty_like(h), dw, ws;
    if (need_w) {
      dw = at::empty_like(weight);
      ws = at::empty({rms_backward_bytes(rows, cols)}, h.options().dtype(at::kByte));
    }
    check(rms_backward(dy.const_data_ptr(), cols, dh.defined() ? dh.const_data_ptr() : nullptr,
                       cols, h.const_data_ptr(), cols, weight.const_data_ptr(),
                       weight.scalar_type() == at::kFloat, rstd.const_data_ptr<float>(),
                       dx.mutable_data_ptr(), need_w ? dw.mutable_data_ptr() : nullptr, rows,
                       cols, type_code(h.scalar_type()), need_w ? ws.mutable_data_ptr() : nullptr,
                       stream_of(h)),
          "rxmet_rms_quantize_backward");
    if (at::GradMode::is_enabled()) {
      // create_graph: the kernel's gradients have no graph, so going through them has to fail
      auto leaf = [](const Tensor &t) { return t.defined() ? t.detach().requires_grad_() : t; };
      const auto outs = std::make_shared<torch::autograd::DelayedError>(
                            "rms_norm_quantize_dequantize cannot be differentiated twice", 2)
                            ->apply({leaf(dx), leaf(dw)});
      dx = outs[0];
      dw = outs[1];
    }
    return {dx, dw, ctx->saved_data["residual"].toBool() ? dx : Tensor(), Tensor()};
  }
};

py::object rms_norm_quantize_dequantize(const Tensor &x, const Tensor &weight,
                                        const OptTensor &residual, double eps) {
  int64_t a, b, c;
  if (!rms_forward || type_code(x.scalar_type()) < 0 || !plain(x) || !as_rows(x, a, b, c) ||
      b > RXMET_ROW_MAX ||
      !((weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat) &&
        is(weight, weight.scalar_type(), x) && vector_of(weight, b)) ||
      (residual && !(is(*residual, x.scalar_type(), x) && residual->sizes() == x.sizes() &&
                     as_rows(*residual, a, b, c))))
    return py::none();
  const auto r = RmsQuantDequant::apply(x, weight, residual, eps);
  return py::make_tuple(r[0], r[1]);
}

py::object linear_int8(const Tensor &codes, const Tensor &scales, const Tensor &weight,
                       const Tensor &weight_scales, const OptTensor &bias, int act,
                       const OptTensor &residual, at::ScalarType type) {
  int64_t M, K, xs, N, k2, ws, rr, rc, rs = 0;
  if (!linear || type_code(type) < 0 || !plain(codes) || codes.scalar_type() != at::kChar ||
      !as_rows(codes, M, K, xs) || !is(weight, at::kChar, codes) || weight.dim() != 2 ||
      !as_rows(weight, N, k2, ws) || k2 != K || K > RXMET_LINEAR_INT8_K_MAX || N < 1 ||
      !is(scales, at::kFloat, codes) || !scales.is_contiguous() ||
      scales.sizes() != codes.sizes().slice(0, codes.dim() - 1) ||
      !is(weight_scales, at::kFloat, codes) || !vector_of(weight_scales, N))
    return py::none();
  if (bias && !(is(*bias, type, codes) && vector_of(*bias, N))) return py::none();
  auto shape = codes.sizes().vec();
  shape.back() = N;
  if (residual && !(is(*residual, type, codes) && residual->sizes() == at::IntArrayRef(shape) &&
                    as_rows(*residual, rr, rc, rs)))
    return py::none();
  const c10::DeviceGuard guard(codes.device());
  const Tensor y = at::empty(shape, codes.options().dtype(type));
  const int64_t bytes = linear_bytes(codes.const_data_ptr<int8_t>(), xs,
                                     weight.const_data_ptr<int8_t>(), ws, M, N, K);
  Tensor work;
  if (bytes > 0) work = at::empty({bytes}, codes.options().dtype(at::kByte));
  check(linear(codes.const_data_ptr<int8_t>(), xs, scales.const_data_ptr<float>(),
               weight.const_data_ptr<int8_t>(), ws, weight_scales.const_data_ptr<float>(),
               ptr(bias), ptr(residual), rs, y.mutable_data_ptr(), M, N, K, act, type_code(type),
               bytes > 0 ? work.mutable_data_ptr() : nullptr, stream_of(codes)),
        "rxmet_linear_int8");
  return py::cast(y);
}

// The cache and the table as the library takes them; false where decoder_ops.py has to look.
bool cache_of(const Tensor &k, const Tensor &v, const Tensor &ks, const Tensor &vs,
              const Tensor &table, rxmet_kv_cache &c, rxmet_kv_table &t) {
  if (!append || !plain(k) || k.scalar_type() != at::kChar || k.dim() != 4 || !k.is_contiguous())
    return false;
  const int64_t pages = k.size(0), heads = k.size(1), P = k.size(2), D = k.size(3);
  if (pages < 1 || heads < 1 || heads > 16384 || !(D == 64 || D == 128 || D == 192 || D == 256) ||
      !(P == 16 || P == 32 || P == 64 || P == 128))
    return false;
  if (!is(v, at::kChar, k) || v.dim() != 4 || v.size(0) != pages || v.size(1) != heads ||
      v.size(2) != D || v.size(3) != P || !v.is_contiguous())
    return false;
  for (const Tensor *s : {&ks, &vs})
    if (!is(*s, at::kFloat, k) || s->dim() != 2 || s->size(0) != pages || s->size(1) != heads ||
        !s->is_contiguous())
      return false;
  if (!is(table, at::kInt, k) || table.dim() != 2 || table.size(1) < 1 ||
      (table.stride(1) != 1 && table.size(1) > 1))
    return false;
  c = {k.mutable_data_ptr<int8_t>(), v.mutable_data_ptr<int8_t>(), ks.mutable_data_ptr<float>(),
       vs.mutable_data_ptr<float>(), pages, static_cast<int32_t>(heads), static_cast<int32_t>(P),
       static_cast<int32_t>(D), 0};
  t = {table.const_data_ptr<int32_t>(), table.stride(0), static_cast<int32_t>(table.size(0)),
       static_cast<int32_t>(table.size(1))};
  return true;
}

bool ints(const Tensor &t, int64_t n, const Tensor &like) {
  return is(t, at::kInt, like) && vector_of(t, n);
}
const int32_t *ints_ptr(const OptTensor &t) {
  return t ? t->const_data_ptr<int32_t>() : nullptr;
}

bool kv_append(const Tensor &k, const Tensor &v, const Tensor &ks, const Tensor &vs,
               const Tensor &key, const Tensor &value, const Tensor &table, const Tensor &lengths,
               const OptTensor &cu, std::optional<int64_t> max_new) {
  rxmet_kv_cache c;
  rxmet_kv_table t;
  const int type = type_code(key.scalar_type());
  if (!cache_of(k, v, ks, vs, table, c, t) || type < 0 || !ints(lengths, t.seqs, k) ||
      (cu && !ints(*cu, t.seqs + 1, k)))
    return false;
  for (const Tensor *x : {&key, &value})
    if (!is(*x, key.scalar_type(), k) || x->dim() != 3 || x->size(0) != key.size(0) ||
        x->size(1) != c.heads || x->size(2) != c.dim || x->stride(2) != 1)
      return false;
  const int64_t n = key.size(0);
  if (!cu && n != t.seqs) return false;
  const c10::DeviceGuard guard(k.device());
  check(append(&c, &t, lengths.const_data_ptr<int32_t>(), ints_ptr(cu), n,
               !cu ? 1 : max_new ? *max_new : n, key.const_data_ptr(), key.stride(0),
               key.stride(1), value.const_data_ptr(), value.stride(0), value.stride(1), type,
               stream_of(k)),
        "rxmet_kv_append");
  return true;
}

py::object kv_read(const Tensor &k, const Tensor &v, const Tensor &ks, const Tensor &vs,
                   const Tensor &table, const Tensor &first, const Tensor &cu, int64_t tokens,
                   std::optional<int64_t> max_tokens, at::ScalarType type) {
  rxmet_kv_cache c;
  rxmet_kv_table t;
  if (!cache_of(k, v, ks, vs, table, c, t) || type_code(type) < 0 || tokens < 0 ||
      !ints(first, t.seqs, k) || !ints(cu, t.seqs + 1, k))
    return py::none();
  const c10::DeviceGuard guard(k.device());
  const Tensor key = at::empty({tokens, c.heads, c.dim}, k.options().dtype(type));
  const Tensor value = at::empty_like(key);
  check(read(&c, &t, first.const_data_ptr<int32_t>(), cu.const_data_ptr<int32_t>(), tokens,
             max_tokens ? *max_tokens : tokens, key.mutable_data_ptr(), value.mutable_data_ptr(),
             type_code(type), stream_of(k)),
        "rxmet_kv_read");
  return py::make_tuple(key, value);
}

py::object kv_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ks,
                        const Tensor &vs, const Tensor &table, const Tensor &lengths,
                        const OptTensor &cu, std::optional<int64_t> max_query,
                        std::optional<int64_t> max_length, std::optional<double> scale,
                        bool causal, std::optional<int64_t> window) {
  rxmet_kv_cache c;
  rxmet_kv_table t;
  const int type = type_code(q.scalar_type());
  if (!cache_of(k, v, ks, vs, table, c, t) || (type != RXMET_QDQ_F16 && type != RXMET_QDQ_BF16) ||
      !is(q, q.scalar_type(), k) || q.dim() != 3 || q.size(2) != c.dim || q.stride(2) != 1 ||
      q.size(1) < c.heads || q.size(1) % c.heads != 0 || !ints(lengths, t.seqs, k) ||
      (cu && !ints(*cu, t.seqs + 1, k)) || (!cu && q.size(0) != t.seqs) || (window && *window < 1))
    return py::none();
  const int64_t n = q.size(0), heads = q.size(1);
  const int64_t mq = !cu ? 1 : max_query ? *max_query : n;
  const int64_t ml = max_length ? *max_length : static_cast<int64_t>(t.cols) * c.page_size;
  const int64_t win = window ? *window : 0;
  const c10::DeviceGuard guard(k.device());
  const Tensor out = at::empty({n, heads, c.dim}, q.options().requires_grad(false));
  const int64_t bytes =
      attention_bytes(&c, t.seqs, n, static_cast<int32_t>(heads), mq, ml, win);
  Tensor work;
  if (bytes > 0) work = at::empty({bytes}, k.options().dtype(at::kByte));
  check(attention(&c, &t, lengths.const_data_ptr<int32_t>(), ints_ptr(cu), n, mq, ml,
                  q.const_data_ptr(), q.stride(0), q.stride(1), static_cast<int32_t>(heads),
                  static_cast<float>(scale ? *scale : 1.0 / std::sqrt(c.dim)), causal, win,
                  out.mutable_data_ptr(), type, bytes > 0 ? work.mutable_data_ptr() : nullptr,
                  stream_of(k)),
        "rxmet_kv_attention");
  return py::cast(out);
}

void bind(const std::vector<uintptr_t> &p) {
  TORCH_CHECK(p.size() == 10, "bind_decoder takes ten entry points");
  size_t i = 0;
  auto take = [&](auto &f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(p[i++]); };
  take(rms_forward);
  take(rms_backward);
  take(rms_backward_bytes);
  take(linear);
  take(linear_bytes);
  take(append);
  take(read);
  take(attention);
  take(attention_bytes);
  take(last_error);
}

}  // namespace

void add_decoder(py::module_ &m) {
  m.def("bind_decoder", &bind);
  m.def("rms_norm_quantize", &rms_norm_quantize);
  m.def("quantize_rows", &quantize_rows);
  m.def("rms_norm_quantize_dequantize", &rms_norm_quantize_dequantize);
  m.def("linear_int8", &linear_int8);
  m.def("kv_append", &kv_append);
  m.def("kv_read", &kv_read);
  m.def("kv_attention", &kv_attention);
}

}  // namespace rxmet_torch
