// frozen_ops.cpp -- torch.ops.lycoris_amd.{int8_quantize, int8_matmul, int8_linear, gated_linear} over the C ABI: the 8-bit frozen layer and
// the gated projection.  Host-only, like torch_ops.cpp: checks, output allocation, autograd nodes, Meta kernels for tracing.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/lycoris_amd.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LYC_F32;
    case at::kHalf: return LYC_F16;
    case at::kBFloat16: return LYC_BF16;
    default: TORCH_CHECK(false, "lycoris_amd supports float32/float16/bfloat16 activations, got ", t);
  }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", lyc_last_error()); }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* dptr(const OptTensor& t) { return has(t) ? t->const_data_ptr() : nullptr; }

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
// a node's edges are its PRESENT tensors: the place of an optional one (-1: absent), and whether its gradient is wanted now
int64_t edge(const OptTensor& t, int64_t at) { return has(t) ? at : -1; }
bool wanted(AutogradContext* ctx, const char* which) {
  const int64_t i = ctx->saved_data[which].toInt();
  return i >= 0 && ctx->needs_input_grad(i);
}

void on_device_of(const Tensor& x, const OptTensor& t, const char* what) {
  TORCH_CHECK(!has(t) || t->device() == x.device(), "lycoris_amd: ", what, " is on ", t->device(), ", the activation on ", x.device());
}
void need_hip(const Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda(), "lycoris_amd: ", what, " is on ", x.device(), "; this op runs on the MI355X HIP device");
}

// [.., K] -> contiguous, 16-byte aligned [M, K]
Tensor rows_of(const Tensor& x, int64_t K) {
  if (x.dim() == 2 && x.is_contiguous() && aligned(x)) return x;  // no new tensor: host time per call
  Tensor r = x.reshape({x.numel() / K, K}).contiguous();
  return aligned(r) ? r : r.clone();
}
// an 8-bit operand in rows the kernels can read (16-byte aligned rows); zero_tail: with zeros behind K up to a multiple of 16
Tensor rows8(const Tensor& q, bool zero_tail) {
  const int64_t N = q.size(0), K = q.size(1);
  if (q.stride(1) == 1 && q.stride(0) >= K && q.stride(0) % 16 == 0 && q.stride(0) <= (1 << 22) && aligned(q) && (!zero_tail || K % 16 == 0)) return q;
  Tensor r = at::zeros({N, (K + 15) / 16 * 16}, q.options());
  r.narrow(1, 0, K).copy_(q);
  return r;
}
Tensor scales_of(const Tensor& s, int64_t n, const char* what) {
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.numel() == n, "lycoris_amd: ", what, " must be ", n, " float32 values, got ", s.sizes(), " ", s.scalar_type());
  return s.dim() == 1 && s.is_contiguous() ? s : s.reshape({n}).contiguous();
}
// bias as the kernels read it: the activation type or fp32
OptTensor bias_of(const OptTensor& b, int64_t n, at::ScalarType act) {
  if (!has(b)) return c10::nullopt;
  TORCH_CHECK(b->dim() == 1 && b->numel() == n && b->is_floating_point(), "lycoris_amd: bias must be [", n, "], got ", b->sizes(), " ", b->scalar_type());
  Tensor t = b->contiguous();
  return t.scalar_type() == act || t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
}
int bias_f32(const OptTensor& b) { return has(b) && b->scalar_type() == at::kFloat; }
OptTensor base_of(const OptTensor& b, const Tensor& x, int64_t n) {
  if (!has(b)) return c10::nullopt;
  auto want = x.sizes().vec();
  want.back() = n;
  TORCH_CHECK(b->sizes() == at::IntArrayRef(want) && b->scalar_type() == x.scalar_type(), "lycoris_amd: base must be ", at::IntArrayRef(want), " ",
              x.scalar_type(), ", got ", b->sizes(), " ", b->scalar_type());
  return b->contiguous();
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}
Tensor scratch(const Tensor& x, int64_t bytes, const char* what) {
  TORCH_CHECK(bytes >= 0, what, ": ", lyc_last_error());
  if (bytes == 0) return Tensor();
  return at::empty({bytes}, x.options().dtype(at::kByte));
}
void check_act_x(const Tensor& x, int64_t K, const char* what) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K, what, ": x has ", x.dim() ? x.size(-1) : 0, " features, the weight ", K);
  code_of(x.scalar_type());
}
void check_w8(const Tensor& wq, const char* what) {
  TORCH_CHECK(wq.dim() == 2 && wq.scalar_type() == at::kChar && wq.size(0) > 0 && wq.size(1) > 0, what, ": the 8-bit operand must be a non-empty int8 matrix, got ",
              wq.sizes(), " ", wq.scalar_type());
}
// May the device function be called without another trip through the dispatcher?  Where the dispatcher would go there by itself: what is left
// of the tensors' keys and the thread's, behind autograd and autocast, is the device.  Anything above it has to hear of the operator: an active
// mode (TorchDispatchMode, functorch, the Python dispatcher), a tensor subclass, a functional or batched wrapper, a view with its negation pending.
bool eager(std::initializer_list<const Tensor*> tensors) {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet ks = tls.included_;
  for (const Tensor* t : tensors)
    if (t && t->defined()) ks = ks | t->key_set();
  ks = ks - tls.excluded_ - c10::autograd_dispatch_keyset_with_ADInplaceOrView - c10::autocast_dispatch_keyset -
       c10::DispatchKeySet(c10::DispatchKey::BackendSelect);
  return ks.highestPriorityTypeId() == c10::DispatchKey::CUDA;
}
const Tensor* tensor_of(const OptTensor& t) { return has(t) ? &*t : nullptr; }
void once(const char* what) { TORCH_CHECK(!c10::GradMode::is_enabled(), what, " can be differentiated once only (create_graph is not supported)"); }

// ---- int8_quantize --------------------------------------------------------------------------------------------------------------------
void check_quantize(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "int8_quantize: x must have rows, got ", x.sizes());
  code_of(x.scalar_type());
}
std::tuple<Tensor, Tensor> int8_quantize(const Tensor& x) {
  need_hip(x, "x");
  check_quantize(x);
  const c10::DeviceGuard guard(x.device());
  const int64_t K = x.size(-1), M = x.numel() / K, ldq = (K + 127) / 128 * 128;
  Tensor r = x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= K ? x : x.reshape({M, K}).contiguous();
  Tensor q = at::empty({M, ldq}, x.options().dtype(at::kChar)), scale = at::empty({M}, x.options().dtype(at::kFloat));
  // (the pitch of a single row means nothing and may be anything)
  check_rc(lyc_int8_quantize(r.const_data_ptr(), M > 1 ? r.stride(0) : K, q.mutable_data_ptr<int8_t>(), ldq, scale.mutable_data_ptr<float>(), M, K,
                             code_of(x.scalar_type()), stream_of(x)), "int8_quantize");
  auto lead = x.sizes().vec();
  lead.pop_back();
  auto shape = lead;
  shape.push_back(ldq);
  return {q.view(shape).narrow(-1, 0, K), scale.view(lead)};
}
std::tuple<Tensor, Tensor> int8_quantize_meta(const Tensor& x) {
  check_quantize(x);
  const int64_t K = x.size(-1);
  auto lead = x.sizes().vec();
  lead.pop_back();
  return {at::empty(with_last(x, (K + 127) / 128 * 128), x.options().dtype(at::kChar)).narrow(-1, 0, K), at::empty(lead, x.options().dtype(at::kFloat))};
}

// ---- int8_matmul --------------------------------------------------------------------------------------------------------------------------
void check_matmul(const Tensor& aq, const Tensor& bq) {
  TORCH_CHECK(aq.dim() >= 1 && aq.scalar_type() == at::kChar, "int8_matmul: a must be int8 rows, got ", aq.sizes(), " ", aq.scalar_type());
  check_w8(bq, "int8_matmul");
  TORCH_CHECK(aq.size(-1) == bq.size(1), "int8_matmul: a has rows of ", aq.size(-1), ", b of ", bq.size(1));
}
Tensor int8_matmul(const Tensor& aq, const Tensor& sa, const Tensor& bq, const Tensor& sb, const OptTensor& bias, at::ScalarType dtype) {
  need_hip(aq, "a");
  check_matmul(aq, bq);
  on_device_of(aq, sa, "the scale of a");
  on_device_of(aq, bq, "b");
  on_device_of(aq, sb, "the scale of b");
  on_device_of(aq, bias, "bias");
  const int code = code_of(dtype);
  const c10::DeviceGuard guard(aq.device());
  const int64_t K = bq.size(1), N = bq.size(0), M = aq.numel() / K;
  // rows of one pitch stay where they are ([.., K] slices of what int8_quantize returns)
  Tensor a = rows8(aq.dim() == 2 ? aq : aq.reshape({M, K}), true), b = rows8(bq, false);
  Tensor fa = scales_of(sa, M, "the scale of a"), fb = scales_of(sb, N, "the scale of b");
  OptTensor bi = bias_of(bias, N, dtype);
  Tensor y = at::empty(with_last(aq, N), aq.options().dtype(dtype));
  Tensor ws = scratch(aq, lyc_int8_matmul_workspace_bytes(M, N, K, code), "int8_matmul");
  check_rc(lyc_int8_matmul(a.const_data_ptr<int8_t>(), a.stride(0), fa.const_data_ptr<float>(), b.const_data_ptr<int8_t>(), b.stride(0),
                           fb.const_data_ptr<float>(), dptr(bi), bias_f32(bi), nullptr, y.mutable_data_ptr(), mptr(ws), M, N, K, code, stream_of(aq)), "int8_matmul");
  return y;
}
Tensor int8_matmul_meta(const Tensor& aq, const Tensor& sa, const Tensor& bq, const Tensor& sb, const OptTensor& bias, at::ScalarType dtype) {
  check_matmul(aq, bq);
  code_of(dtype);
  return at::empty(with_last(aq, bq.size(0)), aq.options().dtype(dtype));
}

// ---- int8_linear --------------------------------------------------------------------------------------------------------------------------
Tensor int8_linear(const Tensor& x, const Tensor& wq, const Tensor& sw, const OptTensor& bias, const OptTensor& base) {
  need_hip(x, "x");
  check_w8(wq, "int8_linear");
  const int64_t N = wq.size(0), K = wq.size(1);
  check_act_x(x, K, "int8_linear");
  on_device_of(x, wq, "the weight");
  on_device_of(x, sw, "the scale");
  on_device_of(x, bias, "bias");
  on_device_of(x, base, "base");
  const c10::DeviceGuard guard(x.device());
  const int code = code_of(x.scalar_type());
  Tensor r = rows_of(x, K), w = rows8(wq, false), s = scales_of(sw, N, "the scale");
  OptTensor bi = bias_of(bias, N, x.scalar_type()), ba = base_of(base, x, N);
  const int64_t M = r.size(0);
  Tensor y = at::empty(with_last(x, N), x.options());
  Tensor ws = scratch(x, lyc_int8_linear_workspace_bytes(M, N, K, code, 0), "int8_linear");
  check_rc(lyc_int8_linear_fwd(r.const_data_ptr(), w.const_data_ptr<int8_t>(), w.stride(0), s.const_data_ptr<float>(), dptr(bi), bias_f32(bi), dptr(ba),
                               y.mutable_data_ptr(), mptr(ws), M, N, K, code, stream_of(x)), "int8_linear");
  return y;
}
Tensor int8_linear_meta(const Tensor& x, const Tensor& wq, const Tensor& sw, const OptTensor& bias, const OptTensor& base) {
  check_w8(wq, "int8_linear");
  check_act_x(x, wq.size(1), "int8_linear");
  return at::empty(with_last(x, wq.size(0)), x.options());
}
Tensor int8_linear_bwd(const Tensor& g, const Tensor& wq, const Tensor& sw) {
  const c10::DeviceGuard guard(g.device());
  const int64_t N = wq.size(0), K = wq.size(1);
  const int code = code_of(g.scalar_type());
  Tensor r = rows_of(g, N), w = rows8(wq, false), s = scales_of(sw, N, "the scale");
  const int64_t M = r.size(0);
  Tensor dx = at::empty(with_last(g, K), g.options());
  Tensor ws = scratch(g, lyc_int8_linear_workspace_bytes(M, N, K, code, 1), "int8_linear backward");
  check_rc(lyc_int8_linear_bwd(r.const_data_ptr(), w.const_data_ptr<int8_t>(), w.stride(0), s.const_data_ptr<float>(), dx.mutable_data_ptr(),
                               mptr(ws), M, N, K, code, stream_of(g)), "int8_linear backward");
  return dx;
}
Tensor int8_linear_bwd_meta(const Tensor& g, const Tensor& wq, const Tensor& sw) { return at::empty(with_last(g, wq.size(1)), g.options()); }

struct Int8LinearFn : public torch::autograd::Function<Int8LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wq, const Tensor& sw, const OptTensor& bias, const OptTensor& base) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("lycoris_amd::int8_linear", "")
                         .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&)>();
    ctx->save_for_backward({wq, sw});  // not x: the layer is frozen
    ctx->saved_data["dt"] = (int64_t)x.scalar_type();
    ctx->saved_data["base"] = edge(base, 3 + has(bias));
    return eager({&x, &wq, &sw, tensor_of(bias), tensor_of(base)}) ? int8_linear(x, wq, sw, bias, base) : op.call(x, wq, sw, bias, base);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("int8_linear");
    variable_list out(5);
    if (!grads[0].defined()) return out;
    auto s = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("lycoris_amd::_int8_linear_backward", "")
                         .typed<Tensor(const Tensor&, const Tensor&, const Tensor&)>();
    Tensor g = grads[0].to((at::ScalarType)ctx->saved_data["dt"].toInt());
    if (ctx->needs_input_grad(0)) out[0] = eager({&g, &s[0], &s[1]}) ? int8_linear_bwd(g, s[0], s[1]) : op.call(g, s[0], s[1]);
    if (wanted(ctx, "base")) out[4] = g;
    return out;
  }
};
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return has(t) && t->requires_grad(); }
// A dual tensor need not require a gradient, so it has to be asked for by itself: passed below autograd, its tangent would be lost without a word.
void no_tangent(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative; an input carries a tangent");
}
// A leaf has one gradient accumulator for as long as any graph on it lives, bound to the stream of the first.  A backward pass captured on
// another stream while such an eager graph lives makes the engine synchronise the two streams, which destroys the capture, and the process with
// it when the capture ends.  Found out here, while it is still an error that can be caught.
void capture_safe(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs) {
    if (!t || !t->defined() || !t->is_cuda() || !t->requires_grad() || t->grad_fn()) continue;
    const auto current = c10::hip::getCurrentHIPStream(t->device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream.has_value() || stream->id() == current.id(), what, ": a graph is being captured while an eager autograd graph on one of the "
                "inputs, made on another stream, is alive; drop its outputs (or detach them) before the capture");
  }
}
Tensor int8_linear_autograd(const Tensor& x, const Tensor& wq, const Tensor& sw, const OptTensor& bias, const OptTensor& base) {
  TORCH_CHECK(!wants(sw) && !wants(bias), "int8_linear: the layer is frozen, its scale and bias cannot require a gradient");
  no_tangent({&x, &sw, tensor_of(bias), tensor_of(base)}, "int8_linear");
  if (eager({&x, &wq, &sw, tensor_of(bias), tensor_of(base)}) && !(c10::GradMode::is_enabled() && (wants(x) || wants(base)))) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return int8_linear(x, wq, sw, bias, base);
  }
  capture_safe({&x, tensor_of(base)}, "int8_linear");
  return Int8LinearFn::apply(x, wq, sw, bias, base);
}

// ---- gated_linear -------------------------------------------------------------------------------------------------------------------------
void check_gated(const Tensor& x, const Tensor& w, const OptTensor& sw, int64_t act) {
  TORCH_CHECK(w.dim() == 2 && w.size(0) > 0 && w.size(0) % 2 == 0 && w.size(1) > 0, "gated_linear: the weight must be [2 F, I], got ", w.sizes());
  check_act_x(x, w.size(1), "gated_linear");
  if (has(sw)) check_w8(w, "gated_linear");
  else TORCH_CHECK(w.scalar_type() == x.scalar_type(), "gated_linear: the weight is ", w.scalar_type(), ", the activation ", x.scalar_type(),
                   "; an int8 weight needs its scale");
  TORCH_CHECK(act >= 0 && act <= 2, "gated_linear: unknown activation ", act);
}
struct GatedArgs {
  Tensor w, s;
  const float* sw = nullptr;
  int64_t ldw;
  GatedArgs(const Tensor& w_, const OptTensor& sw_) {
    if (has(sw_)) {
      w = rows8(w_, false);
      s = scales_of(*sw_, w_.size(0), "the scale");
      sw = s.const_data_ptr<float>();
    } else {
      w = w_.contiguous();
      if (!aligned(w)) w = w.clone();
    }
    ldw = w.stride(0);
  }
};
// what the backward pass reads p from: 3 bytes an element for 16-bit activations, 4 for fp32
Tensor pre_of(const Tensor& x, int64_t M, int64_t N) {
  return at::empty({M * N * (x.scalar_type() == at::kFloat ? 4 : 3)}, x.options().dtype(at::kByte));
}
std::tuple<Tensor, Tensor> gated_fwd(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act,
                                     bool gate_first, bool keep) {
  need_hip(x, "x");
  check_gated(x, w, sw, act);
  on_device_of(x, w, "the weight");
  on_device_of(x, sw, "the scale");
  on_device_of(x, bias, "bias");
  on_device_of(x, base, "base");
  const c10::DeviceGuard guard(x.device());
  const int code = code_of(x.scalar_type());
  const int64_t F = w.size(0) / 2, I = w.size(1);
  GatedArgs a(w, sw);
  Tensor r = rows_of(x, I);
  OptTensor bi = bias_of(bias, 2 * F, x.scalar_type()), ba = base_of(base, x, 2 * F);
  const int64_t M = r.size(0);
  Tensor h = at::empty(with_last(x, F), x.options()), pre = pre_of(x, keep ? M : 0, 2 * F);
  Tensor ws = scratch(x, lyc_gated_linear_workspace_bytes(M, I, F, code, a.sw ? LYC_GATED_INT8 : 0), "gated_linear");
  check_rc(lyc_gated_linear_fwd(r.const_data_ptr(), a.w.const_data_ptr(), a.ldw, a.sw, dptr(bi), bias_f32(bi), dptr(ba), h.mutable_data_ptr(),
                                keep ? pre.mutable_data_ptr() : nullptr, mptr(ws), M, I, F, (int)act, gate_first, code, stream_of(x)),
           "gated_linear");
  return {h, pre};
}
Tensor gated_linear(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act, bool gate_first) {
  return std::get<0>(gated_fwd(x, w, sw, bias, base, act, gate_first, false));
}
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act,
                                         bool gate_first) {
  return gated_fwd(x, w, sw, bias, base, act, gate_first, true);
}
Tensor gated_linear_meta(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act, bool gate_first) {
  check_gated(x, w, sw, act);
  return at::empty(with_last(x, w.size(0) / 2), x.options());
}
std::tuple<Tensor, Tensor> gated_forward_meta(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act,
                                              bool gate_first) {
  return {gated_linear_meta(x, w, sw, bias, base, act, gate_first), pre_of(x, x.numel() / w.size(1), w.size(0))};
}
// (dbase [M, 2 F], dx, dw, dbias); what is not asked for comes back empty
std::tuple<Tensor, Tensor, Tensor, Tensor> gated_backward_meta(const Tensor& g, const Tensor& pre, const Tensor& x, const Tensor& w, const OptTensor& sw,
                                                               int64_t act, bool gate_first, bool dbase, bool dx, bool dw, bool dbias, bool dbias_f32) {
  auto e = [&](bool want, at::IntArrayRef shape) { return want ? at::empty(shape, g.options()) : at::empty({0}, g.options()); };
  return {e(dbase, with_last(g, w.size(0))), e(dx, with_last(g, w.size(1))), e(dw, w.sizes()),
          dbias ? at::empty({w.size(0)}, dbias_f32 ? g.options().dtype(at::kFloat) : g.options()) : e(false, {})};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> gated_backward(const Tensor& g, const Tensor& pre, const Tensor& x, const Tensor& w, const OptTensor& sw,
                                                          int64_t act, bool gate_first, bool dbase, bool dx, bool dw, bool dbias, bool dbias_f32) {
  const c10::DeviceGuard guard(g.device());
  const int code = code_of(g.scalar_type());
  const int64_t F = w.size(0) / 2, I = w.size(1);
  auto out = gated_backward_meta(g, pre, x, w, sw, act, gate_first, dbase, dx, dw, dbias, dbias_f32);
  Tensor gr = rows_of(g, F);
  const int64_t M = gr.size(0);
  if (M == 0) {
    if (dw) std::get<2>(out).zero_();
    if (dbias) std::get<3>(out).zero_();
    return out;
  }
  GatedArgs a(w, sw);
  Tensor xr = dw ? rows_of(x, I) : Tensor();
  const int flags = LYC_GATED_BACKWARD | (a.sw ? LYC_GATED_INT8 : 0) | (dbase ? LYC_GATED_DBASE : 0) | (dx ? LYC_GATED_DX : 0) | (dw ? LYC_GATED_DW : 0) |
                    (dbias ? LYC_GATED_DBIAS : 0);
  Tensor ws = scratch(g, lyc_gated_linear_workspace_bytes(M, I, F, code, flags), "gated_linear backward");
  auto p = [](bool want, const Tensor& t) { return want ? t.mutable_data_ptr() : nullptr; };
  check_rc(lyc_gated_linear_bwd(gr.const_data_ptr(), pre.const_data_ptr(), dw ? xr.const_data_ptr() : nullptr, a.w.const_data_ptr(), a.ldw, a.sw,
                                p(dbase, std::get<0>(out)), p(dx, std::get<1>(out)), p(dw, std::get<2>(out)), p(dbias, std::get<3>(out)),
                                mptr(ws), M, I, F, (int)act, gate_first, code | (dbias_f32 ? LYC_F32_DBIAS : 0), stream_of(g)), "gated_linear backward");
  return out;
}

struct GatedLinearFn : public torch::autograd::Function<GatedLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act,
                        bool gate_first) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("lycoris_amd::_gated_linear_forward", "")
                         .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, int64_t, bool)>();
    auto [h, pre] = eager({&x, &w, tensor_of(sw), tensor_of(bias), tensor_of(base)}) ? gated_forward(x, w, sw, bias, base, act, gate_first) : op.call(x, w, sw, bias, base, act, gate_first);
    // x is read by dw alone
    ctx->save_for_backward({pre, w.requires_grad() ? x : Tensor(), w, has(sw) ? *sw : Tensor()});
    ctx->saved_data["bias"] = edge(bias, 2 + has(sw));
    ctx->saved_data["base"] = edge(base, 2 + has(sw) + has(bias));
    ctx->saved_data["dt"] = (int64_t)x.scalar_type();
    ctx->saved_data["act"] = act;
    ctx->saved_data["gf"] = gate_first;
    ctx->saved_data["bdt"] = (int64_t)(has(bias) ? bias->scalar_type() : x.scalar_type());
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_linear");
    variable_list out(7);
    if (!grads[0].defined()) return out;
    auto s = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("lycoris_amd::_gated_linear_backward", "")
                         .typed<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, int64_t,
                                                                           bool, bool, bool, bool, bool, bool)>();
    const bool dx = ctx->needs_input_grad(0), dw = ctx->needs_input_grad(1), dbias = wanted(ctx, "bias"), dbase = wanted(ctx, "base");
    if (!(dx || dw || dbias || dbase)) return out;
    OptTensor sw = opt(s[3]);
    Tensor g = grads[0].to((at::ScalarType)ctx->saved_data["dt"].toInt());
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool gf = ctx->saved_data["gf"].toBool();
    const Tensor& xs = s[1].defined() ? s[1] : g;
    const auto bdt = (at::ScalarType)ctx->saved_data["bdt"].toInt();
    const bool df = bdt != g.scalar_type();  // the kernels read any other type of bias as fp32, and its gradient is the fp32 sum
    auto [b, x, w, bi] = eager({&g, &s[0], &xs, &s[2], tensor_of(sw)}) ? gated_backward(g, s[0], xs, s[2], sw, act, gf, dbase, dx, dw, dbias, df)
                                                                  : op.call(g, s[0], xs, s[2], sw, act, gf, dbase, dx, dw, dbias, df);
    if (dx) out[0] = x;
    if (dw) out[1] = w;
    if (dbias) out[3] = bi.to(bdt);
    if (dbase) out[4] = b;
    return out;
  }
};
Tensor gated_linear_autograd(const Tensor& x, const Tensor& w, const OptTensor& sw, const OptTensor& bias, const OptTensor& base, int64_t act, bool gate_first) {
  TORCH_CHECK(!wants(sw), "gated_linear: an 8-bit weight is frozen, its scale cannot require a gradient");
  no_tangent({&x, &w, tensor_of(sw), tensor_of(bias), tensor_of(base)}, "gated_linear");
  if (!c10::GradMode::is_enabled() || !(wants(x) || wants(w) || wants(bias) || wants(base))) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("lycoris_amd::gated_linear", "")
                         .typed<Tensor(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, int64_t, bool)>();
    return eager({&x, &w, tensor_of(sw), tensor_of(bias), tensor_of(base)}) ? gated_linear(x, w, sw, bias, base, act, gate_first) : op.call(x, w, sw, bias, base, act, gate_first);
  }
  capture_safe({&x, &w, tensor_of(bias), tensor_of(base)}, "gated_linear");
  return GatedLinearFn::apply(x, w, sw, bias, base, act, gate_first);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lycoris_amd, m) {
  m.def("int8_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_matmul(Tensor aq, Tensor a_scale, Tensor bq, Tensor b_scale, Tensor? bias, ScalarType dtype) -> Tensor");
  m.def("int8_linear(Tensor x, Tensor wq, Tensor w_scale, Tensor? bias=None, Tensor? base=None) -> Tensor");
  m.def("_int8_linear_backward(Tensor g, Tensor wq, Tensor w_scale) -> Tensor");
  m.def("gated_linear(Tensor x, Tensor weight, Tensor? weight_scale, Tensor? bias, Tensor? base, int act, bool gate_first) -> Tensor");
  m.def("_gated_linear_forward(Tensor x, Tensor weight, Tensor? weight_scale, Tensor? bias, Tensor? base, int act, bool gate_first) -> (Tensor, Tensor)");
  m.def("_gated_linear_backward(Tensor g, Tensor pre, Tensor x, Tensor weight, Tensor? weight_scale, int act, bool gate_first, bool dbase, bool dx, bool dw, "
        "bool dbias, bool dbias_f32) -> (Tensor, Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(lycoris_amd, CUDA, m) {
  m.impl("int8_quantize", int8_quantize);
  m.impl("int8_matmul", int8_matmul);
  m.impl("int8_linear", int8_linear);
  m.impl("_int8_linear_backward", int8_linear_bwd);
  m.impl("gated_linear", gated_linear);
  m.impl("_gated_linear_forward", gated_forward);
  m.impl("_gated_linear_backward", gated_backward);
}
TORCH_LIBRARY_IMPL(lycoris_amd, Meta, m) {
  m.impl("int8_quantize", int8_quantize_meta);
  m.impl("int8_matmul", int8_matmul_meta);
  m.impl("int8_linear", int8_linear_meta);
  m.impl("_int8_linear_backward", int8_linear_bwd_meta);
  m.impl("gated_linear", gated_linear_meta);
  m.impl("_gated_linear_forward", gated_forward_meta);
  m.impl("_gated_linear_backward", gated_backward_meta);
}
TORCH_LIBRARY_IMPL(lycoris_amd, Autograd, m) {
  m.impl("int8_linear", int8_linear_autograd);
  m.impl("gated_linear", gated_linear_autograd);
}
