// The layer's operators on torch tensors: checks, outputs, workspaces and autograd around the C ABI.
//
// In C++ because their host time counts: a decoding step's norm or rotary embedding runs for 3 to 4 us, and a training step
// of a short batch for 20, while a Python Function's way through autograd takes over 100 (measured, forward and backward of
// the rotary embedding: 118 us from Python).  Nothing is computed here; libnsa_b200.so does that.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/nsa_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- types, checks, launches
int code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return NSA_BF16;
    case at::kHalf: return NSA_FP16;
    case at::kFloat: return NSA_FP32;
    case at::kFloat8_e4m3fn: return NSA_FP8_E4M3;
    case at::kFloat8_e5m2: return NSA_FP8_E5M2;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t);
  }
  return -1;
}
at::ScalarType type_of(int64_t c) {
  return c == NSA_BF16 ? at::kBFloat16 : c == NSA_FP16 ? at::kHalf : c == NSA_FP8_E4M3 ? at::kFloat8_e4m3fn : c == NSA_FP8_E5M2 ? at::kFloat8_e5m2 : at::kFloat;
}
bool is16(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool is8(const Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2; }
bool is_real(const Tensor& t) { return is16(t) || t.scalar_type() == at::kFloat; }

void need_cuda(const Tensor& t) { TORCH_CHECK(t.is_cuda(), "nsa_from_scratch_b200 kernels need CUDA tensors (there is no CPU path)"); }
// `t` lies where x does and is dense
void operand(const Tensor& t, const char* name, const Tensor& x) {
  need_cuda(t);
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the first operand on ", x.device());
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " is not contiguous");
}
void first(const Tensor& x, const char* name) {
  need_cuda(x);
  TORCH_CHECK_VALUE(x.is_contiguous(), name, " is not contiguous");
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const optional<Tensor>& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
bool given(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
bool wants(const optional<Tensor>& t) { return given(t) && t->requires_grad(); }
// Forward-mode differentiation has no rules here: a tangent is refused, not dropped
bool tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool tangent(const optional<Tensor>& t) { return t.has_value() && tangent(*t); }
template <typename... T> void no_tangents(const char* what, const T&... t) {
  if (C10_UNLIKELY((tangent(t) || ...)) && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    TORCH_CHECK(false, what, ": forward-mode differentiation is not provided; gradients are those of backward()");
}
// a size that the kernels take
int32_t size32(int64_t n, const char* what) {
  TORCH_CHECK_VALUE(n <= NSA_MAX_SIZE, what, ": ", n, " is more than the kernels' 32-bit sizes hold");
  return (int32_t)n;
}
void ok(int rc, const char* what) { TORCH_CHECK(rc == NSA_OK, what, " failed (status ", rc, "): ", nsa_last_error()); }
nsa_stream_t stream(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }
// a new dense tensor beside `like`, without the dispatcher's way to it (0.3 us each; a rotary embedding makes three)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt)); }
Tensor fresh(const Tensor& like) { return fresh(like.sizes(), like.scalar_type(), like); }
// the workspace that a call asks for; lives until the call's launches are queued (the allocator orders reuse on the stream)
template <typename A> Tensor workspace(A& a, int64_t need, const char* what, const Tensor& like) {
  if (need < 0) ok((int)need, what);
  if (need == 0) return Tensor();
  Tensor ws = fresh({need}, at::kByte, like);
  a.ws = ws.data_ptr();
  a.ws_bytes = need;
  return ws;
}
// Bits of the tensor inputs whose gradients this backward is asked for; the inputs of bit i in `present` have an edge.
int64_t asked(AutogradContext* ctx, int64_t present) {
  int64_t bits = 0;
  size_t edge = 0;
  for (int i = 0; present >> i; ++i)
    if (present >> i & 1) bits |= (int64_t)ctx->needs_input_grad(edge++) << i;
  return bits;
}
// The results of a backward under create_graph: they refuse a second differentiation instead of passing for constants.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (auto& g : grads)
    if (g.defined()) some.push_back(g);
  auto guard = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int)some.size());
  for (auto& g : some) g = g.detach().set_requires_grad(true);
  some = (*guard)(std::move(some));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = some[i++];
  return grads;
}

// ---------------------------------------------------------------- norm
nsa_norm_args check_norm(const Tensor& x, const Tensor& w, const optional<Tensor>& res, double eps, const char* what) {
  first(x, "x");
  operand(w, "weight", x);
  TORCH_CHECK_TYPE(is_real(x), what, ": x must be bf16, fp16 or fp32, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 1 && w.size(0) == x.size(-1), what, ": weight shape ", w.sizes(), " does not match x ", x.sizes());
  TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, what, ": weight must have x's dtype or fp32, got ", w.scalar_type(), " beside ",
                   x.scalar_type());
  nsa_norm_args a = {};
  a.hidden = size32(x.size(-1), what);
  a.rows = a.hidden ? x.numel() / a.hidden : 0;
  a.x_dtype = a.res_dtype = a.y_dtype = code(x.scalar_type());
  a.w_dtype = code(w.scalar_type());
  a.eps = (float)eps;
  a.x = x.data_ptr();
  a.weight = w.data_ptr();
  if (given(res)) {
    operand(*res, "residual", x);
    TORCH_CHECK_VALUE(res->sizes() == x.sizes(), what, ": residual shape ", res->sizes(), " does not match x ", x.sizes());
    TORCH_CHECK_TYPE(res->scalar_type() == x.scalar_type() || res->scalar_type() == at::kFloat, what, ": residual must have x's dtype or fp32, got ", res->scalar_type(),
                     " beside ", x.scalar_type());
    a.res_dtype = code(res->scalar_type());
    a.residual = res->data_ptr();
  }
  return a;
}
// launches with outputs y (and scale, rstd) given; returns h
Tensor launch_norm(nsa_norm_args a, const Tensor& x, const optional<Tensor>& res, const Tensor& y, const Tensor& scale, const Tensor& rstd) {
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor h;
  if (given(res)) h = fresh(*res);
  a.y = y.data_ptr();
  a.h = ptr(h);
  a.scale = (float*)ptr(scale);
  a.rstd = (float*)ptr(rstd);
  ok(nsa_rms_norm(&a, stream(x)), "nsa_rms_norm");
  return h;
}

struct RmsNorm : Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const optional<Tensor>& res, double eps) {
    const nsa_norm_args a = check_norm(x, w, res, eps, "rms_norm");
    const Tensor y = fresh(x), rstd = fresh({a.rows}, at::kFloat, x);
    const Tensor h = launch_norm(a, x, res, y, Tensor(), rstd);
    ctx->save_for_backward({h.defined() ? h : x, w, rstd});
    ctx->saved_data["flags"] = (int64_t)(code(x.scalar_type()) | (h.defined() ? 16 : 0));
    ctx->set_materialize_grads(false);
    return h.defined() ? variable_list{y, h} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1], &rstd = saved[2];
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const at::ScalarType xt = type_of(flags & 15);
    const bool has_stream = flags & 16;
    const c10::cuda::CUDAGuard guard(h.device());
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros(h.sizes(), h.options().dtype(xt));
    const Tensor dh = has_stream && grads[1].defined() ? grads[1].contiguous() : Tensor();
    const Tensor dx = fresh(h.sizes(), xt, h);
    const Tensor dres = has_stream && h.scalar_type() != xt ? fresh(h) : Tensor();
    const Tensor dw = ctx->needs_input_grad(1) ? fresh(w) : Tensor();
    nsa_norm_bwd_args a = {};
    a.dy = dy.data_ptr(); a.dh = ptr(dh); a.h = h.data_ptr(); a.weight = w.data_ptr(); a.rstd = (const float*)rstd.data_ptr();
    a.dx = dx.data_ptr(); a.dres = ptr(dres); a.dweight = ptr(dw);
    a.hidden = (int32_t)h.size(-1);
    a.rows = rstd.numel();
    a.x_dtype = code(xt); a.res_dtype = code(h.scalar_type()); a.w_dtype = code(w.scalar_type());
    const Tensor ws = workspace(a, nsa_rms_norm_bwd_ws_bytes(a.rows, a.hidden), "nsa_rms_norm_bwd", h);
    ok(nsa_rms_norm_bwd(&a, stream(h)), "nsa_rms_norm_bwd");
    // the same values reach x and the residual
    return first_order({dx, dw, has_stream ? (dres.defined() ? dres : dx) : Tensor(), Tensor()});
  }
};

variable_list rms_norm(const Tensor& x, const Tensor& w, const optional<Tensor>& res, double eps) {
  no_tangents("rms_norm", x, w, res);
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants(res))) return RmsNorm::apply(x, w, res, eps);
  const nsa_norm_args a = check_norm(x, w, res, eps, "rms_norm");
  const Tensor y = fresh(x);
  const Tensor h = launch_norm(a, x, res, y, Tensor(), Tensor());
  return h.defined() ? variable_list{y, h} : variable_list{y};
}

variable_list rms_norm_fp8(const Tensor& x, const Tensor& w, const optional<Tensor>& res, double eps, int64_t fmt) {
  no_tangents("rms_norm_fp8", x, w, res);
  at::NoGradGuard off;
  nsa_norm_args a = check_norm(x, w, res, eps, "rms_norm_fp8");
  a.y_dtype = (int32_t)fmt;
  const Tensor q = fresh(x.sizes(), type_of(fmt), x);
  const Tensor scale = fresh(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  const Tensor h = launch_norm(a, x, res, q, scale, Tensor());
  return h.defined() ? variable_list{q, scale, h} : variable_list{q, scale};
}

variable_list quantize_rows(const Tensor& x, int64_t fmt) {
  no_tangents("quantize_rows_to_fp8", x);
  at::NoGradGuard off;
  first(x, "x");
  TORCH_CHECK_TYPE(is_real(x) && x.dim() >= 1, "quantize_rows_to_fp8: x must be a bf16, fp16 or fp32 tensor of rows, got ", x.scalar_type());
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor q = fresh(x.sizes(), type_of(fmt), x);
  const Tensor scale = fresh(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  ok(nsa_quantize_rows_fp8(x.data_ptr(), q.data_ptr(), (float*)scale.data_ptr(), scale.numel(), size32(x.size(-1), "quantize_rows_to_fp8"), code(x.scalar_type()), (int)fmt,
                           stream(x)),
     "nsa_quantize_rows_fp8");
  return {q, scale};
}

// ---------------------------------------------------------------- rotary embedding
bool pitched(const Tensor& t) {
  const int64_t D = t.size(3);
  return (t.stride(3) == 1 || D == 1) && (t.stride(2) == D || t.size(2) == 1);
}
nsa_rope_axes_args check_rope(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pos, const Tensor& inv, at::IntArrayRef sections, int64_t dtype) {
  need_cuda(q);
  operand(pos, "positions", q);
  operand(inv, "inv_freq", q);
  TORCH_CHECK_VALUE(q.dim() == 4, "rope_axes_to_heads: q must be [B,T,H,D], got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3), n = (int64_t)sections.size();
  for (const Tensor* t : {&k, &v}) {
    need_cuda(*t);
    TORCH_CHECK_VALUE(t->device() == q.device(), "k and v must be where q is, on ", q.device());
    TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == B && t->size(1) == T && t->size(3) == D && t->size(2) == k.size(2), "rope_axes_to_heads: k/v shapes ", k.sizes(), "/",
                      v.sizes(), " do not match q ", q.sizes());
    TORCH_CHECK_TYPE(t->scalar_type() == q.scalar_type(), "rope_axes_to_heads: q, k and v must share a dtype (fp32, bf16 or fp16)");
  }
  TORCH_CHECK_TYPE(is_real(q), "rope_axes_to_heads: q, k and v must share a dtype (fp32, bf16 or fp16)");
  int64_t sum = 0, least = 0;
  for (const int64_t s : sections) { sum += s; least = std::min(least, s); }
  TORCH_CHECK_VALUE(D % 2 == 0 && n >= 1 && n <= 8 && least >= 0 && sum == D / 2, "rope_axes_to_heads: 1 to 8 sections that add up to D/2 = ", D / 2, " are needed, got ", sections);
  TORCH_CHECK_VALUE(pos.dim() == 3 && pos.size(0) == n && pos.size(1) == B && pos.size(2) == T && (pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong),
                    "rope_axes_to_heads: positions must be [", n, ",", B, ",", T, "] int32 or int64, got ", pos.sizes(), " ", pos.scalar_type());
  TORCH_CHECK_VALUE(inv.dim() == 1 && inv.size(0) == D / 2 && inv.scalar_type() == at::kDouble, "rope_axes_to_heads: inv_freq must be [", D / 2, "] fp64, got ", inv.sizes(), " ",
                    inv.scalar_type());
  TORCH_CHECK_VALUE(pitched(q) && pitched(k) && pitched(v), "q, k or v is not contiguous in its heads and columns");
  nsa_rope_axes_args a = {};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.positions = pos.data_ptr(); a.inv_freq = (const double*)inv.data_ptr();
  a.q_batch = q.stride(0); a.q_token = q.stride(1);
  a.k_batch = k.stride(0); a.k_token = k.stride(1);
  a.v_batch = v.stride(0); a.v_token = v.stride(1);
  a.B = size32(B, "rope_axes_to_heads"); a.T = size32(T, "rope_axes_to_heads");
  a.H = size32(q.size(2), "rope_axes_to_heads"); a.Hkv = size32(k.size(2), "rope_axes_to_heads"); a.D = size32(D, "rope_axes_to_heads");
  a.n_axes = (int32_t)n;
  for (int64_t i = 0; i < n; ++i) a.sections[i] = (int32_t)sections[i];
  a.pos64 = pos.scalar_type() == at::kLong;
  a.x_dtype = code(q.scalar_type());
  a.y_dtype = (int32_t)dtype;
  return a;
}
variable_list launch_rope(nsa_rope_axes_args a, const Tensor& like, at::ScalarType out) {
  const c10::cuda::CUDAGuard guard(like.device());
  const int64_t B = a.B, T = a.T, D = a.D;
  variable_list y(3);
  for (int i = 0; i < 3; ++i) {
    const int64_t h = i == 0 ? a.H : a.Hkv;
    y[i] = a.backward ? fresh({B, T, h, D}, out, like) : fresh({B, h, T, D}, out, like);
  }
  a.q_out = y[0].data_ptr(); a.k_out = y[1].data_ptr(); a.v_out = y[2].data_ptr();
  ok(nsa_rope_axes(&a, stream(like)), "nsa_rope_axes");
  return y;
}

struct RopeAxes : Function<RopeAxes> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pos, const Tensor& inv, at::IntArrayRef sections,
                               int64_t dtype) {
    const nsa_rope_axes_args a = check_rope(q, k, v, pos, inv, sections, dtype);
    ctx->save_for_backward({pos, inv});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["types"] = (int64_t)(a.x_dtype | (a.y_dtype << 4));
    return launch_rope(a, q, type_of(dtype));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const int64_t types = ctx->saved_data["types"].toInt();
    const Tensor dq = grads[0].contiguous(), dk = grads[1].contiguous(), dv = grads[2].contiguous();
    nsa_rope_axes_args a = {};
    a.q = dq.data_ptr(); a.k = dk.data_ptr(); a.v = dv.data_ptr();
    a.positions = saved[0].data_ptr(); a.inv_freq = (const double*)saved[1].data_ptr();
    a.B = (int32_t)dq.size(0); a.H = (int32_t)dq.size(1); a.T = (int32_t)dq.size(2); a.D = (int32_t)dq.size(3); a.Hkv = (int32_t)dk.size(1);
    a.n_axes = (int32_t)sections.size();
    for (size_t i = 0; i < sections.size(); ++i) a.sections[i] = (int32_t)sections[i];
    a.pos64 = saved[0].scalar_type() == at::kLong;
    a.x_dtype = (int32_t)(types & 15); a.y_dtype = (int32_t)(types >> 4);
    a.backward = 1;
    auto y = launch_rope(a, dq, type_of(a.x_dtype));
    return first_order({y[0], y[1], y[2], Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

variable_list rope_axes(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pos, const Tensor& inv, const std::vector<int64_t>& sections, int64_t dtype) {
  no_tangents("rope_axes_to_heads", q, k, v, inv);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) return RopeAxes::apply(q, k, v, pos, inv, at::IntArrayRef(sections), dtype);
  return launch_rope(check_rope(q, k, v, pos, inv, sections, dtype), q, type_of(dtype));
}

// ---------------------------------------------------------------- projections
// t, where it is given, is [lead..., last] (last < 0: [lead...]) of dtype
void rows_like(const optional<Tensor>& t, const char* name, at::IntArrayRef lead, int64_t last, const Tensor& x, at::ScalarType dtype, const char* what) {
  if (!given(t)) return;
  operand(*t, name, x);
  auto same = [&] {
    const size_t n = lead.size();
    if (t->scalar_type() != dtype || (size_t)t->dim() != n + (last >= 0) || t->sizes().slice(0, n) != lead) return false;
    return last < 0 || t->size(-1) == last;
  };
  if (same()) return;
  auto shape = lead.vec();
  if (last >= 0) shape.push_back(last);
  TORCH_CHECK_VALUE(false, what, ": ", name, " must be ", at::IntArrayRef(shape), " ", dtype, ", got ", t->sizes(), " ", t->scalar_type());
}
nsa_linear_args check_linear(const Tensor& x, const Tensor& w, const optional<Tensor>& bias, const optional<Tensor>& res, const optional<Tensor>& xs,
                             const optional<Tensor>& ws, int64_t act, int64_t y_dtype, const char* what) {
  first(x, "x");
  operand(w, "weight", x);
  if (given(xs)) {
    TORCH_CHECK_TYPE(is8(x) && w.scalar_type() == x.scalar_type(), what, ": x and weight must share an fp8 dtype, got ", x.scalar_type(), " and ", w.scalar_type());
  } else {
    TORCH_CHECK_TYPE(is16(x) && w.scalar_type() == x.scalar_type(), what, ": x and weight must both be bf16 or both fp16, got ", x.scalar_type(), " and ", w.scalar_type());
  }
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1) && w.numel() > 0, what, ": x ", x.sizes(), " does not match weight ", w.sizes());
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const at::ScalarType yt = type_of(y_dtype);
  rows_like(xs, "x_scale", lead, -1, x, at::kFloat, what);
  rows_like(ws, "w_scale", {}, w.size(0), x, at::kFloat, what);
  rows_like(bias, "bias", {}, w.size(0), x, yt, what);
  rows_like(res, "residual", lead, w.size(0), x, yt, what);
  nsa_linear_args a = {};
  a.x = x.data_ptr(); a.w = w.data_ptr(); a.bias = ptr(bias); a.residual = ptr(res); a.x_scale = (const float*)ptr(xs); a.w_scale = (const float*)ptr(ws);
  a.N = size32(w.size(0), what); a.K = size32(w.size(1), what); a.M = size32(x.numel() / w.size(1), what);
  a.dtype = code(x.scalar_type());
  a.y_dtype = (int32_t)y_dtype;
  a.act = (int32_t)act;
  return a;
}
Tensor launch_linear(nsa_linear_args a, const Tensor& x, Tensor* slope) {
  const c10::cuda::CUDAGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = a.N;
  const Tensor y = fresh(shape, type_of(a.y_dtype), x);
  a.y = y.data_ptr();
  if (slope != nullptr) {
    *slope = fresh(shape, at::kShort, x);
    a.slope = slope->data_ptr();
  }
  const Tensor ws = workspace(a, nsa_linear_ws_bytes(&a), "nsa_linear", x);
  ok(nsa_linear(&a, stream(x)), "nsa_linear");
  return y;
}

struct Linear : Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const optional<Tensor>& bias, const optional<Tensor>& res, int64_t act) {
    const nsa_linear_args a = check_linear(x, w, bias, res, {}, {}, act, code(x.scalar_type()), "linear");
    Tensor slope;
    const Tensor y = launch_linear(a, x, act != NSA_ACT_NONE && (x.requires_grad() || w.requires_grad() || wants(bias)) ? &slope : nullptr);
    ctx->save_for_backward({x, w, slope});
    ctx->saved_data["present"] = (int64_t)(3 | (given(bias) ? 4 : 0) | (given(res) ? 8 : 0));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
    const int64_t need = asked(ctx, ctx->saved_data["present"].toInt());
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor dy = grads[0].contiguous();
    Tensor dx, dw, db;
    if (need & 1) dx = fresh(x);
    if (need & 2) dw = fresh(w);
    if (need & 4) db = fresh({w.size(0)}, x.scalar_type(), x);
    if (need & 7) {
      nsa_linear_bwd_args a = {};
      a.dy = dy.data_ptr(); a.x = x.data_ptr(); a.w = w.data_ptr(); a.slope = ptr(slope);
      a.dx = ptr(dx); a.dw = ptr(dw); a.dbias = ptr(db);
      a.N = (int32_t)w.size(0); a.K = (int32_t)w.size(1); a.M = (int32_t)(x.numel() / w.size(1));
      a.dtype = code(x.scalar_type());
      a.has_act = slope.defined();
      const Tensor ws = workspace(a, nsa_linear_bwd_ws_bytes(&a), "nsa_linear_bwd", x);
      ok(nsa_linear_bwd(&a, stream(x)), "nsa_linear_bwd");
    }
    return first_order({dx, dw, db, need & 8 ? dy : Tensor(), Tensor()});
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const optional<Tensor>& bias, const optional<Tensor>& res, int64_t act) {
  no_tangents("linear", x, w, bias, res);
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants(bias) || wants(res))) return Linear::apply(x, w, bias, res, act);
  need_cuda(x);
  return launch_linear(check_linear(x, w, bias, res, {}, {}, act, is16(x) ? code(x.scalar_type()) : NSA_BF16, "linear"), x, nullptr);
}
Tensor linear_fp8(const Tensor& x, const Tensor& w, const Tensor& xs, const Tensor& ws, const optional<Tensor>& bias, const optional<Tensor>& res, int64_t act, int64_t dtype) {
  no_tangents("linear_fp8", xs, ws, bias, res);
  at::NoGradGuard off;
  return launch_linear(check_linear(x, w, bias, res, xs, ws, act, dtype, "linear_fp8"), x, nullptr);
}

// ---------------------------------------------------------------- gated feed-forward block
nsa_gated_mlp_args check_mlp(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const optional<Tensor>& res, int64_t act) {
  first(x, "x");
  operand(wg, "w_gate", x);
  operand(wu, "w_up", x);
  operand(wd, "w_down", x);
  const auto t = x.scalar_type();
  TORCH_CHECK_TYPE(is16(x) && wg.scalar_type() == t && wu.scalar_type() == t && wd.scalar_type() == t, "gated_mlp: x and the weights must all be bf16 or all fp16, got ", t, ", ",
                   wg.scalar_type(), ", ", wu.scalar_type(), ", ", wd.scalar_type());
  TORCH_CHECK_VALUE(wg.dim() == 2 && x.dim() >= 1 && x.size(-1) == wg.size(1) && wu.sizes() == wg.sizes() && wd.dim() == 2 && wd.size(0) == wg.size(1) &&
                        wd.size(1) == wg.size(0) && wg.numel() > 0,
                    "gated_mlp: x ", x.sizes(), " and weights ", wg.sizes(), ", ", wu.sizes(), ", ", wd.sizes(), " do not match");
  rows_like(res, "residual", x.sizes(), -1, x, t, "gated_mlp");
  nsa_gated_mlp_args a = {};
  a.x = x.data_ptr(); a.wg = wg.data_ptr(); a.wu = wu.data_ptr(); a.wd = wd.data_ptr(); a.residual = ptr(res);
  a.F = size32(wg.size(0), "gated_mlp"); a.N = size32(wg.size(1), "gated_mlp"); a.M = size32(x.numel() / wg.size(1), "gated_mlp");
  a.dtype = code(t);
  a.act = (int32_t)act;
  return a;
}
// kept: NULL, or what the backward needs (p, s and low hold bits, h numbers; rows padded to a multiple of 8)
Tensor launch_mlp(nsa_gated_mlp_args a, const Tensor& x, Tensor* kept) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = fresh(x);
  a.y = y.data_ptr();
  if (kept != nullptr) {
    for (int i = 0; i < 4; ++i) kept[i] = fresh({(int64_t)a.M, ((int64_t)a.F + 7) / 8 * 8}, i < 3 ? at::kShort : x.scalar_type(), x);
    a.p = kept[0].data_ptr(); a.s = kept[1].data_ptr(); a.low = kept[2].data_ptr(); a.h = kept[3].data_ptr();
  }
  const Tensor ws = workspace(a, nsa_gated_mlp_ws_bytes(&a), "nsa_gated_mlp", x);
  ok(nsa_gated_mlp(&a, stream(x)), "nsa_gated_mlp");
  return y;
}

struct GatedMlp : Function<GatedMlp> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const optional<Tensor>& res, int64_t act) {
    const nsa_gated_mlp_args a = check_mlp(x, wg, wu, wd, res, act);
    Tensor kept[4];
    const Tensor y = launch_mlp(a, x, x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad() ? kept : nullptr);
    ctx->save_for_backward({x, wg, wu, wd, kept[0], kept[1], kept[2], kept[3]});
    ctx->saved_data["present"] = (int64_t)(15 | (given(res) ? 16 : 0));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t need = asked(ctx, ctx->saved_data["present"].toInt());
    const c10::cuda::CUDAGuard guard(s[0].device());
    const Tensor dy = grads[0].contiguous();
    Tensor d[4];
    for (int i = 0; i < 4; ++i)
      if (need & (1 << i)) d[i] = fresh(s[i]);
    if (need & 15) {
      nsa_gated_mlp_bwd_args a = {};
      a.dy = dy.data_ptr(); a.x = s[0].data_ptr(); a.wg = s[1].data_ptr(); a.wu = s[2].data_ptr(); a.wd = s[3].data_ptr();
      a.p = s[4].data_ptr(); a.s = s[5].data_ptr(); a.low = s[6].data_ptr(); a.h = s[7].data_ptr();
      a.dx = ptr(d[0]); a.dwg = ptr(d[1]); a.dwu = ptr(d[2]); a.dwd = ptr(d[3]);
      a.F = (int32_t)s[1].size(0); a.N = (int32_t)s[1].size(1); a.M = (int32_t)(s[0].numel() / s[1].size(1));
      a.dtype = code(s[0].scalar_type());
      const Tensor ws = workspace(a, nsa_gated_mlp_bwd_ws_bytes(&a), "nsa_gated_mlp_bwd", s[0]);
      ok(nsa_gated_mlp_bwd(&a, stream(s[0])), "nsa_gated_mlp_bwd");
    }
    return first_order({d[0], d[1], d[2], d[3], need & 16 ? dy : Tensor(), Tensor()});
  }
};

Tensor gated_mlp(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const optional<Tensor>& res, int64_t act) {
  no_tangents("gated_mlp", x, wg, wu, wd, res);
  if (at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad() || wants(res)))
    return GatedMlp::apply(x, wg, wu, wd, res, act);
  return launch_mlp(check_mlp(x, wg, wu, wd, res, act), x, nullptr);
}

}  // namespace

PYBIND11_MODULE(_nsa_torch, m) {
  m.doc() = "The layer's operators on torch tensors (norm.py, rotary.py and projections.py are their public side)";
  m.attr("abi_version") = NSA_ABI_VERSION;       // of the structs that this module fills
  // torch's wrapper: its exception types, and the interpreter's lock is released meanwhile
  using torch::wrap_pybind_function_no_gil;
  m.def("rms_norm", wrap_pybind_function_no_gil(rms_norm));
  m.def("rms_norm_fp8", wrap_pybind_function_no_gil(rms_norm_fp8));
  m.def("quantize_rows", wrap_pybind_function_no_gil(quantize_rows));
  m.def("rope_axes", wrap_pybind_function_no_gil(rope_axes));
  m.def("linear", wrap_pybind_function_no_gil(linear));
  m.def("linear_fp8", wrap_pybind_function_no_gil(linear_fp8));
  m.def("gated_mlp", wrap_pybind_function_no_gil(gated_mlp));
}
