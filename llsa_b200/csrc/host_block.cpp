// Host path of the operators around the attention of a block: layer norm with modulation, projections with their epilogues, rotary positions over
// several axes.  As in host.cpp: one dispatcher operator each way with C++ autograd over the C ABI.
//
//   llsa_b200::layer_norm_fwd / layer_norm_bwd,  linear_fwd / linear_bwd,  rope_axes (its own backward)
#include "host_common.h"

namespace {

using namespace llsa_host;

// ------------------------------------------------------------------ checks and views
void same_device(const Tensor& x, std::initializer_list<Tensor> ts) {
  need_cuda(x);
  for (const Tensor& t : ts)
    if (t.defined()) {
      need_cuda(t);
      TORCH_CHECK(t.device() == x.device(), "llsa_b200: all operands must be on one device, got ", x.device(), " and ", t.device());
    }
}
void no_tangents(const char* what, std::initializer_list<Tensor> ts) {      // they would be dropped without a word
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "llsa_b200: no forward-mode derivative of ", what);
}
bool any_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// Whether the i-th of the operands that were given wants a gradient (an absent one has no edge), counted along the argument list
struct Edges {
  torch::autograd::AutogradContext* ctx;
  size_t next = 0;
  bool wants(const Tensor& t) { return t.defined() && ctx->needs_input_grad(next++); }
};
Tensor unit_columns(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
// A result laid out as x is, where that leaves the last dimension dense
Tensor like_rows(const Tensor& x) {
  Tensor y = at::empty_like(x);
  return y.size(-1) == 1 || y.stride(-1) == 1 ? y : at::empty(x.sizes(), x.options());
}
void check_param(const char* name, const Tensor& t, const Tensor& x, at::IntArrayRef shape) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), "llsa_b200: ", name, " must be float32 or of the input's type, got ",
                   t.scalar_type());
  TORCH_CHECK(t.sizes() == shape, "llsa_b200: ", name, " must be ", shape, ", got ", t.sizes());
}

// ------------------------------------------------------------------ layer norm
// [B, N, C] view of [..., C]; B is the first dimension
Tensor samples(const Tensor& x) {
  const int64_t C = x.size(-1);
  if (x.dim() == 1) return x.view({1, 1, C});
  if (x.dim() == 2) return x.unsqueeze(1);
  return x.dim() == 3 ? x : x.reshape({x.size(0), -1, C});
}

std::vector<Tensor> layer_norm_fwd(const Tensor& x_, const OptTensor& weight, const OptTensor& bias, const OptTensor& scale, const OptTensor& shift,
                                   double eps, bool want_stats) {
  const Tensor w = or_none(weight), b = or_none(bias), s = or_none(scale), t = or_none(shift);
  same_device(x_, {w, b, s, t});
  check_float({&x_});
  TORCH_CHECK(x_.dim() >= 1 && x_.size(-1) >= 1, "llsa_b200: layer_norm wants [..., C] with C >= 1, got ", x_.sizes());
  TORCH_CHECK(x_.dim() >= 2 || !(s.defined() || t.defined()), "llsa_b200: a scale or shift per sample wants [B, ..., C]");
  const int64_t C = x_.size(-1);
  check_param("weight", w, x_, {C});
  check_param("bias", b, x_, {C});
  check_param("scale", s, x_, {x_.size(0), C});
  check_param("shift", t, x_, {x_.size(0), C});
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.dim() > 3 ? x_.contiguous() : unit_columns(x_), y = like_rows(x);
  if (x.numel() == 0) return want_stats ? std::vector<Tensor>{y, at::empty({0}, x.options().dtype(at::kFloat))} : std::vector<Tensor>{y};
  const Tensor x3 = samples(x), y3 = samples(y);
  std::vector<Tensor> out = {y};
  LlsaTensor st;
  if (want_stats) {
    out.push_back(at::empty({x3.size(0) * x3.size(1) * 2}, x.options().dtype(at::kFloat)));
    st = packed(out[1].data_ptr(), LLSA_F32, {x3.size(0), x3.size(1), 2});
  }
  const LlsaTensor xd = desc(x3), yd = desc(y3);
  const Tensor p[4] = {w, b, s, t};
  Tensor keep[4];
  LlsaTensor pd[4];
  const LlsaTensor* pp[4] = {};
  for (int i = 0; i < 4; ++i)
    if (p[i].defined()) {
      keep[i] = unit_columns(p[i]);
      pd[i] = desc(keep[i]);
      pp[i] = &pd[i];
    }
  mark("layer_norm");
  ok(llsa_layer_norm_fwd(&xd, pp[0], pp[1], pp[2], pp[3], (float) eps, &yd, want_stats ? &st : nullptr, at::cuda::getCurrentCUDAStream(x.device().index())),
     "layer_norm_fwd");
  mark("end");
  return out;
}

// want: 1 weight, 2 bias, 4 scale, 8 shift.  Returns dx and the gradients asked for, in that order; shift's gradient is of shift_type, which is given where the
// forward had a shift.
std::vector<Tensor> layer_norm_bwd(const Tensor& dy_, const Tensor& x_, const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
                                   const Tensor& stats, int64_t want, std::optional<at::ScalarType> shift_type, at::ScalarType bias_type) {
  const Tensor w = or_none(weight), b = or_none(bias), s = or_none(scale);
  same_device(x_, {dy_, w, b, s, stats});
  check_float({&x_, &dy_});
  TORCH_CHECK(dy_.sizes() == x_.sizes(), "llsa_b200.layer_norm_bwd: dy must be ", x_.sizes(), ", got ", dy_.sizes());
  const int64_t C = x_.size(-1);
  check_param("weight", w, x_, {C});
  check_param("bias", b, x_, {C});
  check_param("scale", s, x_, {x_.size(0), C});
  TORCH_CHECK(s.defined() || !(want & 4), "llsa_b200.layer_norm_bwd: scale is missing");
  TORCH_CHECK(shift_type || !(want & 8), "llsa_b200.layer_norm_bwd: shift's type is missing");
  const c10::cuda::CUDAGuard guard(x_.device());
  const at::ScalarType types[4] = {w.defined() ? w.scalar_type() : at::kFloat, bias_type, s.defined() ? s.scalar_type() : at::kFloat, shift_type.value_or(at::kFloat)};
  const bool empty = x_.numel() == 0;
  Tensor dx = at::empty(x_.sizes(), x_.options());
  std::vector<Tensor> out = {dx};
  LlsaTensor gd[4], part;
  const LlsaTensor* gp[4] = {};
  for (int i = 0; i < 4; ++i)
    if (want >> i & 1) {
      const at::TensorOptions o = x_.options().dtype(types[i]);
      const std::vector<int64_t> shape = i < 2 ? std::vector<int64_t>{C} : std::vector<int64_t>{x_.size(0), C};
      out.push_back(empty ? at::zeros(shape, o) : at::empty(shape, o));
      gd[i] = desc(out.back());
      gp[i] = &gd[i];
    }
  if (empty) return out;
  // All rows in one where nothing is per sample: by what the forward had, not by what is asked for, so that a gradient's sums are over the same parts, and its
  // bits the same, whichever others are asked for.  The library goes by samples for a scale or a gradient of the shift: one that nobody asked for goes to scratch.
  // dx alone depends on neither, where its rows are those of one matrix.
  const bool per_sample = s.defined() || shift_type;
  auto one_matrix = [](const Tensor& t) { return t.size(0) == 1 || (t.size(1) > 1 && t.stride(0) == t.size(1) * t.stride(1)); };
  auto view = [&](const Tensor& t) { return per_sample ? samples(t) : t.reshape({1, -1, C}); };
  const Tensor x = view(unit_columns(x_)), dy = view(unit_columns(dy_)), dx3 = view(dx);
  TORCH_CHECK(stats.is_contiguous() && stats.numel() == x.size(0) * x.size(1) * 2 && stats.scalar_type() == at::kFloat,
              "llsa_b200.layer_norm_bwd: `stats` is not from the matching layer_norm_fwd");
  const LlsaTensor xd = desc(x), dyd = desc(dy), dxd = desc(dx3), st = packed(stats.data_ptr(), LLSA_F32, {x.size(0), x.size(1), 2});
  const Tensor p[3] = {w, b, s};
  Tensor keep[3], partial, unasked;
  LlsaTensor pd[3];
  const LlsaTensor* pp[3] = {};
  for (int i = 0; i < 3; ++i)
    if (p[i].defined()) {
      keep[i] = unit_columns(p[i]);
      pd[i] = desc(keep[i]);
      pp[i] = &pd[i];
    }
  if (per_sample && !s.defined() && !(want & 8) && (want || !one_matrix(x) || !one_matrix(dy))) {
    unasked = at::empty({x.size(0), C}, x.options().dtype(at::kFloat));
    gd[3] = desc(unasked);
    gp[3] = &gd[3];
  }
  const bool sums = want || unasked.defined();
  if (sums) {
    partial = at::empty({llsa_layer_norm_bwd_partial_elems(x.size(0), x.size(1), C, per_sample)}, x.options().dtype(at::kFloat));
    part = desc(partial);
  }
  mark("layer_norm_bwd");
  ok(llsa_layer_norm_bwd(&dyd, &xd, pp[0], pp[1], pp[2], &st, &dxd, gp[0], gp[1], gp[2], gp[3], sums ? &part : nullptr,
                         at::cuda::getCurrentCUDAStream(x.device().index())),
     "layer_norm_bwd");
  mark("end");
  return out;
}

// ------------------------------------------------------------------ projection
// Room for a matrix whose rows start on 16-byte boundaries
Tensor padded(std::array<int64_t, 2> shape, const Tensor& like) {
  const int64_t per = 16 / like.element_size(), ld = (shape[1] + per - 1) / per * per;
  return at::empty_strided(shape, {ld, 1}, like.options());
}

// [M, C] with unit column stride and, for bf16, rows on 16-byte boundaries where `aligned` (a copy in padded rows where the tensor has none)
Tensor matrix(const Tensor& t, int64_t M, int64_t C, bool aligned) {
  const Tensor m = t.reshape({M, C});
  const int64_t per = 16 / m.element_size();
  const bool rows = (C == 1 || m.stride(1) == 1) && (M == 1 || m.stride(0) >= C);
  const bool fits = !aligned || m.scalar_type() != at::kBFloat16 || ((uintptr_t) m.data_ptr() % 16 == 0 && (M == 1 || m.stride(0) % per == 0));
  if (rows && fits) return m;
  Tensor c = aligned ? padded({M, C}, m) : at::empty({M, C}, m.options());
  c.copy_(m);
  return c;
}

// A vector, dense and on a 16-byte boundary
Tensor aligned_vector(const Tensor& t) {
  const Tensor c = cont(t);
  return (uintptr_t) c.data_ptr() % 16 ? c.clone() : c;
}

struct Shape {
  int64_t M, K, F, B;
  Shape(const Tensor& x, const Tensor& w, const Tensor& gate) {
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "llsa_b200: linear wants x [..., K] and weight [F, K], got ", x.sizes(), " and ",
                w.sizes());
    K = w.size(1);
    F = w.size(0);
    TORCH_CHECK(K >= 1 && F >= 1, "llsa_b200: linear wants at least one feature on either side, got ", w.sizes());
    M = x.numel() / K;
    B = gate.defined() ? x.size(0) : 1;
    TORCH_CHECK(!gate.defined() || (x.dim() >= 2 && gate.dim() == 2 && gate.size(0) == B && gate.size(1) == F),
                "llsa_b200: gate must be [B, F] with x [B, ..., K]");
  }
};
// What the library says (llsa_linear_keeps_product), from sizes alone
bool keeps_product(const Shape& s, at::ScalarType type, int64_t act, bool gate) {
  if (s.M == 0) return false;
  const int t = dtype_code(type);
  char* at = (char*) 256;      // no memory is looked at
  const LlsaTensor x = packed(at, t, {s.M, (s.K + 7) / 8 * 8}), w = packed(at, t, {s.F, (s.K + 7) / 8 * 8}), g = packed(at, t, {s.B, s.F});
  LlsaTensor xk = x, wk = w;
  xk.shape[1] = wk.shape[1] = s.K;
  LlsaLinearArgs a;
  memset(&a, 0, sizeof(a));
  a.x = &xk; a.weight = &wk; a.activation = (int32_t) act;
  if (gate) a.gate = &g;
  const int keeps = llsa_linear_keeps_product(&a);
  TORCH_CHECK(keeps >= 0, "llsa_b200.linear_fwd failed: ", llsa_last_error_string());
  return keeps;
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

LlsaLinearArgs linear_args(int64_t act, const Status& status) {
  LlsaLinearArgs a;
  memset(&a, 0, sizeof(a));
  a.activation = (int32_t) act;
  a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  a.status = status.ptr();
  return a;
}

// Rows that are no multiple of 16 bytes cost a copy of x and the weight, which a backward wants as well.  [y], then with want_pre z, with want_copies and such rows the
// copies of x [M, K] and of the weight.
bool rows_want_copies(const Tensor& x, int64_t K) { return x.scalar_type() == at::kBFloat16 && K % 8; }
std::vector<Tensor> linear_fwd(const Tensor& x_, const Tensor& w_, const OptTensor& bias, const OptTensor& residual, const OptTensor& gate, int64_t act,
                               bool want_pre, bool want_copies) {
  const Tensor b_ = or_none(bias), r_ = or_none(residual), g_ = or_none(gate);
  same_device(x_, {w_, b_, r_, g_});
  check_float({&x_, &w_});
  for (const Tensor& t : {b_, r_, g_})
    if (t.defined()) check_float({&x_, &t});
  const Shape s(x_, w_, g_);
  TORCH_CHECK(!b_.defined() || (b_.dim() == 1 && b_.size(0) == s.F), "llsa_b200: bias must be [F]");
  const std::vector<int64_t> shape = with_last(x_, s.F);
  TORCH_CHECK(!r_.defined() || r_.sizes() == at::IntArrayRef(shape), "llsa_b200: residual must be ", at::IntArrayRef(shape));
  TORCH_CHECK(!g_.defined() || r_.defined(), "llsa_b200: a gate goes with a residual");
  TORCH_CHECK(!g_.defined() || act == LLSA_ACT_NONE, "llsa_b200: a gate goes with no activation");
  const c10::cuda::CUDAGuard guard(x_.device());
  std::vector<Tensor> out = {at::empty(shape, x_.options())};
  const bool keep = want_pre && keeps_product(s, x_.scalar_type(), act, g_.defined());
  if (want_pre) out.push_back(at::empty({keep ? s.M : 0, s.F}, x_.options()));
  if (s.M == 0) {
    if (want_copies && rows_want_copies(x_, s.K)) {
      out.push_back(padded({s.M, s.K}, x_));
      out.push_back(padded({s.F, s.K}, x_).copy_(w_));
    }
    return out;
  }
  const Tensor x = matrix(x_, s.M, s.K, true), w = matrix(w_, s.F, s.K, true), y = out[0].view({s.M, s.F});
  const LlsaTensor xd = desc(x), wd = desc(w), yd = desc(y);
  const Status status(x);
  LlsaLinearArgs a = linear_args(act, status);
  a.x = &xd; a.weight = &wd; a.y = &yd;
  Tensor b, r, g;
  LlsaTensor bd, rd, gd, pd;
  if (b_.defined()) { b = aligned_vector(b_); bd = desc(b); a.bias = &bd; }
  if (r_.defined()) { r = matrix(r_, s.M, s.F, false); rd = desc(r); a.residual = &rd; }
  if (g_.defined()) { g = unit_columns(g_); gd = desc(g); a.gate = &gd; }
  if (keep) { pd = desc(out[1]); a.pre = &pd; }
  mark("linear");
  ok(llsa_linear_fwd(&a, at::cuda::getCurrentCUDAStream(x.device().index())), "linear_fwd");
  mark("end");
  status.check("linear_fwd");
  if (want_copies && rows_want_copies(x_, s.K)) {      // an output must not be an input, such as rows that came padded
    out.push_back(x.is_alias_of(x_) ? padded({s.M, s.K}, x_).copy_(x) : x);
    out.push_back(w.is_alias_of(w_) ? padded({s.F, s.K}, x_).copy_(w) : w);
  }
  return out;
}

// want: 1 x, 2 weight, 4 bias, 8 gate; the gradients asked for, in that order
std::vector<Tensor> linear_bwd(const Tensor& dy_, const Tensor& x_, const Tensor& w_, const OptTensor& bias, const OptTensor& pre, const OptTensor& gate,
                               const OptTensor& x_copy, const OptTensor& w_copy, int64_t act, int64_t want) {
  const Tensor b_ = or_none(bias), p_ = or_none(pre), g_ = or_none(gate);
  same_device(x_, {dy_, w_, b_, p_, g_, or_none(x_copy), or_none(w_copy)});
  check_float({&x_, &w_, &dy_});
  for (const Tensor& t : {b_, p_, g_})
    if (t.defined()) check_float({&x_, &t});
  const Shape s(x_, w_, g_);
  TORCH_CHECK(dy_.sizes() == at::IntArrayRef(with_last(x_, s.F)), "llsa_b200.linear_bwd: dy must be ", at::IntArrayRef(with_last(x_, s.F)), ", got ",
              dy_.sizes());
  TORCH_CHECK(g_.defined() || !(want & 8), "llsa_b200.linear_bwd: gate is missing");
  const c10::cuda::CUDAGuard guard(x_.device());
  auto room = [&](std::vector<int64_t> shape) { return s.M ? at::empty(shape, x_.options()) : at::zeros(shape, x_.options()); };
  std::vector<Tensor> out;
  Tensor dx, dw, db, dg;
  if (want & 1) out.push_back(dx = room(x_.sizes().vec()));
  if (want & 2) out.push_back(dw = room({s.F, s.K}));
  if (want & 4) out.push_back(db = room({s.F}));
  if (want & 8) out.push_back(dg = room({s.B, s.F}));
  if (s.M == 0 || !want) return out;
  const Tensor x = matrix(x_copy ? *x_copy : x_, s.M, s.K, true), w = matrix(w_copy ? *w_copy : w_, s.F, s.K, true);
  const bool long_samples = g_.defined() && !keeps_product(s, x_.scalar_type(), act, true);
  const Tensor dy = matrix(dy_, s.M, s.F, long_samples);
  const Status status(x);
  LlsaLinearArgs a = linear_args(act, status);
  const LlsaTensor xd = desc(x), wd = desc(w), dyd = desc(dy);
  a.x = &xd; a.weight = &wd; a.dy = &dyd;
  Tensor b, g;
  LlsaTensor bd, gd, pd, o[4];
  if (b_.defined()) {
    TORCH_CHECK(b_.dim() == 1 && b_.size(0) == s.F, "llsa_b200: bias must be [F]");
    b = aligned_vector(b_);
    bd = desc(b);
    a.bias = &bd;
  }
  if (g_.defined()) { g = unit_columns(g_); gd = desc(g); a.gate = &gd; }
  if (p_.defined() && p_.numel()) {
    TORCH_CHECK(p_.dim() == 2 && p_.size(0) == s.M && p_.size(1) == s.F && p_.is_contiguous(), "llsa_b200.linear_bwd: `pre` is not from the matching linear_fwd");
    pd = desc(p_);
    a.pre = &pd;
  }
  if (want & 1) { o[0] = desc(dx.view({s.M, s.K})); a.dx = &o[0]; }
  if (want & 2) { o[1] = desc(dw); a.dweight = &o[1]; }
  if (want & 4) { o[2] = desc(db); a.dbias = &o[2]; }
  if (want & 8) { o[3] = desc(dg); a.dgate = &o[3]; }
  a.workspace_bytes = llsa_linear_bwd_workspace_bytes(&a);
  TORCH_CHECK(a.workspace_bytes >= 0, "llsa_b200.linear_bwd failed: ", llsa_last_error_string());
  const Tensor ws = byte_buffer(a.workspace_bytes, x);
  a.workspace = a.workspace_bytes ? ws.data_ptr() : nullptr;
  mark("linear_bwd");
  ok(llsa_linear_bwd(&a, at::cuda::getCurrentCUDAStream(x.device().index())), "linear_bwd");
  mark("end");
  status.check("linear_bwd");
  return out;
}

// ------------------------------------------------------------------ rotary positions
Tensor rope_axes(const Tensor& x_, const Tensor& positions, at::IntArrayRef axes_dims, double theta, bool inverse) {
  same_device(x_, {positions});
  check_float({&x_});
  TORCH_CHECK(x_.dim() == 4, "llsa_b200: rope_axes wants x [B,H,N,D], got ", x_.sizes());
  const at::ScalarType pt = positions.scalar_type();
  TORCH_CHECK_TYPE(pt == at::kInt || pt == at::kLong || pt == at::kFloat, "llsa_b200: positions must be int32, int64 or float32, got ", pt);
  TORCH_CHECK(axes_dims.size() >= 1 && axes_dims.size() <= 4, "llsa_b200: rope_axes wants 1 to 4 axes, got ", axes_dims.size());
  const int64_t A = (int64_t) axes_dims.size();
  TORCH_CHECK((positions.dim() == 2 || (positions.dim() == 3 && positions.size(0) == x_.size(0))) && positions.size(-2) == x_.size(2) && positions.size(-1) == A,
              "llsa_b200: positions must be [N, A] or [B, N, A] with N = ", x_.size(2), ", A = ", A, ", got ", positions.sizes());
  int32_t dims[4];
  int64_t sum = 0;
  for (int64_t a = 0; a < A; ++a) {
    TORCH_CHECK(axes_dims[a] >= 2 && axes_dims[a] % 2 == 0 && axes_dims[a] <= 512, "llsa_b200: the channels of an axis are a positive even number, got ", axes_dims[a]);
    dims[a] = (int32_t) axes_dims[a];
    sum += axes_dims[a];
  }
  TORCH_CHECK(sum == x_.size(3), "llsa_b200: the axes have ", sum, " channels together, x has ", x_.size(3));
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = unit_columns(x_), y = like_rows(x), pos = unit_columns(positions);
  if (x.numel() == 0) return y;
  const LlsaTensor xd = desc(x), yd = desc(y), pd = desc(pos);
  mark("rope_axes");
  ok(llsa_rope_axes(&xd, &pd, (int) A, dims, theta, inverse, &yd, at::cuda::getCurrentCUDAStream(x.device().index())), "rope_axes");
  mark("end");
  return y;
}

// ------------------------------------------------------------------ autograd
template <typename Sig>
const c10::TypedOperatorHandle<Sig>& op(const char* name) {      // once per signature: each operator here has its own
  static const auto handle = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<Sig>();
  return handle;
}
using NormFwd = std::vector<Tensor>(const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, double, bool);
using NormBwd = std::vector<Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const Tensor&, int64_t,
                                    std::optional<at::ScalarType>, at::ScalarType);
using LinearFwd = std::vector<Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, int64_t, bool, bool);
using LinearBwd = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                      const OptTensor&, int64_t, int64_t);
using Rope = Tensor(const Tensor&, const Tensor&, at::IntArrayRef, double, bool);
const auto& norm_fwd_op() { return op<NormFwd>("llsa_b200::layer_norm_fwd"); }
const auto& norm_bwd_op() { return op<NormBwd>("llsa_b200::layer_norm_bwd"); }
const auto& linear_fwd_op() { return op<LinearFwd>("llsa_b200::linear_fwd"); }
const auto& linear_bwd_op() { return op<LinearBwd>("llsa_b200::linear_bwd"); }
const auto& rope_op() { return op<Rope>("llsa_b200::rope_axes"); }

// A backward operator, recorded where its caller differentiates again: its own node then raises
template <typename F>
auto below_unless_recorded(F&& call) {
  if (at::GradMode::is_enabled()) return call();
  at::AutoDispatchBelowADInplaceOrView below;
  return call();
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, const OptTensor& s,
                               const OptTensor& t, double eps) {
    variable_list out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      out = norm_fwd_op().call(x, w, b, s, t, eps, true);
    }
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1]});
    ctx->save_for_backward({x, or_none(w), or_none(b), or_none(s), out[1]});
    ctx->saved_data["shift"] = t.has_value();
    ctx->saved_data["shift_type"] = (int64_t) (t ? t->scalar_type() : at::kFloat);
    return out;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    variable_list g(6);
    if (!grads[0].defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const Tensor shift = ctx->saved_data["shift"].toBool() ? s[0] : Tensor();      // only whether it was there
    Edges e{ctx};
    const bool wx = e.wants(s[0]);
    int64_t want = 0;
    for (int i = 0; i < 4; ++i)
      if (e.wants(i < 3 ? s[1 + i] : shift)) want |= 1 << i;
    std::optional<at::ScalarType> shift_type;
    if (shift.defined()) shift_type = (at::ScalarType) ctx->saved_data["shift_type"].toInt();
    const auto bias_type = s[2].defined() ? s[2].scalar_type() : at::kFloat;
    const std::vector<Tensor> r =
        below_unless_recorded([&] { return norm_bwd_op().call(grads[0], s[0], opt(s[1]), opt(s[2]), opt(s[3]), s[4], want, shift_type, bias_type); });
    if (wx) g[0] = r[0];
    size_t at = 1;
    for (int i = 0; i < 4; ++i)
      if (want >> i & 1) g[1 + i] = r[at++];
    return g;
  }
};

std::vector<Tensor> layer_norm_autograd(const Tensor& x, const OptTensor& w, const OptTensor& b, const OptTensor& s, const OptTensor& t, double eps,
                                        bool want_stats) {
  no_tangents("layer_norm", {x, or_none(w), or_none(b), or_none(s), or_none(t)});
  if (any_grad({x, or_none(w), or_none(b), or_none(s), or_none(t)})) return NormFunction::apply(x, w, b, s, t, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return norm_fwd_op().call(x, w, b, s, t, eps, want_stats);
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r,
                               const OptTensor& gate, int64_t act) {
    // z is kept where a gate's gradient or, of fp32 data, an activation's slope will ask for it
    const bool pre = (act != LLSA_ACT_NONE && x.scalar_type() == at::kFloat) || (gate && gate->requires_grad());
    variable_list out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      out = linear_fwd_op().call(x, w, b, r, gate, act, pre, true);
    }
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable(variable_list(out.begin() + 1, out.end()));
    const bool copies = out.size() > 2u + pre;
    ctx->save_for_backward({x, w, pre ? out[1] : Tensor(), or_none(gate), or_none(b), copies ? out[1 + pre] : Tensor(), copies ? out[2 + pre] : Tensor()});
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = r.has_value();
    return out;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    variable_list g(6);
    if (!grads[0].defined()) return g;
    const variable_list s = ctx->get_saved_variables();
    const int64_t act = ctx->saved_data["act"].toInt();
    Edges e{ctx};
    int64_t want = 0;
    if (e.wants(s[0])) want |= 1;
    if (e.wants(s[1])) want |= 2;
    if (e.wants(s[4])) want |= 4;
    const bool want_residual = e.wants(ctx->saved_data["residual"].toBool() ? s[0] : Tensor());
    if (e.wants(s[3])) want |= 8;
    if (want) {
      const std::vector<Tensor> r =
          below_unless_recorded([&] { return linear_bwd_op().call(grads[0], s[0], s[1], opt(s[4]), opt(s[2]), opt(s[3]), opt(s[5]), opt(s[6]), act, want); });
      size_t at = 0;
      if (want & 1) g[0] = r[at++];
      if (want & 2) g[1] = r[at++];
      if (want & 4) g[2] = r[at++];
      if (want & 8) g[4] = r[at++];
    }
    if (want_residual) g[3] = grads[0];
    return g;
  }
};

std::vector<Tensor> linear_autograd(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, const OptTensor& gate, int64_t act,
                                    bool want_pre, bool want_copies) {
  no_tangents("linear", {x, w, or_none(b), or_none(r), or_none(gate)});
  if (any_grad({x, w, or_none(b), or_none(r), or_none(gate)})) return LinearFunction::apply(x, w, b, r, gate, act);
  at::AutoDispatchBelowADInplaceOrView below;
  return linear_fwd_op().call(x, w, b, r, gate, act, want_pre, want_copies);
}

struct RopeFunction : torch::autograd::Function<RopeFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& positions, at::IntArrayRef axes_dims, double theta,
                        bool inverse) {
    ctx->save_for_backward({positions});
    auto& d = ctx->saved_data;
    d["axes"] = axes_dims.vec();
    d["theta"] = theta;
    d["inverse"] = inverse;
    at::AutoDispatchBelowADInplaceOrView below;
    return rope_op().call(x, positions, axes_dims, theta, inverse);
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    variable_list g(5);
    if (!grads[0].defined()) return g;
    auto& d = ctx->saved_data;
    const std::vector<int64_t> axes = d["axes"].toIntVector();
    // a rotation again, and differentiable as one
    g[0] = rope_op().call(grads[0], ctx->get_saved_variables()[0], axes, d["theta"].toDouble(), !d["inverse"].toBool());
    return g;
  }
};

Tensor rope_axes_autograd(const Tensor& x, const Tensor& positions, at::IntArrayRef axes_dims, double theta, bool inverse) {
  no_tangents("rope_axes", {x, positions});
  TORCH_CHECK(!(at::GradMode::is_enabled() && positions.requires_grad()), "llsa_b200: positions carry no gradient");
  if (any_grad({x})) return RopeFunction::apply(x, positions, axes_dims, theta, inverse);
  at::AutoDispatchBelowADInplaceOrView below;
  return rope_op().call(x, positions, axes_dims, theta, inverse);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(llsa_b200, m) {
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? shift, float eps, bool want_stats) -> Tensor[]");
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor stats, int want, ScalarType? shift_type, "
        "ScalarType bias_type) -> Tensor[]");
  m.def("linear_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, Tensor? gate, int activation, bool want_pre, bool want_copies) -> "
        "Tensor[]");
  m.def("linear_bwd(Tensor dy, Tensor x, Tensor weight, Tensor? bias, Tensor? pre, Tensor? gate, Tensor? x_copy, Tensor? w_copy, int activation, int want) -> Tensor[]");
  m.def("rope_axes(Tensor x, Tensor positions, int[] axes_dims, float theta, bool inverse) -> Tensor");
}
TORCH_LIBRARY_IMPL(llsa_b200, CUDA, m) {
  m.impl("layer_norm_fwd", layer_norm_fwd);
  m.impl("layer_norm_bwd", layer_norm_bwd);
  m.impl("linear_fwd", linear_fwd);
  m.impl("linear_bwd", linear_bwd);
  m.impl("rope_axes", rope_axes);
}
TORCH_LIBRARY_IMPL(llsa_b200, CPU, m) {      // refuse with the library's own words
  m.impl("layer_norm_fwd", layer_norm_fwd);
  m.impl("layer_norm_bwd", layer_norm_bwd);
  m.impl("linear_fwd", linear_fwd);
  m.impl("linear_bwd", linear_bwd);
  m.impl("rope_axes", rope_axes);
}
TORCH_LIBRARY_IMPL(llsa_b200, Autograd, m) {
  m.impl("layer_norm_fwd", layer_norm_autograd);
  m.impl("layer_norm_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_fwd", linear_autograd);
  m.impl("linear_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("rope_axes", rope_axes_autograd);
}
