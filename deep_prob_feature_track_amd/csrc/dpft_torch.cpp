// dpft_torch.cpp -- libdpft_torch.so: the normalisation entry points of libdpft_ic.so as torch
// operators, with their gradients.
//
//   dpft::group_norm_act           y, differentiable once in x, weight and bias
//   dpft::group_norm_act_forward   y, statistics [2,N,groups], q, scale (empty where not asked for)
//   dpft::group_norm_act_backward  dx, dweight, dbias (empty where not asked for)
//   dpft::act_checkpoint / act_restore
//
// In C++ because the autograd engine runs a backward pass on a thread of its own: a Python function
// there pays for a cold thread and the interpreter lock (a small forward and backward pass: 150 us).
// The operators launch on the current stream of the tensors' device and never synchronise.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "dpft_ic.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

constexpr int64_t kBlock8 = 32;

int32_t type_code(at::ScalarType t, const char* what) {
  if (t == at::kFloat) return DPFT_TYPE_F32;
  if (t == at::kBFloat16) return DPFT_TYPE_BF16;
  TORCH_CHECK_TYPE(t == at::kHalf, what, ": float32, bfloat16 or float16 (got ", t, ")");
  return DPFT_TYPE_F16;
}

// A traced call's channels are what it was traced with; its batch and pixels may be symbols.
int64_t channels(const Tensor& t, int64_t dim) { return t.sym_size(dim).guard_int(__FILE__, __LINE__); }

void check_param(const MaybeTensor& p, const char* name, const Tensor& x, int64_t C) {
  if (!p || !p->defined()) return;
  TORCH_CHECK_VALUE(p->dim() == 1 && channels(*p, 0) == C, name, " must hold one value per channel (", C, "), got ",
                    p->sym_sizes());
  type_code(p->scalar_type(), name);
  TORCH_CHECK_VALUE(p->device() == x.device(), name, " is on ", p->device(), ", expected ", x.device());
}

bool given(const MaybeTensor& t) { return t && t->defined(); }

// The operators have no forward-mode derivative.  A tangent would be lost without a word below autograd, whether or
// not anything requires a gradient: every way in asks for it.
void refuse_tangents(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "group_norm_act has no forward-mode derivative (an input carries a tangent)");
}
void refuse_tangents(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias) {
  refuse_tangents({&x});
  if (weight) refuse_tangents({&*weight});
  if (bias) refuse_tangents({&*bias});
}
void* ptr(const MaybeTensor& t) { return given(t) && t->numel() ? t->data_ptr() : nullptr; }
Tensor dense(const MaybeTensor& t) { return given(t) ? t->contiguous() : Tensor(); }

// Everything that the arguments have to meet, on any device and in a trace.
DpftGroupNorm check_args(const Tensor& x, int64_t groups, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                         int64_t act, bool packed) {
  refuse_tangents(x, weight, bias);
  TORCH_CHECK_VALUE(x.dim() == 4, "group_norm_act needs a map [N,C,H,W], got ", x.sym_sizes());
  const int64_t C = channels(x, 1);
  TORCH_CHECK_VALUE(groups >= 1 && C >= 1 && C % groups == 0, "groups=", groups, " does not divide C=", C);
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative (got ", eps, ")");
  check_param(weight, "weight", x, C);
  check_param(bias, "bias", x, C);
  if (given(weight) && given(bias))
    TORCH_CHECK_TYPE(weight->scalar_type() == bias->scalar_type(), "weight and bias must have one dtype (got ",
                     weight->scalar_type(), ", ", bias->scalar_type(), ")");
  TORCH_CHECK_VALUE(!packed || (x.scalar_type() == at::kFloat && C % 4 == 0), "packed=True needs fp32 and C % 4 == 0, got ",
                    x.scalar_type(), " ", x.sym_sizes());
  TORCH_CHECK_VALUE(C <= INT32_MAX, "too large: ", x.sym_sizes());
  DpftGroupNorm d{};
  d.C = (int32_t)C;
  d.groups = (int32_t)groups;
  d.act = (int32_t)act;
  d.x_type = type_code(x.scalar_type(), "group_norm_act");
  d.param_type = given(weight) ? type_code(weight->scalar_type(), "weight")
                 : given(bias) ? type_code(bias->scalar_type(), "bias")
                               : DPFT_TYPE_F32;
  d.flags = packed ? DPFT_GN_PACKED : 0;
  d.eps = (float)eps;
  return d;
}

// ... and the sizes of a map with memory.
DpftGroupNorm sized(DpftGroupNorm d, const Tensor& x) {
  TORCH_CHECK_VALUE(x.size(0) <= INT32_MAX, "too large: ", x.sizes());
  d.pixels = x.size(2) * x.size(3);
  d.N = (int32_t)x.size(0);
  return d;
}

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == DPFT_OK, what, " failed (", rc, "): ", dpft_last_error()); }

// Stored channels_last (a copy where it is not); and 16-byte aligned (a tensor with memory).
Tensor ordered(const Tensor& x) {
  return x.is_contiguous(at::MemoryFormat::ChannelsLast) ? x : x.contiguous(at::MemoryFormat::ChannelsLast);
}
Tensor nhwc(const Tensor& x) {
  const Tensor r = ordered(x);
  return reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 ? r.clone(at::MemoryFormat::ChannelsLast) : r;
}
Tensor empty_nhwc(const Tensor& x) { return at::empty(x.sizes(), x.options(), at::MemoryFormat::ChannelsLast); }
Tensor none(const Tensor& x) { return at::empty({0}, x.options()); }
void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

struct Workspace {  // of one call: calls on other streams and captured ones share nothing
  size_t bytes;
  Tensor t;
  Workspace(const DpftGroupNorm& d, const Tensor& x) : bytes(dpft_group_norm_workspace_size(&d)) {
    if (bytes == 0) check_rc(DPFT_E_INVALID, "dpft_group_norm_workspace_size");
    t = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  }
};

int64_t blocks_of(int64_t n) { return (n + kBlock8 - 1) / kBlock8; }

// ------------------------------------------------------------------ group norm
std::tuple<Tensor, Tensor, Tensor, Tensor> forward_outputs(const Tensor& x, int64_t groups, bool packed, bool stats,
                                                           bool checkpoint) {
  Tensor y = packed ? at::empty({x.size(0), x.size(1) / 4, x.size(2), x.size(3), 4}, x.options()) : empty_nhwc(x);
  Tensor stat = stats ? at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat)) : none(x);
  Tensor q = checkpoint ? at::empty({x.numel()}, x.options().dtype(at::kChar)) : none(x);
  Tensor scale = checkpoint ? at::empty({blocks_of(x.numel())}, x.options().dtype(at::kByte)) : none(x);
  return {y, stat, q, scale};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> forward_hip(const Tensor& x0, int64_t groups, const MaybeTensor& weight,
                                                       const MaybeTensor& bias, double eps, int64_t act, bool packed,
                                                       bool stats, bool checkpoint) {
  const DpftGroupNorm d = sized(check_args(x0, groups, weight, bias, eps, act, packed), x0);
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = nhwc(x0), w = dense(weight), b = dense(bias);
  auto out = forward_outputs(x, groups, packed, stats, checkpoint);
  if (x.numel() == 0) return out;
  auto& [y, stat, q, scale] = out;
  const Workspace ws(d, x);
  float* mean = stats ? stat.data_ptr<float>() : nullptr;
  check_rc(dpft_group_norm_act(&d, x.data_ptr(), ptr(w), ptr(b), y.data_ptr(), mean,
                               stats ? mean + (int64_t)d.N * groups : nullptr, static_cast<int8_t*>(ptr(q)),
                               static_cast<uint8_t*>(ptr(scale)), ws.t.data_ptr(), ws.bytes, stream_of(x)),
           "dpft_group_norm_act");
  return out;
}
std::tuple<Tensor, Tensor, Tensor, Tensor> forward_meta(const Tensor& x, int64_t groups, const MaybeTensor& weight,
                                                        const MaybeTensor& bias, double eps, int64_t act, bool packed,
                                                        bool stats, bool checkpoint) {
  check_args(x, groups, weight, bias, eps, act, packed);
  const auto N = x.sym_size(0), C = x.sym_size(1), H = x.sym_size(2), W = x.sym_size(3), n = x.sym_numel();
  Tensor y = packed ? at::empty_symint({N, C / 4, H, W, 4}, x.options())
                    : at::empty_symint({N, C, H, W}, x.options(), at::MemoryFormat::ChannelsLast);
  Tensor stat = stats ? at::empty_symint({2, N, groups}, x.options().dtype(at::kFloat)) : none(x);
  Tensor q = checkpoint ? at::empty_symint({n}, x.options().dtype(at::kChar)) : none(x);
  Tensor scale = checkpoint ? at::empty_symint({(n + kBlock8 - 1) / kBlock8}, x.options().dtype(at::kByte)) : none(x);
  return {y, stat, q, scale};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> forward_cpu(const Tensor& x, int64_t groups, const MaybeTensor& weight,
                                                       const MaybeTensor& bias, double eps, int64_t act, bool packed,
                                                       bool, bool) {
  check_args(x, groups, weight, bias, eps, act, packed);
  TORCH_CHECK(false, "group_norm_act needs a device tensor; there is no CPU fallback");
}

std::tuple<Tensor, Tensor, Tensor> backward_outputs(const Tensor& dy, const MaybeTensor& weight, const MaybeTensor& bias,
                                                    bool need_x, bool need_w, bool need_b) {
  return {need_x ? empty_nhwc(dy) : none(dy), need_w ? at::empty_like(*weight) : none(dy),
          need_b ? at::empty_like(*bias) : none(dy)};
}

// x, or its checkpoint (q, scale) where x is empty.
std::tuple<Tensor, Tensor, Tensor> backward_hip(const Tensor& dy0, const Tensor& x, const Tensor& q, const Tensor& scale,
                                                const MaybeTensor& weight, const MaybeTensor& bias, const Tensor& stat,
                                                int64_t groups, double eps, int64_t act, bool need_x, bool need_w,
                                                bool need_b) {
  refuse_tangents({&x});
  const DpftGroupNorm d = sized(check_args(dy0, groups, weight, bias, eps, act, false), dy0);
  const int64_t n = dy0.numel();
  const bool from_x = x.numel() != 0 && q.numel() == 0 && x.sizes() == dy0.sizes() && x.scalar_type() == dy0.scalar_type(),
             from_q = x.numel() == 0 && q.numel() == n && scale.numel() == blocks_of(n) && q.is_contiguous() &&
                      scale.is_contiguous() && q.scalar_type() == at::kChar && scale.scalar_type() == at::kByte;
  TORCH_CHECK_VALUE((n == 0 || from_x || from_q) && stat.is_contiguous() && stat.scalar_type() == at::kFloat &&
                        stat.numel() == 2 * d.N * groups && (!need_w || given(weight)) && (!need_b || given(bias)),
                    "group_norm_act_backward: dy, x, its checkpoint and statistics do not belong together");
  for (const Tensor& t : {x, q, scale, stat})
    TORCH_CHECK_VALUE(t.device() == dy0.device(), "group_norm_act_backward: tensors on ", t.device(), " and ", dy0.device());
  const c10::DeviceGuard guard(dy0.device());
  const Tensor dy = nhwc(dy0), w = dense(weight), b = dense(bias), xs = x.numel() ? nhwc(x) : x;
  auto out = backward_outputs(dy, w, b, need_x, need_w, need_b);
  auto& [dx, dw, db] = out;
  if (n == 0) {
    dw.zero_();
    db.zero_();
    return out;
  }
  const Workspace ws(d, dy);
  const float* mean = stat.data_ptr<float>();
  check_rc(dpft_group_norm_act_backward(&d, dy.data_ptr(), ptr(xs), static_cast<int8_t*>(ptr(q)),
                                        static_cast<uint8_t*>(ptr(scale)), ptr(w), ptr(b), mean,
                                        mean + (int64_t)d.N * groups, ptr(dx), ptr(dw), ptr(db), ws.t.data_ptr(), ws.bytes,
                                        stream_of(dy)),
           "dpft_group_norm_act_backward");
  return out;
}
std::tuple<Tensor, Tensor, Tensor> backward_meta(const Tensor& dy, const Tensor& x, const Tensor&, const Tensor&,
                                                 const MaybeTensor& weight, const MaybeTensor& bias, const Tensor&, int64_t,
                                                 double, int64_t, bool need_x, bool need_w, bool need_b) {
  refuse_tangents({&x});
  refuse_tangents(dy, weight, bias);
  return {need_x ? at::empty_symint(dy.sym_sizes(), dy.options(), at::MemoryFormat::ChannelsLast) : none(dy),
          need_w ? at::empty_like(*weight) : none(dy), need_b ? at::empty_like(*bias) : none(dy)};
}

auto& forward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("dpft::group_norm_act_forward", "")
                       .typed<decltype(forward_hip)>();
  return op;
}
auto& backward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("dpft::group_norm_act_backward", "")
                       .typed<decltype(backward_hip)>();
  return op;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const MaybeTensor& weight, const MaybeTensor& bias,
                        int64_t groups, double eps, int64_t act, bool checkpoint) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = x0.dim() == 4 && x0.is_cuda() ? ordered(x0) : x0;  // a copy is made once, and kept
    auto [y, stat, q, scale] = forward_op().call(x, groups, weight, bias, eps, act, false, true, checkpoint);
    ctx->save_for_backward({checkpoint ? none(x) : x, q, scale, given(weight) ? *weight : Tensor(),
                            given(bias) ? *bias : Tensor(), stat});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "group_norm_act is differentiable once (create_graph=True is refused)");
    if (!grads[0].defined()) return variable_list(7);
    const auto saved = ctx->get_saved_variables();
    const bool has_w = saved[3].defined(), has_b = saved[4].defined();  // one edge for each tensor that was given
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
               need_b = has_b && ctx->needs_input_grad(1 + has_w);
    auto opt = [](const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    auto [dx, dw, db] =
        backward_op().call(grads[0], saved[0], saved[1], saved[2], opt(saved[3]), opt(saved[4]), saved[5],
                           ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(),
                           ctx->saved_data["act"].toInt(), need_x, need_w, need_b);
    variable_list out(7);
    if (need_x) out[0] = dx;
    if (need_w) out[1] = dw;
    if (need_b) out[2] = db;
    return out;
  }
};

bool wants_grad(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias) {
  return at::GradMode::is_enabled() &&
         (x.requires_grad() || (given(weight) && weight->requires_grad()) || (given(bias) && bias->requires_grad()));
}
Tensor act_autograd(const Tensor& x, int64_t groups, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                    int64_t act, bool packed, bool checkpoint) {
  refuse_tangents(x, weight, bias);
  if (!wants_grad(x, weight, bias)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return std::get<0>(forward_op().call(x, groups, weight, bias, eps, act, packed, false, false));
  }
  TORCH_CHECK(!packed, "packed=True is the solver's input at inference: it has no backward");
  return GroupNormAct::apply(x, weight, bias, groups, eps, act, checkpoint);
}
Tensor act_plain(const Tensor& x, int64_t groups, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                 int64_t act, bool packed, bool) {
  return std::get<0>(forward_op().call(x, groups, weight, bias, eps, act, packed, false, false));
}

// ------------------------------------------------------------------ 8-bit checkpoints
void check_checkpoint(const Tensor& x) { type_code(x.scalar_type(), "act_checkpoint"); }
std::tuple<Tensor, Tensor> checkpoint_hip(const Tensor& x0) {
  check_checkpoint(x0);
  const c10::DeviceGuard guard(x0.device());
  TORCH_CHECK_VALUE(x0.is_non_overlapping_and_dense(), "act_checkpoint: x must fill its memory");
  const Tensor x = reinterpret_cast<uintptr_t>(x0.data_ptr()) % 16 ? x0.clone(at::MemoryFormat::Preserve) : x0;
  const int64_t n = x.numel();
  Tensor q = at::empty({n}, x.options().dtype(at::kChar)), scale = at::empty({blocks_of(n)}, x.options().dtype(at::kByte));
  if (n)
    check_rc(dpft_act_checkpoint(x.data_ptr(), type_code(x.scalar_type(), "x"), n, q.data_ptr<int8_t>(),
                                 scale.data_ptr<uint8_t>(), stream_of(x)),
             "dpft_act_checkpoint");
  return {q, scale};
}
std::tuple<Tensor, Tensor> checkpoint_meta(const Tensor& x) {
  check_checkpoint(x);
  return {at::empty({x.numel()}, x.options().dtype(at::kChar)), at::empty({blocks_of(x.numel())}, x.options().dtype(at::kByte))};
}
std::tuple<Tensor, Tensor> checkpoint_cpu(const Tensor& x) {
  check_checkpoint(x);
  TORCH_CHECK(false, "act_checkpoint needs a device tensor; there is no CPU fallback");
}

Tensor restore_output(const Tensor& q, const Tensor& scale, at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType dtype) {
  type_code(dtype, "act_restore");
  Tensor out = at::empty_strided(size, stride, q.options().dtype(dtype));
  TORCH_CHECK_VALUE(q.scalar_type() == at::kChar && scale.scalar_type() == at::kByte && q.is_contiguous() &&
                        scale.is_contiguous() && q.device() == scale.device() && out.is_non_overlapping_and_dense() &&
                        q.numel() == out.numel() && scale.numel() == blocks_of(q.numel()),
                    "act_restore: not a checkpoint of that shape");
  return out;
}
Tensor restore_hip(const Tensor& q, const Tensor& scale, at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType dtype) {
  const c10::DeviceGuard guard(q.device());
  Tensor out = restore_output(q, scale, size, stride, dtype);
  if (out.numel())
    check_rc(dpft_act_restore(q.data_ptr<int8_t>(), scale.data_ptr<uint8_t>(), q.numel(), out.data_ptr(),
                              type_code(dtype, "act_restore"), stream_of(q)),
             "dpft_act_restore");
  return out;
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(dpft, m) {
  m.def("group_norm_act(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, bool packed, bool checkpoint) -> Tensor");
  m.def("group_norm_act_forward(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, bool packed, bool stats, bool checkpoint) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("group_norm_act_backward(Tensor dy, Tensor x, Tensor q, Tensor scale, Tensor? weight, Tensor? bias, Tensor stat, int groups, float eps, int act, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)");
  m.def("act_checkpoint(Tensor x) -> (Tensor, Tensor)");
  m.def("act_restore(Tensor q, Tensor scale, int[] size, int[] stride, ScalarType dtype) -> Tensor");
}
TORCH_LIBRARY_IMPL(dpft, CUDA, m) {
  m.impl("group_norm_act", act_plain);
  m.impl("group_norm_act_forward", forward_hip);
  m.impl("group_norm_act_backward", backward_hip);
  m.impl("act_checkpoint", checkpoint_hip);
  m.impl("act_restore", restore_hip);
}
TORCH_LIBRARY_IMPL(dpft, CPU, m) {
  m.impl("group_norm_act", act_plain);
  m.impl("group_norm_act_forward", forward_cpu);
  m.impl("act_checkpoint", checkpoint_cpu);
}
TORCH_LIBRARY_IMPL(dpft, Meta, m) {
  m.impl("group_norm_act", act_plain);
  m.impl("group_norm_act_forward", forward_meta);
  m.impl("group_norm_act_backward", backward_meta);
  m.impl("act_checkpoint", checkpoint_meta);
  m.impl("act_restore", restore_output);
}
TORCH_LIBRARY_IMPL(dpft, Autograd, m) { m.impl("group_norm_act", act_autograd); }
