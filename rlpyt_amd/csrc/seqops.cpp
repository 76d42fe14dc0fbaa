// Call path of the sequence operators' small calls: allocations, launches (through the C entry points of
// include/rlpyt_hip.h) and autograd nodes in C++.  A scan of 85 x 32 x 512 runs 19 us on the device; with a Python
// autograd.Function and ctypes its two directions took 118 us of host time, most of it in the backward thread, where
// Python's allocations and calls take twice as long.  Arguments are checked by rlpyt_amd/ops_seq.py.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/rlpyt_hip.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct HipFailure : std::runtime_error {   // rlpyt_amd._lib.HipError
  using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
  if (rc != RLPYT_OK)
    throw HipFailure(std::string(what) + " failed (rc=" + std::to_string(rc) + "): " + rlpyt_hip_last_error());
}

int code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }
Tensor bytes(int64_t n, const Tensor& like) {
  return n ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor();
}

// The gradients of a backward pass that builds a graph raise when they are differentiated.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<size_t> places;
  variable_list in;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      places.push_back(i);
      in.push_back(grads[i].detach().set_requires_grad(true));
    }
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "rlpyt_amd: the sequence operators can be differentiated once", (int64_t)in.size());
  const variable_list out = (*node)(std::move(in));
  for (size_t i = 0; i < places.size(); ++i) grads[places[i]] = out[i];
  return grads;
}

// A captured backward pass would wait for the stream of the node that gathers a leaf's gradient.  Where an eager graph of the
// leaf lives, that is the eager graph's, which a capture cannot wait for (the process ends): refused here.
void check_leaves(const char* what, std::initializer_list<const Tensor*> inputs) {
  const Tensor& first = **inputs.begin();
  const c10::DeviceGuard guard(first.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto current = c10::hip::getCurrentHIPStream(first.device().index());
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto other = node->stream();
    if (other && other->id() != current.id())
      throw std::runtime_error(std::string(what) + ": a result computed from the same leaf on another stream is still held; "
                               "drop it before its backward pass is captured");
  }
}

// ---- gated linear recurrence ------------------------------------------------------------------------------
// An empty [T, B, D] whose rows lie in memory in the order of x's: time or batch first.  (By its strides: a transposed view made
// under a node could not be written in place.)
Tensor like_rows(const Tensor& x) {
  if (x.is_contiguous()) return at::empty_like(x);
  const int64_t T = x.size(0), B = x.size(1), D = x.size(2);
  if (T > 1 && B > 1 && x.stride(1) > x.stride(0)) return at::empty_strided({T, B, D}, {D, T * D, 1}, x.options());
  return at::empty({T, B, D}, x.options());
}

struct Scan {
  Tensor h, hn, states;
};
Scan scan_forward(const Tensor& x, const Tensor& gate, const Tensor& h0, const Tensor& reset, const Tensor& lengths,
                  bool keep) {
  const c10::DeviceGuard guard(x.device());
  const int64_t T = x.size(0), B = x.size(1), D = x.size(2);
  const auto f32 = x.options().dtype(at::kFloat);
  Scan s;
  s.h = like_rows(x);
  s.hn = at::empty({B, D}, f32);
  if (keep) s.states = at::empty({rlpyt_gated_scan_state_rows(T), B, D}, f32);
  const Tensor first = h0.defined() ? h0.detach().to(at::kFloat).contiguous() : h0;
  const Tensor ws = bytes(rlpyt_gated_scan_workspace_bytes(T, B, D), x);
  check(rlpyt_gated_scan_fwd(code(x.scalar_type()), ptr(x), x.stride(0), x.stride(1), ptr(gate), gate.stride(0),
                             gate.stride(1), ptr<float>(first), ptr<uint8_t>(reset), ptr<int64_t>(lengths), ptr(s.h),
                             s.h.stride(0), s.h.stride(1), ptr<float>(s.hn), ptr<float>(s.states), T, B, D, ptr(ws),
                             stream_of(x)),
        "rlpyt_gated_scan_fwd");
  return s;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& h0,
                               const Maybe& reset, const Maybe& lengths) {
    Scan s = scan_forward(x, gate, or_none(h0), or_none(reset), or_none(lengths), true);
    ctx->save_for_backward({x, gate, or_none(reset), or_none(lengths), s.states});
    ctx->set_materialize_grads(false);
    if (h0) ctx->saved_data["h0"] = (int64_t)h0->scalar_type();
    return {s.h, s.hn};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dh = grads[0], dhn = grads[1];
    if (!dh.defined() && !dhn.defined()) return variable_list(5);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate = saved[1];
    const c10::DeviceGuard guard(x.device());
    const int64_t T = x.size(0), B = x.size(1), D = x.size(2);
    const auto f32 = x.options().dtype(at::kFloat);
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      if (!dh.defined()) dh = at::zeros({D}, x.options()).expand({T, B, D});
      if (dh.scalar_type() != x.scalar_type() || (dh.stride(2) != 1 && D != 1)) dh = dh.to(x.scalar_type()).contiguous();
      if (dhn.defined()) dhn = dhn.to(at::kFloat).contiguous();
      const auto h0 = ctx->saved_data.find("h0");
      const bool need = h0 != ctx->saved_data.end() && ctx->needs_input_grad(2);
      Tensor dx = like_rows(x), dgate = like_rows(x), dh0;
      if (need) dh0 = at::empty({B, D}, f32);
      const Tensor ws = bytes(rlpyt_gated_scan_workspace_bytes(T, B, D), x);
      check(rlpyt_gated_scan_bwd(code(x.scalar_type()), ptr(x), x.stride(0), x.stride(1), ptr(gate), gate.stride(0),
                                 gate.stride(1), ptr(dh), dh.stride(0), dh.stride(1), ptr<float>(dhn),
                                 ptr<uint8_t>(saved[2]), ptr<int64_t>(saved[3]), ptr<float>(saved[4]), ptr(dx),
                                 dx.stride(0), dx.stride(1), ptr(dgate), dgate.stride(0), dgate.stride(1),
                                 ptr<float>(dh0), T, B, D, ptr(ws), stream_of(x)),
            "rlpyt_gated_scan_bwd");
      out[0] = dx, out[1] = dgate;
      if (need) out[2] = dh0.to((at::ScalarType)h0->second.toInt());
    }
    return once(out);
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& reset,
                                      const Maybe& lengths) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (h0 && h0->requires_grad()))) {
    const Tensor state = or_none(h0);
    check_leaves("gated_scan", {&x, &gate, &state});
    const variable_list out = GatedScan::apply(x, gate, h0, reset, lengths);
    return {out[0], out[1]};
  }
  const Scan s = scan_forward(x, gate, or_none(h0), or_none(reset), or_none(lengths), false);
  return {s.h, s.hn};
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state, const Maybe& reset) {
  const c10::DeviceGuard guard(x.device());
  const int64_t B = x.size(0), D = x.size(1);
  const Tensor y = at::empty({B, D}, x.options());
  check(rlpyt_gated_scan_step(code(x.scalar_type()), ptr(x), x.stride(0), ptr(gate), gate.stride(0),
                              ptr<uint8_t>(or_none(reset)), ptr<float>(state), ptr(y), B, D, stream_of(x)),
        "rlpyt_gated_scan_step");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();   // written through a raw pointer
  return y;
}

// ---- clipped policy loss with a KL term ----------------------------------------------------------------------
struct Coeffs {
  double low, high, kl, entropy, grad_scale;
};
struct Loss {
  Tensor loss, scalars, grad;
};
Loss loss_forward(const Tensor& rows, const Tensor& action, const Tensor& old_logp, const Tensor& advantage,
                  const Tensor& ref_logp, const Tensor& valid, const Coeffs& c, bool want_grad) {
  const c10::DeviceGuard guard(rows.device());
  const int64_t N = rows.size(0), V = rows.size(1);
  const auto f32 = rows.options().dtype(at::kFloat);
  Loss l;
  l.loss = at::empty({}, f32);
  l.scalars = at::empty({5}, f32);
  if (want_grad) l.grad = at::empty({N, V}, rows.options());
  const int type = code(rows.scalar_type());
  const Tensor ws = bytes(rlpyt_policy_loss_workspace_bytes(type, N, V), rows);
  check(rlpyt_policy_kl_loss_fwd_bwd(type, ptr(rows), rows.stride(0), ptr<int64_t>(action), ptr<float>(old_logp),
                                     ptr<float>(advantage), ptr<float>(ref_logp), ptr<float>(valid), N, V, c.low, c.high,
                                     c.kl, c.entropy, c.grad_scale, ptr<float>(l.loss), ptr<float>(l.scalars),
                                     ptr(l.grad), ptr(ws), stream_of(rows)),
        "rlpyt_policy_kl_loss_fwd_bwd");
  return l;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& rows, const Tensor& action,
                               const Tensor& old_logp, const Tensor& advantage, const Maybe& ref_logp,
                               const Maybe& valid, const Coeffs& c, int64_t unit_seed) {
    Loss l = loss_forward(rows, action, old_logp, advantage, or_none(ref_logp), or_none(valid), c, true);
    ctx->saved_data["grad"] = l.grad;
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->saved_data["factor"] = 1.0 / c.grad_scale;
    ctx->saved_data["unit"] = unit_seed;
    ctx->mark_non_differentiable({l.scalars});
    return {l.loss, l.scalars};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto it = ctx->saved_data.find("grad");
    if (it == ctx->saved_data.end())
      throw std::runtime_error("policy_kl_loss: its gradient went out with the first backward pass (it is scaled in place); "
                               "run the loss again");
    Tensor grad = it->second.toTensor();
    ctx->saved_data.erase(it);
    variable_list out(9);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(grad.device());
      const Tensor g = grads[0].to(at::kFloat);
      const double factor = ctx->saved_data["factor"].toDouble();
      // the standing scalar 1 of ops.unit_seed is known to be 1
      if (factor != 1.0 || (int64_t)g.data_ptr() != ctx->saved_data["unit"].toInt())
        check(rlpyt_scale_unless_one(code(grad.scalar_type()), ptr(grad), grad.numel(), ptr<float>(g), (float)factor,
                                     stream_of(grad)),
              "rlpyt_scale_unless_one");
      out[0] = grad.view(ctx->saved_data["shape"].toIntVector());
    }
    return once(out);
  }
};

std::tuple<Tensor, Tensor> policy_kl_loss(const Tensor& logits, const Tensor& rows, const Tensor& action,
                                          const Tensor& old_logp, const Tensor& advantage, const Maybe& ref_logp,
                                          const Maybe& valid, double low, double high, double kl, double entropy,
                                          double grad_scale, int64_t unit_seed) {
  const Coeffs c = {low, high, kl, entropy, grad_scale};
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    check_leaves("policy_kl_loss", {&logits});
    const variable_list out =
        PolicyLoss::apply(logits, rows, action, old_logp, advantage, ref_logp, valid, c, unit_seed);
    return {out[0], out[1]};
  }
  const Loss l = loss_forward(rows, action, old_logp, advantage, or_none(ref_logp), or_none(valid), c, false);
  return {l.loss, l.scalars};
}

std::tuple<Tensor, Tensor> action_logp(const Tensor& logits, const Tensor& rows, const Tensor& action) {
  const c10::DeviceGuard guard(rows.device());
  const int64_t N = rows.size(0), V = rows.size(1);
  const auto f32 = rows.options().dtype(at::kFloat);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const Tensor logp = at::empty(lead, f32), entropy = at::empty(lead, f32);
  const int type = code(rows.scalar_type());
  const Tensor ws = bytes(rlpyt_policy_loss_workspace_bytes(type, N, V), rows);
  check(rlpyt_action_logp(type, ptr(rows), rows.stride(0), ptr<int64_t>(action), N, V, ptr<float>(logp),
                          ptr<float>(entropy), ptr(ws), stream_of(rows)),
        "rlpyt_action_logp");
  return {logp, entropy};
}
}  // namespace

PYBIND11_MODULE(_seqops, m) {
  pybind11::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const HipFailure& e) {
      const auto type = pybind11::module_::import("rlpyt_amd._lib").attr("HipError");
      PyErr_SetString(type.ptr(), e.what());
    }
  });
  m.attr("abi_version") = RLPYT_HIP_ABI_VERSION;
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_step", &gated_scan_step);
  m.def("policy_kl_loss", &policy_kl_loss);
  m.def("action_logp", &action_logp);
}
