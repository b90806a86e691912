// Token log-probabilities and the losses over them as torch operators with their backwards in C++:
//
//   token_logprobs(Tensor logits, Tensor targets, float temperature, int ignore_index, bool entropy)
//       -> (Tensor, Tensor)
//   preference_loss(Tensor logps, Tensor? reference, Tensor? offsets, Tensor? mask, int kind, float beta,
//       float smoothing, bool average, int reduction) -> (Tensor, Tensor, Tensor)
//   policy_loss(Tensor logps, Tensor old, Tensor advantages, Tensor? reference, Tensor? offsets,
//       Tensor? mask, float clip_low, float clip_high, float kl_coef, int reduction)
//       -> (Tensor, Tensor, Tensor)
//
// As in ti_torch.cpp there are no kernels here: outputs and workspaces are torch's, the stream is
// torch's current one, and the C ABI of libtorchisotonic_amd.so does the work. Nothing here waits for
// the GPU.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>
#include <tuple>

#include "torchisotonic_amd.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Three = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == TI_OK, "torchisotonic_amd.", what, ": ", ti_last_error(), " (status ", rc, ")");
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const std::optional<at::Tensor>& t) { return t.has_value() ? ptr(*t) : nullptr; }

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dtype_code(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return TI_F32;
    case at::kDouble: return TI_F64;
    case at::kBFloat16: return TI_BF16;
    case at::kHalf: return TI_F16;
    default: TORCH_CHECK(false, "torchisotonic_amd.", what, ": no kernel for ", t.scalar_type());
  }
}

// (the kernels' gradients are no functions that autograd could differentiate again)
void once(const char* what) {
  TORCH_CHECK(!c10::GradMode::is_enabled(), "torchisotonic_amd.", what, " is not twice differentiable");
}

// Whether a backward may follow (asked outside the autograd node's forward, which runs untracked).
bool tracked(const at::Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }

// There are no forward-mode derivatives: a dual tensor raises, whether it requires a gradient or not, as its result
// without a tangent would read as a derivative of zero.
void no_tangents(std::initializer_list<const at::Tensor*> tensors, const char* what) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : tensors)
    TORCH_CHECK(t == nullptr || !t->defined() || !t->_fw_grad(0).defined(), "torchisotonic_amd.", what,
                " has no forward-mode derivative (jvp)");
}
const at::Tensor* some(const std::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

// A saved tensor as the kernels take it. (What comes back is what saved-tensor hooks made of it: a copy, maybe in
// another layout, so that nothing of the layout it was saved in holds.)
at::Tensor saved_as(const at::Tensor& t, int64_t numel, at::ScalarType type, const at::Device& device, const char* what) {
  TORCH_CHECK(t.defined() && t.numel() == numel && t.scalar_type() == type && t.device() == device, "torchisotonic_amd.",
              what, " backward: a saved tensor came back with another size, type or device");
  return t.contiguous();
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// --- token log-probabilities -------------------------------------------------------------------

// Where the rows of a [..., vocab] tensor begin: two strides over the leading dimensions taken as
// one index. A tensor whose leading dimensions are no two-level grid of rows, or whose rows are not
// contiguous, is copied.
struct Rows {
  at::Tensor logits;
  int64_t inner = 1, outer_stride = 0, row_stride = 0;
};

std::optional<Rows> rows_of(const at::Tensor& z) {
  const int64_t last = z.dim() - 1;
  if (z.size(last) > 1 && z.stride(last) != 1) return std::nullopt;
  // the leading dimensions of more than one index, those that continue one another joined
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};
  int levels = 0;
  for (int64_t d = last - 1; d >= 0; --d) {
    if (z.size(d) == 1) continue;
    if (levels > 0 && z.stride(d) == stride[levels - 1] * size[levels - 1]) {
      size[levels - 1] *= z.size(d);
      continue;
    }
    if (levels == 2) return std::nullopt;
    size[levels] = z.size(d);
    stride[levels] = z.stride(d);
    ++levels;
  }
  return Rows{z, size[0], stride[1], stride[0]};
}

struct Logprobs {
  at::Tensor logp, entropy, stats;  // entropy and stats undefined where not wanted
  Rows where;
};

// The checks and the launch of one call, with the statistics a backward reads or without.
Logprobs logprobs_of(const at::Tensor& logits, const at::Tensor& targets, double temperature, int64_t ignore_index,
                     bool entropy, bool want) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() >= 1 && logits.size(-1) >= 1,
              "torchisotonic_amd.token_logprobs: logits must be [..., vocab] on a ROCm device");
  TORCH_CHECK(targets.device() == logits.device() && targets.scalar_type() == at::kLong && targets.is_contiguous() &&
                  targets.sizes() == logits.sizes().slice(0, logits.dim() - 1),
              "torchisotonic_amd.token_logprobs: targets must be contiguous int64 of logits' leading shape and device");
  const int dtype = dtype_code(logits, "token_logprobs");
  const int64_t rows = targets.numel(), vocab = logits.size(-1);
  const auto acc = logits.options().dtype(dtype == TI_F64 ? at::kDouble : at::kFloat).requires_grad(false);
  const c10::DeviceGuard guard(logits.device());
  Logprobs out;
  out.logp = at::empty(targets.sizes(), acc);
  if (entropy) out.entropy = at::empty(targets.sizes(), acc);
  if (want) out.stats = at::empty({2, rows}, acc);
  out.where.logits = logits;
  if (rows == 0) return out;
  std::optional<Rows> r = rows_of(logits);
  out.where = r.has_value() ? *r : *rows_of(logits.contiguous());
  size_t bytes = 0;
  check(ti_logprobs_workspace(rows, vocab, dtype, &bytes), "token_logprobs");
  const at::Tensor ws = bytes > 0 ? workspace(bytes, logits) : at::Tensor();
  check(ti_logprobs(ptr(out.where.logits), targets.data_ptr<int64_t>(), ptr(out.logp), ptr(out.entropy), ptr(out.stats),
                    rows, vocab, out.where.inner, out.where.outer_stride, out.where.row_stride, ignore_index,
                    temperature, dtype, ptr(ws), bytes, stream_of(logits)),
        "token_logprobs");
  return out;
}

struct LogprobsFn : public torch::autograd::Function<LogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& targets,
                               double temperature, int64_t ignore_index, bool entropy) {
    Logprobs out = logprobs_of(logits, targets, temperature, ignore_index, entropy, true);
    ctx->set_materialize_grads(false);  // (an output that no gradient comes for costs no launch)
    ctx->save_for_backward({out.where.logits, targets, out.stats, out.entropy});
    ctx->saved_data["i"] = ignore_index;
    ctx->saved_data["t"] = temperature;
    if (entropy) return {out.logp, out.entropy};
    return {out.logp};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("token_logprobs");
    variable_list none(5);
    const at::Tensor g = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    const at::Tensor ge = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    if (!g.defined() && !ge.defined()) return none;
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &up = g.defined() ? g : ge;
    const c10::DeviceGuard guard(up.device());
    const int64_t rows = up.numel();
    TORCH_CHECK(logits.device() == up.device() && logits.dim() == up.dim() + 1 &&
                    logits.sizes().slice(0, up.dim()) == up.sizes() &&
                    (logits.scalar_type() == at::kDouble) == (up.scalar_type() == at::kDouble),
                "torchisotonic_amd.token_logprobs backward: the saved logits came back with another size, type or device");
    at::Tensor out = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
    none[0] = out;
    if (rows == 0) return none;
    const at::Tensor t = saved_as(saved[1], rows, at::kLong, up.device(), "token_logprobs");
    const at::Tensor stats = saved_as(saved[2], 2 * rows, up.scalar_type(), up.device(), "token_logprobs");
    const at::Tensor h = ge.defined() ? saved_as(saved[3], rows, up.scalar_type(), up.device(), "token_logprobs") : at::Tensor();
    std::optional<Rows> r = rows_of(logits);
    const Rows where = r.has_value() ? *r : *rows_of(logits.contiguous());
    check(ti_logprobs_bwd(ptr(where.logits), t.data_ptr<int64_t>(), ptr(stats), ptr(h), ptr(g), ptr(ge), ptr(out), rows,
                          logits.size(-1), where.inner, where.outer_stride, where.row_stride,
                          ctx->saved_data["i"].toInt(), ctx->saved_data["t"].toDouble(),
                          dtype_code(logits, "token_logprobs"), stream_of(logits)),
          "token_logprobs backward");
    return none;
  }
};

// (the entropy undefined, in Python None, where not wanted)
std::tuple<at::Tensor, at::Tensor> token_logprobs(const at::Tensor& logits, const at::Tensor& targets,
                                                  double temperature, int64_t ignore_index, bool entropy) {
  no_tangents({&logits}, "token_logprobs");
  if (!tracked(logits)) {
    const Logprobs out = logprobs_of(logits, targets, temperature, ignore_index, entropy, false);
    return {out.logp, out.entropy};
  }
  const variable_list out = LogprobsFn::apply(logits, targets, temperature, ignore_index, entropy);
  return {out[0], entropy ? out[1] : at::Tensor()};
}

// --- the losses --------------------------------------------------------------------------------

// The sequences of token arrays: [sequences, len], or packed with offsets, or (without) all one.
struct Sequences {
  int64_t total, count, len;
  const int64_t* offsets;
};

Sequences sequences_of(const at::Tensor& logps, const std::optional<at::Tensor>& offsets, const char* what) {
  TORCH_CHECK(logps.is_cuda() && logps.is_contiguous() && (logps.dim() == 1 || logps.dim() == 2),
              "torchisotonic_amd.", what, ": logps must be 1-D or [sequences, tokens], contiguous, on a ROCm device");
  if (offsets.has_value()) {
    TORCH_CHECK(logps.dim() == 1 && offsets->dim() == 1 && offsets->numel() >= 1 &&
                    offsets->scalar_type() == at::kLong && offsets->is_contiguous() &&
                    offsets->device() == logps.device(),
                "torchisotonic_amd.", what, ": offsets must be 1-D int64, contiguous, on logps' device, with 1-D logps");
    TORCH_CHECK(offsets->numel() > 1 || logps.numel() == 0, "torchisotonic_amd.", what, ": offsets must run from 0 to ",
                logps.numel());
    return {logps.numel(), offsets->numel() - 1, 0, offsets->data_ptr<int64_t>()};
  }
  if (logps.dim() == 1) return {logps.numel(), 1, logps.numel(), nullptr};
  return {logps.numel(), logps.size(0), logps.size(1), nullptr};
}

void check_like(const at::Tensor& logps, const std::optional<at::Tensor>& t, at::ScalarType type, const char* name,
                const char* what) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->sizes() == logps.sizes() && t->device() == logps.device() && t->scalar_type() == type &&
                  t->is_contiguous(),
              "torchisotonic_amd.", what, ": ", name, " must match logps");
}

struct Preference {
  at::Tensor loss, rewards, slopes;  // slopes undefined where not wanted
  Sequences seq;
};

// The checks and the launches of one call, with the slopes a backward spreads or without.
Preference preference_of(const at::Tensor& logps, const std::optional<at::Tensor>& ref,
                         const std::optional<at::Tensor>& offsets, const std::optional<at::Tensor>& mask, int64_t kind,
                         double beta, double smoothing, bool average, int64_t reduction, bool want) {
  const Sequences s = sequences_of(logps, offsets, "preference_loss");
  TORCH_CHECK(s.count % 2 == 0, "torchisotonic_amd.preference_loss: the sequences must be pairs");
  check_like(logps, ref, logps.scalar_type(), "reference", "preference_loss");
  check_like(logps, mask, at::kBool, "mask", "preference_loss");
  const int64_t pairs = s.count / 2;
  const bool each = reduction == TI_REDUCE_NONE;
  const c10::DeviceGuard guard(logps.device());
  const auto options = logps.options().requires_grad(false);
  Preference out;
  out.seq = s;
  out.rewards = at::empty({2, pairs}, options);
  if (want) out.slopes = at::empty({s.count}, options);
  if (pairs == 0) {
    out.loss = each ? at::empty({0}, options) : at::zeros({}, options);
    return out;
  }
  out.loss = each ? at::empty({pairs}, options) : at::empty({}, options);
  size_t bytes = 0;
  check(ti_preference_workspace(s.total, s.count, &bytes), "preference_loss");
  const at::Tensor ws = workspace(bytes, logps);
  char* rewards = static_cast<char*>(ptr(out.rewards));
  check(ti_preference(ptr(logps), ptr(ref), static_cast<const uint8_t*>(ptr(mask)), s.offsets, s.total, s.count, s.len,
                      static_cast<int>(kind), beta, smoothing, average ? 1 : 0, static_cast<int>(reduction),
                      ptr(out.loss), rewards, rewards + pairs * out.rewards.element_size(), ptr(out.slopes),
                      dtype_code(logps, "preference_loss"), ptr(ws), bytes, stream_of(logps)),
        "preference_loss");
  return out;
}

struct PreferenceFn : public torch::autograd::Function<PreferenceFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logps, const std::optional<at::Tensor>& ref,
                               const std::optional<at::Tensor>& offsets, const std::optional<at::Tensor>& mask,
                               int64_t kind, double beta, double smoothing, bool average, int64_t reduction) {
    const Preference out =
        preference_of(logps, ref, offsets, mask, kind, beta, smoothing, average, reduction, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({out.slopes, offsets.value_or(at::Tensor()), mask.value_or(at::Tensor())});
    c10::List<int64_t> p({out.seq.total, out.seq.count, out.seq.len, reduction == TI_REDUCE_NONE ? 1 : 0});
    for (const int64_t n : logps.sizes()) p.push_back(n);
    ctx->saved_data["p"] = p;
    ctx->mark_non_differentiable({out.rewards});
    return {out.loss, out.rewards};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("preference_loss");
    variable_list none(9);
    if (!grads[0].defined()) return none;
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
    const at::Tensor g = grads[0].contiguous();
    const c10::DeviceGuard guard(g.device());
    at::Tensor out = at::empty(at::IntArrayRef(p).slice(4), g.options());
    if (p[1] == 0) {
      out.zero_();
    } else {
      const at::Tensor slopes = saved_as(saved[0], p[1], g.scalar_type(), g.device(), "preference_loss");
      const at::Tensor offsets = saved[1].defined()
                                     ? saved_as(saved[1], p[1] + 1, at::kLong, g.device(), "preference_loss")
                                     : at::Tensor();
      const at::Tensor mask =
          saved[2].defined() ? saved_as(saved[2], p[0], at::kBool, g.device(), "preference_loss") : at::Tensor();
      check(ti_preference_bwd(static_cast<const uint8_t*>(ptr(mask)), static_cast<const int64_t*>(ptr(offsets)), p[0],
                              p[1], p[2], ptr(slopes), ptr(g), static_cast<int>(p[3]), ptr(out),
                              dtype_code(slopes, "preference_loss"), stream_of(slopes)),
            "preference_loss backward");
    }
    none[0] = out;
    return none;
  }
};

Three preference_loss(const at::Tensor& logps, const std::optional<at::Tensor>& ref,
                      const std::optional<at::Tensor>& offsets, const std::optional<at::Tensor>& mask, int64_t kind,
                      double beta, double smoothing, bool average, int64_t reduction) {
  no_tangents({&logps, some(ref)}, "preference_loss");
  if (!tracked(logps)) {
    const Preference out = preference_of(logps, ref, offsets, mask, kind, beta, smoothing, average, reduction, false);
    return {out.loss, out.rewards[0], out.rewards[1]};
  }
  const variable_list out = PreferenceFn::apply(logps, ref, offsets, mask, kind, beta, smoothing, average, reduction);
  const at::NoGradGuard untracked;
  return {out[0], out[1][0], out[1][1]};
}

// One call of the policy loss: the loss, kl and clip fraction into more, and the gradient into grad (if any).
struct PolicyCall {
  at::Tensor logps, old, advantages, ref, mask, offsets;
  double clip_low, clip_high, kl_coef;
  int64_t reduction;

  // The sequences, once every tensor is checked.
  Sequences checked() const {
    auto maybe = [](const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; };
    const Sequences s = sequences_of(logps, maybe(offsets), "policy_loss");
    check_like(logps, old, logps.scalar_type(), "old_logps", "policy_loss");
    check_like(logps, maybe(ref), logps.scalar_type(), "reference_logps", "policy_loss");
    check_like(logps, maybe(mask), at::kBool, "mask", "policy_loss");
    TORCH_CHECK((advantages.sizes() == logps.sizes() || (advantages.dim() == 1 && advantages.numel() == s.count)) &&
                    advantages.device() == logps.device() && advantages.scalar_type() == logps.scalar_type() &&
                    advantages.is_contiguous(),
                "torchisotonic_amd.policy_loss: advantages must be one a token or one a sequence, and match logps");
    return s;
  }

  void operator()(const Sequences& s, const at::Tensor& loss, const at::Tensor& more, const at::Tensor& grad) const {
    const bool each = advantages.sizes() == logps.sizes();
    size_t bytes = 0;
    check(ti_policy_workspace(s.total, s.count, &bytes), "policy_loss");
    const at::Tensor ws = workspace(bytes, logps);
    char* m = static_cast<char*>(more.data_ptr());
    check(ti_policy(ptr(logps), ptr(old), ptr(advantages), each ? 1 : 0, ptr(ref),
                    static_cast<const uint8_t*>(ptr(mask)), s.offsets, s.total, s.count, s.len, clip_low, clip_high,
                    kl_coef, static_cast<int>(reduction), ptr(loss), m, m + more.element_size(), ptr(grad),
                    dtype_code(logps, "policy_loss"), ptr(ws), bytes, stream_of(logps)),
          "policy_loss");
  }
};

// The forward writes the gradient with the loss, in the one read of the tokens, and the backward hands
// it out, times the upstream gradient (a kernel that leaves it as it is where that is one). A second
// backward of the same node computes it again.
struct PolicyFn : public torch::autograd::Function<PolicyFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logps, const at::Tensor& old,
                               const at::Tensor& advantages, const std::optional<at::Tensor>& ref,
                               const std::optional<at::Tensor>& offsets, const std::optional<at::Tensor>& mask,
                               double clip_low, double clip_high, double kl_coef, int64_t reduction, bool want) {
    const PolicyCall call{logps, old, advantages, ref.value_or(at::Tensor()), mask.value_or(at::Tensor()),
                          offsets.value_or(at::Tensor()), clip_low, clip_high, kl_coef, reduction};
    const Sequences s = call.checked();
    const c10::DeviceGuard guard(logps.device());
    // (the loss a tensor of its own: a view made here could not be changed in place by the caller)
    at::Tensor loss, more, grad;
    if (s.count == 0) {
      loss = at::zeros({}, logps.options());
      more = at::zeros({2}, logps.options());
      if (want) grad = at::zeros_like(logps);
    } else {
      loss = at::empty({}, logps.options());
      more = at::empty({2}, logps.options());
      if (want) grad = at::empty_like(logps);
      call(s, loss, more, grad);
    }
    if (want) {
      ctx->save_for_backward({logps, old, advantages, call.ref, call.mask, call.offsets});
      ctx->saved_data["grad"] = grad;
      ctx->saved_data["p"] = c10::List<double>(
          {clip_low, clip_high, kl_coef, static_cast<double>(reduction), static_cast<double>(s.total)});
    }
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({more});
    return {loss, more};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("policy_loss");
    variable_list none(11);
    if (!grads[0].defined()) return none;
    const at::Tensor g = grads[0].contiguous();
    const c10::DeviceGuard guard(g.device());
    at::Tensor grad;
    if (const auto held = ctx->saved_data.find("grad"); held != ctx->saved_data.end()) {
      grad = held->second.toTensor();
      ctx->saved_data.erase(held);
    } else {
      variable_list t = ctx->get_saved_variables();
      for (at::Tensor& saved : t)
        if (saved.defined()) saved = saved_as(saved, saved.numel(), saved.scalar_type(), g.device(), "policy_loss");
      const c10::List<double> p = ctx->saved_data["p"].toDoubleList();
      TORCH_CHECK(t[0].scalar_type() == g.scalar_type() && t[0].numel() == static_cast<int64_t>(p.get(4)),
                  "torchisotonic_amd.policy_loss backward: a saved tensor came back with another size or type");
      const PolicyCall call{t[0], t[1], t[2], t[3], t[4], t[5], p.get(0), p.get(1), p.get(2), static_cast<int64_t>(p.get(3))};
      const Sequences s = call.checked();
      grad = at::empty_like(t[0]);
      if (s.count == 0) grad.zero_();
      else call(s, at::empty({}, g.options()), at::empty({2}, g.options()), grad);
    }
    check(ti_policy_bwd(ptr(grad), grad.numel(), ptr(g), dtype_code(g, "policy_loss"), stream_of(g)),
          "policy_loss backward");
    none[0] = grad;
    return none;
  }
};

Three policy_loss(const at::Tensor& logps, const at::Tensor& old, const at::Tensor& advantages,
                  const std::optional<at::Tensor>& ref, const std::optional<at::Tensor>& offsets,
                  const std::optional<at::Tensor>& mask, double clip_low, double clip_high, double kl_coef,
                  int64_t reduction) {
  no_tangents({&logps, &old, &advantages, some(ref)}, "policy_loss");
  const variable_list out = PolicyFn::apply(logps, old, advantages, ref, offsets, mask, clip_low, clip_high, kl_coef,
                                            reduction, tracked(logps));
  const at::NoGradGuard untracked;
  return {out[0], out[1][0], out[1][1]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torchisotonic_amd, m) {
  m.def("token_logprobs(Tensor logits, Tensor targets, float temperature, int ignore_index, bool entropy) "
        "-> (Tensor, Tensor)",
        &token_logprobs);
  m.def("preference_loss(Tensor logps, Tensor? reference, Tensor? offsets, Tensor? mask, int kind, float beta, "
        "float smoothing, bool average, int reduction) -> (Tensor, Tensor, Tensor)",
        &preference_loss);
  m.def("policy_loss(Tensor logps, Tensor old, Tensor advantages, Tensor? reference, Tensor? offsets, Tensor? mask, "
        "float clip_low, float clip_high, float kl_coef, int reduction) -> (Tensor, Tensor, Tensor)",
        &policy_loss);
}
