// torch operators on a decoder's logits over the C ABI of libkvm_amd.so
// (include/kvm_amd.h): kvm_amd::sample_tokens, kvm_amd::top_logits and
// kvm_amd::head_loss with its autograd function.  Host code only: they check
// their tensors, describe the logits' rows as they lie in memory, and call the
// library on torch's current stream of the logits' device.  Invalid arguments
// are raised as ValueError, other failures as RuntimeError.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <vector>

#include "../../include/kvm_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxVocab = 1 << 20;

void check(int rc, const char *what) {
  if (rc == KVM_OK) return;
  if (rc == KVM_EINVAL) TORCH_CHECK_VALUE(false, what, ": ", kvm_last_error());
  TORCH_CHECK(false, what, ": ", kvm_last_error());
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// The graph capture that the current stream of t's device is part of (0: none).
int64_t capture_of(const Tensor &t) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const auto stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  if (hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? int64_t(id) : 0;
}

int64_t type_code(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return KVM_BF16;
    case at::kHalf: return KVM_F16;
    case at::kFloat: return KVM_F32;
    default: TORCH_CHECK_VALUE(false, name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  }
  return -1;
}

// Rows of a tensor [..., V] in the order of its leading axes, as it lies in
// memory where V is contiguous and the leading axes collapse to two.
bool row_layout(const Tensor &t, kvm_logits *L) {
  const auto sizes = t.sizes(), strides = t.strides();
  const int64_t dims = t.dim();
  if (sizes[dims - 1] > 1 && strides[dims - 1] != 1) return false;
  int64_t n[2] = {1, 1}, st[2] = {0, 0};  // inner, outer
  int found = 0;
  for (int64_t i = dims - 2; i >= 0; --i) {
    if (sizes[i] == 1) continue;
    if (found && strides[i] == n[found - 1] * st[found - 1]) {
      n[found - 1] *= sizes[i];
    } else if (found == 2) {
      return false;
    } else {
      n[found] = sizes[i];
      st[found] = strides[i];
      ++found;
    }
  }
  L->inner = n[0];
  L->s_inner = st[0];
  L->outer = n[1];
  L->s_outer = st[1];
  return true;
}

// The descriptor of logits and, in *held, the tensor it points to (a copy
// where the layout needs one).
kvm_logits rows_of(const Tensor &t, const char *name, Tensor *held) {
  kvm_logits L{};
  L.dtype = type_code(t, name);
  TORCH_CHECK_VALUE(t.dim() >= 1, name, " must have a vocabulary axis");
  TORCH_CHECK(t.is_cuda(), name, " must be a ROCm device tensor");
  L.vocab = t.size(-1);
  TORCH_CHECK_VALUE(L.vocab >= 1 && L.vocab <= kMaxVocab, name, ": the vocabulary must have 1 to ", kMaxVocab,
                    " entries, got ", L.vocab);
  *held = t;
  if (!row_layout(t, &L)) {
    *held = t.contiguous();
    row_layout(*held, &L);
  }
  L.data = held->data_ptr();
  return L;
}

at::IntArrayRef rows_shape(const Tensor &t) { return t.sizes().slice(0, t.dim() - 1); }

void check_rows(const Tensor &t, const Tensor &logits, const char *name) {
  TORCH_CHECK_VALUE(t.sizes() == rows_shape(logits), name, " must have the rows' shape ", rows_shape(logits),
                    ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == logits.device(), name, " must be on the logits' device");
}

// A setting of every row, as the kernel reads it; undefined where it is a number.
Tensor setting(const OptTensor &v, const Tensor &logits, const char *name, at::ScalarType type) {
  if (!v.has_value()) return {};
  TORCH_CHECK_VALUE(v->device() == logits.device(), name, " must be on the logits' device");
  if (v->dim() == 0) return v->to(type).expand(rows_shape(logits)).contiguous();
  check_rows(*v, logits, name);
  return v->to(type).contiguous();
}

template <class T>
const T *data_of(const Tensor &t) {
  return t.defined() ? static_cast<const T *>(t.data_ptr()) : nullptr;
}

std::tuple<Tensor, Tensor> sample_tokens(const Tensor &logits, const Tensor &uniforms, const OptTensor &temperature,
                                         const OptTensor &top_k, const OptTensor &top_p, const OptTensor &min_p,
                                         double temperature_all, int64_t top_k_all, double top_p_all,
                                         double min_p_all) {
  Tensor held;
  kvm_sample_desc d{};
  d.logits = rows_of(logits, "logits", &held);
  check_rows(uniforms, logits, "uniforms");
  const c10::DeviceGuard guard(logits.device());
  const Tensor u = uniforms.to(at::kFloat).contiguous(), t = setting(temperature, logits, "temperature", at::kFloat),
               k = setting(top_k, logits, "top_k", at::kInt), p = setting(top_p, logits, "top_p", at::kFloat),
               m = setting(min_p, logits, "min_p", at::kFloat);
  const Tensor tokens = at::empty(rows_shape(logits), logits.options().dtype(at::kLong));
  const Tensor logprobs = at::empty(rows_shape(logits), logits.options().dtype(at::kFloat));
  d.uniforms = data_of<float>(u);
  d.temperature = data_of<float>(t);
  d.top_k = data_of<int32_t>(k);
  d.top_p = data_of<float>(p);
  d.min_p = data_of<float>(m);
  d.temperature_all = temperature_all;
  d.top_k_all = top_k_all;
  d.top_p_all = top_p_all;
  d.min_p_all = min_p_all;
  d.tokens = tokens.data_ptr<int64_t>();
  d.logprobs = logprobs.data_ptr<float>();
  if (tokens.numel()) check(kvm_sample(&d, stream_of(logits)), "sample_tokens");
  return {tokens, logprobs};
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor &logits, int64_t k, double temperature) {
  Tensor held;
  const kvm_logits L = rows_of(logits, "logits", &held);
  TORCH_CHECK_VALUE(k >= 1 && k <= L.vocab, "k must be in [1, ", L.vocab, "], got ", k);
  const c10::DeviceGuard guard(logits.device());
  std::vector<int64_t> shape = rows_shape(logits).vec();
  const Tensor rest = at::empty(shape, logits.options().dtype(at::kFloat));
  shape.push_back(k);
  const Tensor values = at::empty(shape, logits.options());
  const Tensor indices = at::empty(shape, logits.options().dtype(at::kLong));
  if (rest.numel())
    check(kvm_top_logits(&L, k, temperature, values.data_ptr(), indices.data_ptr<int64_t>(), rest.data_ptr<float>(),
                         stream_of(logits)),
          "top_logits");
  return {values, indices, rest};
}

enum Reduction : int64_t { kMean = 0, kSum = 1, kNone = 2 };

struct LossArgs {
  Tensor labels, values, indices, rest;  // checked; undefined where absent
  double temperature, label_weight;
  int64_t ignore_index, reduction;
};

// A tensor shaped as the logits whose rows start at the same offset modulo 16
// bytes as the logits' rows (the kernel stores it in the chunks it loads), with
// as little padding between them as that takes.
Tensor gradient_like(const Tensor &logits, const kvm_logits &L, int64_t *g_outer, int64_t *g_inner,
                     bool strides_only = false) {
  const int64_t size = logits.element_size(), n = 16 / size;
  auto mod = [n](int64_t v) { return ((v % n) + n) % n; };
  const int64_t gi = L.inner > 1 ? L.vocab + mod(L.s_inner - L.vocab) : L.vocab;
  const int64_t go = L.outer > 1 ? L.inner * gi + mod(L.s_outer - L.inner * gi) : L.inner * gi;
  const int64_t offset = int64_t(reinterpret_cast<uintptr_t>(L.data) % 16) / size;
  *g_outer = go;
  *g_inner = gi;
  if (strides_only) return {};
  if (gi == L.vocab && go == L.inner * gi && offset == 0) return at::empty(logits.sizes(), logits.options());
  return at::empty({offset + L.outer * go}, logits.options())
      .as_strided({L.outer, L.inner, L.vocab}, {go, gi, 1}, offset)
      .view(logits.sizes());
}

// The loss, and with grad its gradient for an upstream gradient of one;
// *row_losses receives the losses of the rows, and behind them the scratch of
// a mean.  With upstream, *grad and *row_losses are those of such a call, and
// the gradient is made again times upstream; the result is then nothing.
Tensor run_loss(const Tensor &logits, const LossArgs &a, Tensor *grad, Tensor *row_losses,
                const Tensor &upstream = {}) {
  const c10::DeviceGuard guard(logits.device());
  Tensor held;
  kvm_head_loss_desc d{};
  d.logits = rows_of(logits, "logits", &held);
  const int64_t rows = d.logits.outer * d.logits.inner;
  d.labels = data_of<int64_t>(a.labels);
  d.ignore_index = a.ignore_index;
  d.label_weight = a.label_weight;
  if (a.values.defined()) {
    d.k = a.values.size(-1);
    d.t_values = a.values.data_ptr();
    d.t_dtype = type_code(a.values, "teacher values");
    d.t_indices = data_of<int64_t>(a.indices);
    d.t_rest = data_of<float>(a.rest);
  }
  d.temperature = a.temperature;
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor loss;
  Tensor &per_row = *row_losses;
  if (!upstream.defined() || a.reduction == kNone)  // the losses a caller got are left as they are
    per_row = a.reduction == kNone ? at::empty(rows_shape(logits), f32) : at::empty({rows + 1}, f32);
  d.row_loss = per_row.data_ptr<float>();
  if (a.reduction != kNone) {
    if (!upstream.defined()) {
      loss = at::empty({}, f32);
      d.loss = loss.data_ptr<float>();
    }
    if (a.reduction == kMean) d.inv_count = d.row_loss + rows;
  } else {
    loss = per_row;
  }
  if (grad) {
    const Tensor fresh = gradient_like(logits, d.logits, &d.g_outer, &d.g_inner, upstream.defined());
    if (fresh.defined()) *grad = fresh;
    d.grad = grad->data_ptr();
    d.upstream = data_of<float>(upstream);
    d.upstream_stride = upstream.defined() && upstream.dim() ? 1 : 0;
  }
  check(kvm_head_loss(&d, stream_of(logits)), "head_loss");
  return loss;
}

class HeadLoss : public torch::autograd::Function<HeadLoss> {
 public:
  // The gradient for an upstream gradient of one is made with the loss, while
  // a row is in registers, and kept for the backward.
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &logits, const LossArgs &a) {
    Tensor grad, rows;
    const Tensor loss = run_loss(logits, a, &grad, &rows);
    ctx->save_for_backward({logits, a.labels, a.values, a.indices, a.rest});
    ctx->saved_data["grad"] = grad;
    if (a.reduction != kNone && logits.scalar_type() == at::kHalf) ctx->saved_data["rows"] = rows;
    ctx->saved_data["capture"] = capture_of(logits);
    ctx->saved_data["temperature"] = a.temperature;
    ctx->saved_data["label_weight"] = a.label_weight;
    ctx->saved_data["ignore_index"] = a.ignore_index;
    ctx->saved_data["reduction"] = a.reduction;
    return loss;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list ups) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0];
    torch::autograd::variable_list out(2);
    if (!ups[0].defined()) return out;
    Tensor grad;
    {
      const at::AutoGradMode no_grad(false);
      const c10::DeviceGuard guard(logits.device());
      const LossArgs a{saved[1], saved[2], saved[3], saved[4], ctx->saved_data["temperature"].toDouble(),
                       ctx->saved_data["label_weight"].toDouble(), ctx->saved_data["ignore_index"].toInt(),
                       ctx->saved_data["reduction"].toInt()};
      auto it = ctx->saved_data.find("grad");
      Tensor rows;
      if (auto kept = ctx->saved_data.find("rows"); kept != ctx->saved_data.end()) rows = kept->second.toTensor();
      if (it == ctx->saved_data.end()) {  // a retained graph, again
        run_loss(logits, a, &grad, &rows);
      } else if (ctx->saved_data["capture"].toInt() == capture_of(logits)) {
        grad = it->second.toTensor();  // handed out once, as what is below may change it
        ctx->saved_data.erase(it);
      } else {
        // A copy where the loss or the gradient is captured without the other,
        // of which one may run again without the other.
        int64_t outer, inner;
        Tensor held;
        grad = gradient_like(logits, rows_of(logits, "logits", &held), &outer, &inner);
        grad.copy_(it->second.toTensor());
      }
      const Tensor up = ups[0].to(at::kFloat).contiguous();
      if (grad.scalar_type() == at::kHalf) {
        // fp16 ends at 2^-24, where the gradient of a mean over a batch often
        // lies, and a loss scaled against that has its factor here: the gradient
        // is made again, rounded with the factor in it.  The traffic is the same.
        run_loss(logits, a, &grad, &rows, up);
      } else {
        Tensor held;
        const kvm_logits L = rows_of(grad, "gradient", &held);
        check(kvm_scale_rows(&L, up.data_ptr<float>(), up.dim() ? 1 : 0, stream_of(grad)), "head_loss backward");
      }
    }
    if (at::GradMode::is_enabled()) {
      auto twice = std::make_shared<torch::autograd::DelayedError>(
          "the losses on logits are differentiable once: their gradient has no gradient", 1);
      out[0] = (*twice)({grad.detach().requires_grad_(true)})[0];
    } else {
      out[0] = grad;
    }
    return out;
  }
};

Tensor head_loss(const Tensor &logits, const OptTensor &labels, const OptTensor &t_values, const OptTensor &t_indices,
                 const OptTensor &t_rest, double temperature, double label_weight, int64_t ignore_index,
                 int64_t reduction) {
  Tensor held;
  rows_of(logits, "logits", &held);  // its checks; a copy, where one is needed, is differentiable
  TORCH_CHECK_VALUE(reduction >= kMean && reduction <= kNone, "unknown reduction");
  LossArgs a{{}, {}, {}, {}, temperature, label_weight, ignore_index, reduction};
  if (labels.has_value()) {
    TORCH_CHECK_VALUE(labels->scalar_type() == at::kLong || labels->scalar_type() == at::kInt,
                      "labels must be int64 or int32, got ", labels->scalar_type());
    check_rows(*labels, logits, "labels");
    a.labels = labels->to(at::kLong).contiguous();
  }
  if (t_values.has_value()) {
    TORCH_CHECK_VALUE(t_indices.has_value(), "a teacher needs indices");
    type_code(*t_values, "teacher values");
    TORCH_CHECK_VALUE(t_indices->scalar_type() == at::kLong || t_indices->scalar_type() == at::kInt,
                      "teacher indices must be int64 or int32, got ", t_indices->scalar_type());
    TORCH_CHECK_VALUE(t_values->dim() == logits.dim() && rows_shape(*t_values) == rows_shape(logits) &&
                          t_indices->sizes() == t_values->sizes(),
                      "teacher values and indices must have the rows' shape ", rows_shape(logits),
                      " and one more axis, got ", t_values->sizes(), " and ", t_indices->sizes());
    TORCH_CHECK_VALUE(t_values->size(-1) >= 1, "a teacher needs one or more values per row");
    TORCH_CHECK_VALUE(t_values->device() == logits.device() && t_indices->device() == logits.device(),
                      "the teacher's tensors must be on the logits' device");
    a.values = t_values->detach().contiguous();
    a.indices = t_indices->to(at::kLong).contiguous();
    if (t_rest.has_value()) {
      check_rows(*t_rest, logits, "the teacher's rest");
      a.rest = t_rest->detach().to(at::kFloat).contiguous();
    }
  }
  const bool differentiable = at::GradMode::is_enabled() && logits.requires_grad();
  if (logits.numel() == 0) {  // no rows: an empty loss, or 0, that a graph still reaches
    const Tensor empty = logits.to(at::kFloat).sum(-1);
    return reduction == kNone ? empty : empty.sum();
  }
  if (differentiable)
    return HeadLoss::apply(held, a);
  const at::AutoGradMode no_grad(false);
  Tensor rows;
  return run_loss(held, a, nullptr, &rows);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(kvm_amd, m) {
  m.def(
      "sample_tokens(Tensor logits, Tensor uniforms, Tensor? temperature, Tensor? top_k, Tensor? top_p, "
      "Tensor? min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all) -> (Tensor, Tensor)",
      sample_tokens);
  m.def("top_logits(Tensor logits, int k, float temperature) -> (Tensor, Tensor, Tensor)", top_logits);
  m.def(
      "head_loss(Tensor logits, Tensor? labels, Tensor? t_values, Tensor? t_indices, Tensor? t_rest, "
      "float temperature, float label_weight, int ignore_index, int reduction) -> Tensor",
      head_loss);
}
