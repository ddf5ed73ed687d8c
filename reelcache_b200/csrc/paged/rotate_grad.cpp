// The multi-axis rotation as a differentiable function. It is linear and orthogonal, so its gradient is the same
// rotation turned back, which is again this function (gradients of any order). The node lives in C++ because a training
// step calls it once per layer on tensors that take a few microseconds: a Python node costs several times that.
#include <torch/extension.h>

#include <vector>

namespace rc {

bool rotary_rows_ok(const at::Tensor& t);
void rotate_launch(const at::Tensor& q, at::Tensor& q_out, const at::Tensor& k, at::Tensor& k_out,
                   const at::Tensor& positions, const at::Tensor& turns, const std::vector<int64_t>& sections,
                   bool halves, double sign);

namespace {

at::Tensor dense_rows(const at::Tensor& t) { return !t.defined() || rotary_rows_ok(t) ? t : t.contiguous(); }

// The rotation of one or two tensors (the second may be undefined; then one comes back).
std::vector<at::Tensor> rotated(const at::Tensor& first, const at::Tensor& second, const at::Tensor& positions,
                                const at::Tensor& turns, const std::vector<int64_t>& sections, bool halves, double sign) {
  const at::Tensor x = dense_rows(first), y = dense_rows(second);
  std::vector<at::Tensor> out = {at::empty(x.sizes(), x.options())};
  at::Tensor none;
  if (y.defined()) out.push_back(at::empty(y.sizes(), y.options()));
  rotate_launch(x, out[0], y, y.defined() ? out[1] : none, positions, turns, sections, halves, sign);
  return out;
}

struct Rotate : public torch::autograd::Function<Rotate> {
  static std::vector<at::Tensor> forward(torch::autograd::AutogradContext* ctx, const at::Tensor& first,
                                         const c10::optional<at::Tensor>& second, const at::Tensor& positions,
                                         const at::Tensor& turns, std::vector<int64_t> sections, bool halves,
                                         double sign) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, turns});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["halves"] = halves;
    ctx->saved_data["sign"] = sign;
    return rotated(first, second.value_or(at::Tensor()), positions, turns, sections, halves, sign);
  }

  static std::vector<at::Tensor> backward(torch::autograd::AutogradContext* ctx, std::vector<at::Tensor> grads) {
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> sections = ctx->saved_data["sections"].toIntVector();
    const bool halves = ctx->saved_data["halves"].toBool();
    const double sign = -ctx->saved_data["sign"].toDouble();
    std::vector<at::Tensor> out(7);  // one per input; only the rotated tensors have a gradient
    std::vector<int> with;           // outputs that were used
    for (int i = 0; i < static_cast<int>(grads.size()); ++i)
      if (grads[i].defined()) with.push_back(i);
    if (with.empty()) return out;
    c10::optional<at::Tensor> second;
    if (with.size() > 1) second = grads[with[1]];
    const std::vector<at::Tensor> back = apply(grads[with[0]], second, saved[0], saved[1], sections, halves, sign);
    for (size_t i = 0; i < with.size(); ++i) out[with[i]] = back[i];
    return out;
  }
};

}  // namespace

std::vector<at::Tensor> rotate(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions,
                               const at::Tensor& turns, const std::vector<int64_t>& sections, bool halves) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad())))
    return Rotate::apply(q, k, positions, turns, sections, halves, 1.0);
  return rotated(q, k.value_or(at::Tensor()), positions, turns, sections, halves, 1.0);
}

}  // namespace rc
