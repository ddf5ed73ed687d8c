// The multi-axis rotation as a differentiable function. It is linear and orthogonal, so its gradient is the same
// rotation turned back, which is again this function (gradients of any order). The node is written out in C++ because a
// training step calls it once per layer on tensors that take a few microseconds: a Python function costs several times
// that, and a generic C++ one a dictionary per call.
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <memory>
#include <vector>

#include "rope_plan.h"

namespace rc {

bool rotary_rows_ok(const at::Tensor& t);
void rotate_launch(const at::Tensor& q, at::Tensor& q_out, const at::Tensor& k, at::Tensor& k_out,
                   const at::Tensor& positions, const RopePlan& plan, double sign);

namespace {

using torch::autograd::Variable;
using torch::autograd::variable_list;

at::Tensor dense_rows(const at::Tensor& t) { return !t.defined() || rotary_rows_ok(t) ? t : t.contiguous(); }

variable_list turned(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                     const std::shared_ptr<RopePlan>& plan, double sign);

struct RotateBackward : public torch::autograd::Node {
  std::shared_ptr<RopePlan> plan;
  torch::autograd::SavedVariable positions;
  double sign = 1.0;

  variable_list apply(variable_list&& grads) override {
    // an output that was not used has no gradient; an input that needs none gets none
    at::Tensor q = grads[0], k = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!task_should_compute_output(0)) q = at::Tensor();
    if (!task_should_compute_output(1)) k = at::Tensor();
    if (!q.defined() && !k.defined()) return variable_list(2);
    const at::Tensor at = positions.unpack();
    return turned(q, k, at, plan, -sign);
  }
  void release_variables() override { positions.reset_data(); }
  std::string name() const override { return "RotateBackward"; }
};

variable_list turned(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                     const std::shared_ptr<RopePlan>& plan, double sign) {
  refuse_tangents({&q, &k, &positions}, "rotate");
  RC_CHECK(!torch::autograd::compute_requires_grad(positions), "rotate has no gradient with respect to positions");
  std::shared_ptr<RotateBackward> node;
  if (torch::autograd::compute_requires_grad(q, k)) {
    node = std::shared_ptr<RotateBackward>(new RotateBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k));
    node->plan = plan;
    node->positions = torch::autograd::SavedVariable(positions, false);
    node->sign = sign;
  }
  variable_list out(2);
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor x = dense_rows(q), y = dense_rows(k);
    if (x.defined()) out[0] = at::empty(x.sizes(), x.options());
    if (y.defined()) out[1] = at::empty(y.sizes(), y.options());
    rotate_launch(x, out[0], y, out[1], positions, *plan, sign);
  }
  if (node) {
    for (at::Tensor& t : out) {
      if (t.defined()) torch::autograd::set_history(t, node);
      else node->add_input_metadata(torch::autograd::Node::undefined_input());
    }
  }
  return out;
}

}  // namespace

std::pair<at::Tensor, c10::optional<at::Tensor>> rotate(const at::Tensor& q, const c10::optional<at::Tensor>& k,
                                                        const at::Tensor& positions, std::shared_ptr<RopePlan> plan) {
  variable_list out = turned(q, k.value_or(at::Tensor()), positions, plan, 1.0);
  return {out[0], out[1].defined() ? c10::optional<at::Tensor>(out[1]) : c10::nullopt};
}

}  // namespace rc
