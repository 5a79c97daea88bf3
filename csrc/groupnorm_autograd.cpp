// Group norm's node in autograd. It is C++ and not a Python function because
// the smallest calls are all launch: a backward pass that has to come back to
// Python's thread costs more than its kernels.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <vector>

namespace eg {

std::vector<torch::Tensor> group_norm_fwd(torch::Tensor, torch::Tensor,
                                          torch::Tensor, long, double, long,
                                          c10::optional<torch::Tensor>);
torch::Tensor group_norm_only(torch::Tensor, torch::Tensor, torch::Tensor,
                              long, double, long,
                              c10::optional<torch::Tensor>);
std::vector<torch::Tensor> group_norm_bwd(
    torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor,
    long, long, c10::optional<torch::Tensor>, c10::optional<torch::Tensor>,
    bool, bool, c10::optional<torch::Tensor>, c10::optional<torch::Tensor>);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

c10::optional<torch::Tensor> if_defined(const torch::Tensor& t) {
  return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt;
}

// a result that raises where it is differentiated again
torch::Tensor once(const torch::Tensor& t) {
  auto fake = t.detach();
  fake.set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "group_norm has no second derivative", 1);
  return (*node)({fake})[0];
}

// Leaves with gradients already there (views into the flat space) get theirs
// added in place, like those of the other layers; a standalone parameter gets
// its gradient from autograd. The leaves are kept, and not their gradients:
// what .grad is when the backward pass runs is what counts, for it may have
// been replaced or cleared since.
struct Direct {
  torch::Tensor gamma, beta;
};

bool ready(const torch::Tensor& t) {
  return t.requires_grad() && t.is_leaf() && t.grad().defined();
}

void give(const torch::Tensor& leaf, const torch::Tensor& d) {
  auto& grad = leaf.mutable_grad();
  if (grad.defined()) grad.add_(d);
  else grad = d;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Variable forward(AutogradContext* ctx, const Variable& x,
                          const Variable& gamma, const Variable& beta,
                          const c10::optional<Variable>& residual,
                          const Direct& direct, long groups, double eps,
                          long act) {
    auto out = group_norm_fwd(x, gamma, beta, groups, eps, act, residual);
    // a ReLU's gradient needs the bits that the pass left (out[2]) in the
    // residual's place, and without an activation it needs neither
    ctx->save_for_backward({x, gamma, beta, out[1],
                            act == 2 && residual ? *residual : torch::Tensor(),
                            out[2]});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["groups"] = (int64_t)groups;
    ctx->saved_data["act"] = (int64_t)act;
    if (direct.gamma.defined()) {
      ctx->saved_data["gamma"] = direct.gamma;
      ctx->saved_data["beta"] = direct.beta;
    }
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const long groups = ctx->saved_data["groups"].toInt();
    const long act = ctx->saved_data["act"].toInt();
    const bool want_x = ctx->needs_input_grad(0);
    const bool want_g = ctx->needs_input_grad(1);
    const bool want_b = ctx->needs_input_grad(2);
    const bool want_r = ctx->saved_data["residual"].toBool() &&
                        ctx->needs_input_grad(3);
    const auto kept = ctx->saved_data.find("gamma");
    const bool direct = kept != ctx->saved_data.end();
    torch::Tensor gamma, beta;
    c10::optional<torch::Tensor> dgamma, dbeta;
    if (direct) {
      gamma = kept->second.toTensor();
      beta = ctx->saved_data["beta"].toTensor();
      if (gamma.grad().defined() && beta.grad().defined()) {
        dgamma = gamma.grad();
        dbeta = beta.grad();
      }
    }
    const bool again = at::GradMode::is_enabled();
    torch::Tensor dy;
    std::vector<torch::Tensor> d;
    {
      at::NoGradGuard no_grad;
      dy = grads[0].contiguous();
      d = group_norm_bwd(dy, saved[0], saved[3], saved[1], saved[2], groups,
                         act, if_defined(saved[4]), if_defined(saved[5]),
                         want_x, want_r && act, dgamma, dbeta);
      if (direct && !dgamma) {
        give(gamma, d[2]);
        give(beta, d[3]);
      }
    }
    if (want_r && !act) d[1] = dy;
    variable_list out(8);
    if (want_x) out[0] = d[0];
    if (want_g && !direct) out[1] = d[2];
    if (want_b && !direct) out[2] = d[3];
    if (want_r) out[3] = d[1];
    if (again)
      for (auto& t : out)
        if (t.defined()) t = once(t);
    return out;
  }
};

}  // namespace

torch::Tensor group_norm(torch::Tensor x, torch::Tensor gamma,
                         torch::Tensor beta,
                         c10::optional<torch::Tensor> residual, long groups,
                         double eps, long act) {
  const torch::Tensor res = residual ? *residual : torch::Tensor();
  // a tangent would be dropped wherever the call does not go through the node
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const auto* t : std::initializer_list<const torch::Tensor*>{
             &x, &gamma, &beta, &res})
      TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                  "group_norm has no forward-mode derivative");
  const bool wanted =
      at::GradMode::is_enabled() &&
      (x.requires_grad() || gamma.requires_grad() || beta.requires_grad() ||
       (res.defined() && res.requires_grad()));
  if (!wanted) return group_norm_only(x, gamma, beta, groups, eps, act, residual);
  const bool in_place = ready(gamma) && ready(beta);
  const bool captured = c10::hip::currentStreamCaptureStatusMayInitCtx() !=
                        c10::hip::CaptureStatus::None;
  if (captured) {
    auto refuse = [](const torch::Tensor& t) {
      TORCH_CHECK(!(t.defined() && t.requires_grad() && t.is_leaf()),
                  "group_norm: a captured backward pass cannot accumulate "
                  "into this leaf; give gamma and beta pre-allocated "
                  "gradients, both of them, and make x and the residual in "
                  "the captured region");
    };
    refuse(x);
    refuse(res);
    if (!in_place) {
      refuse(gamma);
      refuse(beta);
    }
  }
  Direct direct;
  if (in_place) {
    direct = {gamma, beta};
    // Autograd then has nothing to bring gamma and beta, and is not told of
    // them where x or the residual carries the graph.
    const bool carried =
        x.requires_grad() || (res.defined() && res.requires_grad());
    if (carried || captured) {
      gamma = gamma.detach();
      beta = beta.detach();
    }
    // In a captured region a leaf of the call's own carries it: the engine
    // ends by waiting for its leaves' streams, and one that an eager graph
    // holds has that graph's, which is not captured.
    if (captured && !carried) gamma.set_requires_grad(true);
  }
  return GroupNorm::apply(x, gamma, beta, residual, direct, groups, eps, act);
}

}  // namespace eg
