// token_logprobs (logprobs.cu) as one differentiable function of the logits. The node is C++ so that a
// small fine-tuning batch is not bound by the interpreter: forward and backward of 4 rows took 80 us
// of host time as a Python node.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace hrm {

std::vector<at::Tensor> token_logprobs_fwd(const at::Tensor& logits, const at::Tensor& tokens, int64_t k, bool keep);
void token_logprobs_bwd(const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& stats,
                        const c10::optional<at::Tensor>& g_lp, const c10::optional<at::Tensor>& g_h,
                        const at::Tensor& grad);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens, int64_t k) {
    auto out = token_logprobs_fwd(logits, tokens, k, true);
    ctx->save_for_backward({logits, tokens, out.back()});
    out.pop_back();
    ctx->set_materialize_grads(false);
    if (k > 0) ctx->mark_non_differentiable({out[2], out[3]});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!grads[0].defined() && !grads[1].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto rows = [](const at::Tensor& g) {
      return g.defined() ? c10::optional<at::Tensor>(g.detach().contiguous()) : c10::nullopt;
    };
    at::Tensor grad = at::empty_like(saved[0].detach());
    token_logprobs_bwd(saved[0].detach(), saved[1], saved[2], rows(grads[0]), rows(grads[1]), grad);
    if (at::GradMode::is_enabled()) {  // a graph of the gradient: an error where it is differentiated
      auto once = std::make_shared<torch::autograd::DelayedError>("token_logprobs is differentiable once", 1);
      variable_list in{grad};
      in[0].set_requires_grad(true);
      grad = (*once)(std::move(in))[0];
    }
    return {grad, at::Tensor(), at::Tensor()};
  }
};

}  // namespace

// logprob, entropy and for k > 0 top_ids, top_logprobs of logits [N, V]; differentiable where the logits are.
std::vector<at::Tensor> token_logprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t k) {
  // a dual tensor need not require a gradient, and its tangent would be lost in the kernel's outputs
  TORCH_CHECK(!logits._fw_grad(/*level=*/0).defined(), "token_logprobs has no forward-mode derivative");
  if (at::GradMode::is_enabled() && logits.requires_grad()) return TokenLogprobs::apply(logits, tokens, k);
  return token_logprobs_fwd(logits, tokens, k, false);
}

}  // namespace hrm
