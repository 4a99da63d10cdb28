"""Training through ``token_logprobs``: the GPU head's logits are differentiable."""
import pytest
import torch

from gpu_utils import assert_close, random_packing

pytestmark = pytest.mark.gpu


def _model(device):
    from hrm_text_b200.runtime.factory import arch_preset, build_model
    cfg = arch_preset("hrm", "L") | dict(n_layers=2, hidden_size=256, num_heads=2, H_cycles=1, L_cycles=1, bp_max_steps=2,
                                         vocab_size=1024, max_seq_len=1024)
    torch.manual_seed(0)
    return build_model(cfg, device).to(torch.bfloat16)


def _batch(T, device):
    cu, pl, pos, total = random_packing(T, seed=1, max_doc=200)
    g = torch.Generator().manual_seed(1)
    inputs, labels = (torch.randint(0, 1024, (T,), generator=g, dtype=torch.int32) for _ in range(2))
    labels[total:] = -100
    labels[::5] = -100
    return {k: t.to(device) for k, t in dict(inputs=inputs, labels=labels, position_ids=pos, prefix_lens=pl, cu_seqlens=cu).items()}


@pytest.mark.parametrize("T", [512, 96])  # 96 rows take the decode form of the head's product
def test_gradients_equal_the_fused_loss(cuda_device, T):
    """Minus the mean log probability is the cross-entropy that the fused head computes from the same weights."""
    from hrm_text_b200.ops.logprobs import token_logprobs
    model, batch = _model(cuda_device), _batch(T, cuda_device)
    grads, losses = [], []
    for fused in (True, False):
        model.zero_grad()
        if fused:
            loss = model(carry=None, batch=dict(batch), bp_steps=2)[1]
        else:
            labels = batch["labels"].long()
            logits = model(carry=None, batch={k: v for k, v in batch.items() if k != "labels"}, bp_steps=2)[-1]
            assert logits.requires_grad and logits.dtype == torch.bfloat16
            loss = -token_logprobs(logits, labels).logprobs.sum() / (labels != -100).sum()
        loss.backward()
        losses.append(loss.item())
        grads.append({n: p.grad.float().clone() for n, p in model.named_parameters() if p.grad is not None})
    assert abs(losses[0] - losses[1]) < 2e-3 * losses[0]  # bf16 logits
    assert grads[0].keys() == grads[1].keys() and "lm_head.weight" in grads[0]
    for name in grads[0]:
        assert_close(grads[1][name], grads[0][name], 8e-2, name)


def test_head_gradients_match_fp32(cuda_device):
    from hrm_text_b200.ops.loss import lm_head_logits
    torch.manual_seed(1)
    for rows in (7, 300):
        x = torch.randn(2, rows, 256, device=cuda_device).bfloat16().requires_grad_()
        w = (torch.randn(320, 256, device=cuda_device) / 16).bfloat16().requires_grad_()
        y = lm_head_logits(x, w)
        assert y.shape == (2, rows, 320)
        g = torch.randn_like(y)
        y.backward(g)
        xr, wr = (t.detach().float().requires_grad_() for t in (x, w))
        yr = xr @ wr.t()
        yr.backward(g.float())
        # products of 256 to 600 terms in fp32, rounded once to bf16
        for a, b in ((y, yr), (x.grad, xr.grad), (w.grad, wr.grad)):
            assert_close(a, b, 2.0 ** -7, "logits")


def test_main_grad_takes_the_weight_gradient(cuda_device):
    from hrm_text_b200.ops.loss import lm_head_logits
    torch.manual_seed(2)
    x = torch.randn(300, 256, device=cuda_device).bfloat16()
    w = torch.randn(320, 256, device=cuda_device).bfloat16().requires_grad_()
    w.main_grad = torch.ones(320, 256, device=cuda_device)
    g = torch.randn(300, 320, device=cuda_device).bfloat16()
    lm_head_logits(x, w).backward(g)
    assert w.grad is None
    assert_close(w.main_grad - 1, g.float().t() @ x.float(), 2.0 ** -7, "main_grad")


def test_no_graph_without_gradients(cuda_device):
    model, batch = _model(cuda_device), _batch(512, cuda_device)
    del batch["labels"]
    with torch.no_grad():
        assert not model(carry=None, batch=batch, bp_steps=2)[-1].requires_grad
