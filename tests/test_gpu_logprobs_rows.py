"""Log probabilities where the rows decide which kernel runs, and the row's first places.

Rows run on 1024, 128 or 64 threads (many threads a row for few rows). Tolerances: a thread adds V / (2 threads)
terms in each of two chains, then the chains and the threads are joined and a running maximum moves a few times, so S is
good to r = (V / (2 threads) + 40) 2^-24 + 2^-18 (the second for the exponentials: 2^-22 each, and the rounding of
their arguments, 2^-24 |x - m| with |x - m| < 60 where a term counts). All terms of W have one sign, so W / S is good to
2 r |W / S| and the entropy to r (1 + 2 |log S - H|). A log probability takes two more roundings of itself.
Gradients: p to r + 2^-17, H as above, one rounding to the logits' type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(n, v, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(n, v, generator=g, device=device) * 3
    x[:, :: max(1, v // 3)] += 8
    return x.to(dtype), torch.randint(0, v, (n,), generator=g, device=device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [6, 700])
def test_nan_at_the_first_id(cuda_device, dtype, n):
    """NaN is above everything, lowest id first, also where a row is too long or too even to be ranked by counting."""
    from hrm_text_b200.models.paged import token_logprobs_reference
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(n, 32768, dtype, cuda_device, seed=1)
    logits[0, 0] = math.nan
    logits[1] = math.nan
    logits[2, ::2] = math.nan
    logits[3, 0], logits[3, 77] = math.inf, math.nan
    logits[4] = 1.0                              # equal values: id 0 first
    logits[5, 1:] = -math.inf
    for k in (1, 5, 64):
        got = token_logprobs(logits, tokens, k)
        want = token_logprobs_reference(logits[:6].double(), tokens[:6], k)
        assert torch.equal(got.top_ids[:6], want[2])
        assert got.top_ids[0, 0] == 0 and got.top_ids[1].tolist() == list(range(k)) and got.top_ids[3, 0] == 77


def test_rows_past_32_bits_of_statistics(cuda_device):
    """The statistics are three numbers a row: from 715,827,883 rows on their index passes 31 bits."""
    from hrm_text_b200.ops.logprobs import token_logprobs
    n = 715_827_883 + 40
    leaf = torch.tensor([[0.5, 2.0]], device=cuda_device).bfloat16().requires_grad_()
    tokens = torch.ones(n, dtype=torch.long, device=cuda_device)
    tokens[-1] = 0
    got = token_logprobs(leaf.expand(n, 2), tokens)
    want = torch.log_softmax(torch.tensor([0.5, 2.0]), -1).tolist()
    assert torch.allclose(got.logprobs[-50:-1].cpu(), torch.full((49,), want[1]), rtol=0, atol=2.0 ** -18)
    assert abs(got.logprobs[-1].item() - want[0]) < 2.0 ** -18
    logits = leaf.detach().expand(n, 2).requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(logits, tokens).logprobs.sum(), logits)
    p = math.exp(want[1])
    rest = torch.tensor([p - 1, 1 - p]).bfloat16().expand(49, 2)  # bf16 gradients, to one step of theirs
    assert torch.allclose(grad[-50:-1].float().cpu(), rest.float(), rtol=2.0 ** -7, atol=0)
    assert torch.allclose(grad[-1].float().cpu(), torch.tensor([p, -p]), rtol=2.0 ** -7, atol=0)


def test_forward_gradients_are_refused(cuda_device):
    import torch.autograd.forward_ad as fwd
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(2, 100, torch.float32, cuda_device)
    for leaf in (logits, logits.clone().requires_grad_()):
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward"):
            token_logprobs(fwd.make_dual(leaf, torch.ones_like(leaf)), tokens)
    token_logprobs(logits, tokens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_an_id_outside_the_vocabulary(cuda_device, dtype):
    """Its log probability is NaN and so is the gradient of it; the entropy, and the entropy's gradient, do not depend on it."""
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(5, 1001, dtype, cuda_device, seed=2)
    inside = tokens.clone()
    tokens[1], tokens[2], tokens[3] = 1001, -1, -100
    g_lp, g_h = (torch.randn(5, device=cuda_device) for _ in range(2))

    def grad(ids, use_lp, use_h):
        leaf = logits.clone().requires_grad_()
        got = token_logprobs(leaf, ids)
        outs = [o for o, use in ((got.logprobs, use_lp), (got.entropy, use_h)) if use]
        return torch.autograd.grad(outs, leaf, [g for g, use in ((g_lp, use_lp), (g_h, use_h)) if use])[0]

    entropy = grad(inside, 0, 1)
    assert torch.isfinite(entropy).all() and torch.equal(grad(tokens, 0, 1), entropy)
    both = grad(tokens, 1, 1)
    assert both[1:3].isnan().all() and torch.equal(both[3], entropy[3])  # -100 keeps the entropy's gradient
    assert torch.equal(both[[0, 4]], grad(inside, 1, 1)[[0, 4]])
    alone = grad(tokens, 1, 0)
    assert alone[1:3].isnan().all() and (alone[3] == 0).all()


def test_strides_of_a_single_column(cuda_device):
    from hrm_text_b200.ops.logprobs import token_logprobs
    wide, _ = _rows(4, 10, torch.float32, cuda_device)
    column = wide[:, ::3][:, :1]                 # [4, 1] with a column stride of 3, which nothing uses
    assert column.stride(1) == 3
    got = token_logprobs(column, torch.zeros(4, dtype=torch.long, device=cuda_device), 1)
    assert (got.logprobs == 0).all() and (got.top_ids == 0).all()
    leaf = column.detach().requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, torch.zeros(4, dtype=torch.long, device=cuda_device)).logprobs.sum(), leaf)
    assert (grad == 0).all()


def _threads(n, v, dtype, device):
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    return 1024 if n <= 2 * sms else 64 if v * dtype.itemsize < 8192 else 128


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 5, 511, 1001, 2047, 4097, 32003, 32768, 151937])
def test_many_rows_match_64_bits(cuda_device, dtype, v):
    """More rows than are given 1024 threads each, at any start in memory, with masked, tied, NaN and ignored ones among them."""
    from hrm_text_b200.models.paged import token_logprobs_reference
    from hrm_text_b200.ops.logprobs import token_logprobs
    n = 2 * torch.cuda.get_device_properties(cuda_device).multi_processor_count + 5
    whole, tokens = _rows(n, v + 3, dtype, cuda_device, seed=v)
    logits, tokens = whole[:, 1:v + 1], tokens % v
    if v > 500:
        logits[0, 5:] = -math.inf
        logits[1] = -math.inf
        logits[2] = torch.finfo(dtype).min
        logits[3, ::7] = 12.0                    # more equal values than are ranked by counting
        logits[4, v // 2] = math.nan
        logits[5, 3] = math.inf
        tokens[6], tokens[7] = -100, v
    threads = _threads(n, v, dtype, cuda_device)
    assert threads < 1024
    r = (v / (2 * threads) + 40) * 2.0 ** -24 + 2.0 ** -18
    for k in (0, min(5, v), min(64, v)):
        got = token_logprobs(logits, tokens, k)
        lp, h, ids, top = token_logprobs_reference(logits.double(), tokens, k)
        log_s = torch.logsumexp(logits.double(), -1) - logits.double().amax(-1)
        slack = (r * (1 + 2 * (log_s - h).abs()) + 2.0 ** -22 * h.abs()).nan_to_num(0.0, posinf=0.0)
        torch.testing.assert_close(got.logprobs.double(), lp, rtol=2.0 ** -22, atol=r, equal_nan=True)
        off = torch.where(h.isnan() & got.entropy.isnan(), 0.0, (got.entropy.double() - h).abs())
        assert (off <= slack).all()
        if k:
            assert torch.equal(got.top_ids, ids)
            torch.testing.assert_close(got.top_logprobs.double(), top, rtol=2.0 ** -22, atol=r, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [5, 1001, 4097, 32768])
def test_many_rows_gradient(cuda_device, dtype, v):
    """From the statistics of the 64- and 128-thread forward kernels."""
    from hrm_text_b200.ops.logprobs import token_logprobs
    n = 2 * torch.cuda.get_device_properties(cuda_device).multi_processor_count + 5
    logits, tokens = _rows(n, v, dtype, cuda_device, seed=v + 1)
    logits[1, v // 2:] = -math.inf
    logits[2] = -math.inf
    tokens[0], tokens[1], tokens[3] = -100, 0, v - 1
    g_lp, g_h = (torch.randn(n, device=cuda_device) for _ in range(2))
    leaf = logits.clone().requires_grad_()
    got = token_logprobs(leaf, tokens)
    (grad,) = torch.autograd.grad((got.logprobs, got.entropy), leaf, (g_lp, g_h))
    x = logits.double()
    empty = (x == -math.inf).all(-1, keepdim=True)
    logp = torch.log_softmax(torch.where(empty, torch.zeros_like(x), x), -1)
    p = torch.where(empty, torch.zeros_like(x), logp.exp())
    finite = torch.where(p > 0, logp, torch.zeros_like(logp))
    h = -(p * finite).sum(-1, keepdim=True)
    hot = torch.zeros_like(x).scatter_(1, tokens.clamp_min(0)[:, None], 1.0) * ((tokens >= 0)[:, None] & ~empty)
    glp, gh = (g_lp.double() * (tokens >= 0))[:, None], g_h.double()[:, None]
    want = glp * (hot - p) - gh * p * (finite + h)
    r = (v / (2 * _threads(n, v, dtype, cuda_device)) + 40) * 2.0 ** -24 + 2.0 ** -17
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    bound = half * want.abs() + 4 * r * (glp.abs() + gh.abs()) * (p + hot) * (1 + h + finite.abs()) + 1e-12
    assert grad.dtype == dtype and ((grad.double() - want).abs() <= bound).all()
