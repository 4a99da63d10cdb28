"""Log probabilities, entropy and top-k of logits rows, and their gradient, against 64 bits.

Tolerances. Forward: exp2 is good to 2^-21, S is a sum of positive terms in fp32 (512 threads' sums of at
most V / 512 terms, joined in a tree), so log S is good to about (V / 512 + 20) 2^-24 + 2^-21 < 2^-16 for
V <= 200,000; the products x log2(e) round at 2^-24 |x| <= 2^-17 for the logits here: 2^-15 + 2^-20 |value|
covers both. The entropy has W / S of the same accuracy times |y - m| <= 60: 2^-13. Gradients: p to 2^-15
relative, then one rounding to the logits' type.
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


def _check(got, logits, tokens, k):
    from hrm_text_b200.models.paged import token_logprobs_reference
    lp, h, ids, top = token_logprobs_reference(logits.double(), tokens, k)
    torch.testing.assert_close(got.logprobs.double(), lp, rtol=2.0 ** -20, atol=2.0 ** -15, equal_nan=True)
    torch.testing.assert_close(got.entropy.double(), h, rtol=2.0 ** -20, atol=2.0 ** -13, equal_nan=True)
    if k:
        assert torch.equal(got.top_ids, ids)
        torch.testing.assert_close(got.top_logprobs.double(), top, rtol=2.0 ** -20, atol=2.0 ** -15, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (2, 5, 5), (3, 64, 64), (7, 511, 3), (5, 2048, 64), (33, 32768, 5), (4, 32003, 20),
                                   (2, 151937, 64), (1, 8192, 0)])
def test_matches_64_bits(cuda_device, dtype, n, v, k):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(n, v, dtype, cuda_device, seed=v)
    _check(token_logprobs(logits, tokens, k), logits, tokens, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_id(cuda_device, dtype):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits = torch.zeros(4, 9001, dtype=dtype, device=cuda_device)
    logits[1] = -3.0
    logits[1, 5000:5004] = 2.0
    logits[2, ::7] = 1.0                     # many equal values: more than are ranked by counting
    logits[3, 100], logits[3, 50] = 0.0, -0.0
    tokens = torch.tensor([0, 5001, 6, 8999], device=cuda_device)
    _check(token_logprobs(logits, tokens, 64), logits, tokens, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows(cuda_device, dtype):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(8, 3000, dtype, cuda_device)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf                    # nothing left
    logits[1, 5:] = -math.inf
    logits[2, :2999] = -math.inf             # one token left
    logits[3] = low                          # all equal, as low as the type goes
    logits[4, 1000:] = low
    logits[5, 77] = math.nan
    logits[6, 3] = math.inf
    tokens[:] = torch.tensor([4, 2, 2999, 9, 10, 1, 3, -100], device=cuda_device)
    got = token_logprobs(logits, tokens, 5)
    _check(got, logits, tokens, 5)
    assert got.logprobs[0] == -math.inf and got.entropy[0] == 0 and got.logprobs[2] == 0 and got.logprobs[7] == 0
    tokens[:] = torch.tensor([0, 6, 0, 0, 0, 0, 0, 3000], device=cuda_device)  # 6: masked, 3000: no token
    got = token_logprobs(logits, tokens)
    assert got.logprobs[1] == -math.inf and got.logprobs[7].isnan() and not got.entropy[7].isnan()


@pytest.mark.parametrize("n", [3, 700])  # many threads a row, and few
def test_few_tokens_left_by_a_mask(cuda_device, n):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(n, 9000, torch.float32, cuda_device, seed=4)
    keep = torch.zeros_like(logits, dtype=torch.bool)
    for i in range(n):                       # left: a few at the start, in the middle, at the end; or a run of 300
        keep[i, [(i * 7) % 50, 20, 4000 + i, 8999]] = True
        if i % 3 == 1:
            keep[i, 60:360] = True
        if i % 3 == 2:
            keep[i] = False
            keep[i, 63] = True
    logits.masked_fill_(~keep, -math.inf)
    logits[0, 20] = math.nan
    for k in (1, 20, 64):
        got = token_logprobs(logits, tokens, k)
        from hrm_text_b200.models.paged import token_logprobs_reference
        want = token_logprobs_reference(logits.double(), tokens, k)
        assert torch.equal(got.top_ids, want[2])
        torch.testing.assert_close(got.top_logprobs.double(), want[3], rtol=2.0 ** -20, atol=2.0 ** -15, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(1, 1), (3, 5), (9, 1001), (6, 32768)])
def test_gradient_matches_formula(cuda_device, dtype, n, v):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(n, v, dtype, cuda_device, seed=n)
    if n > 2:
        tokens[0] = -100
        logits[1, v // 2:] = -math.inf
        tokens[1] = 0
        logits[2] = -math.inf
    g_lp, g_h = (torch.randn(n, device=cuda_device) for _ in range(2))
    x = logits.double()
    empty = (x == -math.inf).all(-1, keepdim=True)
    logp = torch.log_softmax(torch.where(empty, torch.zeros_like(x), x), -1)
    p = torch.where(empty, torch.zeros_like(x), logp.exp())
    finite = torch.where(p > 0, logp, torch.zeros_like(logp))
    h = -(p * finite).sum(-1, keepdim=True)
    hot = torch.zeros_like(x).scatter_(1, tokens.clamp_min(0)[:, None], 1.0) * ((tokens >= 0)[:, None] & ~empty)
    glp = (g_lp.double() * (tokens >= 0))[:, None]
    for use_lp, use_h in ((1, 1), (1, 0), (0, 1)):
        leaf = logits.clone().requires_grad_()
        got = token_logprobs(leaf, tokens, top_k=1)
        outs = [o for o, use in ((got.logprobs, use_lp), (got.entropy, use_h)) if use]
        grads = [g for g, use in ((g_lp, use_lp), (g_h, use_h)) if use]
        (grad,) = torch.autograd.grad(outs, leaf, grads)
        want = use_lp * glp * (hot - p) - use_h * g_h.double()[:, None] * p * (finite + h)
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        bound = half * want.abs() + 2.0 ** -13 * (use_lp * glp.abs() + use_h * g_h.double().abs()[:, None]) * (p + hot) * (1 + h + finite.abs()) + 1e-12
        assert grad.dtype == dtype and torch.isfinite(grad.float()).all()
        assert ((grad.double() - want).abs() <= bound).all()


def test_gradient_matches_differences(cuda_device):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(2, 40, torch.float32, cuda_device)
    logits = logits / 3
    leaf = logits.clone().requires_grad_()
    got = token_logprobs(leaf, tokens)
    (grad,) = torch.autograd.grad((got.logprobs * 1.5 - got.entropy * 0.7).sum(), leaf)
    step = 2.0 ** -6  # central differences: step^2 / 6 of a third derivative of order one, values good to 2^-18 / step
    for j in range(40):
        moved = []
        for sign in (1, -1):
            x = logits.clone()
            x[:, j] += sign * step
            out = token_logprobs(x, tokens)
            moved.append(out.logprobs * 1.5 - out.entropy * 0.7)
        diff = (moved[0] - moved[1]) / (2 * step)
        torch.testing.assert_close(diff, grad[:, j], rtol=0, atol=2.0 ** -11)


def test_gradient_once_and_through_shapes(cuda_device):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(6, 64, torch.float32, cuda_device)
    leaf = logits.view(2, 3, 64).clone().requires_grad_()
    got = token_logprobs(leaf, tokens.view(2, 3), top_k=2)
    assert not got.top_ids.requires_grad and not got.top_logprobs.requires_grad
    (grad,) = torch.autograd.grad(got.logprobs.sum(), leaf, create_graph=True)
    flat = logits.clone().requires_grad_()
    (want,) = torch.autograd.grad(token_logprobs(flat, tokens).logprobs.sum(), flat)
    assert torch.equal(grad.detach().view(6, 64), want)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.sum().backward()
    with torch.no_grad():
        assert not token_logprobs(leaf, tokens.view(2, 3)).logprobs.requires_grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_shapes_and_streams(cuda_device, dtype):
    from hrm_text_b200.ops.logprobs import token_logprobs
    wide, _ = _rows(6, 1003, dtype, cuda_device)
    view = wide[::2, 1:1000]                                # rows start at any element
    tokens = torch.tensor([0, 5, 998], device=cuda_device, dtype=torch.int32)
    _check(token_logprobs(view, tokens, 3), view, tokens.long(), 3)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = token_logprobs(wide.view(2, 3, 1003), torch.ones(2, 3, dtype=torch.long, device=cuda_device), 2)
    torch.cuda.current_stream().wait_stream(other)
    assert got.logprobs.shape == (2, 3) and got.top_ids.shape == (2, 3, 2)
    one = token_logprobs(wide, torch.ones(6, dtype=torch.long, device=cuda_device), 2)
    assert torch.equal(got.logprobs.flatten(), one.logprobs) and torch.equal(got.top_ids.view(6, 2), one.top_ids)
    leaf = view.detach().requires_grad_()                   # the gradient of a strided view
    (grad,) = torch.autograd.grad(token_logprobs(leaf, tokens).logprobs.sum(), leaf)
    dense = view.contiguous().requires_grad_()
    (want,) = torch.autograd.grad(token_logprobs(dense, tokens).logprobs.sum(), dense)
    torch.testing.assert_close(grad, want, rtol=2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18, atol=1e-9)


def test_refusals(cuda_device):
    from hrm_text_b200.ops.logprobs import token_logprobs
    logits, tokens = _rows(3, 100, torch.float32, cuda_device)
    for bad in (65, -1, 101):
        with pytest.raises(ValueError, match="top_k"):
            token_logprobs(logits, tokens, bad)
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(logits, tokens[:2])
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(logits, tokens.float())
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(logits.cpu(), tokens.cpu())
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        token_logprobs(logits.half(), tokens)
    with pytest.raises(RuntimeError, match="rows contiguous"):
        token_logprobs(logits.t(), torch.zeros(100, dtype=torch.long, device=cuda_device))
    assert token_logprobs(logits[:0], tokens[:0], 2).top_ids.shape == (0, 2)
