"""Log probabilities of given tokens, entropy and likeliest alternatives of logits rows
(csrc/kernels/logprobs.cu), differentiable with respect to the logits.

Sampling gives token ids only (``inference.engine.sample``); this gives what scoring, ranking of
generations and fine-tuning on log probabilities need, in one pass over the logits. The reference
has no counterpart: its harness compares generated text (evaluation/benchmarks.py).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from .._native import cuda

MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """fp32 ``logprobs``, ``entropy`` (natural logarithm) ``[...]``; ``top_ids`` int64 and ``top_logprobs``
    fp32 ``[..., top_k]``, likeliest first, lowest id first among equals (``None`` for ``top_k`` 0)."""

    logprobs: Tensor
    entropy: Tensor
    top_ids: Optional[Tensor]
    top_logprobs: Optional[Tensor]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, tokens: Tensor, top_k: int):
        *out, stats = cuda().token_logprobs_fwd(logits, tokens, top_k, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(out[2], out[3])
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_h, _ids, _top):
        if g_lp is None and g_h is None:
            return None, None, None
        logits, tokens, stats = ctx.saved_tensors
        grad = torch.empty_like(logits)
        rows = [None if g is None else g.contiguous() for g in (g_lp, g_h)]
        cuda().token_logprobs_bwd(logits, tokens, stats, rows[0], rows[1], grad)
        return grad, None, None


def token_logprobs(logits: Tensor, tokens: Tensor, top_k: int = 0) -> TokenLogprobs:
    """``log softmax(logits)[tokens]``, the entropy of ``softmax(logits)`` and its ``top_k`` likeliest tokens.

    ``logits [..., V]`` fp32 or bf16 (rows contiguous, any row stride), ``tokens [...]`` integer ids; a token of
    -100 (``IGNORE_LABEL_ID``) has log probability 0 and no gradient, any other id outside the vocabulary
    gives NaN. A row of minus infinities has log probability -inf, entropy 0 and no gradient. ``logprobs``
    and ``entropy`` are differentiable; the top log probabilities are not.
    """
    if not logits.is_cuda:
        raise RuntimeError("hrm_text_b200.ops.logprobs takes CUDA tensors only (models.paged has the CPU oracle)")
    if tokens.shape != logits.shape[:-1] or tokens.is_floating_point() or tokens.dtype == torch.bool:
        raise ValueError(f"tokens must be integers of shape {tuple(logits.shape[:-1])}, got {tokens.dtype} {tuple(tokens.shape)}")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"top_k must be 0 to {MAX_TOP_K} and at most the vocabulary, got {top_k}")
    lead = logits.shape[:-1]
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    ids = tokens if tokens.dim() == 1 and tokens.dtype == torch.int64 else tokens.reshape(-1).to(torch.int64)
    ids = ids.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _TokenLogprobs.apply(rows, ids, top_k)
    else:
        out = cuda().token_logprobs_fwd(rows, ids, top_k, False)
    if logits.dim() != 2:
        out = [out[0].view(lead), out[1].view(lead), out[2].view(*lead, top_k), out[3].view(*lead, top_k)]
    return TokenLogprobs(out[0], out[1], *((out[2], out[3]) if top_k else (None, None)))
