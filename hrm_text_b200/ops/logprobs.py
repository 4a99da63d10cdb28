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

MAX_TOP_K = 64  # groups of threads in the kernel


class TokenLogprobs(NamedTuple):
    """fp32 ``logprobs``, ``entropy`` (natural logarithm) ``[...]``; ``top_ids`` int64 and ``top_logprobs``
    fp32 ``[..., top_k]``, likeliest first, lowest id first among equals (``None`` for ``top_k`` 0)."""

    logprobs: Tensor
    entropy: Tensor
    top_ids: Optional[Tensor]
    top_logprobs: Optional[Tensor]


def token_logprobs(logits: Tensor, tokens: Tensor, top_k: int = 0) -> TokenLogprobs:
    """``log softmax(logits)[tokens]``, the entropy of ``softmax(logits)`` and its ``top_k`` likeliest tokens.

    ``logits [..., V]`` fp32 or bf16 (rows contiguous, any row stride), ``tokens [...]`` integer ids; a token of
    -100 (``IGNORE_LABEL_ID``) has log probability 0 and no gradient of it, any other id outside the vocabulary
    gives NaN for both. A row's entropy, and the entropy's gradient, do not depend on its token: mask them
    where a padded row must not count. A row of minus infinities has log probability -inf, entropy 0 and no gradient. ``logprobs``
    and ``entropy`` are differentiable (once, backwards only); the top log probabilities are not.
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
    out = cuda().token_logprobs(rows, ids, top_k)
    if logits.dim() != 2:
        out = [o.view(lead + o.shape[1:]) for o in out]
    return TokenLogprobs(*out) if top_k else TokenLogprobs(out[0], out[1], None, None)
