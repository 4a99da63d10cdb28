"""Inference: checkpoint loading and batched generation with static KV caches.

Behaviour follows the reference's simple_inference_engine.py:
* ``inference_load_checkpoint`` (:37-90) rebuilds the model from ``all_config.yaml`` /
  ``train_metadata.yaml``, loads the DCP checkpoint on one process, optionally swaps in the EMA
  weights, casts to the forward dtype and loads the tokenizer;
* ``inference_generate`` (:115-197) is a generator doing continuous batching over
  ``batch_size`` slots: a free slot is filled by a bidirectional prefill of one prompt (the
  PrefixLM prefix), then all active slots decode one token per step; finished generations are
  yielded as ``(prompt_id, text)``; prompts that do not fit the context yield ``""``;
* sampling is greedy for ``temp < 1e-5`` and Gumbel-max otherwise (:93-102).

Every module call of the recurrent model has its own static cache (one per call and layer,
``model.create_cache``). ``kv_cache="int8"`` or ``"fp8"`` holds keys and values in 8 bits in blocks of one
pool (``ops.paged``). A prompt reserves the blocks of its own longest generation until it ends, so that a
step never runs out; with ``num_blocks`` below every slot at its longest, as many prompts run together
as fit. ``logprobs`` adds the log probability, entropy and likeliest alternatives of every generated token
(``ops.logprobs``; of the bf16 logits that the token is drawn from). Both are additions to the reference.
"""
from __future__ import annotations

import os
from dataclasses import dataclass
from typing import Any, Generator, Iterator, Optional

import numpy as np
import torch
from torch import Tensor, nn

from ..config import PretrainConfig
from ..data.dataset import V1DatasetMeta
from ..ops.logprobs import MAX_TOP_K
from ..ops.paged import MAX_REQUESTS, BlockTables
from ..optim.adam_atan2 import AdamATan2
from ..runtime.checkpoint import checkpoint_dir, latest_epoch
from ..runtime.factory import build_model, model_config_dict


@dataclass
class InferenceCheckpoint:
    model: nn.Module
    carry: Any
    tokenizer: Any
    tokenizer_info: dict

    def tokenize_prompt(self, condition: str, prompt: str) -> np.ndarray:
        info = self.tokenizer_info
        cond = "".join(info["condition_mapping"][c] for c in condition.split(","))
        text = f'{info["boq"]}{cond}{prompt}{info["eoq"]}'
        return np.asarray(self.tokenizer(text, add_special_tokens=False)["input_ids"], dtype=np.int64)

    def decode_generation(self, tokens: np.ndarray, eos_id: int) -> str:
        if tokens.size and tokens[-1] == eos_id:
            tokens = tokens[:-1]
        return self.tokenizer.decode(tokens.tolist())


def load_model_from_checkpoint(ckpt_path: str, ckpt_epoch: Optional[int] = None, use_ema: bool = True,
                               device: Optional[torch.device] = None):
    """Model (eval mode, forward dtype) + carry + metadata, from a training checkpoint directory."""
    import yaml
    import torch.distributed.checkpoint as dcp
    from torch.distributed.checkpoint.state_dict import get_optimizer_state_dict
    device = device or (torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available()
                        else torch.device("cpu"))
    with open(os.path.join(ckpt_path, "all_config.yaml")) as f:
        cfg = PretrainConfig(**yaml.safe_load(f))
    with open(os.path.join(ckpt_path, "train_metadata.yaml")) as f:
        meta = V1DatasetMeta(**yaml.safe_load(f))
    model_cfg = model_config_dict(cfg.arch.model_dump(), meta.model_dump(), cfg.data.model_dump())
    model = build_model(model_cfg, device)
    optim = AdamATan2(model.parameters(), lr=torch.tensor(0.0), betas=(cfg.beta1, cfg.beta2),
                      weight_decay=cfg.weight_decay, ema=cfg.ema)
    if ckpt_epoch is None:
        ckpt_epoch = latest_epoch(ckpt_path)
        if ckpt_epoch is None:
            raise ValueError(f"No checkpoint files found in {ckpt_path}")
    dcp.load({"model": model.state_dict(), "optim": get_optimizer_state_dict(model, optim)},
             checkpoint_id=checkpoint_dir(ckpt_path, ckpt_epoch), no_dist=True)
    carry_file = os.path.join(ckpt_path, f"carry_epoch_{ckpt_epoch}.0.pt")
    carry = torch.load(carry_file, map_location=device, weights_only=False) if os.path.exists(carry_file) else None
    if use_ema:
        optim.swap_ema()
    model = model.to(getattr(torch, cfg.fwd_bwd_dtype)).eval()
    return model, carry, cfg, meta


def inference_load_checkpoint(ckpt_path: str, ckpt_epoch: Optional[int], ckpt_use_ema: bool) -> InferenceCheckpoint:
    from transformers import AutoTokenizer
    model, carry, _cfg, meta = load_model_from_checkpoint(ckpt_path, ckpt_epoch, ckpt_use_ema)
    tokenizer = AutoTokenizer.from_pretrained(meta.tokenizer_info["tokenizer_path"], use_fast=True)
    return InferenceCheckpoint(model=model, carry=carry, tokenizer=tokenizer, tokenizer_info=meta.tokenizer_info)


_SAMPLE_CALLS = [0]


def sample(logits: Tensor, temp: float, generator: Optional[torch.Generator] = None) -> Tensor:
    """Greedy for ``temp < 1e-5``; else Gumbel-max sampling at temperature ``temp``.

    On CUDA one fused kernel does the scaling, the Gumbel noise (counter-based, seeded from
    ``generator`` or torch's default seed, advanced every call) and the argmax.
    """
    if logits.is_cuda and logits.dim() == 2 and logits.dtype in (torch.float32, torch.bfloat16):
        from .._native import cuda
        seed = generator.initial_seed() if generator is not None else torch.initial_seed()
        _SAMPLE_CALLS[0] += 1
        return cuda().sample_tokens(logits.contiguous(), float(temp), int(seed) & 0x7FFFFFFFFFFFFFFF, _SAMPLE_CALLS[0])
    if temp < 1e-5:
        return logits.argmax(-1)
    scaled = logits.float() / temp
    u = torch.rand(scaled.shape, device=scaled.device, generator=generator).clamp_min(torch.finfo(torch.float32).tiny)
    return (scaled - torch.log(-torch.log(u))).argmax(-1)


@torch.inference_mode()
def prefill(model: nn.Module, carry, tokens: Tensor, cache) -> Tensor:
    """Bidirectional pass over one prompt into ``cache``; returns the last position's logits."""
    batch = {"inputs": tokens[None], "position_ids": torch.arange(tokens.numel(), device=tokens.device),
             "cache": cache, "cache_lengths": 0}
    return model(carry=carry, batch=batch)[-1][0, -1]


@torch.inference_mode()
def decode_step(model: nn.Module, carry, last_tokens: Tensor, cache, cache_lengths: Tensor) -> Tensor:
    batch = {"inputs": last_tokens[:, None], "position_ids": cache_lengths[:, None], "cache": cache,
             "cache_lengths": cache_lengths}
    return model(carry=carry, batch=batch)[-1][:, -1]


class DecodeGraph:
    """The decode step (all ``batch_size`` slots, one token each) captured in one CUDA graph.

    The step's work is a fixed sequence of device operations on static shapes (embedding,
    per module call and layer the RMSNorm / GEMM / decode-attention kernels, the LM-head GEMM),
    so it is captured once per cache and replayed for every generated token; the per-step
    inputs (last tokens, cache lengths) are copied into static buffers. Capture writes junk
    keys / values at position 0 of every slot, so it must happen before any prompt is
    prefilled into the cache.
    """

    def __init__(self, model: nn.Module, carry, cache, batch_size: int, device: torch.device, warmup: int = 2):
        self.tokens = torch.zeros(batch_size, dtype=torch.long, device=device)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        stream = torch.cuda.Stream(device=device)
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(stream):
            for _ in range(warmup):
                decode_step(model, carry, self.tokens, cache, self.lengths)
        torch.cuda.current_stream(device).wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=stream):
            self.logits = decode_step(model, carry, self.tokens, cache, self.lengths)

    def __call__(self, last_tokens: Tensor, cache_lengths: Tensor) -> Tensor:
        self.tokens.copy_(last_tokens, non_blocking=True)
        self.lengths.copy_(cache_lengths, non_blocking=True)
        self.graph.replay()
        return self.logits


KV_CACHES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


@torch.inference_mode()
def paged_prefill(model: nn.Module, carry, tokens: Tensor, cache, tables: BlockTables, slot: int) -> Tensor:
    """Bidirectional pass over one prompt into the (empty) request ``slot``; returns the last position's logits."""
    new = torch.zeros_like(tables.lengths)
    new[slot] = tokens.numel()
    plan = tables.step(new, tokens.numel())
    batch = {"inputs": tokens[None], "position_ids": plan.positions, "cache": cache, "cache_lengths": plan, "prompt": True}
    return model(carry=carry, batch=batch)[-1][0, -1]


@torch.inference_mode()
def paged_decode_step(model: nn.Module, carry, last_tokens: Tensor, cache, tables: BlockTables, active: Tensor) -> Tensor:
    """One token for every request with ``active [B]`` (int32) 1; logits ``[B, V]`` (rows of the others are arbitrary)."""
    B = active.numel()
    plan = tables.step(active, B, max_new=1)
    row = torch.where(active > 0, plan.cu_new[:-1], B).long()  # a request's row among the packed ones
    packed = last_tokens.new_zeros(B + 1).scatter_(0, row, last_tokens)
    batch = {"inputs": packed[:B, None], "position_ids": plan.positions[:, None], "cache": cache, "cache_lengths": plan}
    return model(carry=carry, batch=batch)[-1][:, -1][row.clamp_max(B - 1)]


class PagedDecodeGraph:
    """``paged_decode_step`` in one CUDA graph, blocks assigned inside it. Warming up writes junk into the blocks of
    requests that are then freed, so it must happen while the tables are empty."""

    def __init__(self, model: nn.Module, carry, cache, tables: BlockTables, warmup: int = 2):
        device, B = tables.lengths.device, tables.lengths.numel()
        self.tokens = torch.zeros(B, dtype=torch.long, device=device)
        self.active = torch.zeros(B, dtype=torch.int32, device=device)
        self.active[0] = 1
        stream = torch.cuda.Stream(device=device)
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(stream):
            for _ in range(warmup):
                paged_decode_step(model, carry, self.tokens, cache, tables, self.active)
            tables.truncate(torch.zeros_like(tables.lengths))
        torch.cuda.current_stream(device).wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=stream):
            self.logits = paged_decode_step(model, carry, self.tokens, cache, tables, self.active)

    def __call__(self, last_tokens: Tensor, active: Tensor) -> Tensor:
        self.tokens.copy_(last_tokens, non_blocking=True)
        self.active.copy_(active, non_blocking=True)
        self.graph.replay()
        return self.logits


@dataclass
class GeneratedLogprobs:
    """Per generated token: log probability and entropy ``[n]``, the likeliest tokens and theirs ``[n, k]`` (float32 / int64)."""

    logprobs: np.ndarray
    entropy: np.ndarray
    top_ids: np.ndarray
    top_logprobs: np.ndarray


def _logprobs_to_host(logits: Tensor, tokens: Tensor, top_k: int) -> np.ndarray:
    """``[B, 2 + 2 * top_k]`` float64: log probability, entropy, top log probabilities, top ids."""
    if logits.is_cuda:
        from ..ops.logprobs import token_logprobs
        lp, h, ids, top = token_logprobs(logits, tokens, top_k)
    else:
        from ..models.paged import token_logprobs_reference
        lp, h, ids, top = token_logprobs_reference(logits.float(), tokens, top_k)
    parts = [lp[:, None], h[:, None]] + ([top, ids] if top_k else [])
    return torch.cat([p.double() for p in parts], dim=1).cpu().numpy()


class _StaticSlots:
    """bf16 caches of the full context length for every slot."""

    def __init__(self, model, carry, batch_size, max_tokens, dtype, device, use_cuda_graph):
        self.model, self.carry, self.max_tokens = model, carry, max_tokens
        self.cache = model.create_cache(max_batch_size=batch_size, max_seq_len=max_tokens, dtype=dtype, device=device)
        self.graphed = None
        if use_cuda_graph and device.type == "cuda" and dtype == torch.bfloat16:
            self.graphed = DecodeGraph(model, carry, self.cache, batch_size, device)  # before any prefill (see DecodeGraph)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)

    def fits(self, prompt_len: int) -> bool:
        return True

    def admit(self, i: int, tokens: Tensor, most: int) -> Tensor:
        logits = prefill(self.model, self.carry, tokens, _slot_view(self.cache, i))
        self.lengths[i] = tokens.numel()
        return logits

    def release(self, i: int) -> None:
        pass

    def decode(self, last: Tensor, stopped: np.ndarray) -> Tensor:
        if self.graphed is not None:
            logits = self.graphed(last, self.lengths)
        else:
            logits = decode_step(self.model, self.carry, last, self.cache, self.lengths)
        self.lengths.add_(1).clamp_max_(self.max_tokens - 1)
        return logits


class _PagedSlots:
    """8-bit caches in blocks from one pool; a prompt is admitted when its blocks for the longest possible
    generation are free, so a step never runs out."""

    def __init__(self, model, carry, batch_size, max_tokens, code, device, use_cuda_graph, block_size, num_blocks):
        if batch_size > MAX_REQUESTS:
            raise ValueError(f"a paged cache serves at most {MAX_REQUESTS} slots, got {batch_size}")
        self.model, self.carry, self.block_size, self.device = model, carry, block_size, device
        width = -(-max_tokens // block_size)
        self.spare = batch_size * width if num_blocks is None else num_blocks
        if self.spare < width:
            raise ValueError(f"the pool of {self.spare} blocks does not hold one request of {max_tokens} tokens")
        self.tables = BlockTables(self.spare, block_size, batch_size, width, device)
        self.cache = model.create_cache(paged=self.tables, dtype=code, device=device)
        self.held = [0] * batch_size
        self.graphed = PagedDecodeGraph(model, carry, self.cache, self.tables) if use_cuda_graph and device.type == "cuda" else None

    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.block_size)

    def fits(self, most: int) -> bool:
        return self._blocks(most) <= self.spare

    def admit(self, i: int, tokens: Tensor, most: int) -> Tensor:
        self.held[i] = self._blocks(most)
        self.spare -= self.held[i]
        return paged_prefill(self.model, self.carry, tokens, self.cache, self.tables, i)

    def release(self, i: int) -> None:
        keep = torch.full_like(self.tables.lengths, torch.iinfo(torch.int32).max)
        keep[i] = 0
        self.tables.truncate(keep)
        self.tables.check()  # a step that did not fit would have decoded nothing
        self.spare += self.held[i]
        self.held[i] = 0

    def decode(self, last: Tensor, stopped: np.ndarray) -> Tensor:
        active = torch.as_tensor(~stopped, dtype=torch.int32).to(self.device)
        if self.graphed is not None:
            return self.graphed(last, active)
        return paged_decode_step(self.model, self.carry, last, self.cache, self.tables, active)


def _slot_view(cache, i: int):
    return torch.utils._pytree.tree_map(lambda x: x[i:i + 1] if isinstance(x, Tensor) else x, cache)


@torch.inference_mode()
def generate_tokens(model: nn.Module, carry, prompts: Iterator[tuple[int, np.ndarray]], max_tokens: int,
                    max_generation: int, batch_size: int, stop_token: int, temp: float = 0.0,
                    device: Optional[torch.device] = None, use_cuda_graph: bool = True, kv_cache: str = "bf16",
                    block_size: int = 64, num_blocks: Optional[int] = None,
                    logprobs: Optional[int] = None) -> Generator[tuple, None, None]:
    """Continuous-batching generation over token prompts; yields ``(prompt_id, generated_ids)``.

    On a CUDA device with bf16 weights the decode step runs as one captured CUDA graph
    (``DecodeGraph``, ``PagedDecodeGraph``). ``kv_cache`` ``"int8"`` / ``"fp8"`` keeps the caches in 8 bits in
    blocks of ``block_size`` tokens from a pool of ``num_blocks`` (default: room for every slot at its longest;
    with fewer, prompts wait until blocks are free). With ``logprobs=k`` (0 to 64) yields ``(prompt_id, generated_ids,
    GeneratedLogprobs)``, the ``k`` likeliest tokens among it."""
    device = device or next(model.parameters()).device
    dtype = next(model.parameters()).dtype
    if logprobs is not None:
        most = min(MAX_TOP_K, model.lm_head.weight.shape[0])
        if not 0 <= logprobs <= most:
            raise ValueError(f"logprobs must be 0 to {most} (or None), got {logprobs}")
    if kv_cache == "bf16":
        slots = _StaticSlots(model, carry, batch_size, max_tokens, dtype, device, use_cuda_graph)
    elif kv_cache in KV_CACHES:
        slots = _PagedSlots(model, carry, batch_size, max_tokens, KV_CACHES[kv_cache], device,
                            use_cuda_graph and dtype == torch.bfloat16, block_size, num_blocks)
    else:
        raise ValueError(f'kv_cache must be "bf16", "int8" or "fp8", got {kv_cache!r}')
    last = torch.zeros(batch_size, dtype=torch.long, device=device)
    generated = np.zeros((batch_size, max_tokens), dtype=np.int64)
    scores = None if logprobs is None else np.zeros((batch_size, max_tokens, 2 + 2 * logprobs))
    g_start = np.zeros(batch_size, dtype=np.int64)
    g_len = np.zeros(batch_size, dtype=np.int64)
    stopped = np.ones(batch_size, dtype=bool)
    ids = [-1] * batch_size

    def next_prompt():
        for pid, tok in prompts:
            if tok.size >= max_tokens:
                yield (pid, np.zeros(0, dtype=np.int64)) + (() if scores is None else (_scores(np.zeros((0, 2 + 2 * logprobs))),))
                continue
            return pid, tok
        return -1, None

    def _scores(x: np.ndarray) -> GeneratedLogprobs:
        f = x.astype(np.float32)
        return GeneratedLogprobs(f[:, 0], f[:, 1], x[:, 2 + logprobs:].astype(np.int64), f[:, 2:2 + logprobs])

    def finished(i: int):
        span = slice(g_start[i], g_len[i])
        out = (ids[i], generated[i, span].copy())
        return out if scores is None else out + (_scores(scores[i, span]),)

    pending_id, pending = yield from next_prompt()
    while True:
        for i in np.nonzero(stopped)[0]:
            if ids[i] != -1:
                yield finished(i)
                ids[i] = -1
                slots.release(int(i))
            if pending is None:
                continue
            start = max(pending.size, max_tokens - max_generation)
            most = pending.size + max_tokens - start
            if not slots.fits(most):
                continue
            tok = torch.as_tensor(pending, device=device)
            logits = slots.admit(int(i), tok, most)[None]
            token = sample(logits, temp)
            first = int(token[0])
            last[i] = first
            ids[i] = pending_id
            g_start[i] = start
            g_len[i] = start + 1
            generated[i, start] = first
            if scores is not None:
                scores[i, start] = _logprobs_to_host(logits, token, logprobs)[0]
            stopped[i] = first == stop_token or g_len[i] >= max_tokens
            pending_id, pending = yield from next_prompt()
        if not stopped.all():
            logits = slots.decode(last, stopped)
            last = sample(logits, temp)
            active = ~stopped
            g_len[active] += 1
            host = last.cpu().numpy()
            generated[active, g_len[active] - 1] = host[active]
            if scores is not None:
                scores[active, g_len[active] - 1] = _logprobs_to_host(logits, last, logprobs)[active]
            stopped |= (host == stop_token) | (g_len >= max_tokens)
        elif pending is None:
            break
    for i in range(batch_size):
        if ids[i] != -1:
            yield finished(i)


def inference_generate(ckpt: InferenceCheckpoint, iterator: Iterator[tuple[int, tuple[str, str]]], max_tokens: int,
                       max_generation: int, batch_size: int, temp: float = 0.0, kv_cache: str = "bf16",
                       block_size: int = 64, num_blocks: Optional[int] = None) -> Generator[tuple[int, str], None, None]:
    """Text in, text out: ``iterator`` yields ``(prompt_id, (condition, prompt))``; the caches as in ``generate_tokens``."""
    stop = ckpt.tokenizer.convert_tokens_to_ids(ckpt.tokenizer_info["eoa"])
    tokenized = ((pid, ckpt.tokenize_prompt(*p)) for pid, p in iterator)
    for pid, toks in generate_tokens(ckpt.model, ckpt.carry, tokenized, max_tokens, max_generation, batch_size,
                                     stop, temp, kv_cache=kv_cache, block_size=block_size, num_blocks=num_blocks):
        yield pid, ckpt.decode_generation(toks, stop) if toks.size else ""
