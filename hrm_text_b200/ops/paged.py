"""Paged 8-bit KV cache: block tables on the device, quantising append, attention, read-back.

A paged cache stores the keys and values of one attention layer in blocks of ``block_size``
tokens, as int8 or e4m3 codes with one fp32 scale for each block and head. Requests own blocks
through ``BlockTables``, which all layers of a model share. One step of generation is

    plan = tables.step(new_tokens, num_tokens, max_new=1) # once: blocks, slots, positions
    for every layer:
        paged_append(key, value, cache, plan)             # [num_tokens, heads, 128] bf16
        y = paged_attention(query, cache, plan, gate=gate)
    tables.truncate(keep)                                 # a request that ends frees its blocks

Nothing here reads a device value on the host, so a step can be captured in a CUDA graph and
replayed. Everything runs on the current stream; a plan, its tables and the caches are used in stream order. These
calls are for inference: their results carry no gradient.
On CUDA the kernels of csrc/kernels/paged_*.cu run. ``BlockTables`` on the CPU, and
``models.paged`` for the rest, are the plain torch oracle of the same operations.

The reference keeps one bf16 cache of the full context length for each slot
(models/layers.py:105-113, simple_inference_engine.py:118-131).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from .._native import cuda

BLOCK_SIZES = (16, 32, 64, 128)
CODE_TYPES = (torch.int8, torch.float8_e4m3fn)
UNIT_KEYS, PAIR_COST = 128, 3  # how attention work is counted (csrc/kernels/paged.h)
MAX_REQUESTS = 8192

STATUS = {1: "the pool has too few free blocks", 2: "more new tokens than num_tokens", 3: "a request outgrows its table",
          4: "a negative number of new tokens", 5: "a request has more new tokens than max_new",
          6: "lengths outside the table or free blocks outside the stack (a state from outside)"}


class OutOfBlocks(RuntimeError):
    """A step could not be held, or a state could not be stepped or truncated; nothing of it was done."""


class PagedKV8(NamedTuple):
    """One layer's cache: codes ``[num_blocks, heads, block_size, 128]``, scales ``[num_blocks, heads]`` fp32."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor
    value_scales: Tensor

    @classmethod
    def create(cls, num_blocks: int, block_size: int, num_heads: int, dtype: torch.dtype = torch.int8,
               device=None, head_dim: int = 128) -> "PagedKV8":
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if dtype not in CODE_TYPES:
            raise ValueError(f"a paged cache holds int8 or float8_e4m3fn, got {dtype}")
        if head_dim != 128:
            raise ValueError(f"the paged cache is specialised for head_dim 128, got {head_dim}")
        # zeros: codes that no request has written are still finite when a masked key reads them
        codes = [torch.zeros((num_blocks, num_heads, block_size, head_dim), dtype=torch.uint8, device=device).view(dtype)
                 for _ in range(2)]
        scales = [torch.zeros((num_blocks, num_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])

    @property
    def block_size(self) -> int:
        return self.keys.shape[2]


class StepPlan(NamedTuple):
    """What one step's layers need; all tensors int32 on the tables' device.

    ``slots`` / ``positions`` ``[num_tokens]``: cache slot and position of each packed new token, requests
    in order (slot -1, position 0 in the rows after the last one). ``cu_new [R + 1]``: first packed row of
    each request. ``kv_lengths [R]``: tokens of each request after the step. ``runs``, ``num_runs``,
    ``cu_units``: work lists of the append and attention kernels. ``tables`` is the live table.
    """

    tables: Tensor
    slots: Tensor
    positions: Tensor
    runs: Tensor
    meta: Tensor  # cu_new, cu_units, kv_lengths, num_runs
    block_size: int
    num_blocks: int
    max_new: int

    @property
    def cu_new(self) -> Tensor:
        return self.meta[:self.tables.shape[0] + 1]

    @property
    def cu_units(self) -> Tensor:
        R = self.tables.shape[0]
        return self.meta[R + 1:2 * R + 2]

    @property
    def kv_lengths(self) -> Tensor:
        return self.meta[2 * self.tables.shape[0] + 2:-1]

    @property
    def num_runs(self) -> Tensor:
        return self.meta[-1:]


class BlockTables:
    """Which blocks each request owns, and the pool they come from (csrc/kernels/paged_tables.cu).

    ``tables [R, max_blocks]`` block ids (-1 where none), ``lengths [R]`` tokens, ``free`` a stack of
    block ids whose first ``num_free`` entries are free.
    """

    def __init__(self, num_blocks: int, block_size: int, max_requests: int, max_blocks: int, device=None):
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if not 1 <= max_requests <= MAX_REQUESTS:
            raise ValueError(f"max_requests must be 1 to {MAX_REQUESTS}, got {max_requests}")
        if num_blocks < 0 or max_blocks < 1 or max(num_blocks, max_blocks) * block_size >= 1 << 31:
            raise ValueError("num_blocks * block_size and max_blocks * block_size must fit in 31 bits")
        self.block_size = block_size
        i32 = dict(dtype=torch.int32, device=device)
        self.tables = torch.full((max_requests, max_blocks), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.free = torch.arange(num_blocks - 1, -1, -1, **i32)  # low ids are handed out first
        self.num_free = torch.full((1,), num_blocks, **i32)
        self.status = torch.zeros(2, **i32)
        self._state = (self.tables, self.lengths, self.free, self.num_free, self.status, torch.zeros(1, **i32), block_size)

    @classmethod
    def restore(cls, tables: Tensor, lengths: Tensor, free: Tensor, num_free: Tensor, block_size: int) -> "BlockTables":
        """Tables in a given state (copied): a server's state moved or resumed."""
        out = cls(free.numel(), block_size, tables.shape[0], tables.shape[1], device=tables.device)
        for mine, given in ((out.tables, tables), (out.lengths, lengths), (out.free, free), (out.num_free, num_free)):
            mine.copy_(given.reshape(mine.shape))
        return out

    def _check(self, value: Tensor, name: str) -> None:
        if value.dtype is not torch.int32 or value.shape != self.lengths.shape or not value.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [{self.lengths.numel()}] on the tables' device")

    def step(self, new_tokens: Tensor, num_tokens: int, max_new: Optional[int] = None) -> StepPlan:
        """Give every request room for ``new_tokens [R]`` more tokens (int32, on the tables' device).

        ``num_tokens`` is the number of packed rows of the step, at least the sum of ``new_tokens``;
        ``max_new`` bounds one request's (a decode step: 1; attention takes a kernel for few rows where it is small). A step that does not fit does nothing: its plan is
        empty, and ``check`` raises.
        """
        self._check(new_tokens, "new_tokens")
        if num_tokens < 0:
            raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
        max_new = num_tokens if max_new is None else min(int(max_new), num_tokens)
        if self.tables.is_cuda:
            return StepPlan(self.tables, *cuda().paged_step(*self._state, new_tokens, num_tokens, max_new), self.block_size,
                            self.free.shape[0], max_new)
        from ..models.paged import step_reference
        return step_reference(self, new_tokens, num_tokens, max_new)

    def truncate(self, keep: Tensor) -> None:
        """Cut every request to at most ``keep [R]`` tokens (int32) and free its surplus blocks. A block that stays in
        part keeps its codes and scales, a scale that tokens now cut had widened among them."""
        self._check(keep, "keep")
        if self.tables.is_cuda:
            cuda().paged_truncate(*self._state, keep)
        else:
            from ..models.paged import truncate_reference
            truncate_reference(self, keep)

    def check(self) -> None:
        """Raise ``OutOfBlocks`` if a step since the last check did not fit, or a call met a state that cannot be (waits for
        the device)."""
        code, request = self.status.tolist()
        if code:
            self.status.zero_()
            raise OutOfBlocks(STATUS[code] + (f" (request {request})" if request >= 0 else ""))


def _check_plan(cache: PagedKV8, plan: StepPlan, rows: int) -> None:
    if not cache.keys.is_cuda:
        raise RuntimeError("hrm_text_b200.ops.paged takes CUDA caches only (models.paged has the CPU oracle)")
    blocks, _, size, _ = cache.keys.shape
    if plan.block_size != size or plan.num_blocks > blocks:
        raise ValueError(f"the plan is for {plan.num_blocks} blocks of {plan.block_size} tokens, the cache has {blocks} of {size}")
    if rows != plan.slots.numel():
        raise ValueError(f"the plan has {plan.slots.numel()} rows, got {rows}")


def paged_append(key: Tensor, value: Tensor, cache: PagedKV8, plan: StepPlan) -> None:
    """Quantise the step's new ``key, value [num_tokens, heads, 128]`` bf16 into ``cache``.

    Rows may have any token and head stride that is a multiple of 16 bytes. A block's scale is the largest
    magnitude it has held over 127 (int8) or 448 (e4m3); where it grows, the block's older codes are
    rounded again. An infinity or NaN makes its block and head read as NaN.
    """
    _check_plan(cache, plan, key.shape[0])
    cuda().paged_append(key, value, cache.keys, cache.values, cache.key_scales, cache.value_scales, plan.runs, plan.meta)


def paged_read(cache: PagedKV8, slots: Tensor) -> tuple[Tensor, Tensor]:
    """Keys and values ``[N, heads, 128]`` bf16 of ``slots [N]`` (int32, as in a plan; -1 reads zeros)."""
    if not cache.keys.is_cuda:
        raise RuntimeError("hrm_text_b200.ops.paged takes CUDA caches only (models.paged has the CPU oracle)")
    if slots.dtype != torch.int32 or slots.dim() != 1:
        raise ValueError("slots must be int32 [N]")
    return cuda().paged_read(*cache, slots.contiguous())


def paged_attention(query: Tensor, cache: PagedKV8, plan: StepPlan, causal: bool = True,
                    gate: Optional[Tensor] = None) -> Tensor:
    """Attention of the step's new tokens over their requests' cached tokens, the new ones included.

    ``query [num_tokens, q_heads, 128]`` bf16, ``q_heads`` a multiple of the cache's heads (query head ``i`` reads
    cache head ``i // (q_heads / heads)``). Each new token sees the tokens up to itself (``causal``) or all of its
    request. With ``gate`` (like ``query``) the result is ``sigmoid(gate) * attention``. Rows of no request are
    zero. Returns ``[num_tokens, q_heads, 128]`` bf16.
    """
    _check_plan(cache, plan, query.shape[0])
    return cuda().paged_attention(query, *cache, plan.tables, plan.meta, plan.max_new, causal, gate)
