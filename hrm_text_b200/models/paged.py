"""Plain torch forms of the paged 8-bit KV cache and the token log probabilities.

The oracle of ``ops.paged`` and ``ops.logprobs``, and what the models run on the CPU: loops over
requests and blocks, fp32 arithmetic in the kernels' order where the result is a code or an id
(so those agree exactly). ``paged_cached_attention`` is the models' attention over a paged cache.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from ..ops.paged import PAIR_COST, UNIT_KEYS, BlockTables, PagedKV8, StepPlan, paged_append, paged_attention

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def step_reference(tables: BlockTables, new_tokens: Tensor, rows: int, max_new: int) -> StepPlan:
    """``BlockTables.step`` on host tensors."""
    size, R = tables.block_size, tables.lengths.numel()
    i32 = dict(dtype=torch.int32)
    plan = StepPlan(tables.tables, torch.empty(rows, **i32), torch.empty(rows, **i32),
                    torch.empty((min(rows, rows // size + 2 * R), 4), **i32), torch.empty(3 * R + 3, **i32), size,
                    tables.free.numel(), max_new)
    lengths, new = tables.lengths.tolist(), new_tokens.tolist()
    blocks = lambda n: -(-n // size)  # noqa: E731
    code, at, most = 0, -1, tables.tables.shape[1] * size
    for i, (length, n) in enumerate(zip(lengths, new)):
        fault = 6 if not 0 <= length <= most else 4 if n < 0 else 5 if n > plan.max_new else 3 if length + n > most else 0
        if fault:
            code, at = fault, i
            break
    need = [max(0, blocks(length + n) - blocks(length)) for length, n in zip(lengths, new)]
    if not code:
        code = 6 if not 0 <= int(tables.num_free) <= tables.free.numel() else 2 if sum(new) > rows else 1 if sum(need) > int(tables.num_free) else 0
    if code:
        new, need = [0] * len(new), [0] * len(new)
        if int(tables.status[0]) == 0:
            tables.status.copy_(torch.tensor([code, at], dtype=torch.int32))
    top, rank, row, units, runs = int(tables.num_free), 0, 0, 0, []
    plan.slots.fill_(-1)
    plan.positions.zero_()
    for i, (length, n) in enumerate(zip(lengths, new)):
        plan.cu_new[i], plan.cu_units[i], plan.kv_lengths[i] = row, units, length + n
        have = blocks(length)
        for j in range(need[i]):
            tables.tables[i, have + j] = tables.free[top - 1 - (rank + j)]
        rank += need[i]
        done = 0
        while done < n:
            pos = length + done
            block, off = int(tables.tables[i, pos // size]), pos % size
            take = min(size - off, n - done)
            runs.append((block, off, take, row + done))
            plan.slots[row + done:row + done + take] = block * size + off + torch.arange(take, dtype=torch.int32)
            plan.positions[row + done:row + done + take] = pos + torch.arange(take, dtype=torch.int32)
            done += take
        row += n
        units += -(-(length + n) // UNIT_KEYS) + PAIR_COST if n else 0
    plan.cu_new[-1], plan.cu_units[-1], plan.num_runs[0] = row, units, len(runs)
    if runs:
        plan.runs[:len(runs)] = torch.tensor(runs, dtype=torch.int32)
    tables.lengths += torch.tensor(new, dtype=torch.int32)
    tables.num_free -= rank
    return plan


def truncate_reference(tables: BlockTables, keep: Tensor) -> None:
    size = tables.block_size
    blocks = lambda n: -(-n // size)  # noqa: E731
    kept = torch.minimum(tables.lengths, keep.clamp_min(0))
    wild = (tables.lengths < 0) | (tables.lengths > size * tables.tables.shape[1])
    surplus = sum(blocks(n) - blocks(k) for k, n in zip(kept.tolist(), tables.lengths.tolist()))
    if wild.any() or not 0 <= int(tables.num_free) <= tables.free.numel() - surplus:
        if int(tables.status[0]) == 0:
            tables.status.copy_(torch.tensor([6, int(wild.int().argmax()) if wild.any() else -1], dtype=torch.int32))
        return
    gone = [(i, b) for i, (k, n) in enumerate(zip(kept.tolist(), tables.lengths.tolist())) for b in range(blocks(k), blocks(n))]
    top = int(tables.num_free)
    for rank, (i, b) in enumerate(gone):
        tables.free[top + len(gone) - 1 - rank] = tables.tables[i, b]
        tables.tables[i, b] = -1
    tables.lengths.copy_(kept)
    tables.num_free += len(gone)


def _codes(x: Tensor, dtype: torch.dtype) -> Tensor:
    x = x.clamp(-QMAX[dtype], QMAX[dtype])
    return x.round().to(dtype) if dtype == torch.int8 else x.to(dtype)


def paged_append_reference(key: Tensor, value: Tensor, cache: PagedKV8, plan: StepPlan) -> None:
    for block, off, take, row in plan.runs[:int(plan.num_runs)].tolist():
        for x, codes, scales in ((key, cache.keys, cache.key_scales), (value, cache.values, cache.value_scales)):
            x = x[row:row + take].float().transpose(0, 1)  # [heads, take, 128]
            before = scales[block].clone() if off else torch.zeros_like(scales[block])
            top = x.abs().amax((1, 2))
            finite = torch.isfinite(x).all(-1).all(-1) & ~before.isnan()
            now = top * torch.tensor(1 / QMAX[codes.dtype], dtype=torch.float32)
            now = torch.where(top > 0, now.clamp_min(2.0 ** -100), now)
            now = torch.where(finite, torch.maximum(now.nan_to_num(0.0), before.nan_to_num(0.0)), torch.nan)
            inv = torch.where(now > 0, 1 / now, torch.zeros_like(now))
            moved = finite & (before > 0) & (now != before)
            old = codes[block, :, :off].float()
            again = _codes(old * (before * inv).nan_to_num(0.0)[:, None, None], codes.dtype).float()
            codes[block, :, :off] = torch.where(moved[:, None, None], again, old).to(codes.dtype)
            fresh = torch.where(finite[:, None, None], x, torch.zeros_like(x)) * inv[:, None, None]
            codes[block, :, off:off + take] = _codes(fresh, codes.dtype)
            scales[block] = now


def paged_read_reference(cache: PagedKV8, slots: Tensor) -> tuple[Tensor, Tensor]:
    size, ids = cache.block_size, slots.long()
    valid = (ids >= 0) & (ids < cache.keys.shape[0] * size)
    block, off = ids.clamp(0, cache.keys.shape[0] * size - 1) // size, ids.clamp_min(0) % size
    out = [torch.where(valid[:, None, None], c.float()[block, :, off] * s[block][..., None], 0.0).to(torch.bfloat16)
           for c, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales))]
    return out[0], out[1]


def paged_attention_reference(query: Tensor, cache: PagedKV8, plan: StepPlan, causal: bool = True,
                              gate: Optional[Tensor] = None, dtype: torch.dtype = torch.float32) -> Tensor:
    """``dtype`` is the arithmetic's; the result has the query's type."""
    heads, size = cache.keys.shape[1], cache.block_size
    group = query.shape[1] // heads
    out = torch.zeros(query.shape, dtype=dtype, device=query.device)
    cu = plan.cu_new.tolist()
    for i, length in enumerate(plan.kv_lengths.tolist()):
        n = cu[i + 1] - cu[i]
        if n == 0:
            continue
        ids = plan.tables[i, :-(-length // size)].long()
        k, v = ((c[ids].to(dtype) * s[ids].to(dtype)[..., None, None]).transpose(0, 1).reshape(heads, -1, 128)[:, :length]
                for c, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)))
        q = query[cu[i]:cu[i + 1]].to(dtype).view(n, heads, group, 128)
        a = torch.einsum("nhgd,hkd->hngk", q, k) / math.sqrt(128)
        last = torch.arange(length - n, length, device=a.device) if causal else torch.full((n,), length - 1, device=a.device)
        unseen = torch.arange(length, device=a.device)[None] > last[:, None]
        a = a.masked_fill(unseen[None, :, None], -math.inf)
        # a NaN value is one for the rows that see it: a weight of zero times NaN would be for all
        poison = v.isnan().any(-1).to(dtype) @ (~unseen).t().to(dtype) > 0  # [heads, n]
        o = torch.einsum("hngk,hkd->nhgd", a.softmax(-1), v.nan_to_num(0.0, math.inf, -math.inf))
        out[cu[i]:cu[i + 1]] = o.masked_fill(poison.t()[:, :, None, None], math.nan).reshape(n, heads * group, 128)
    if gate is not None:
        out = out * torch.sigmoid(gate.to(dtype))
    return out.to(query.dtype)


def token_logprobs_reference(logits: Tensor, tokens: Tensor, top_k: int = 0, ignore: int = -100):
    """``(logprobs, entropy, top_ids, top_logprobs)`` of ``logits [N, V]`` in their own type."""
    empty = (logits == -math.inf).all(-1)
    logp = torch.log_softmax(torch.where(empty[:, None], torch.zeros_like(logits), logits), -1)
    logp = torch.where(empty[:, None], torch.full_like(logp, -math.inf), logp)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.where(p.isnan(), p, torch.zeros_like(p))).sum(-1)
    skip = tokens == ignore
    wild = ~skip & ((tokens < 0) | (tokens >= logits.shape[1]))
    lp = logp.gather(1, tokens.clamp(0, logits.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where(skip, torch.zeros_like(lp), torch.where(wild, torch.full_like(lp, math.nan), lp))
    # NaN above everything, then by value (-0 and 0 are equal), the lowest id first among equals
    order = torch.sort(torch.where(logits.isnan(), torch.full_like(logits, math.inf), logits) + 0.0, dim=-1, descending=True,
                       stable=True).indices
    first = torch.sort(logits.isnan().gather(1, order).to(torch.int8), dim=-1, descending=True, stable=True).indices
    order = order.gather(1, first)
    top = order[:, :top_k]
    return lp, entropy, top, logp.gather(1, top)


def paged_cached_attention(gate: Tensor, query: Tensor, key: Tensor, value: Tensor, cache: PagedKV8, plan: StepPlan,
                           is_causal: bool, prompt: bool) -> Tensor:
    """``sigmoid(gate) * attention`` of a step's packed rows (``[..., heads, 128]`` with as many rows as the plan).

    The step's keys and values go into the cache. A ``prompt`` (one request's tokens into an empty cache) attends to its own
    keys and values as they are, bidirectionally unless the layer is causal, on CUDA by the PrefixLM kernel; any other
    step's tokens attend to the cache up to themselves.
    """
    from .layers import prefixlm_attention_reference
    shape, dtype = query.shape, query.dtype
    gate, query, key, value = (t.reshape(-1, *t.shape[-2:]) for t in (gate, query, key, value))
    if cache.keys.is_cuda:  # the kernels' type
        gate, query, key, value = (t.to(torch.bfloat16) for t in (gate, query, key, value))
    append = paged_append if cache.keys.is_cuda else paged_append_reference
    append(key, value, cache, plan)
    if prompt and cache.keys.is_cuda and query.shape == key.shape:  # the kernel reads the gate and applies it
        from ..ops.attention import PackedSeq, attention_fwd
        n, heads, _ = query.shape
        i32 = dict(dtype=torch.int32, device=query.device)
        packed = PackedSeq(plan.positions, torch.tensor([0, n], **i32), torch.tensor([0 if is_causal else n], **i32))
        gqkv = torch.cat([gate, query, key, value], dim=1).view(n, -1)
        out = attention_fwd(gqkv, heads, packed.schedule(is_causal))[1]
    elif prompt:
        n = query.shape[0]
        cu, prefix = torch.tensor([0, n]), torch.tensor([n])
        out = torch.sigmoid(gate.float()).to(query.dtype) * prefixlm_attention_reference(query, key, value, is_causal, prefix, cu)
    else:
        attend = paged_attention if cache.keys.is_cuda else paged_attention_reference
        out = attend(query, cache, plan, True, gate)
    return out.view(shape).to(dtype)
