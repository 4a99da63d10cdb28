"""Cases of the paged 8-bit KV cache and the token log probabilities, for timing and comparison.

Four kinds of case, each one call (or one pair of calls) as the generation path makes it:

* ``plan``      ``BlockTables.truncate`` back to the lengths before the step, then ``BlockTables.step``;
* ``append``    ``paged_append`` of new keys and values, then ``paged_read`` of every token of the touched blocks;
* ``attend``    ``paged_attention`` of new tokens' queries against the blocks;
* ``logprobs``  ``token_logprobs``, with its gradient where ``grad`` is true.

``run`` computes them in elementary torch operations in 32 bits (``own`` false) or through
``hrm_text_b200.ops`` (``own`` true) on the same inputs; ``exact`` computes them in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

HEAD = 128
QMAX = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def _blocks(tokens, size):
    return (tokens + size - 1) // size


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of the majority-vote batch (25 samples): latency counts
        dict(name="plan decode", kind="plan", requests=25, size=16, low=1, high=4000, new=1, new_low=1),
        # a whole batch of prompts admitted at once: 512 requests, about half a million tokens
        dict(name="plan admit", kind="plan", requests=512, size=64, low=0, high=0, new=2048, new_low=1),
        # decode step of size L (10 heads): one token for each of 33 slots, blocks partly filled
        dict(name="append decode int8", kind="append", code="int8", requests=33, heads=10, size=64, low=1, high=1024,
             new=1, new_low=1),
        # prompts of size XL (12 heads) written after prefill, ragged, into blocks of 32
        dict(name="append prompts fp8", kind="append", code="fp8", requests=8, heads=12, size=32, low=0, high=0,
             new=2500, new_low=300),
        # the smallest attention call: one sequence, one token, a short context
        dict(name="attend one int8", kind="attend", code="int8", requests=1, heads=10, group=1, size=16, low=777,
             high=777, new=1, new_low=1, gate=True, causal=True),
        # decode of size L at the evaluation's batch and a context around 512
        dict(name="attend batch int8", kind="attend", code="int8", requests=33, heads=10, group=1, size=64, low=200,
             high=1000, new=1, new_low=1, gate=True, causal=True),
        # decode of size XL with contexts up to the models' 4096 tokens, 100 slots
        dict(name="attend context fp8", kind="attend", code="fp8", requests=100, heads=12, group=1, size=32, low=1,
             high=4096, new=1, new_low=1, gate=True, causal=True),
        # shared key heads and long contexts: four query heads to a key head
        dict(name="attend long int8", kind="attend", code="int8", requests=16, heads=8, group=4, size=64, low=4000,
             high=40000, new=1, new_low=1, gate=False, causal=True),
        # a few tokens for each request at once (a verified draft, a short continuation), ragged
        dict(name="attend several fp8", kind="attend", code="fp8", requests=12, heads=10, group=2, size=128, low=300,
             high=6000, new=7, new_low=1, gate=False, causal=True),
        # log probabilities beside a decode step's sampled tokens, with five alternatives
        dict(name="logprobs decode", kind="logprobs", rows=33, vocab=32768, dtype="bf16", top=5, grad=False),
        # scoring given answers: a packed batch of 4096 tokens with fp32 logits of an odd vocabulary
        dict(name="logprobs score", kind="logprobs", rows=4096, vocab=32003, dtype="fp32", top=1, grad=False),
        # fine-tuning on log probabilities with an entropy term: both gradients
        dict(name="logprobs train", kind="logprobs", rows=8192, vocab=32768, dtype="bf16", top=0, grad=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "logprobs", "logprobs"])
    size = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        requests = _log_int(rng, 1, 1000)
        most = min(4096, 500_000 // requests)
        if rng.random() < 0.5:  # a decode step
            return dict(kind=kind, requests=requests, size=size, low=1, high=_log_int(rng, 16, 8000), new=1, new_low=1)
        return dict(kind=kind, requests=requests, size=size, low=0, high=_log_int(rng, 1, 4000),
                    new=_log_int(rng, 2, max(2, most)), new_low=rng.choice([0, 1]))
    code = rng.choice(["int8", "fp8"])
    heads = rng.choice([1, 2, 5, 8, 10, 12, 14, 20])
    if kind == "append":
        requests = _log_int(rng, 1, 100)
        if rng.random() < 0.5:
            return dict(kind=kind, code=code, requests=requests, heads=heads, size=size, low=1,
                        high=_log_int(rng, 2, 2000), new=rng.choice([1, 1, 3, 7]), new_low=1)
        return dict(kind=kind, code=code, requests=requests, heads=heads, size=size, low=0,
                    high=_log_int(rng, 1, 300), new=_log_int(rng, 8, max(8, 120_000 // (requests * heads))), new_low=1)
    if kind == "attend":
        requests = _log_int(rng, 1, 200)
        group = rng.choice([1, 1, 1, 2, 4, 7, 8])
        new = rng.choice([1, 1, 1, 2, 5, 8])
        most = min(65536, 2_400_000 // (requests * heads))
        high = _log_int(rng, 8, max(8, most))
        return dict(kind=kind, code=code, requests=requests, heads=heads, group=group, size=size,
                    low=max(1, int(high * rng.choice([0.02, 0.3, 1.0]))), high=high, new=new, new_low=1,
                    gate=rng.random() < 0.5, causal=rng.random() < 0.8)
    vocab = rng.choice([_log_int(rng, 1000, 150_000), 32768, 65536])
    grad = rng.random() < 0.4
    dtype = rng.choice(["bf16", "fp32"])
    rows = _log_int(rng, 1, max(2, (268_000_000 if not grad else 200_000_000) // vocab // (2 if dtype == "fp32" else 1)))
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=0 if grad else rng.choice([0, 1, 5, 20]), grad=grad)


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached and new tokens of each request, from the case alone (so ``work`` can count them)."""
    n = case["requests"]
    g = torch.Generator().manual_seed(1000 * n + case["high"] + case["new"])
    draw_ = lambda low, high: (low + (torch.rand(n, generator=g) * (high - low + 1)).long()).clamp_(low, high)  # noqa: E731
    old, new = draw_(case["low"], case["high"]), draw_(case["new_low"], case["new"])
    if case["kind"] == "attend":  # high is the whole length, new tokens among it
        new = torch.minimum(new, old)
        old = old - new
    return old, new


def _paged(case, gen, dev):
    """Block tables of a server that has run for a while: block ids in no order."""
    size = case["size"]
    old, new = _lengths(case)
    have, width = _blocks(old, size), int(_blocks(old + new, size).max())
    most = int(_blocks(old + new, size).sum())
    spare = most // 8 + 3
    ids = torch.randperm(most + spare, generator=gen, device=dev).to(torch.int32)
    old, new, have = old.to(dev), new.to(dev), have.to(dev)
    first = torch.cumsum(have, 0) - have
    col = torch.arange(max(1, width), device=dev)
    held = col[None] < have[:, None]
    tables = torch.where(held, ids[(first[:, None] + col[None]).clamp_max(most - 1)], -1).to(torch.int32)
    used = int(have.sum())
    free = torch.cat([ids[used:], ids[:used]])  # the stack [0, count), then what is in use
    count = torch.tensor([most + spare - used], dtype=torch.int32, device=dev)
    return dict(tables=tables.contiguous(), lengths=old.to(torch.int32), new=new.to(torch.int32), free=free,
                count=count, blocks=most + spare, total=int(new.sum()), longest=int(new.max()))


def _filled(case, blocks, gen, dev):
    """Codes and scales of a cache in use: normal values, each block with a range of its own."""
    code, heads, size = case["code"], case["heads"], case["size"]
    out = []
    for _ in range(2):
        x = torch.empty((blocks, heads, size, HEAD), dtype=CODE[code], device=dev)
        for i in range(0, blocks, 4096):
            r = torch.randn(x[i:i + 4096].shape, generator=gen, device=dev) * (QMAX[code] / 4)
            r = r.clamp_(-QMAX[code], QMAX[code])
            x[i:i + 4096] = (r.round_() if code == "int8" else r).to(CODE[code])
        s = (torch.rand((blocks, heads), generator=gen, device=dev) + 0.5) * (4 / QMAX[code])
        out += [x, s]
    return dict(k=out[0], ks=out[1], v=out[2], vs=out[3])


def _rows_of(lengths, starts, counts, total):
    """Request and position of each of ``total`` packed rows; request -1 in the rows after the last one."""
    cu = torch.cumsum(counts.long(), 0)
    t = torch.arange(total, device=lengths.device)
    req = torch.searchsorted(cu, t, right=True)
    real = req < lengths.numel()
    req = req.clamp_max(lengths.numel() - 1)
    return req, starts.long()[req] + t - (cu - counts.long())[req], real


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    normal = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        logits = torch.empty((n, v), dtype=dtype, device=dev)
        for i in range(0, n, 2048):
            logits[i:i + 2048] = normal(*logits[i:i + 2048].shape) * 2.5
        tokens = torch.randint(0, v, (n,), generator=gen, device=dev)
        # a trained model's mass lies on a few tokens, the given one often among them
        peak = torch.randint(0, v, (n, 4), generator=gen, device=dev)
        peak[:, 0] = torch.where(torch.rand((n,), generator=gen, device=dev) < 0.6, tokens, peak[:, 0])
        logits.scatter_(1, peak, (normal(n, 4) * 2 + 11).to(dtype))
        st = dict(case, logits=logits, tokens=tokens)
        if case["grad"]:
            st.update(g_lp=normal(n) / n, g_h=normal(n) * (0.01 / n), leaf=logits.detach().requires_grad_())
        return st
    st = dict(case, **_paged(case, gen, dev))
    total = st["total"]
    if kind == "plan":
        st.update(base=st["lengths"].clone(), rows=total + total % 3)
        if own:
            from hrm_text_b200.ops.paged import BlockTables
            st["handle"] = BlockTables.restore(st["tables"], st["lengths"], st["free"], st["count"], case["size"])
        return st
    st.update(_filled(case, st["blocks"], gen, dev))
    heads = case["heads"]
    if kind == "append":
        loud = torch.exp(normal(1, heads, 1) * 0.3)  # heads differ in range
        st.update(key=(normal(total, heads, HEAD) * loud).bfloat16(), value=(normal(total, heads, HEAD) * loud).bfloat16())
        start = (st["lengths"] // case["size"]) * case["size"]  # every token of the touched blocks is read back
        count = st["lengths"] + st["new"] - start
        st.update(read_start=start, read_count=count, read_total=int(count.sum()))
    else:
        hq = heads * case["group"]
        st.update(query=(normal(total, hq, HEAD) * 1.5).bfloat16())
        if case["gate"]:
            st.update(gate_rows=normal(total, hq, HEAD).bfloat16())
    _advance(st)  # blocks of the step's tokens are assigned before its layers run
    if kind == "append":
        req, pos, _ = _rows_of(st["lengths"], st["read_start"], st["read_count"], st["read_total"])
        st["read_slots"] = _slots(st, req, pos).to(torch.int32)
    if own:
        from hrm_text_b200.ops.paged import BlockTables, PagedKV8
        back = st["lengths"] - st["new"]
        st["handle"] = BlockTables.restore(st["tables"], st["lengths"], st["free"], st["count"], case["size"])
        st["handle"].truncate(back)
        st["step"] = st["handle"].step(st["new"], total, max_new=st["longest"])
        st["cache"] = PagedKV8(st["k"], st["v"], st["ks"], st["vs"])
    return st


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _truncate(st, base):
    size, tables, lengths = st["size"], st["tables"], st["lengths"]
    kept = torch.minimum(lengths, base)
    col = torch.arange(tables.shape[1], device=tables.device)
    gone = (col[None] >= _blocks(kept, size)[:, None]) & (col[None] < _blocks(lengths, size)[:, None])
    rank = torch.cumsum(gone.flatten().long(), 0)
    freed = rank[-1]
    to = torch.where(gone.flatten(), st["count"].long() + freed - rank, st["free"].numel())
    stack = torch.cat([st["free"], st["free"].new_zeros(1)])
    stack.scatter_(0, to, tables.flatten())
    st["free"].copy_(stack[:-1])
    tables.masked_fill_(gone, -1)
    lengths.copy_(kept)
    st["count"].add_(freed)


def _slots(st, req, pos):
    return st["tables"][req, pos // st["size"]].long() * st["size"] + pos % st["size"]


def _advance(st, rows=None):
    size, tables, lengths, new = st["size"], st["tables"], st["lengths"].long(), st["new"].long()
    rows = st["total"] if rows is None else rows
    have = _blocks(lengths, size)
    need = _blocks(lengths + new, size) - have
    rank = torch.cumsum(need, 0) - need
    col = torch.arange(tables.shape[1], device=tables.device)
    fresh = (col[None] >= have[:, None]) & (col[None] < (have + need)[:, None])
    at = (st["count"].long() - 1 - (rank[:, None] + col[None] - have[:, None])).clamp(0, st["free"].numel() - 1)
    tables.copy_(torch.where(fresh, st["free"][at], tables))
    req, pos, real = _rows_of(lengths, lengths, new, rows)
    slots = torch.where(real, _slots(st, req, pos.clamp_max(size * tables.shape[1] - 1)), -1).to(torch.int32)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)]).to(torch.int32)
    st["lengths"].add_(st["new"])
    st["count"].sub_(need.sum())
    return slots, torch.where(real, pos, 0).to(torch.int32), cu


def _round_code(x, code):
    x = x.clamp(-QMAX[code], QMAX[code])
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _quantise(st, codes, scales, x):
    """New rows into the touched blocks (one group of consecutive rows per block)."""
    code, size = st["code"], st["size"]
    before = st["lengths"] - st["new"]
    req, pos, _ = _rows_of(st["lengths"], before, st["new"], st["total"])
    slot = _slots(st, req, pos)
    block, off = slot // size, slot % size
    x = x.float()
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")
    low = torch.full((scales.shape[0],), size, dtype=torch.long, device=x.device).index_reduce_(0, block, off, "amin")
    touched = low < size
    held = torch.where((low > 0)[:, None], scales, torch.zeros_like(scales))
    fresh = torch.maximum(held, top * torch.tensor(1 / QMAX[code], device=x.device))
    fresh = torch.where(touched[:, None], fresh, scales)
    back = torch.where(fresh > 0, torch.reciprocal(fresh), torch.zeros_like(fresh))
    # old rows of the blocks that got a wider range
    first, cnt = st["read_start"], st["read_count"] - st["new"]
    oreq, opos, oreal = _rows_of(st["lengths"], first, cnt, max(1, int(st["read_total"] - st["total"])))
    oslot = torch.where(oreal, _slots(st, oreq, opos.clamp_max(size * st["tables"].shape[1] - 1)), slot[0])
    ob, oo = oslot // size, oslot % size
    old = codes[ob, :, oo]
    ratio = (scales[ob] * back[ob])[..., None]
    moved = _round_code(old.float() * ratio, code)
    keep = (fresh[ob] == scales[ob])[..., None]
    codes[ob, :, oo] = torch.where(keep, old.float(), moved.float()).to(codes.dtype)
    codes[block, :, off] = _round_code(x * back[block][..., None], code)
    scales.copy_(fresh)


def _append(st):
    size, slots = st["size"], st["read_slots"].long()
    got = []
    for codes, scales, x in ((st["k"], st["ks"], st["key"]), (st["v"], st["vs"], st["value"])):
        _quantise(st, codes, scales, x)
        got.append((codes[slots // size, :, slots % size].float() * scales[slots // size][..., None]).bfloat16())
    return dict(keys=got[0], values=got[1], key_scales=st["ks"], value_scales=st["vs"])


def _attend(st):
    heads, group, size, n = st["heads"], st["group"], st["size"], st["longest"]
    lengths, new, total = st["lengths"].long(), st["new"].long(), st["total"]
    r, width = st["tables"].shape
    blocks = st["tables"].clamp_min(0).long()
    req, pos, _ = _rows_of(lengths, lengths - new, new, total)
    nth = pos - (lengths - new)[req]
    q = torch.zeros((r, n, heads * group, HEAD), dtype=torch.float32, device=blocks.device)
    q[req, nth] = st["query"].float()
    q = q.view(r, n, heads, group, HEAD).permute(0, 2, 1, 3, 4).reshape(r, heads, n * group, HEAD)
    k = st["k"][blocks].float() * st["ks"][blocks][..., None, None]
    k = k.transpose(1, 2).reshape(r, heads, width * size, HEAD)
    a = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(HEAD))
    del k
    key = torch.arange(width * size, device=a.device)
    last = (lengths - new)[:, None] + torch.arange(n, device=a.device)[None]
    last = last if st["causal"] else last.new_zeros(last.shape) + lengths[:, None] - 1
    seen = (key[None, None] <= last[..., None]) & (key[None, None] < lengths[:, None, None])
    a = a.view(r, heads, n, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True).clamp_min(-1e30))
    a = (a / a.sum(-1, keepdim=True).clamp_min(1e-30)).view(r, heads, n * group, -1)
    v = st["v"][blocks].float() * st["vs"][blocks][..., None, None]
    v = v.transpose(1, 2).reshape(r, heads, width * size, HEAD)
    o = torch.matmul(a, v).view(r, heads, n, group, HEAD).permute(0, 2, 1, 3, 4).reshape(r, n, heads * group, HEAD)
    o = o[req, nth]
    if st["gate"]:
        o = o / (1 + torch.exp(-st["gate_rows"].float()))
    return o.bfloat16()


def _logprobs(st):
    x, t, k = st["logits"].float(), st["tokens"], st["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    log_s = torch.log(s)
    lp = d.gather(1, t[:, None]) - log_s
    h = log_s - (e * d).sum(-1, keepdim=True) / s
    out = dict(logprobs=lp[:, 0], entropy=h[:, 0])
    if k:
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        order = (order << 32) - torch.arange(x.shape[1], device=x.device)  # ties go to the lowest index
        ids = torch.topk(order, k, dim=-1).indices
        out.update(top_ids=ids, top_logprobs=d.gather(1, ids) - log_s)
    if st["grad"]:
        p = e / s
        dx = -p * (st["g_lp"][:, None] + st["g_h"][:, None] * (d - log_s + h))
        dx.scatter_add_(1, t[:, None], st["g_lp"][:, None])
        out["grad"] = dx.to(st["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    kind = state["kind"]
    if not own:
        if kind == "plan":
            _truncate(state, state["base"])
            slots, positions, cu = _advance(state, state["rows"])
            return dict(slots=slots, positions=positions, cu=cu, tables=state["tables"], lengths=state["lengths"],
                        free=state["free"], count=state["count"])
        return {"append": _append, "attend": _attend, "logprobs": _logprobs}[kind](state)
    if kind == "plan":
        handle = state["handle"]
        handle.truncate(state["base"])
        step = handle.step(state["new"], state["rows"])
        return dict(slots=step.slots, positions=step.positions, cu=step.cu_new, tables=handle.tables,
                    lengths=handle.lengths, free=handle.free, count=handle.num_free)
    if kind == "append":
        from hrm_text_b200.ops.paged import paged_append, paged_read
        cache = state["cache"]
        paged_append(state["key"], state["value"], cache, state["step"])
        keys, values = paged_read(cache, state["read_slots"])
        return dict(keys=keys, values=values, key_scales=cache.key_scales, value_scales=cache.value_scales)
    if kind == "attend":
        from hrm_text_b200.ops.paged import paged_attention
        return paged_attention(state["query"], state["cache"], state["step"], causal=state["causal"],
                               gate=state["gate_rows"] if state["gate"] else None)
    from hrm_text_b200.ops.logprobs import token_logprobs
    if state["grad"]:
        got = token_logprobs(state["leaf"], state["tokens"])
        (grad,) = torch.autograd.grad((got.logprobs, got.entropy), (state["leaf"],), (state["g_lp"], state["g_h"]))
        return dict(logprobs=got.logprobs.detach(), entropy=got.entropy.detach(), grad=grad)
    got = token_logprobs(state["logits"], state["tokens"], top_k=state["top"])
    out = dict(logprobs=got.logprobs, entropy=got.entropy)
    if state["top"]:
        out.update(top_ids=got.top_ids, top_logprobs=got.top_logprobs)
    return out


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        each = 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=n * v * each * (2 if case["grad"] else 1) + n * (16 + 12 * case["top"]),
                    flops=n * v * (12 if case["grad"] else 6))
    old, new = _lengths(case)
    size, total = case["size"], int(new.sum())
    fresh = int((_blocks(old + new, size) - _blocks(old, size)).sum())
    if kind == "plan":
        return dict(bytes=total * 8 + fresh * 4 * 4 + case["requests"] * 16, flops=total * 8)
    heads = case["heads"]
    if kind == "append":
        touched = _blocks(old + new, size) - old // size
        read = int((old + new - old // size * size).sum())
        return dict(bytes=heads * HEAD * 2 * (3 * total + 3 * read) + int(touched.sum()) * heads * 16,
                    flops=heads * HEAD * 2 * (4 * total + read))
    whole = old + new
    rows = heads * case["group"]
    pages = int(_blocks(whole, size).sum())
    seen = int((new * whole).sum())
    return dict(bytes=heads * (int(whole.sum()) * HEAD * 2 + pages * 8) + pages * 4 +
                total * rows * HEAD * (6 if case["gate"] else 4), flops=4 * HEAD * rows * seen)


# ------------------------------------------------------------------------------------------
# in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------
def _to_e4m3(x):
    exponent = torch.floor(torch.log2(x.abs().clamp_min(1e-300))).clamp_min(-6)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), exponent - 3)
    return (x / step).round() * step


def _exact_append(st):
    size, code = st["size"], st["code"]
    rnd = torch.round if code == "int8" else _to_e4m3
    tables, old = st["tables"].tolist(), (st["lengths"] - st["new"]).tolist()
    new = st["new"].tolist()
    out = {}
    for name, codes, scales, x in (("key", st["k"], st["ks"], st["key"]), ("value", st["v"], st["vs"], st["value"])):
        after, parts, row = scales.double(), [], 0
        for i, (length, count) in enumerate(zip(old, new)):
            done, first = 0, length // size
            while done < count:
                at = length + done
                block, off = tables[i][at // size], at % size
                take = min(size - off, count - done)
                fresh = x[row + done:row + done + take].double()          # [take, heads, 128]
                held = codes[block, :, :off].double().transpose(0, 1)    # [off, heads, 128]
                wide = fresh.abs().amax((0, 2)) / QMAX[code]
                if off:
                    wide = torch.maximum(wide, scales[block].double())
                    kept = torch.where((wide == scales[block].double())[None, :, None], held,
                                       rnd(held * (scales[block].double() / wide)[None, :, None]))
                    parts.append(kept * wide[None, :, None])
                after[block] = wide
                over = wide.clamp_min(1e-300)[None, :, None]
                parts.append(rnd((fresh / over).clamp(-QMAX[code], QMAX[code])) * wide[None, :, None])
                done += take
            if count == 0 and length % size:
                block = tables[i][first]
                parts.append(codes[block, :, :length % size].double().transpose(0, 1) * scales[block].double()[None, :, None])
            row += count
        out[name + "s"], out[name + "_scales"] = torch.cat(parts), after
    return out


def _exact_attend(st):
    heads, group = st["heads"], st["group"]
    out, row = [], 0
    for i, (length, count) in enumerate(zip(st["lengths"].tolist(), st["new"].tolist())):
        ids = st["tables"][i, :_blocks(length, st["size"])].long()
        flat = lambda c, s: (c[ids].double() * s[ids].double()[..., None, None]).transpose(0, 1).reshape(heads, -1, HEAD)[:, :length]  # noqa: E731
        k, v = flat(st["k"], st["ks"]), flat(st["v"], st["vs"])
        q = st["query"][row:row + count].double().view(count, heads, group, HEAD)
        a = torch.einsum("nhgd,hkd->hngk", q, k) / math.sqrt(HEAD)
        if st["causal"]:
            key = torch.arange(length, device=a.device)
            last = torch.arange(length - count, length, device=a.device)
            a = a.masked_fill((key[None] > last[:, None])[None, :, None], -math.inf)
        out.append(torch.einsum("hngk,hkd->nhgd", torch.softmax(a, -1), v).reshape(count, heads * group, HEAD))
        row += count
    o = torch.cat(out)
    return o * torch.sigmoid(st["gate_rows"].double()) if st["gate"] else o


def _exact_logprobs(st):
    parts = []
    for i in range(0, st["rows"], 512):
        x, t = st["logits"][i:i + 512].double(), st["tokens"][i:i + 512]
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        h = -(p * logp).sum(-1)
        one = dict(logprobs=logp.gather(1, t[:, None])[:, 0], entropy=h)
        if st["top"]:
            best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :st["top"]]
            one.update(top_ids=best, top_logprobs=logp.gather(1, best))
        if st["grad"]:
            g = -p * st["g_lp"][i:i + 512, None].double() - p * (logp + h[:, None]) * st["g_h"][i:i + 512, None].double()
            g.scatter_add_(1, t[:, None], st["g_lp"][i:i + 512, None].double())
            one["grad"] = g
        parts.append(one)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](st)
