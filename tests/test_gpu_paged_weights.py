"""Paged attention where the value ranges of a request's blocks, or of its rows' futures, differ widely.

The kernel multiplies a softmax weight by its block's value scale, relative to the largest such product of the
row so far, before it rounds it to f16: each product that counts is good to 2^-11 of itself, and what is lost altogether is
below 2^-24 of the largest. exp2 is good to 2^-21, and scores of magnitude 100 carry 2^-14 of rounding into it. With the
output's own rounding to bf16 that makes 2^-8 |o| + 2^-10 sum p |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.int8, torch.float8_e4m3fn]


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _request(device, dtype, heads, size, lengths):
    """A cache of ones, scales 1, and the plan of the last token of each request."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8
    most = max(lengths)
    bt = BlockTables(sum(-(-n // size) for n in lengths), size, len(lengths), -(-most // size), device)
    cache = PagedKV8.create(bt.free.numel(), size, heads, dtype, device)
    bt.step(_i32([n - 1 for n in lengths], device), sum(lengths) - len(lengths))
    plan = bt.step(_i32([1] * len(lengths), device), len(lengths), max_new=1)
    bt.check()
    for scales in (cache.key_scales, cache.value_scales):
        scales.fill_(1.0)
    return bt, cache, plan


def _bound(out, q, cache, plan, causal=True):
    from hrm_text_b200.models.paged import paged_attention_reference
    want = paged_attention_reference(q.double(), cache, plan, causal, dtype=torch.float64)
    mass = paged_attention_reference(q.double(), cache._replace(values=cache.values.float().abs()), plan, causal, dtype=torch.float64)
    excess = (out.double() - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -10 * mass)
    assert torch.isfinite(out.float()).all() and excess.max() <= 0, float((excess / mass).max())


# a query of sqrt(128) in dim 0 makes the first code of a key its score (natural logarithm)
def _query(rows, heads, device):
    q = torch.zeros(rows, heads, 128, device=device)
    q[:, :, 0] = math.sqrt(128)
    return q.bfloat16()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seed", range(4))
def test_weights_and_ranges_against_each_other(cuda_device, dtype, seed):
    """Blocks whose scores differ by 70 and whose value scales by 2^120: any of them may decide a row."""
    from hrm_text_b200.ops.paged import paged_attention
    g = torch.Generator(device=cuda_device).manual_seed(seed)
    lengths = [700, 33, 4000, 1]
    bt, cache, plan = _request(cuda_device, dtype, 3, 16, lengths)
    blocks = cache.keys.shape[0]
    score = torch.randint(-33, 34, (blocks, 3, 1), generator=g, device=cuda_device)
    codes = torch.randint(-100, 101, cache.values.shape, generator=g, device=cuda_device)
    cache.values.copy_(codes.to(dtype))
    cache.keys[..., 0] = (score + torch.randint(-2, 3, (blocks, 3, 16), generator=g, device=cuda_device)).to(dtype)
    cache.value_scales.copy_(torch.exp2(torch.randint(-60, 61, (blocks, 3), generator=g, device=cuda_device).float()))
    q = _query(4, 3, cuda_device)
    _bound(paged_attention(q, cache, plan), q, cache, plan)


@pytest.mark.parametrize("dtype", TYPES)
def test_all_the_weight_on_small_values(cuda_device, dtype):
    """Blocks of values around 2^-80 with all the weight, among blocks of ordinary values with none."""
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, plan = _request(cuda_device, dtype, 2, 16, [640, 640])
    cache.values.copy_(torch.full_like(cache.values, 64.0, dtype=torch.float32).to(dtype))
    for i in range(2):
        chosen = bt.tables[i, 5 + 13 * i].long()
        cache.value_scales[chosen] = 2.0 ** -80
        cache.keys[chosen, :, :, 0] = torch.tensor(96.0).to(dtype).to(cuda_device)
    q = _query(2, 2, cuda_device)
    out = paged_attention(q, cache, plan)
    assert ((out.double() / (64 * 2.0 ** -80) - 1).abs() <= 2.0 ** -7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_ranges_that_fall_again_and_again(cuda_device, dtype):
    """Values of 2^100, 2^50, 1 and 2^-50 in a request's order: the first decide, and nothing overflows on the way."""
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, plan = _request(cuda_device, dtype, 10, 16, [512] * 60)
    cache.values.copy_(torch.full_like(cache.values, 96.0, dtype=torch.float32).to(dtype))
    for i in range(60):
        for unit, e in enumerate((100, 50, 0, -50)):
            cache.value_scales[bt.tables[i, 8 * unit:8 * unit + 8].long()] = 2.0 ** e
    q = _query(60, 10, cuda_device)
    _bound(paged_attention(q, cache, plan), q, cache, plan)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_small_weights_of_small_values(cuda_device, dtype):
    """Equal products of a small weight and a small scale round alike, so their error does not average out: the
    result is of values around 2^-3 with weights of e^-7 each, after a block of large values with no weight."""
    from hrm_text_b200.ops.paged import paged_attention
    lengths = [1024] * 50
    bt, cache, plan = _request(cuda_device, dtype, 10, 16, lengths)
    cache.values.copy_(torch.full_like(cache.values, 96.0, dtype=torch.float32).to(dtype))
    cache.keys[..., 0] = torch.tensor(-7.0).to(dtype).to(cuda_device)
    cache.value_scales.fill_(16.45 * 2.0 ** -24 * math.exp(7.0))
    first = bt.tables[:, :8].long().flatten()
    cache.value_scales[first] = 1.0
    cache.keys[first, :, :, 0] = torch.tensor(-60.0).to(dtype).to(cuda_device)
    second = bt.tables[:, 8:16].long().flatten()   # each sixteen keys' first has the largest score and no value
    cache.keys[second, :, 0, 0] = torch.tensor(0.0).to(dtype).to(cuda_device)
    cache.values[second, :, 0] = torch.tensor(0.0).to(dtype).to(cuda_device)
    q = _query(50, 10, cuda_device)
    _bound(paged_attention(q, cache, plan), q, cache, plan)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["key", "value"])
def test_nan_does_not_reach_earlier_tokens(cuda_device, dtype, where):
    """A NaN token poisons its own block; a token before that block does not see it, with any neighbours in its tile."""
    from hrm_text_b200.models.paged import paged_append_reference, paged_attention_reference
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(7)
    for old, new in ((14, 3), (127, 2), (30, 7), (300, 6)):
        sides = []
        kv = torch.randn(old + new, 2, 2, 128).bfloat16()
        at = -(-(old + 1) // 16) * 16              # the first token of the block after the first new one's
        kv[at, 0 if where == "key" else 1, 0, 3] = math.nan
        for dev in (cuda_device, torch.device("cpu")):
            bt = BlockTables(64, 16, 1, 40, dev)
            cache = PagedKV8.create(64, 16, 2, dtype, dev)
            append = paged_append if dev == cuda_device else paged_append_reference
            for a, b in ((0, old), (old, old + new)):
                plan = bt.step(_i32([b - a], dev), b - a)
                append(kv[a:b, 0].to(dev), kv[a:b, 1].to(dev), cache, plan)
            sides.append((cache, plan))
        q = torch.randn(new, 2, 128).bfloat16()
        out = paged_attention(q.to(cuda_device), *sides[0]).cpu()
        want = paged_attention_reference(q.double(), *sides[1], dtype=torch.float64)
        before = at - old
        assert 0 < before < new and torch.isfinite(want[:before]).all() and torch.isfinite(want[:, 1]).all()
        assert torch.isfinite(out[:before]).all() and torch.isfinite(out[:, 1]).all()
        assert out[before:, 0].isnan().all() and want[before:, 0].isnan().all()
        ok = torch.isfinite(want)
        top = float(kv[:, 1].float().abs().nan_to_num(0.0).max()) * 1.07  # no read-back value is larger
        assert ((out.double() - want)[ok].abs() <= (2.0 ** -8 * want.abs() + 2.0 ** -10 * top)[ok]).all()


def test_many_requests_in_one_step(cuda_device):
    """A packed step of many requests whose plan does not know that each has few tokens: the grid and the workspace
    stay bounded by what one request can have, and the result does not depend on it."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(8)
    requests, heads, group = 400, 2, 4
    new = [(i * 7) % 48 + 12 for i in range(requests)]
    rows = sum(new)
    assert rows * group / 16 > 1776 * 1.5
    bt = BlockTables(requests * 2, 64, requests, 300, cuda_device)
    cache = PagedKV8.create(requests * 2, 64, heads, torch.int8, cuda_device)
    plan = bt.step(_i32(new, cuda_device), rows)
    x = torch.randn(rows, 2, heads, 128, device=cuda_device).bfloat16()
    paged_append(x[:, 0], x[:, 1], cache, plan)
    q = torch.randn(rows, heads * group, 128, device=cuda_device).bfloat16()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = paged_attention(q, cache, plan)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < (33 << 20) + out.numel() * 2
    _bound(out, q, cache, plan)
    tight = paged_attention(q, cache, plan._replace(max_new=max(new)))
    _bound(tight, q, cache, plan)


def test_half_a_million_rows_in_one_step(cuda_device):
    """More nominal tiles than a launch's second grid dimension takes; no request has more than a thousand tokens."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(9)
    requests, group = 530, 2
    new = [1000] * requests
    rows = sum(new)
    bt = BlockTables(requests * 8, 128, requests, -(-rows // 128), cuda_device)
    cache = PagedKV8.create(requests * 8, 128, 1, torch.float8_e4m3fn, cuda_device)
    plan = bt.step(_i32(new, cuda_device), rows)
    bt.check()
    assert rows * group / 16 > 65535
    x = torch.randn(rows, 2, 1, 128, device=cuda_device).bfloat16()
    paged_append(x[:, 0], x[:, 1], cache, plan)
    q = torch.randn(rows, group, 128, device=cuda_device).bfloat16()
    out = paged_attention(q, cache, plan)
    tight = paged_attention(q, cache, plan._replace(max_new=1000))
    assert torch.isfinite(out.float()).all()
    for i in (0, 1, 263, 529):
        part = slice(i * 1000, (i + 1) * 1000)
        ids = bt.tables[i, :8].long()
        k, v = ((c[ids].double() * s[ids].double()[..., None, None]).reshape(-1, 128)[:1000]
                for c, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)))
        a = torch.einsum("ngd,kd->gnk", q[part].double(), k) / math.sqrt(128)
        a = a.masked_fill(torch.ones(1000, 1000, dtype=torch.bool, device=cuda_device).triu(1), -math.inf).softmax(-1)
        o, mass = (a @ v).transpose(0, 1), (a @ v.abs()).transpose(0, 1)
        for got in (out, tight):
            assert ((got[part].double() - o).abs() <= 2.0 ** -8 * o.abs() + 2.0 ** -10 * mass).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_grid_follows_the_step(cuda_device, dtype):
    """What the plan says of one request's new tokens bounds the grid only: the work is cut by what the step has, so
    the same step gives the same bits with a loose bound and with a tight one."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(11)
    for new, width in (([65, 3, 0, 700, 1], 12), ([90] * 300, 20), ([0, 0, 130], 40)):
        rows = sum(new) + 2
        bt = BlockTables(sum(-(-n // 64) for n in new) + 1, 64, len(new), width, cuda_device)
        cache = PagedKV8.create(bt.free.numel(), 64, 2, dtype, cuda_device)
        plan = bt.step(_i32(new, cuda_device), rows)
        bt.check()
        x = torch.randn(rows, 2, 2, 128, device=cuda_device).bfloat16()
        paged_append(x[:, 0], x[:, 1], cache, plan)
        q = torch.randn(rows, 4, 128, device=cuda_device).bfloat16()
        out = paged_attention(q, cache, plan)
        assert (out[sum(new):] == 0).all()
        _bound(out[:sum(new)], q[:sum(new)], cache, plan)
        assert torch.equal(out, paged_attention(q, cache, plan._replace(max_new=max(new))))


def _states():
    """(lengths, free blocks, request at fault) that no steps lead to, for tables of 3 requests of 4 blocks and a pool of 8."""
    return [([3, 65, 0], 6, 1), ([3, 0, -1], 6, 2), ([3, 2 ** 31 - 1, 0], 6, 1), ([-(2 ** 31), 70, 0], 6, 0), ([3, 0, 0], 9, -1),
            ([3, 0, 0], -1, -1), ([3, 0, 0], 2 ** 31 - 1, -1)]


@pytest.mark.parametrize("lengths,free,at", _states())
def test_states_that_cannot_be_change_nothing(cuda_device, lengths, free, at):
    from hrm_text_b200.ops.paged import BlockTables, OutOfBlocks
    for dev in (cuda_device, torch.device("cpu")):
        bt = BlockTables(8, 16, 3, 4, dev)
        bt.step(_i32([3, 17, 0], dev), 20)
        bt.lengths.copy_(_i32(lengths, dev))
        bt.num_free.fill_(free)
        before = [t.clone() for t in (bt.tables, bt.lengths, bt.free, bt.num_free)]
        words = "outside" + (rf".*request {at}" if at >= 0 else "")
        for call in (lambda: bt.step(_i32([1, 1, 1], dev), 3), lambda: bt.truncate(_i32([0, 0, 0], dev)),
                     lambda: bt.truncate(_i32([1 << 30] * 3, dev))):
            plan = call()
            assert plan is None or (plan.slots == -1).all() and int(plan.num_runs) == 0
            for t, was in zip((bt.tables, bt.lengths, bt.free, bt.num_free), before):
                assert torch.equal(t, was)
            with pytest.raises(OutOfBlocks, match=words):
                bt.check()
            bt.check()
        bt.lengths.copy_(_i32([3, 17, 0], dev))
        bt.num_free.fill_(5)
        assert bt.step(_i32([1, 1, 1], dev), 3).slots.min() >= 0


def test_a_full_stack_takes_no_more_blocks(cuda_device):
    """A restored state in which blocks are both owned and free."""
    from hrm_text_b200.ops.paged import BlockTables, OutOfBlocks
    for dev in (cuda_device, torch.device("cpu")):
        bt = BlockTables(8, 16, 3, 4, dev)
        bt.step(_i32([3, 17, 0], dev), 20)
        twin = BlockTables.restore(bt.tables, bt.lengths, bt.free, torch.full_like(bt.num_free, 6), 16)
        twin.truncate(_i32([3, 0, 0], dev))          # two more fit exactly
        twin.check()
        assert int(twin.num_free) == 8 and twin.lengths.tolist() == [3, 0, 0]
        twin.truncate(_i32([0, 0, 0], dev))
        with pytest.raises(OutOfBlocks, match="outside"):
            twin.check()
        assert int(twin.num_free) == 8 and twin.lengths.tolist() == [3, 0, 0]


def test_strides_of_a_single_row(cuda_device):
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(3)
    bt = BlockTables(4, 16, 1, 4, cuda_device)
    cache = PagedKV8.create(4, 16, 1, torch.int8, cuda_device)
    plan = bt.step(_i32([1], cuda_device), 1)
    wide = torch.randn(3, 259, device=cuda_device).bfloat16()
    odd = torch.as_strided(wide, (1, 1, 128), (259, 131, 1))   # one row and one head: nothing steps by 259 or 131
    paged_append(odd, odd, cache, plan)
    out = paged_attention(odd, cache, plan, gate=odd)
    want = odd.contiguous().float()
    assert ((out.float() - want * torch.sigmoid(want)).abs() <= 0.02).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("chunk,group,size", [(700, 2, 64), (5000, 1, 16), (130, 7, 32)])
def test_late_tiles_see_exactly_their_keys(cuda_device, dtype, chunk, group, size):
    """Each new token's own key has nearly all its weight, and the next token's key would have as much if it were seen."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(chunk)
    heads, old = 2, [300, 1000]
    bt = BlockTables(2 * (-(-(1000 + chunk) // size) + 1), size, 2, -(-(1000 + chunk) // size), cuda_device)
    cache = PagedKV8.create(bt.free.numel(), size, heads, dtype, cuda_device)
    k, v = (torch.randn(sum(old), heads, 128, device=cuda_device).bfloat16() for _ in range(2))
    paged_append(k, v, cache, bt.step(_i32(old, cuda_device), sum(old)))
    plan = bt.step(_i32([chunk, 1], cuda_device), chunk + 1)
    bt.check()
    k, v = (torch.randn(chunk + 1, heads, 128, device=cuda_device).bfloat16() for _ in range(2))
    paged_append(k, v, cache, plan)
    after = torch.cat([k[1:], k[:1]]).float()
    q = (4 * (k.float() + after)).repeat_interleave(group, 1).bfloat16()
    out = paged_attention(q, cache, plan)
    own = v.float().repeat_interleave(group, 1)
    assert ((out.float() - own).abs().mean((1, 2)) < 0.3).all()   # more than 0.5 where another token's value is mixed in
    # with all the weight on one key the rest is lost below 2^-24 of it: 2^-8 |o| for bf16 and 2^-10 of the largest value
    from hrm_text_b200.models.paged import paged_attention_reference
    want = paged_attention_reference(q.double(), cache, plan, dtype=torch.float64)
    top = float(cache.value_scales.max()) * (127 if dtype == torch.int8 else 448)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * top).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most", [5, 17, 32])
def test_few_rows_with_a_loose_bound(cuda_device, dtype, most):
    """One to four tiles of rows a request, nominally many: cut as with the tight bound, to the same bits."""
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention
    torch.manual_seed(most)
    new = [1 + (i * 5) % most for i in range(80)]
    old = [(i * 37) % 900 for i in range(80)]
    bt = BlockTables(80 * 30, 32, 80, 30, cuda_device)
    cache = PagedKV8.create(80 * 30, 32, 3, dtype, cuda_device)
    for step in (old, new):
        rows = sum(step)
        plan = bt.step(_i32(step, cuda_device), rows)
        x = torch.randn(rows, 2, 3, 128, device=cuda_device).bfloat16()
        paged_append(x[:, 0], x[:, 1], cache, plan)
    bt.check()
    q = torch.randn(rows, 6, 128, device=cuda_device).bfloat16()
    out = paged_attention(q, cache, plan)
    _bound(out, q, cache, plan)
    assert torch.equal(out, paged_attention(q, cache, plan._replace(max_new=max(new))))
