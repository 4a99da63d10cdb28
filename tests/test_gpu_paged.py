"""Paged 8-bit KV cache kernels against the plain torch forms (in 64 bits where they round).

Tolerances. Block tables, slots and codes are compared exactly: the oracle rounds in fp32 in the same
order. Attention: the output is rounded to bf16 (at most 2^-8 of itself), P to f16 (2^-11 each, so at most
2^-11 of the weighted mean of |v|, itself at most sqrt(mean v^2)), the queries are exact in f16, exp2 is good to
2^-21 and scores of magnitude 30 carry 2^-19 of rounding into it. Held to 2^-9 |o| + 2^-10 max|v|, which is tighter
than their sum where one key has nearly all the weight and looser where many share it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.int8, torch.float8_e4m3fn]


def _tables(device, requests, size, lengths, max_len, spare=5):
    from hrm_text_b200.ops.paged import BlockTables
    blocks = sum(-(-n // size) for n in lengths) + requests * 3 + spare
    bt = BlockTables(blocks, size, requests, -(-max_len // size), device)
    g = torch.Generator().manual_seed(5)
    bt.free.copy_(bt.free[torch.randperm(blocks, generator=g).to(device)])  # ids in no order
    return bt


def _twin(bt):
    from hrm_text_b200.ops.paged import BlockTables
    return BlockTables.restore(bt.tables.cpu(), bt.lengths.cpu(), bt.free.cpu(), bt.num_free.cpu(), bt.block_size)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _same_plan(a, b):
    n = int(b.num_runs)
    for name in ("slots", "positions", "cu_new", "kv_lengths", "cu_units", "num_runs", "tables"):
        assert torch.equal(getattr(a, name).cpu(), getattr(b, name).cpu()), name
    assert torch.equal(a.runs[:n].cpu(), b.runs[:n].cpu()), "runs"


def _same_state(a, b):
    for name in ("tables", "lengths", "free", "num_free", "status"):
        assert torch.equal(getattr(a, name).cpu(), getattr(b, name).cpu()), name


@pytest.mark.parametrize("requests,size,most", [(1, 16, 1), (1, 128, 700), (33, 16, 70), (300, 32, 40), (1025, 64, 9)])
def test_steps_match_reference(cuda_device, requests, size, most):
    g = torch.Generator().manual_seed(requests + size)
    bt = _tables(cuda_device, requests, size, [6 * most] * requests, 8 * most + size)
    ref = _twin(bt)
    for k in range(4):
        new = torch.randint(0, most + 1, (requests,), generator=g).int()
        if k == 1:
            new = (new > 0).int()  # a decode step in which some requests do not take part
        before = ref.lengths.clone()
        pad = k * 3
        rows = int(new.sum()) + pad
        a, b = bt.step(new.to(cuda_device), rows), ref.step(new, rows)
        _same_plan(a, b)
        _same_state(bt, ref)
        assert torch.equal(a.slots[rows - pad:].cpu(), torch.full((pad,), -1, dtype=torch.int32))
        if k == 2:  # undone exactly
            free = ref.free.clone()
            bt.truncate(before.to(cuda_device)), ref.truncate(before)
            _same_state(bt, ref)
            assert torch.equal(ref.free, free) and torch.equal(bt.lengths.cpu(), before)
    keep = torch.where(torch.arange(requests) % 3 == 0, torch.zeros(requests), ref.lengths / 2).int()
    keep[-1] = 1 << 30  # more than it has: kept whole
    bt.truncate(keep.to(cuda_device)), ref.truncate(keep)
    _same_state(bt, ref)


@pytest.mark.parametrize("new,rows,max_new,words", [
    ([40, 40, 0], 80, None, "free blocks"), ([9, 9, 0], 17, None, "num_tokens"), ([1, 65, 0], 80, None, "table"),
    ([1, -1, 0], 80, None, "negative"), ([1, 2, 0], 80, 1, "max_new")])
def test_step_that_does_not_fit_does_nothing(cuda_device, new, rows, max_new, words):
    from hrm_text_b200.ops.paged import BlockTables, OutOfBlocks
    for dev in (cuda_device, torch.device("cpu")):
        bt = BlockTables(4, 16, 3, 4, dev)
        bt.step(_i32([3, 0, 0], dev), 3)
        before = [t.clone() for t in (bt.tables, bt.lengths, bt.free, bt.num_free)]
        plan = bt.step(_i32(new, dev), rows, max_new)
        assert (plan.slots == -1).all() and (plan.cu_new == 0).all() and int(plan.num_runs) == 0
        for t, was in zip((bt.tables, bt.lengths, bt.free, bt.num_free), before):
            assert torch.equal(t, was)
        with pytest.raises(OutOfBlocks, match=words):
            bt.check()
        bt.check()  # said once
        assert bt.step(_i32([1, 1, 1], dev), 3).slots.min() >= 0


def _filled(device, dtype, heads, size, lengths, steps=(), extra=64):
    """A cache and its tables after appending ``lengths`` at once, then ``steps`` of new tokens."""
    from hrm_text_b200.ops.paged import PagedKV8, paged_append
    torch.manual_seed(sum(lengths) + heads)
    most = max(lengths) + sum(max(s) for s in steps) + extra
    bt = _tables(device, len(lengths), size, [most] * len(lengths), most)
    cache = PagedKV8.create(bt.free.numel(), size, heads, dtype, device)
    plan = None
    for new in (lengths, *steps):
        rows = sum(new)
        plan = bt.step(_i32(new, device), rows)
        k, v = (torch.randn(rows, heads, 128, device=device).bfloat16() for _ in range(2))
        paged_append(k, v, cache, plan)
    return bt, cache, plan


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_append_matches_reference_exactly(cuda_device, dtype, size):
    from hrm_text_b200.models.paged import paged_append_reference, paged_read_reference
    from hrm_text_b200.ops.paged import PagedKV8, paged_append, paged_read
    torch.manual_seed(size)
    heads, lengths = 3, [1, 0, size, size + 1, 3 * size - 1, 7]
    bt = _tables(cuda_device, len(lengths), size, [8 * size] * len(lengths), 8 * size)
    ref = _twin(bt)
    cache = PagedKV8.create(bt.free.numel(), size, heads, dtype, cuda_device)
    host = PagedKV8.create(bt.free.numel(), size, heads, dtype)
    for k, new in enumerate((lengths, [1] * 6, [2, 0, 5, size, 1, size // 2], [1] * 6)):
        rows = sum(new) + 2
        plan, hplan = bt.step(_i32(new, cuda_device), rows), ref.step(_i32(new, "cpu"), rows)
        # ranges grow from step to step, so older tokens are rounded again; one head stays all zero,
        # the rows come out of a wider tensor
        wide = torch.randn(rows, 4, heads, 128) * (1.7 ** k)
        wide[:, :, 1] = 0
        wide = wide.bfloat16()
        dwide = wide.to(cuda_device)
        paged_append(dwide[:, 2], dwide[:, 3], cache, plan)
        paged_append_reference(wide[:, 2], wide[:, 3], host, hplan)
        for a, b in zip(cache, host):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)), k
    slots = torch.cat([plan.slots, _i32([-1, 0, 1 << 30], cuda_device)])
    got, want = paged_read(cache, slots), paged_read_reference(host, slots.cpu())
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_error_is_half_a_step(cuda_device, dtype):
    """Read back, a token is within half a code step (int8) or 2^-4 of itself (e4m3), plus bf16's 2^-8."""
    from hrm_text_b200.ops.paged import PagedKV8, paged_append, paged_read
    torch.manual_seed(3)
    bt = _tables(cuda_device, 2, 32, [100, 100], 100)
    cache = PagedKV8.create(bt.free.numel(), 32, 2, dtype, cuda_device)
    plan = bt.step(_i32([70, 31], cuda_device), 101)
    k, v = (torch.randn(101, 2, 128, device=cuda_device).bfloat16() for _ in range(2))
    paged_append(k, v, cache, plan)
    for x, y, s in zip((k, v), paged_read(cache, plan.slots), (cache.key_scales, cache.value_scales)):
        scale = s[(plan.slots // 32).long()][..., None]
        half = 0.5 * scale if dtype == torch.int8 else x.float().abs() / 16 + scale * 2.0 ** -10
        assert ((x.float() - y.float()).abs() <= half * (1 + 1e-5) + x.float().abs() * 2.0 ** -8).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_extremes(cuda_device, dtype):
    """NaN and infinity poison their block and head only, and only until the block is written anew; the
    smallest and largest finite values stay finite."""
    from hrm_text_b200.ops.paged import PagedKV8, paged_append, paged_attention, paged_read
    bt = _tables(cuda_device, 3, 16, [16] * 3, 64)
    cache = PagedKV8.create(bt.free.numel(), 16, 2, dtype, cuda_device)
    k = torch.ones(30, 2, 128, device=cuda_device).bfloat16()
    k[3, 0, 5], k[13, 1, 0] = float("nan"), float("inf")
    k[20:25] *= 1e-40
    k[25:30] *= 3e38
    plan = bt.step(_i32([10, 10, 10], cuda_device), 30)
    paged_append(k, k, cache, plan)
    got = paged_read(cache, plan.slots)[0].float()
    assert got[:10, 0].isnan().all() and not got[:10, 1].isnan().any()
    assert got[10:20, 1].isnan().all() and not got[10:20, 0].isnan().any()
    assert torch.isfinite(got[20:]).all()
    assert torch.isfinite(cache.keys.float()).all() and torch.isfinite(cache.values.float()).all()
    out = paged_attention(torch.ones(30, 2, 128, device=cuda_device).bfloat16(), cache, plan, causal=False).float()
    assert out[:10, 0].isnan().all() and torch.isfinite(out[:10, 1]).all()
    assert out[10:20, 1].isnan().all() and torch.isfinite(out[10:20, 0]).all()
    paged_append(k[:3], k[:3], cache, bt.step(_i32([1, 1, 1], cuda_device), 3))  # stays poisoned
    assert paged_read(cache, plan.slots)[0][:10, 0].isnan().all()
    bt.truncate(_i32([0, 0, 0], cuda_device))
    plan = bt.step(_i32([2, 2, 2], cuda_device), 6)
    fine = torch.ones(6, 2, 128, device=cuda_device).bfloat16()
    paged_append(fine, fine, cache, plan)
    out = paged_attention(fine, cache, plan).float()
    torch.testing.assert_close(out, torch.ones_like(out), rtol=2.0 ** -7, atol=0)


def _close(out, want, cache):
    out, want = out.double(), want.double()
    assert torch.isfinite(out).all()
    top = (cache.value_scales.max() * (127 if cache.keys.dtype == torch.int8 else 448)).double()
    excess = (out - want).abs() - (2.0 ** -9 * want.abs() + 2.0 ** -10 * top)
    assert excess.max() <= 0, float(excess.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,size,lengths,last", [
    (10, 1, 16, [1], [1]),                          # two tokens in all
    (2, 1, 64, [127, 128, 129, 1, 63], [1] * 5),    # around a unit of 128 keys and a block
    (3, 4, 32, [500, 33, 2000], [1, 1, 1]),
    (1, 8, 128, [4000], [1]),                       # one pair over many CTAs
    (5, 2, 16, [300, 0, 40, 1000], [3, 2, 0, 8]),   # a request that starts, one that sits out
    (2, 7, 64, [100, 900], [5, 2]),                 # 35 rows: more than one tile of 32
    (4, 3, 32, [700] * 40, [1] * 40),
    (20, 1, 128, [5] * 260, [1] * 260),             # more requests than threads of a CTA
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_matches_64_bits(cuda_device, dtype, heads, group, size, lengths, last, causal):
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, _ = _filled(cuda_device, dtype, heads, size, lengths)
    rows = sum(last) + 3
    plan = bt.step(_i32(last, cuda_device), rows)
    from hrm_text_b200.ops.paged import paged_append
    x = torch.randn(rows, 3, heads, 128, device=cuda_device).bfloat16()
    paged_append(x[:, 0], x[:, 1], cache, plan)
    q = (torch.randn(rows, heads * group, 128, device=cuda_device) * 2).bfloat16()
    gate = torch.randn(rows, 2, heads * group, 128, device=cuda_device).bfloat16()[:, 1]
    for gt in (None, gate):
        out = paged_attention(q, cache, plan, causal, gt)
        want = paged_attention_reference(q, cache, plan, causal, gt, dtype=torch.float64)
        want64 = paged_attention_reference(q.double(), cache, plan, causal, gt, dtype=torch.float64)
        assert torch.equal(want, want64.bfloat16())
        _close(out, want64, cache)
        assert (out[sum(last):] == 0).all()  # rows of no request
    assert torch.equal(out, paged_attention(q, cache, plan, causal, gt))  # the same bits again


@pytest.mark.parametrize("chunk,group", [(700, 2), (5000, 1)])  # 88 and 313 tiles of rows
def test_attention_many_new_tokens(cuda_device, chunk, group):
    """A chunk of a prompt on a cached beginning, beside a decoding request; the workspace stays bounded."""
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import paged_append, paged_attention
    bt, cache, _ = _filled(cuda_device, torch.int8, 2, 64, [300, 1000], extra=chunk + 64)
    plan = bt.step(_i32([chunk, 1], cuda_device), chunk + 1)
    bt.check()
    x = torch.randn(chunk + 1, 2, 2, 128, device=cuda_device).bfloat16()
    paged_append(x[:, 0], x[:, 1], cache, plan)
    q = torch.randn(chunk + 1, 2 * group, 128, device=cuda_device).bfloat16()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = paged_attention(q, cache, plan)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < (64 << 20) + out.numel() * 2
    rows = torch.arange(0, chunk + 1, 37, device=cuda_device)
    rows[-1] = chunk
    want = paged_attention_reference(q.double(), cache, plan, dtype=torch.float64)
    _close(out[rows], want[rows], cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_peaked_scores_and_ranges(cuda_device, dtype):
    """Scores of hundreds, blocks whose value ranges differ by 2^60, rows of tiny or huge queries."""
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, _ = _filled(cuda_device, dtype, 2, 16, [1500, 40, 600])
    plan = bt.step(_i32([1, 1, 1], cuda_device), 3)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    cache.value_scales.mul_(torch.exp2(torch.randint(-30, 30, cache.value_scales.shape, generator=g, device=cuda_device).float()))
    q = torch.randn(3, 4, 128, device=cuda_device)
    q[0] *= 100
    q[1] *= 1e-20
    q[2, 1] = 0
    q[2, 2, 64:] *= 2.0 ** -12
    q = q.bfloat16()
    out = paged_attention(q, cache, plan)
    want = paged_attention_reference(q.double(), cache, plan, dtype=torch.float64)
    # each weighted value is rounded relative to itself, so the error is held to the mean of |v|
    mass = paged_attention_reference(q.double(), cache._replace(values=cache.values.float().abs()), plan, dtype=torch.float64)
    excess = (out.double() - want).abs() - (2.0 ** -9 * want.abs() + 2.0 ** -9 * mass)
    assert torch.isfinite(out.float()).all() and excess.max() <= 0


def test_attention_ignores_what_lies_beyond(cuda_device):
    """Codes after a request's last token, and blocks of others, do not reach its output."""
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, plan = _filled(cuda_device, torch.int8, 2, 32, [50, 10], steps=[[1, 1]])
    q = torch.randn(2, 2, 128, device=cuda_device).bfloat16()
    out = paged_attention(q, cache, plan)
    mine = torch.zeros(cache.keys.shape[0], 32, dtype=torch.bool, device=cuda_device)
    for i, n in enumerate(plan.kv_lengths.tolist()):
        for p in range(n):
            mine[plan.tables[i, p // 32], p % 32] = True
    for codes in (cache.keys, cache.values):
        codes.masked_fill_(~mine[:, None, :, None], 127)
    assert torch.equal(out, paged_attention(q, cache, plan))


def test_attention_strided_queries_and_streams(cuda_device):
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import paged_attention
    bt, cache, _ = _filled(cuda_device, torch.int8, 4, 32, [300, 77])
    plan = bt.step(_i32([1, 2], cuda_device), 3)
    wide = torch.randn(3, 4, 4, 128, device=cuda_device).bfloat16()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        out = paged_attention(wide[:, 1], cache, plan, gate=wide[:, 0])
    torch.cuda.current_stream().wait_stream(other)
    want = paged_attention_reference(wide[:, 1].double(), cache, plan, gate=wide[:, 0], dtype=torch.float64)
    _close(out, want, cache)
    swapped = wide.permute(0, 2, 1, 3)[:, :, 1]  # heads a stride of four rows apart
    _close(paged_attention(swapped, cache, plan),
           paged_attention_reference(swapped.double(), cache, plan, dtype=torch.float64), cache)


def test_cache_past_32_bit_offsets(cuda_device):
    """Blocks whose bytes lie beyond 2^32 of the codes."""
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention, paged_read
    heads, size, blocks = 16, 128, 17000  # 4.46 GB of codes each for keys and values
    cache = PagedKV8.create(blocks, size, heads, torch.int8, cuda_device)
    bt = BlockTables(blocks, size, 2, 4, cuda_device)
    bt.free.copy_(torch.arange(blocks, dtype=torch.int32, device=cuda_device))  # the highest ids first
    plan = bt.step(_i32([300, 129], cuda_device), 429)
    assert int(plan.slots.min()) // size * size * heads * 128 > 1 << 32
    k, v = (torch.randn(429, heads, 128, device=cuda_device).bfloat16() for _ in range(2))
    paged_append(k, v, cache, plan)
    back = paged_read(cache, plan.slots)[0]
    assert (back.float() - k.float()).abs().max() < 0.05
    q = torch.randn(429, heads, 128, device=cuda_device).bfloat16()
    _close(paged_attention(q, cache, plan), paged_attention_reference(q.double(), cache, plan, dtype=torch.float64), cache)


def test_decode_step_in_a_graph_crosses_blocks(cuda_device):
    from hrm_text_b200.models.paged import paged_attention_reference
    from hrm_text_b200.ops.paged import paged_append, paged_attention
    bt, cache, _ = _filled(cuda_device, torch.int8, 2, 16, [14, 30, 1], extra=200)
    ones = _i32([1, 1, 1], cuda_device)
    source, x = (torch.randn(3, 4, 2, 128, device=cuda_device).bfloat16() for _ in range(2))
    queries, kept = torch.empty_like(x), torch.empty_like(x[:, 1])

    def step():  # with copies, which are no kernels, before and after the calls
        bt.truncate(bt.lengths.clone())
        plan = bt.step(ones, 3, max_new=1)
        x.copy_(source)
        paged_append(x[:, 2], x[:, 3], cache, plan)
        queries.copy_(source)
        out = paged_attention(queries[:, 1], cache, plan, gate=queries[:, 0])
        kept.copy_(out)
        return plan, kept

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step()
    for _ in range(40):
        source.copy_(torch.randn_like(x.float()))
        graph.replay()
        want = paged_attention_reference(x[:, 1].double(), cache, plan, gate=x[:, 0], dtype=torch.float64)
        _close(out, want, cache)
    bt.check()
    assert bt.lengths.tolist() == [14 + 41, 30 + 41, 1 + 41]


def test_refusals(cuda_device):
    from hrm_text_b200.ops.paged import BlockTables, PagedKV8, paged_append, paged_attention, paged_read
    bt = BlockTables(8, 16, 2, 4, cuda_device)
    cache = PagedKV8.create(8, 16, 2, torch.int8, cuda_device)
    plan = bt.step(_i32([2, 1], cuda_device), 3)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="block_size"):
        BlockTables(8, 24, 2, 4, cuda_device)
    with pytest.raises(ValueError, match="max_requests"):
        BlockTables(8, 16, 0, 4, cuda_device)
    with pytest.raises(ValueError, match="int8 or float8"):
        PagedKV8.create(8, 16, 2, torch.uint8, cuda_device)
    with pytest.raises(ValueError, match="head_dim 128"):
        PagedKV8.create(8, 16, 2, torch.int8, cuda_device, head_dim=64)
    with pytest.raises(ValueError, match="new_tokens"):
        bt.step(torch.ones(2, device=cuda_device), 2)
    with pytest.raises(ValueError, match="new_tokens"):
        bt.step(_i32([1], cuda_device), 2)
    with pytest.raises(ValueError, match="keep"):
        bt.truncate(_i32([1, 1, 1], cuda_device))
    with pytest.raises(ValueError, match="rows"):
        paged_append(x[:2], x[:2], cache, plan)
    with pytest.raises(ValueError, match="blocks of 16"):
        paged_attention(x, PagedKV8.create(8, 32, 2, torch.int8, cuda_device), plan)
    with pytest.raises(ValueError, match="8 blocks"):
        paged_append(x, x, PagedKV8.create(7, 16, 2, torch.int8, cuda_device), plan)
    with pytest.raises(RuntimeError, match="bf16"):
        paged_append(x.float(), x.float(), cache, plan)
    with pytest.raises(RuntimeError, match="bf16"):
        paged_attention(x.half(), cache, plan)
    with pytest.raises(RuntimeError, match="multiple"):
        paged_attention(torch.zeros(3, 3, 128, dtype=torch.bfloat16, device=cuda_device), cache, plan)
    with pytest.raises(RuntimeError, match="gate"):
        paged_attention(x, cache, plan, gate=x[:, :1])
    with pytest.raises(RuntimeError, match="aligned"):
        paged_append(torch.zeros(3, 2, 129, dtype=torch.bfloat16, device=cuda_device)[..., 1:], x, cache, plan)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(x.cpu(), PagedKV8.create(8, 16, 2), plan)
    with pytest.raises(ValueError, match="slots"):
        paged_read(cache, plan.slots.long())
    # nothing to do is not an error
    empty = bt.step(_i32([0, 0], cuda_device), 0)
    paged_append(x[:0], x[:0], cache, empty)
    assert paged_attention(x[:0], cache, empty).shape == (0, 2, 128)
    assert paged_read(cache, plan.slots[:0])[0].shape == (0, 2, 128)
