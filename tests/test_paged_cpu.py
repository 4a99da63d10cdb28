"""Paged 8-bit cache and token log probabilities on the CPU: the oracle itself, and generation with it."""
import math

import numpy as np
import pytest
import torch

from hrm_text_b200.inference.engine import generate_tokens
from hrm_text_b200.models.paged import (paged_append_reference, paged_attention_reference, paged_read_reference,
                                        token_logprobs_reference)
from hrm_text_b200.ops.paged import BlockTables, OutOfBlocks, PagedKV8
from hrm_text_b200.runtime.factory import arch_preset, build_model


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_step_assigns_blocks_in_order_and_truncate_undoes_it():
    bt = BlockTables(6, 16, 3, 4)
    plan = bt.step(_i32(17, 0, 3), 22)
    assert bt.tables.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    assert plan.slots.tolist() == [*range(16), 16, 32, 33, 34, -1, -1]
    assert plan.positions.tolist() == [*range(17), 0, 1, 2, 0, 0]
    assert plan.cu_new.tolist() == [0, 17, 17, 20] and plan.kv_lengths.tolist() == [17, 0, 3]
    assert plan.runs[:int(plan.num_runs)].tolist() == [[0, 0, 16, 0], [1, 0, 1, 16], [2, 0, 3, 17]]
    before = (bt.tables.clone(), bt.free.clone(), bt.num_free.clone())
    bt.step(_i32(16, 1, 0), 17)
    assert int(bt.num_free) == 1
    bt.truncate(_i32(17, 0, 3))
    assert all(torch.equal(a, b) for a, b in zip(before, (bt.tables, bt.free, bt.num_free)))
    with pytest.raises(OutOfBlocks, match="free blocks"):
        bt.step(_i32(40, 0, 30), 70)
        bt.check()
    assert bt.lengths.tolist() == [17, 0, 3]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_append_keeps_older_tokens_when_the_range_grows(dtype):
    torch.manual_seed(0)
    bt, cache = BlockTables(4, 16, 1, 4), PagedKV8.create(4, 16, 2, dtype)
    rows = torch.randn(20, 2, 128) * torch.linspace(0.1, 3, 20)[:, None, None]
    for t in range(20):
        paged_append_reference(rows[t:t + 1], -rows[t:t + 1], cache, bt.step(_i32(1), 1))
    keys, values = paged_read_reference(cache, torch.arange(20, dtype=torch.int32))
    assert torch.equal(keys, -values)
    # each growth of the scale rounds an older code once more: the steps of the scales it had add up
    scale = cache.key_scales[torch.arange(20) // 16][..., None]
    bound = 4 * scale if dtype == torch.int8 else rows.abs() / 2 + 4 * scale * 2.0 ** -9
    assert ((keys.float() - rows).abs() <= bound + rows.abs() * 2.0 ** -8).all()


def test_attention_is_softmax_over_the_read_back_tokens():
    torch.manual_seed(1)
    bt, cache = BlockTables(12, 16, 2, 6), PagedKV8.create(12, 16, 2)
    paged_append_reference(torch.randn(50, 2, 128), torch.randn(50, 2, 128), cache, bt.step(_i32(30, 20), 50))
    plan = bt.step(_i32(2, 1), 4)
    paged_append_reference(torch.randn(4, 2, 128), torch.randn(4, 2, 128), cache, plan)
    q, gate = torch.randn(4, 4, 128), torch.randn(4, 4, 128)
    out = paged_attention_reference(q, cache, plan, True, gate, dtype=torch.float64)
    assert (out[3] == 0).all()
    for row, (i, length) in enumerate([(0, 31), (0, 32), (1, 21)]):
        slots = bt.tables[i].repeat_interleave(16)[:length] * 16 + torch.arange(length) % 16
        for h in range(4):
            k, v = ((c[slots // 16, h // 2, slots % 16].double() * s[slots // 16, h // 2][:, None].double())
                    for c, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)))
            want = torch.softmax(k @ q[row, h].double() / math.sqrt(128), 0) @ v * torch.sigmoid(gate[row, h].double())
            torch.testing.assert_close(out[row, h], want.float(), rtol=1e-6, atol=1e-7)  # rounded once, to fp32


def test_logprobs_reference_gradcheck_and_masks():
    torch.manual_seed(2)
    x = torch.randn(3, 7, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([0, 6, 3])
    assert torch.autograd.gradcheck(lambda x: token_logprobs_reference(x, t)[:2], (x,))
    y = torch.full((2, 5), -math.inf)
    y[1, 2] = 1.0
    lp, h, ids, top = token_logprobs_reference(y, torch.tensor([0, 2]), 2)
    assert lp.tolist() == [-math.inf, 0.0] and h.tolist() == [0.0, 0.0]
    assert ids.tolist() == [[0, 1], [2, 0]] and top[1].tolist() == [0.0, -math.inf]


def _model():
    cfg = arch_preset("hrm", "L") | dict(vocab_size=256, max_seq_len=128, n_layers=2, hidden_size=256, num_heads=2)
    torch.manual_seed(0)
    return build_model(cfg).eval()


def _prompts():
    rng = np.random.default_rng(0)
    return [(i, rng.integers(0, 256, n)) for i, n in enumerate([5, 17, 9, 33])] + [(9, np.arange(70) % 256)]


def _run(model, prompts, **kw):
    args = dict(max_tokens=64, max_generation=6, batch_size=2, stop_token=-1, temp=0.0, device=torch.device("cpu"))
    return {out[0]: out[1:] for out in generate_tokens(model, None, iter(prompts), **(args | kw))}


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_generation_with_a_paged_cache(code):
    """Greedy tokens follow the bf16-cache run until a near tie; a small pool changes nothing but the waiting."""
    model, prompts = _model(), _prompts()
    whole = _run(model, prompts, kv_cache=code, block_size=16, logprobs=2)
    small = _run(model, prompts, kv_cache=code, block_size=16, num_blocks=4, logprobs=2)
    plain = _run(model, prompts, logprobs=2)
    assert sorted(whole) == sorted(small) == sorted(plain) == [0, 1, 2, 3, 9]
    for pid in whole:
        assert whole[pid][0].tolist() == small[pid][0].tolist()
        np.testing.assert_array_equal(whole[pid][1].logprobs, small[pid][1].logprobs)
    assert whole[9][0].size == 0 and whole[9][1].top_ids.shape == (0, 2)
    for pid, prompt in prompts[:4]:
        # the first token comes from the prompt's own pass, which the cache does not change
        assert whole[pid][0][0] == plain[pid][0][0]
        np.testing.assert_allclose(whole[pid][1].logprobs[0], plain[pid][1].logprobs[0], rtol=1e-5)
        same = 0
        while same < 6 and whole[pid][0][same] == plain[pid][0][same]:
            same += 1
        got, want = whole[pid][1], plain[pid][1]
        # 8-bit keys and values move a log probability by their relative error (2^-8 int8, 2^-4 e4m3) times its spread
        assert np.abs(got.logprobs[:same] - want.logprobs[:same]).max() < (0.1 if code == "int8" else 0.6)
        if same < 6:  # the tokens part where the two likeliest were close
            assert want.top_logprobs[same, 0] - want.top_logprobs[same, 1] < (0.2 if code == "int8" else 1.2)


def test_generated_logprobs_are_the_tokens_own():
    out = _run(_model(), _prompts(), kv_cache="int8", block_size=16, logprobs=3)
    for tokens, lp in out.values():
        assert lp.logprobs.shape == lp.entropy.shape == tokens.shape and lp.top_ids.shape == (tokens.size, 3)
        np.testing.assert_array_equal(lp.top_ids[:, 0], tokens)  # greedy
        np.testing.assert_array_equal(lp.top_logprobs[:, 0], lp.logprobs)
        assert (lp.entropy >= 0).all() and (lp.logprobs <= 0).all()


def test_generation_refusals():
    model = _model()
    with pytest.raises(ValueError, match="kv_cache"):
        _run(model, _prompts(), kv_cache="int4")
    with pytest.raises(ValueError, match="does not hold one request"):
        _run(model, _prompts(), kv_cache="int8", block_size=16, num_blocks=3)
    with pytest.raises(ValueError, match="block_size"):
        _run(model, _prompts(), kv_cache="int8", block_size=20)
