"""The paged cache's and the log probabilities' oracle and entry points at their limits, on the CPU."""
import math

import numpy as np
import pytest
import torch

from hrm_text_b200.inference.engine import generate_tokens
from hrm_text_b200.models.paged import paged_append_reference, paged_attention_reference, token_logprobs_reference
from hrm_text_b200.ops.paged import BlockTables, OutOfBlocks, PagedKV8
from hrm_text_b200.runtime.factory import arch_preset, build_model


def test_likeliest_order_is_nan_then_infinity_then_the_lowest_id():
    nan, inf = math.nan, math.inf
    rows = torch.tensor([[inf, 1.0, nan, inf, nan], [-nan, nan, 0.0, -inf, inf], [-0.0, 0.0, -inf, 0.0, -1.0]])
    for dtype in (torch.float32, torch.float64):
        ids = token_logprobs_reference(rows.to(dtype), torch.zeros(3, dtype=torch.long), 5)[2]
        assert ids.tolist() == [[2, 4, 0, 3, 1], [0, 1, 4, 2, 3], [0, 1, 3, 4, 2]]


def test_attention_oracle_keeps_nan_from_earlier_tokens():
    torch.manual_seed(0)
    bt, cache = BlockTables(4, 16, 1, 4), PagedKV8.create(4, 16, 2)
    x = torch.randn(17, 2, 128)
    value = x.clone()
    value[16, 0, 5] = math.nan
    paged_append_reference(x[:14], value[:14], cache, bt.step(torch.tensor([14], dtype=torch.int32), 14))
    plan = bt.step(torch.tensor([3], dtype=torch.int32), 3)
    paged_append_reference(x[14:], value[14:], cache, plan)
    q = torch.randn(3, 4, 128)
    out = paged_attention_reference(q, cache, plan)
    assert torch.isfinite(out[:2]).all() and torch.isfinite(out[:, 2:]).all() and out[2, :2].isnan().all()
    assert paged_attention_reference(q, cache, plan, causal=False)[:, :2].isnan().all()


@pytest.mark.parametrize("lengths,free,at", [([3, 65, 0], 6, 1), ([3, 0, -1], 6, 2), ([3, 0, 0], 9, -1), ([3, 0, 0], -1, -1)])
def test_states_that_cannot_be_change_nothing(lengths, free, at):
    bt = BlockTables(8, 16, 3, 4)
    bt.step(torch.tensor([3, 17, 0], dtype=torch.int32), 20)
    bt.lengths.copy_(torch.tensor(lengths))
    bt.num_free.fill_(free)
    before = [t.clone() for t in (bt.tables, bt.lengths, bt.free, bt.num_free)]
    for call in (lambda: bt.step(torch.ones(3, dtype=torch.int32), 3), lambda: bt.truncate(torch.zeros(3, dtype=torch.int32))):
        call()
        assert all(torch.equal(t, was) for t, was in zip((bt.tables, bt.lengths, bt.free, bt.num_free), before))
        with pytest.raises(OutOfBlocks, match="outside" + (f".*request {at}" if at >= 0 else "")):
            bt.check()


def _model():
    cfg = arch_preset("hrm", "L") | dict(vocab_size=48, max_seq_len=128, n_layers=2, hidden_size=128, num_heads=1)
    torch.manual_seed(0)
    return build_model(cfg).eval()


@pytest.mark.parametrize("kv_cache", ["bf16", "int8"])
@pytest.mark.parametrize("k", [-1, 49, 65])
def test_alternatives_are_refused_before_a_prompt_is_taken(kv_cache, k):
    taken = []

    def prompts():
        taken.append(0)
        yield 0, np.arange(5)

    with pytest.raises(ValueError, match="logprobs must be 0 to 48"):
        next(generate_tokens(_model(), None, prompts(), max_tokens=32, max_generation=4, batch_size=1, stop_token=-1,
                             kv_cache=kv_cache, logprobs=k))
    assert not taken


class _Words:
    """A tokenizer of numbers."""

    def __call__(self, text, add_special_tokens):
        return {"input_ids": [int(w) for w in text.split()]}

    def decode(self, ids):
        return " ".join(map(str, ids))

    def convert_tokens_to_ids(self, token):
        return -1


def test_text_generation_shares_a_small_pool(monkeypatch):
    """A pool of blocks for one request at its longest: the same texts as with room for all, from a smaller cache."""
    import hrm_text_b200.inference.engine as engine
    info = dict(boq="", eoq="", eoa="", condition_mapping={"direct": ""})
    ckpt = engine.InferenceCheckpoint(_model(), None, _Words(), info)
    prompts = ["3 1 4 1 5", "9 2 6", "5 3 5 8 9 7 9"]
    pools = []
    create = BlockTables.__init__
    monkeypatch.setattr(BlockTables, "__init__", lambda self, num_blocks, *a: (pools.append(num_blocks), create(self, num_blocks, *a))[1])

    def run(**kw):
        return dict(engine.inference_generate(ckpt, ((i, ("direct", p)) for i, p in enumerate(prompts)), 32, 6, 3, kv_cache="int8",
                                              block_size=16, **kw))

    whole, small = run(), run(num_blocks=2)
    assert whole == small and all(len(t.split()) == 6 for t in whole.values()) and pools == [6, 2]

    from evaluation.engines import SimpleEngine
    simple = SimpleEngine.__new__(SimpleEngine)
    simple.ckpt = ckpt
    assert simple.generate(prompts, 3, 32, 6, kv_cache="int8", block_size=16, num_blocks=2) == [whole[i] for i in range(3)]
    assert pools == [6, 2, 2]
