"""Generation with the paged 8-bit cache on the GPU: logits against the CPU oracle of the same cache,
the CUDA-graph step against the eager one, log probabilities of the generated tokens."""
import numpy as np
import pytest
import torch

from gpu_utils import assert_close

pytestmark = pytest.mark.gpu


def _models(device):
    from hrm_text_b200.runtime.factory import arch_preset, build_model
    cfg = arch_preset("hrm", "L") | dict(vocab_size=256, max_seq_len=128, n_layers=2, hidden_size=256, num_heads=2)
    torch.manual_seed(0)
    gpu = build_model(cfg, device).to(torch.bfloat16).eval()
    cpu = build_model(cfg, "cpu").eval()
    cpu.load_state_dict({k: v.float().cpu() for k, v in gpu.state_dict().items()})
    return gpu, cpu


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_prefill_and_decode_match_oracle(cuda_device, code):
    """The models round to bf16 between layers; as for the bf16 cache, logits agree to 5e-2 of their size. Both
    sides quantise, so a code may fall on the other side of a step: that moves e4m3 values by 2^-3, and a
    few of them are averaged away."""
    from hrm_text_b200.inference.engine import paged_decode_step, paged_prefill
    from hrm_text_b200.models.common import oracle_mode
    from hrm_text_b200.ops.paged import BlockTables
    gpu, cpu = _models(cuda_device)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 256, n) for n in (17, 9, 40)]
    sides = []
    for model, dev in ((gpu, cuda_device), (cpu, torch.device("cpu"))):
        tables = BlockTables(24, 16, 3, 8, dev)
        sides.append((model, tables, model.create_cache(paged=tables, dtype=code, device=dev), dev))
    rel = 5e-2 if code == torch.int8 else 1e-1
    for i, pr in enumerate(prompts):
        lg = paged_prefill(gpu, None, torch.as_tensor(pr, device=cuda_device), sides[0][2], sides[0][1], i)
        with oracle_mode():
            lc = paged_prefill(cpu, None, torch.as_tensor(pr), sides[1][2], sides[1][1], i)
        assert_close(lg.float().cpu(), lc, 5e-2, f"prefill logits {i}")
    active = torch.tensor([1, 0, 1], dtype=torch.int32)
    for t in range(4):
        if t == 2:
            active[:] = torch.tensor([1, 1, 0], dtype=torch.int32)
        tok = torch.as_tensor(rng.integers(0, 256, 3))
        lg = paged_decode_step(gpu, None, tok.to(cuda_device), sides[0][2], sides[0][1], active.to(cuda_device))
        with oracle_mode():
            lc = paged_decode_step(cpu, None, tok, sides[1][2], sides[1][1], active)
        on = active > 0
        assert_close(lg.float().cpu()[on], lc[on], rel, f"decode logits step {t}")
    assert torch.equal(sides[0][1].tables.cpu(), sides[1][1].tables)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_graphed_generation_equals_eager(cuda_device, code):
    from hrm_text_b200.inference.engine import generate_tokens
    gpu, _ = _models(cuda_device)
    rng = np.random.default_rng(2)
    prompts = [(i, rng.integers(0, 256, n)) for i, n in enumerate([5, 17, 9, 30, 63])]
    runs = []
    for graph, blocks in ((False, None), (True, None), (True, 5)):
        runs.append({p: (t, s) for p, t, s in generate_tokens(
            gpu, None, iter(prompts), max_tokens=64, max_generation=20, batch_size=3, stop_token=-1, temp=0.0,
            device=cuda_device, use_cuda_graph=graph, kv_cache=code, block_size=16, num_blocks=blocks, logprobs=2)})
    for pid, _ in prompts:
        for other in runs[1:]:
            assert runs[0][pid][0].tolist() == other[pid][0].tolist(), pid
        tokens, scores = runs[1][pid]
        np.testing.assert_array_equal(scores.top_ids[:, 0], tokens)
        np.testing.assert_array_equal(scores.top_logprobs[:, 0], scores.logprobs)
        np.testing.assert_allclose(scores.logprobs, runs[0][pid][1].logprobs, rtol=0, atol=1e-6)
    assert runs[0][4][0].size == 1 and runs[0][0][0].size == 20


def test_paged_decode_step_runs_no_library_gemm(cuda_device):
    from torch.profiler import ProfilerActivity, profile

    from hrm_text_b200.inference.engine import paged_decode_step
    from hrm_text_b200.ops.paged import BlockTables
    gpu, _ = _models(cuda_device)
    tables = BlockTables(16, 16, 4, 4, cuda_device)
    cache = gpu.create_cache(paged=tables, dtype=torch.int8, device=cuda_device)
    tok, active = torch.zeros(4, dtype=torch.long, device=cuda_device), torch.ones(4, dtype=torch.int32, device=cuda_device)
    with torch.inference_mode():
        paged_decode_step(gpu, None, tok, cache, tables, active)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            paged_decode_step(gpu, None, tok, cache, tables, active)
            torch.cuda.synchronize()
    names = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]
    assert any("paged_attention_kernel" in n for n in names) and any("paged_append_kernel" in n for n in names)
    assert not any(s in n.lower() for n in names if "hrm::" not in n for s in ("gemm", "nvjet", "xmma", "cutlass", "gemv"))
