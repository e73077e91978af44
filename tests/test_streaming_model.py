"""Models that keep going at constant cost per token: attention layers with a sliding window and sinks through the whole stack (prompt pass, chunked
prompts, decode, serving engine), and the Mamba / Gated DeltaNet layers on the batched pooled-state operators."""
import pytest
import torch

from metal_marlin_b200 import ops
from metal_marlin_b200.engine.engine import EngineConfig, LLMEngine
from metal_marlin_b200.models.config import ModelConfig, get_preset
from metal_marlin_b200.models.mmfp4_causal_lm import MMFP4ForCausalLM, prefill


def windowed(preset="tiny-llama", window=12, sinks=3):
    cfg = get_preset(preset)
    cfg.sliding_window, cfg.attention_sinks = window, sinks
    return cfg


def test_config_carries_the_sinks():
    cfg = windowed()
    assert ModelConfig.from_dict(cfg.to_dict()).attention_sinks == 3
    assert get_preset("tiny-llama").attention_sinks == 0
    with pytest.raises(ValueError):
        MMFP4ForCausalLM.from_config(windowed("tiny-mla-moe"), device="cpu", seed=0)


def test_decode_with_sinks_agrees_with_recomputation():
    """Every greedy token of the decode path equals the arg-max of a prompt pass over the whole sequence, far past the window."""
    lm = MMFP4ForCausalLM.from_config(windowed(), device="cpu", seed=0)
    prompts = [list(range(3, 40)), [5, 6, 7, 8]]
    out = lm.generate(prompts, max_new_tokens=14)
    for pr, o in zip(prompts, out):
        seq = list(pr)
        for t in o:
            assert int(lm.forward_logits(seq)[-1].argmax()) == t
            seq.append(t)
    # chunked prompts see the same keys
    bt = torch.arange(8, dtype=torch.int32).view(2, 4)
    a = prefill(lm.model, lm.new_cache(8, 16), prompts, bt, chunk_tokens=4096)
    b = prefill(lm.model, lm.new_cache(8, 16), prompts, bt, chunk_tokens=7)
    assert float((a - b).abs().max() / a.abs().max()) < 2e-2
    # the sinks matter: without them the logits behind the window are others
    plain = MMFP4ForCausalLM.from_config(windowed(sinks=0), device="cpu", seed=0)
    c = prefill(plain.model, plain.new_cache(8, 16), prompts, bt)
    assert float((a[0] - c[0]).abs().max()) > 1e-3 * float(a[0].abs().max())
    assert torch.equal(a[1], c[1])                       # four tokens: nothing is behind a window of twelve


@pytest.mark.gpu
@pytest.mark.parametrize("preset", ["tiny-llama", "tiny-jamba", "tiny-qwen3-moe"])
def test_windowed_models_on_the_gpu_match_the_reference_path(preset):
    lm = MMFP4ForCausalLM.from_config(windowed(preset, 40, 5), device="cuda", seed=0)
    V = lm.config.vocab_size
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (150, 9, 61)]
    bt = torch.arange(36, dtype=torch.int32).view(3, 12)
    a = prefill(lm.model, lm.new_cache(36, 16), prompts, bt)
    c = prefill(lm.model, lm.new_cache(36, 16), prompts, bt, chunk_tokens=33)
    with ops.force_reference():
        b = prefill(lm.model, lm.new_cache(36, 16), prompts, bt)
    assert float((a - b).abs().max() / b.abs().max()) < 6e-2
    assert float((a - c).abs().max() / a.abs().max()) < 6e-2
    out_g = lm.generate(prompts, max_new_tokens=12, use_graph=True)
    out_e = lm.generate(prompts, max_new_tokens=12, use_graph=False)
    assert out_g == out_e
    with ops.force_reference():
        ref = lm.generate(prompts, max_new_tokens=12, use_graph=False)
    assert [o[0] for o in out_g] == [r[0] for r in ref]
    assert ops.check_status(torch.device("cuda")) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("preset,kv_dtype", [("tiny-llama", "bf16"), ("tiny-llama", "fp8"), ("tiny-jamba", "bf16"), ("tiny-hybrid-deltanet", "bf16")])
def test_engine_serves_windowed_streams(preset, kv_dtype):
    """Continuous batching (bucketed, padded decode batches, graphs) gives what one sequence alone gives."""
    cfg = windowed(preset, 24, 4)
    lm = MMFP4ForCausalLM.from_config(cfg, device="cuda", seed=1)
    prompts = [list(range(1, 70)), [9, 8, 7], list(range(40, 90)), list(range(5, 25)), [3] * 33]
    kw = dict(num_kv_blocks=64, block_size=16, max_model_len=128, max_chunk=16, max_prefill_tokens=32, kv_cache_dtype=kv_dtype)
    alone = [LLMEngine(lm.model, EngineConfig(use_cuda_graphs=False, **kw)).generate([p], max_new_tokens=3)[0] for p in prompts]
    eng = LLMEngine(lm.model, EngineConfig(use_cuda_graphs=True, **kw))
    got = eng.generate(prompts, max_new_tokens=3)
    same = sum(a == b for g, w in zip(got, alone) for a, b in zip(g, w))
    assert [g[0] for g in got] == [w[0] for w in alone]
    assert same >= 12                                     # 15 tokens; a near tie may fall otherwise at another batch size
    assert ops.check_status(torch.device("cuda")) == 0
