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


@pytest.mark.gpu
@pytest.mark.parametrize("t,n,Hq,Hk,D,window,sinks", [(1024, 1024, 4, 2, 128, 64, 4), (700, 1536, 4, 2, 128, 300, 129), (300, 900, 2, 2, 256, 100, 65),
                                                      (512, 2048, 2, 1, 256, 1000, 1), (640, 640, 2, 2, 128, 4096, 7), (384, 1200, 4, 4, 128, 1, 200),
                                                      (257, 700, 2, 1, 128, 250, 5000), (256, 256, 1, 1, 128, 129, 128)])
def test_prompt_attention_with_sinks_on_the_tensor_cores(t, n, Hq, Hk, D, window, sinks):
    """Tiles of the sinks, a gap, then the window's tiles.  What a kernel may round: P and the output to bf16, which keeps 8 significant bits, so
    half a step is finfo.eps / 2 = 2^-8 of the value (of sum p |v| and of the output); scores in fp32."""
    g = torch.Generator().manual_seed(t + n)
    q, k, v = (torch.randn(m, h, D, generator=g).to(torch.bfloat16).cuda() for m, h in ((t, Hq), (n, Hk), (n, Hk)))
    out = torch.empty(t, Hq, D, dtype=torch.bfloat16, device="cuda")
    ops.fmha_prefill(q, k, v, out, D ** -0.5, window=window, sinks=sinks)
    assert ops.check_status(torch.device("cuda")) == 0
    qd, kd, vd = q.double(), k.double().repeat_interleave(Hq // Hk, 1), v.double().repeat_interleave(Hq // Hk, 1)
    s = torch.einsum("thd,nhd->htn", qd, kd) * D ** -0.5
    m = torch.einsum("thd,nhd->htn", qd.abs(), kd.abs()).amax(-1) * D ** -0.5
    pos, key = torch.arange(n - t, n, device="cuda")[:, None], torch.arange(n, device="cuda")
    p = torch.softmax(s.masked_fill(~((key <= pos) & ((key > pos - window) | (key < sinks))), float("-inf")), -1)
    o, w = torch.einsum("htn,nhd->thd", p, vd), torch.einsum("htn,nhd->thd", p, vd.abs())
    rel = (2 * ((D + 8) * 2.0 ** -23 * m + n * 2.0 ** -23 + 2.0 ** -18)).t()[..., None]
    half = 1.01 * torch.finfo(torch.bfloat16).eps / 2
    gap = (out.double() - o).abs() - ((half + rel) * w + half * (o.abs() + (half + rel) * w))
    assert (gap <= 0).all(), float(gap.max())


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "int8"])
def test_long_prompts_of_a_windowed_model(kv_dtype):
    """Chunked prompts far past the window, several sequences: the gathered sinks and window rows against the reference path."""
    cfg = windowed("tiny-llama", 100, 6)
    cfg.head_dim, cfg.num_attention_heads, cfg.num_key_value_heads = 128, 4, 2
    lm = MMFP4ForCausalLM.from_config(cfg, device="cuda", seed=2)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (900, 640)]
    bt = torch.arange(2 * 60, dtype=torch.int32).view(2, 60)
    calls, real = [], ops.fmha_prefill

    def counting(*a, **kw):
        calls.append((a[1].shape[0], kw.get("sinks")))
        return real(*a, **kw)
    ops.fmha_prefill = counting
    try:
        a = prefill(lm.model, lm.new_cache(120, 16, kv_dtype), prompts, bt, chunk_tokens=300)
        b = prefill(lm.model, lm.new_cache(120, 16, kv_dtype), prompts, bt)
    finally:
        ops.fmha_prefill = real
    assert calls and all(s == 6 for _, s in calls)
    assert min(n for n, _ in calls) < 600                  # only sinks, window and chunk are gathered, not the whole context
    with ops.force_reference():
        c = prefill(lm.model, lm.new_cache(120, 16, kv_dtype), prompts, bt)
    for x in (a, b):
        assert float((x - c).abs().max() / c.abs().max()) < 6e-2
    assert ops.check_status(torch.device("cuda")) == 0
