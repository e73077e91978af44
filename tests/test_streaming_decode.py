"""Decode steps of whole models on the streaming operators, fed with given tokens: every step's logits against the reference path."""
import pytest
import torch

from metal_marlin_b200 import ops
from metal_marlin_b200.models.config import get_preset
from metal_marlin_b200.models.mmfp4_causal_lm import MMFP4ForCausalLM, prefill
from metal_marlin_b200.models.transformer import BatchMeta

LENS, STEPS, BS, NB = (37, 5, 61), 12, 16, 6
ROWS = (0, None, 1, 2)                                  # decode batch: one row of padding between the sequences, its table that of a live one


def model(preset, device, window, sinks, seed=0):
    cfg = get_preset(preset)
    cfg.sliding_window, cfg.attention_sinks = window, sinks
    return MMFP4ForCausalLM.from_config(cfg, device=device, seed=seed)


def texts(vocab):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(0, vocab, (n + STEPS,), generator=g).tolist() for n in LENS]


def tables():
    return torch.randperm(len(LENS) * NB, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(len(LENS), NB)


def decode(lm, kv, seqs, reference):
    """Logits ``[steps, sequences, vocabulary]`` of the decode path over the last STEPS tokens of every sequence."""
    dev, out, bt = lm.model.device, [], tables()
    for i in range(STEPS):
        ids, pos, slots, ctx, rows = [], [], [], [], []
        for r in ROWS:
            p = 0 if r is None else LENS[r] + i
            ids.append(0 if r is None else seqs[r][p])
            pos.append(p)
            slots.append(-1 if r is None else int(bt[r, p // BS]) * BS + p % BS)
            ctx.append(p + 1)
            rows.append(bt[2 if r is None else r].tolist())
        t = lambda v, d=torch.int32: torch.tensor(v, dtype=d, device=dev)
        meta = BatchMeta(positions=t(pos), slots=t(slots, torch.int64), block_tables=t(rows), ctx_lens=t(ctx), decode=True, max_ctx=NB * BS, splits=2)
        with ops.force_reference(reference):
            lg = lm.model.forward(t(ids, torch.int64), kv, meta)
        out.append(lg[[j for j, r in enumerate(ROWS) if r is not None]].float().cpu())
    return torch.stack(out)


def caches(lm, seqs, kv_dtype, count):
    """The same prompts in several caches, written by the reference path."""
    with ops.force_reference():
        kvs = [lm.new_cache(len(LENS) * NB, BS, kv_dtype) for _ in range(count)]
        for kv in kvs:
            prefill(lm.model, kv, [s[:n] for s, n in zip(seqs, LENS)], tables())
    return kvs


def gap(a, b):
    return float((a - b).abs().amax(dim=(1, 2)).max() / b.abs().max())


@pytest.mark.parametrize("preset", ["tiny-llama", "tiny-jamba", "tiny-hybrid-deltanet"])
def test_logits_notice_the_mask(preset):
    """What the comparison below rests on: a window or a number of sinks that is off by one moves the logits by more than twice its tolerance."""
    lm = model(preset, "cpu", 20, 3)
    seqs = texts(lm.config.vocab_size)
    kvs = caches(lm, seqs, "bf16", 3)
    want = decode(lm, kvs[0], seqs, True)
    for kv, (window, sinks) in zip(kvs[1:], ((21, 3), (20, 2))):
        lm.config.sliding_window, lm.config.attention_sinks = window, sinks
        assert gap(decode(lm, kv, seqs, True), want) > 0.12


@pytest.mark.gpu
@pytest.mark.parametrize("preset,kv_dtype", [("tiny-llama", "bf16"), ("tiny-llama", "int8"), ("tiny-llama", "fp4"), ("tiny-jamba", "bf16"), ("tiny-hybrid-deltanet", "bf16"),
                                             ("tiny-qwen3-moe", "bf16")])
def test_decode_steps_agree_with_the_reference_path(preset, kv_dtype):
    """From the same cache, the same tokens, past the window: every step's logits within 6 % of the largest (bf16 activations through the stack; the bound
    that prompt passes are held to), every cache row and recurrent state that no live sequence owns left as it was."""
    lm = model(preset, "cuda", 20, 3)
    seqs = texts(lm.config.vocab_size)
    ref, own = caches(lm, seqs, kv_dtype, 2)
    free = torch.ones(len(LENS) * NB + 1, dtype=torch.bool)
    free[[int(r[0]) for r in tables()]] = False
    for rec in own.rec:
        if rec is not None:
            for pool in rec:
                pool[:-1][free[:-1]] = 7.0
    ops.clear_status("cuda")
    want, got = decode(lm, ref, seqs, True), decode(lm, own, seqs, False)
    assert gap(got, want) < 6e-2
    assert ops.check_status("cuda") == 0
    for rec in own.rec:
        if rec is not None:
            assert all((pool[:-1][free[:-1]] == 7).all() for pool in rec)
    # and a prompt pass over the same tokens, on the reference path
    with ops.force_reference():
        whole = prefill(lm.model, lm.new_cache(len(LENS) * NB, BS, kv_dtype), seqs, tables()).float().cpu()
    assert gap(got[-1:], whole[None]) < 6e-2
