"""What the streaming operators promise beyond their formulas: probabilities of 32 bits, one status word a device, the same answers on the CPU and on the
GPU for bad pages and uneven batches, and decode steps of whole models that agree with the reference path."""
import pytest
import torch

from metal_marlin_b200 import ops
from test_stream_operators import (DEVICES, attention_inputs, attention_oracle, check_attention, check_conv, check_ssm, conv_inputs, conv_oracle, half_step, run_attention,
                                   run_ssm, spans, ssm_inputs, want_ssm)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,G", [(64, 1), (128, 1), (256, 1), (128, 16)])
def test_probabilities_keep_32_bits(device, D, G):
    """Values that cancel: three visible keys of probabilities p0 = 1, p1 and p2 (before the sum), v0 + p1 v1 + p2 v2 = 0 to 2^-16 of v0, so that the output's own
    rounding is far below that of the probabilities.  One element of q and of every key is not zero, so scores are exact products.

    What 32 bits leave, in units of 2^-24 of w = sum p |v|: exponents x = s log2(e) with |x| <= 2 and two roundings, 2 x 2 x ln 2 < 3; the exponential, two
    steps of 2^-23, 4; the sum over the keys, four terms aligned to the largest, 2^-23 each, 8.  Together below 16 x 2^-24 = 2^-20.  Probabilities in
    two bf16 numbers would be up to 2^-17 of p1 off, that is 2^-18 w."""
    B, Hkv, bs, n, window, sinks = 8, 32, 16, 40, 2, 1
    g = torch.Generator().manual_seed(D + G)
    bf = lambda t: t.to(torch.bfloat16).double()
    slots = B * 48
    k, v = torch.zeros(slots, Hkv, D, dtype=torch.float64), torch.zeros(slots, Hkv, D, dtype=torch.float64)
    q = torch.zeros(B, Hkv, G, D, dtype=torch.float64)
    q[:, :, 1:, 0] = bf(torch.rand(B, Hkv, max(G - 1, 1), generator=g))[:, :, : G - 1]
    q[:, :, 0, 0] = 1.0
    first, last = torch.arange(B) * 48, torch.arange(B) * 48 + n - 1
    k[last - 1, :, 0], k[last, :, 0] = (bf(-0.1 - 1.2 * torch.rand(B, Hkv, generator=g)) for _ in range(2))        # scores 0, s1, s2
    p1, p2 = k[last - 1, :, :1].exp(), k[last, :, :1].exp()
    v0 = bf(1 + torch.rand(B, Hkv, D, generator=g))
    v1 = bf(-v0 / p1)
    v2 = bf(-(v0 + p1 * v1) / p2)
    v[first], v[last - 1], v[last] = v0, v1, v2
    tables = torch.arange(3 * B, dtype=torch.int32).view(B, 3)
    ctx = torch.full((B,), n, dtype=torch.int32)
    qb, kb, vb = (t.to(torch.bfloat16).to(device) for t in (q.reshape(B, Hkv * G, D), k, v))
    got = ops.paged_attention(qb, kb, vb, tables.to(device), ctx.to(device), Hq=Hkv * G, Hkv=Hkv, dqk=D, dv=D, block_size=bs, scale=1.0, window=window, sinks=sinks)
    got = got.double().cpu().view(B, Hkv, G, D)[:, :, 0]
    total = 1 + p1 + p2
    o, w = (v0 + p1 * v1 + p2 * v2) / total, (v0 + p1 * v1.abs() + p2 * v2.abs()) / total
    assert float((o.abs() / w).max()) < 2.0 ** -15
    off = (got - o).abs() - half_step(torch.bfloat16) * o.abs()
    assert (off <= 2.0 ** -20 * w).all(), float((off / w).max() * 2 ** 24)


def test_one_status_word_a_device(monkeypatch):
    """"cuda" is the current GPU; its word is that of "cuda:0" there, however it is spelled and whichever is asked for first."""
    real, made = torch.zeros, []

    def zeros(*shape, device=None, **kw):
        made.append(str(device))
        return real(*shape, **kw)
    monkeypatch.setattr(ops, "_status", {})
    monkeypatch.setattr(ops, "native_available", lambda: False)
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    words = [ops.gemm_status(d) for d in ("cuda", "cuda:1", torch.device("cuda"), torch.device("cuda", 1), torch.device("cuda:1"))]
    assert all(w is words[0] for w in words) and made == ["cuda:1"]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert ops.gemm_status("cuda") is ops.gemm_status("cuda:0") is not words[0]
    assert ops.gemm_status("cpu") is ops.gemm_status(torch.device("cpu"))
    assert made == ["cuda:1", "cuda:0", "cpu"]


@pytest.mark.gpu
def test_reports_are_seen_and_cleared_under_every_spelling():
    """A sequence longer than its table: the code that the kernel leaves on cuda:0, read and cleared through both names in turn."""
    q, pool = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda:0"), torch.zeros(32, 1, 64, dtype=torch.bfloat16, device="cuda:0")
    table, ctx = torch.zeros(1, 2, dtype=torch.int32, device="cuda:0"), torch.tensor([33], dtype=torch.int32, device="cuda:0")
    for read, other in (("cuda", "cuda:0"), ("cuda:0", "cuda"), (torch.device("cuda"), q.device), (q.device, torch.device("cuda"))):
        ops.clear_status(read)
        ops.paged_attention(q, pool, pool, table, ctx, Hq=2, Hkv=1, dqk=64, dv=64, block_size=16, scale=1.0, window=8, sinks=2)
        assert ops.check_status(read) == ops.check_status(other) == 131
        ops.clear_status(other)
        assert ops.check_status(read) == 0


def test_bad_indexes_are_no_expired_waits():
    """Codes 130 and 131 of the status word: an index that does not exist.  No wait ran out and no peer is gone."""
    from metal_marlin_b200.parallel import BadIndex, DeviceWaitExpired, PeerFailure, decode_status, raise_for_status
    for code, what in ((130, "row"), (131, "block")):
        kind, ranks, text = decode_status(code)
        assert (kind, ranks) == ("index", []) and what in text
        with pytest.raises(BadIndex) as e:
            raise_for_status(code)
        assert e.value.code == code and what in str(e.value) and "wait" not in str(e.value)
        assert not isinstance(e.value, (DeviceWaitExpired, PeerFailure))
    assert decode_status(128)[0] == "peer" and decode_status(129)[0] == decode_status(132)[0] == "local" and decode_status(140)[0] == "peer"


def test_the_engine_reports_a_bad_index_as_such():
    """The word that the engine polls after a pass."""
    from metal_marlin_b200.engine.engine import EngineConfig, LLMEngine
    from metal_marlin_b200.models.config import get_preset
    from metal_marlin_b200.models.mmfp4_causal_lm import MMFP4ForCausalLM
    from metal_marlin_b200.parallel import BadIndex
    lm = MMFP4ForCausalLM.from_config(get_preset("tiny-llama"), device="cpu", seed=0)
    eng = LLMEngine(lm.model, EngineConfig(num_kv_blocks=16, block_size=16, max_model_len=64, use_cuda_graphs=False))
    ops.gemm_status("cpu")[0] = 131
    with pytest.raises(BadIndex):
        eng._check_device_status()
    assert ops.check_status("cpu") == 0
    eng._check_device_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("block", [-1, -(2 ** 31), 7, 2 ** 31 - 1])
def test_blocks_outside_the_pool_hide_their_tokens(device, block):
    """A page of a sequence that the pool does not have, one step below and above it and at the ends of the type; a sequence with nothing else; one
    that is longer than its table, and one of negative length.  What is left is the attention of the visible tokens alone, and 131 is reported."""
    Hq, Hkv, D, bs, window, sinks = 4, 2, 64, 16, 40, 3
    a = attention_inputs(device, [30, 16, 16, 16], Hq, Hkv, D, bs)                   # seven blocks, five of them in use
    assert a[1].shape[0] == 7 * bs
    use = a[3][0, 0], a[3][0, 1], a[3][1, 0], a[3][2, 0]
    tables = torch.tensor([[use[0], block, use[1]], [block, block, block], [use[2], use[3], use[0]], [use[0], use[1], use[2]]], dtype=torch.int32)
    ctx = [45, 33, 60, -5]                                                           # the third has places for 48
    ops.clear_status(device)
    got = run_attention((*a[:3], tables), ctx, Hq, Hkv, D, bs, window, sinks, device)
    assert ops.check_status(device) == 131
    ops.clear_status(device)
    assert not got[1].any() and not got[3].any()
    # the same tokens as sequences of their own in a dense cache, every one visible: 2 sinks and the window from 5, without the block 16 .. 31; 0 .. 2 and 8 .. 47
    for b, pos in ((0, [p for p in range(45) if (p < 3 or p >= 5) and not 16 <= p < 32]), (2, [p for p in range(48) if p < 3 or p >= 8])):
        slots = torch.tensor([int(tables[b, p // bs]) * bs + p % bs for p in pos])
        n = len(pos)
        k, v = (torch.cat([t[slots], torch.zeros(48 - n, Hkv, D, dtype=torch.float64)]) for t in a[4:6])
        want = attention_oracle(a[0][b: b + 1], k, v, torch.arange(3)[None], [n], Hkv, bs, D ** -0.5, n, 1)
        check_attention(got[b: b + 1], want)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_outside_the_pool_are_skipped_and_reported(device):
    """Prompts and single tokens: a row behind the pool is reported, a negative one is padding, an empty sequence is neither."""
    x, w, b, state, rows, fresh, cu = conv_inputs(device, [3, 0, 4, 5], 8, 4, torch.bfloat16)
    for bad, code in (([1, 99, -1, 2], 0), ([1, 2, 7, -1], 130), ([1, 2, 3, 2 ** 62], 130)):
        pool, rows = state.clone(), torch.tensor(bad)
        ops.clear_status(device)
        out = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device), state=pool, rows=rows.to(device), fresh=fresh.to(device))
        assert ops.check_status(device) == code
        check_conv(out, pool, *conv_oracle(x, w, b, state, spans(cu, fresh, bad), 1))
    p = ssm_inputs(device, [5, 6], 8, 16, torch.bfloat16)
    p["rows"] = torch.tensor([1, 99])
    ops.clear_status(device)
    out, pool = run_ssm(p, device)
    assert ops.check_status(device) == 130
    check_ssm(out, pool, want_ssm(p))
    for rows, code in (([0, -1], 0), ([4, 1], 130)):
        ops.clear_status(device)
        ops.ssm_step(p["x"][:2], p["dt"][:2], p["A"], p["Bm"][:2], p["Cm"][:2], state=p["state"].clone(), rows=torch.tensor(rows, device=device))
        assert ops.check_status(device) == code
    ops.clear_status(device)


def poisoned(device, *shape, dtype):
    """Leaves NaN where the next tensor of this size is likely to be made."""
    torch.full(shape, float("nan"), dtype=dtype, device=device)


# rows in front of the first sequence, lengths, rows behind the last
FRONTS = [(1, [5], 0), (3, [0, 9], 2), (8, [20], 5), (70, [3, 0, 130], 0), (131, [], 9), (7, [0, 0], 3), (64, [1] * 20, 1), (9, [], 0)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("front,lens,tail", FRONTS)
@pytest.mark.parametrize("C,dtype", [(8, "bf16"), (7, "fp32"), (2048, "fp16")])
def test_conv_with_rows_in_front_of_the_first_sequence(device, front, lens, tail, C, dtype):
    """They belong to no sequence: zeros in a new output, left alone in the caller's, and no part of any window."""
    t = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}[dtype]
    x, w, b, state, rows, fresh, cu = conv_inputs(device, [front] + lens, C, 4, t, tail=tail)
    cu, rows, fresh = cu[1:], rows[1:], fresh[1:]
    x[:front] = float("nan")
    want = conv_oracle(torch.nan_to_num(x), w, b, state, spans(cu, fresh, rows.tolist()), 1)
    call = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device), rows=rows.to(device), fresh=fresh.to(device))
    pool = state.clone()
    poisoned(device, *x.shape, dtype=t)
    out = ops.causal_conv(x, w, b, state=pool, **call)
    assert not out[:front].any() and not out[cu[-1]:].any()
    check_conv(out, pool, *want)
    pool, into = state.clone(), torch.full_like(x, 7.0)
    assert ops.causal_conv(x, w, b, state=pool, out=into, **call) is into
    assert (into[:front] == 7).all() and (into[cu[-1]:] == 7).all() and torch.equal(into[front: cu[-1]], out[front: cu[-1]])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("front,lens,tail", FRONTS)
@pytest.mark.parametrize("C,N", [(8, 16), (7, 5), (300, 64)])
def test_scan_with_rows_in_front_of_the_first_sequence(device, front, lens, tail, C, N):
    """The same of the selective scan."""
    p = ssm_inputs(device, [front] + lens, C, N, torch.bfloat16, tail=tail)
    p["cu"], p["rows"], p["fresh"] = p["cu"][1:], p["rows"][1:], p["fresh"][1:]
    want = want_ssm(p)
    for name in ("x", "z", "dt", "Bm", "Cm"):
        p[name][:front] = float("nan")
    poisoned(device, *p["x"].shape, dtype=torch.bfloat16)
    out, state = run_ssm(p, device)
    assert not out[:front].any() and not out[p["cu"][-1]:].any()
    check_ssm(out, state, want)
    into = torch.full((p["x"].shape[0], C), 7.0, dtype=torch.bfloat16, device=device)
    run_ssm(p, device, out=into)
    assert (into[:front] == 7).all() and (into[p["cu"][-1]:] == 7).all() and torch.equal(into[front: p["cu"][-1]], out[front: p["cu"][-1]])


@pytest.mark.parametrize("T,C", [(1, 2 ** 30 + 1), (1, 2 ** 31 - 1), (2 ** 30 + 1, 1)])
def test_sizes_that_the_kernels_do_not_count_are_refused(T, C):
    """Rows and channels are numbered in 32 bits, up to the end of the last tile: more than 2^30 of either is refused.  Shapes alone, nothing is allocated."""
    from metal_marlin_b200 import _build
    m = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="meta", dtype=dtype)
    x, w, A, bc, cu = m(T, C, dtype=torch.bfloat16), m(C, 2), m(C, 1), m(T, 1), m(2, dtype=torch.int32)
    for call in (lambda: ops.causal_conv(x, w, cu_seqlens=cu), lambda: ops.ssm_scan(x, x, A, bc, bc, cu_seqlens=cu)):
        with pytest.raises(ValueError):
            call()
    if T == 1:
        for call in (lambda: ops.causal_conv_step(x, w, state=m(1, C, 1)), lambda: ops.ssm_step(x, x, A, bc, bc, state=m(1, C, 1))):
            with pytest.raises(ValueError):
                call()
    if _build.load():
        with pytest.raises(ValueError):
            torch.ops.mmb200.causal_conv(x, w, None, x, None, None, None, cu, 1, True)
        with pytest.raises(ValueError):
            torch.ops.mmb200.ssm(x, x, A, bc, bc, None, None, None, x, None, None, None, cu, False, True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8", "fp4", "int4"])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (256, 2), (128, 16), (256, 12)])
def test_long_sums_are_rounded_and_not_cut_off(fmt, D, G):
    """Enough rows that nobody shares one: each warp keeps one sum over all visible keys, 64 tiles of its own.  Scores repeat from one round of the warps' tiles
    to the next; values are 256 u in the first round, u with signs in turn in the 62 between, -256 u in the last.  The exact output is zero, while the sum a stays
    near its largest value.

    Rounded to nearest, a + s and then - s gives a again (it is a multiple of a's step within half a step of a; one step more where a tie was met), whatever
    the 62 rounds add up to; the first and the last are the same products with other signs.  A tile's own products may lose two steps of theirs, the first and
    last 256 times as large two of a's each: four steps 2^-23 of at most 257 rounds' worth, against 64 rounds' worth in the denominator, 2.01 x 2^-20 u.
    Sums that every product cuts off drift by up to a step with each: 2^-15 u."""
    B, Hkv, bs, rounds, sinks = 320, 1, 16, 64, 16
    per = 64 if fmt == "bf16" or D == 256 else 128                           # keys of the four warps' tiles
    m = per * rounds
    window, n = m - sinks, m + 100
    g = torch.Generator().manual_seed(D + G)
    pos = torch.cat([torch.arange(sinks), torch.arange(n - window, n)])
    k, v = torch.zeros(n + 12, Hkv, D), torch.zeros(n + 12, Hkv, D)
    k[:, :, 0] = -8.0                                                        # never visible
    k[pos, 0, 0] = -(torch.rand(per, generator=g) * 2)[torch.arange(m) % per]
    sign = torch.ones(rounds)
    sign[2:-1:2], sign[0], sign[-1] = -1.0, 256.0, -256.0
    u = (1 + torch.rand(D, generator=g)).to(torch.bfloat16).float() if fmt == "bf16" else torch.ones(D)
    v[pos, 0] = sign[torch.arange(m) // per][:, None] * u
    assert float(v[pos].double().sum(0).abs().max()) == 0
    kb, vb = k.to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda()
    if fmt != "bf16":
        pools = []
        for t in (kb, vb):
            pool = ops.FP8KV(n + 12, (Hkv, D), "cuda", fmt)
            pool.store(torch.arange(n + 12, device="cuda"), t)
            pools.append(pool)
        kb, vb = pools
    q = torch.zeros(B, Hkv * G, D, dtype=torch.bfloat16)
    q[:, :, 0] = torch.rand(B, Hkv * G, generator=g) + 0.5
    tables = torch.arange((n + 12) // bs, dtype=torch.int32).expand(B, -1).contiguous().cuda()
    ctx = torch.full((B,), n, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q.cuda(), kb, vb, tables, ctx, Hq=Hkv * G, Hkv=Hkv, dqk=D, dv=D, block_size=bs, scale=1.0, window=window, sinks=sinks)
    off = got.double().cpu().abs() / u.double()
    assert float(off.max()) <= 2.02 * 2.0 ** -20, float(off.max()) * 2 ** 20
