"""The operators that keep a sequence going at constant cost per token, against their definitions in 64 bits: short causal convolution and
selective scan over pools of per-sequence state, and decode attention with a sliding window and sinks.

Tolerances are sums of what the kernels may round: half a step of the output type (``finfo.eps / 2`` of the value), and for the arithmetic in 32 bits
the terms written at each comparison."""
import math

import pytest
import torch

from metal_marlin_b200 import ops

CPU = torch.device("cpu")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# one fp32 step of the special functions: 2^x and the logarithm are good to 2^-21, and the argument x = v log2(e) with |v| <= 16 adds 2^-20
FN = 2.0 ** -19


def half_step(t):
    return 0.501 * torch.finfo(t).eps


def tiny(t):
    """What values below the smallest normal number of the type may lose."""
    return float(torch.finfo(t).tiny)


def gen(seed, device):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float32).to(device)


def spans(cu, fresh, rows):
    return [(cu[i], cu[i + 1] - cu[i], rows[i], bool(fresh[i])) for i in range(len(cu) - 1)]


# ------------------------------------------------------------------------------------------------------------- oracles (64 bits)
def conv_oracle(x, w, bias, state, seqs, act):
    """``(out, scale of every output, new state)``; rows of no live sequence are zero."""
    x, w, state = x.double().cpu(), w.double().cpu(), state.double().cpu().clone()
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    K = w.shape[1]
    for at, n, row, fresh in seqs:
        if n == 0 or row is None or row < 0 or row >= state.shape[0]:
            continue
        old = torch.zeros_like(state[row]) if fresh else state[row]
        line = torch.cat([old.t(), x[at: at + n]])
        for k in range(K):
            out[at: at + n] += line[k: k + n] * w[:, k]
            mag[at: at + n] += (line[k: k + n] * w[:, k]).abs()
        if bias is not None:
            out[at: at + n] += bias.double().cpu()
            mag[at: at + n] += bias.double().cpu().abs()
        state[row] = line[n:].t()
    return (out * torch.sigmoid(out) if act else out), mag, state


def check_conv(out, state, want, mag, want_state):
    assert torch.equal(state.double().cpu(), want_state)                                     # inputs, moved and never computed with
    # fp32 sums of up to 9 terms: 9 2^-24 of their magnitudes; SiLU has slope at most 1.1 and its exponential is FN off
    tol = half_step(out.dtype) * want.abs() + (1.1 * 9 * 2.0 ** -24 + FN) * mag + tiny(out.dtype)
    assert ((out.double().cpu() - want).abs() <= tol).all(), float(((out.double().cpu() - want).abs() - tol).max())


def ssm_oracle(x, dt, A, Bm, Cm, D, z, bias, softplus, state, seqs):
    """``(out, its error bound apart from the output's rounding, new state, its error bound)``.  The bounds follow the recurrence: every step
    multiplies the state by a factor that is ``c`` off and adds a term that is ``c`` off, where c collects the roundings of d (softplus: FN, and its
    sum with the bias 2^-24 of its parts), of the exponent and of the exponential."""
    x, dt, A, Bm, Cm = (t.double().cpu() for t in (x, dt, A, Bm, Cm))
    state = state.double().cpu().clone()
    bound = torch.zeros_like(state)
    T, Di = x.shape
    raw = dt if bias is None else dt + bias.double().cpu()
    d = torch.logaddexp(raw, torch.zeros((), dtype=torch.float64)) if softplus else raw
    err_d = 2.0 ** -23 * (dt.abs() + (0 if bias is None else bias.double().cpu().abs()))
    if softplus:                                                                             # slope of softplus: its sigmoid
        err_d = err_d * torch.sigmoid(raw) + FN * d
    out, err = torch.zeros_like(x), torch.zeros_like(x)
    for at, n, row, fresh in seqs:
        if n == 0 or row < 0 or row >= state.shape[0]:
            continue
        h = torch.zeros_like(state[row]) if fresh else state[row].clone()
        H, E = h.abs(), torch.zeros_like(h)
        for t in range(at, at + n):
            a = torch.exp(d[t][:, None] * A)
            b = (d[t] * x[t])[:, None] * Bm[t]
            rel_a = (err_d[t][:, None] + 2.0 ** -22 * d[t].abs()[:, None]) * A.abs() + 2.0 ** -20
            err_b = (err_d[t] * x[t].abs())[:, None] * Bm[t].abs() + 2.0 ** -22 * b.abs()
            h, H, E = a * h + b, a * H + b.abs(), a * E + a * H * rel_a + err_b + 2.0 ** -23 * (a * H + b.abs())
            y = (h * Cm[t]).sum(-1)
            m = (H * Cm[t].abs()).sum(-1)
            e = (E * Cm[t].abs()).sum(-1) + (A.shape[1] + 4) * 2.0 ** -24 * m
            if D is not None:
                y, e = y + D.double().cpu() * x[t], e + 2.0 ** -22 * (m + (D.double().cpu() * x[t]).abs())
            if z is not None:
                zf = z[t].double().cpu()
                s = zf * torch.sigmoid(zf)
                e = e * s.abs() + (y.abs() + e) * FN * zf.abs()
                y = y * s
            out[t], err[t] = y, e
        state[row], bound[row] = h, E
    return out, err, state, bound


def check_ssm(out, state, want):
    y, err, st, st_err = want
    tol = half_step(out.dtype) * (y.abs() + err) + err + tiny(out.dtype)
    gap = (out.double().cpu() - y).abs() - tol
    assert (gap <= 0).all(), float(gap.max())
    gap = (state.double().cpu() - st).abs() - (st_err + tiny(torch.float32))
    assert (gap <= 0).all(), float(gap.max())


def attention_oracle(q, k, v, tables, ctx, Hkv, bs, scale, window, sinks, kf=None):
    """``(out, error bound apart from the output's rounding)``; ``k, v`` are double ``[slots, Hkv, D]``."""
    B, Hq, D = q.shape
    out, err = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        n = int(ctx[b])
        pos = [p for p in range(n) if p < sinks or p >= n - window]
        if not pos:
            continue
        slots = torch.tensor([int(tables[b, p // bs]) * bs + p % bs for p in pos])
        kk, vv = k[slots], v[slots]
        qq = q[b].double().cpu().view(Hkv, Hq // Hkv, D)
        s = torch.einsum("hgd,thd->hgt", qq, kk) * scale
        m = torch.einsum("hgd,thd->hgt", qq.abs(), kk.abs()) * abs(scale)
        pr = torch.softmax(s, -1)
        o = torch.einsum("hgt,thd->hgd", pr, vv)
        w = torch.einsum("hgt,thd->hgd", pr, vv.abs())
        # scores: D fp32 products summed (2^-23 a step) and a few roundings of scale; exponentials 2^-21 and their argument; P in two bf16
        # parts 2^-16; sums over the keys 2^-23 a key; numerator and denominator alike
        rel = m.amax(-1) * (D + 8) * 2.0 ** -23 + s.abs().amax(-1) * 2.0 ** -22 + 2.0 ** -16 + len(pos) * 2.0 ** -23
        out[b], err[b] = o.reshape(Hq, D), (2 * rel[..., None] * w).reshape(Hq, D)
    return out, err


def check_attention(got, want):
    o, err = want
    gap = (got.double().cpu() - o).abs() - (half_step(torch.bfloat16) * (o.abs() + err) + err + 1e-30)
    assert (gap <= 0).all(), float(gap.max())


# --------------------------------------------------------------------------------------------------------------------- inputs
def conv_inputs(device, lens, C, K, dtype, seed=0, bias=True, wide=0, tail=0):
    rn = gen(seed, device)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T, S = cu[-1] + tail, len(lens)
    x = rn(T, C + wide).to(dtype)[:, wide // 2: wide // 2 + C]
    w, b = (rn(C, K) * K ** -0.5).to(dtype), ((rn(C) * 0.3).to(dtype) if bias else None)
    state = rn(S + 3, C, K - 1)
    rows = torch.randperm(S + 3, generator=torch.Generator().manual_seed(seed + 1))[:S]
    fresh = torch.arange(S) % 2 == 1
    return x, w, b, state, rows, fresh, cu


def ssm_inputs(device, lens, C, N, dtype, seed=0, tail=0, bc=None, dt_type=None):
    rn = gen(seed, device)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T, S = cu[-1] + tail, len(lens)
    xz = rn(T, 2 * C + 8).to(dtype)
    d = torch.exp(math.log(1e-3) + torch.sigmoid(rn(C) * 1.5) * math.log(100.0))
    p = {"x": xz[:, :C], "z": xz[:, C: 2 * C], "dt": (rn(T, C) * 0.5).to(dt_type or dtype), "dt_bias": d + torch.log(-torch.expm1(-d)),
         "A": -torch.arange(1, N + 1, device=device).float() * torch.exp(rn(C, N) * 0.1), "D": rn(C)}
    BC = rn(T, 2 * N).to(bc or dtype)
    p["Bm"], p["Cm"] = BC[:, :N], BC[:, N:]
    p["state"] = rn(S + 2, C, N) * 0.2
    p["rows"] = torch.randperm(S + 2, generator=torch.Generator().manual_seed(seed + 1))[:S]
    p["fresh"] = torch.arange(S) % 2 == 1
    p["cu"] = cu
    return p


def run_ssm(p, device, out=None, **kw):
    state = p["state"].clone()
    o = ops.ssm_scan(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], cu_seqlens=torch.tensor(p["cu"], dtype=torch.int32, device=device), state=state,
                     rows=p["rows"].to(device), fresh=p["fresh"].to(device), D=p["D"], z=p["z"], dt_bias=p["dt_bias"], dt_softplus=True, out=out, **kw)
    return o, state


def want_ssm(p):
    return ssm_oracle(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], p["D"], p["z"], p["dt_bias"], True, p["state"], spans(p["cu"], p["fresh"], p["rows"].tolist()))


def attention_inputs(device, ctx, Hq, Hkv, D, bs, fmt="bf16", seed=0, sharp=1.0):
    rn = gen(seed, device)
    need = [max(1, (n + bs - 1) // bs) for n in ctx]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tables = torch.full((len(ctx), max(need) + 1), 10 ** 8, dtype=torch.int32)                # entries behind a sequence are never followed
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at: at + n]
        at += n
    slots = (sum(need) + 2) * bs
    q = (rn(len(ctx), Hq, D) * sharp).to(torch.bfloat16)
    k, v = rn(slots, Hkv, D).to(torch.bfloat16), rn(slots, Hkv, D).to(torch.bfloat16)
    if fmt == "bf16":
        return q, k, v, tables, k.double().cpu(), v.double().cpu()
    pools = []
    for t in (k, v):
        pool = ops.FP8KV(slots, (Hkv, D), device, fmt)
        pool.store(torch.arange(slots, device=device), t)
        pools.append(pool)
    exact = []
    for pool in pools:
        codes = pool.data
        if pool.four_bit:
            codes = torch.stack([codes & 0xF, codes >> 4], -1).flatten(-2)
        exact.append((pool._decode(codes).double() * pool.scale.double()[..., None]).cpu())
    return q, pools[0], pools[1], tables, exact[0], exact[1]


def run_attention(a, ctx, Hq, Hkv, D, bs, window, sinks, device, **kw):
    q, k, v, tables = a[:4]
    return ops.paged_attention(q, k, v, tables.to(device), torch.tensor(ctx, dtype=torch.int32, device=device), Hq=Hq, Hkv=Hkv, dqk=D, dv=D,
                               block_size=bs, scale=kw.pop("scale", D ** -0.5), window=window, sinks=sinks, **kw)


# -------------------------------------------------------------------------------------------------------------------- devices
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


CONV_CASES = [
    ([1], 1, 2, "fp32", {}), ([3], 8, 4, "bf16", {}), ([1, 2, 3, 4], 24, 4, "fp16", {}), ([5, 0, 1, 17], 40, 3, "bf16", {"tail": 3}),
    ([33, 64, 7], 65, 4, "bf16", {"wide": 7}), ([8, 9], 16, 8, "fp32", {"bias": False}), ([0, 0, 2], 8, 5, "bf16", {"tail": 9}),
    ([70], 256, 4, "bf16", {"wide": 8}), ([40, 31], 12, 6, "fp16", {}), ([2, 12], 9, 7, "fp32", {"tail": 1}),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,C,K,dtype,kw", CONV_CASES)
@pytest.mark.parametrize("act", [0, 1])
def test_conv_of_ragged_prompts(device, lens, C, K, dtype, kw, act):
    x, w, b, state, rows, fresh, cu = conv_inputs(device, lens, C, K, TYPES[dtype], **kw)
    want = conv_oracle(x, w, b, state, spans(cu, fresh, rows.tolist()), act)
    out = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device), state=state, rows=rows.to(device), fresh=fresh.to(device),
                          act=act)
    assert out.dtype == x.dtype
    check_conv(out, state, *want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("C,K,dtype,out_dtype", [(8, 4, "bf16", "fp32"), (7, 3, "fp16", "fp16"), (260, 4, "bf16", "bf16"), (512, 2, "fp32", "bf16"), (36, 8, "bf16", "bf16")])
def test_conv_of_single_tokens(device, C, K, dtype, out_dtype):
    """Padding rows give zeros and touch nothing; the windows of the others shift by their input."""
    B = 5
    x, w, b, state, _, _, _ = conv_inputs(device, [B], C, K, TYPES[dtype], seed=3, wide=4)
    state = gen(9, device)(9, C, K - 1)
    rows = torch.tensor([4, -1, 0, 8, -7])
    want = conv_oracle(x, w, b, state, [(i, 1, r, False) for i, r in enumerate(rows.tolist())], 1)
    out = ops.causal_conv_step(x, w, b, state=state, rows=rows.to(device), out_dtype=TYPES[out_dtype])
    assert out.dtype == TYPES[out_dtype]
    check_conv(out, state, *want)
    assert not out[1].any() and not out[4].any()


@pytest.mark.parametrize("device", DEVICES)
def test_conv_without_a_pool_and_with_the_callers_out(device):
    x, w, b, _, _, _, cu = conv_inputs(device, [6, 11], 16, 4, torch.bfloat16, tail=4)
    seqs = [(cu[i], cu[i + 1] - cu[i], i, True) for i in range(2)]
    want = conv_oracle(x, w, b, torch.zeros(2, 16, 3), seqs, 1)
    wide = torch.full((21, 40), 7.0, dtype=torch.bfloat16, device=device)
    out = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device), out=wide[:, 8:24])
    check_conv(out[:17], torch.zeros(2, 16, 3), want[0][:17], want[1][:17], torch.zeros(2, 16, 3, dtype=torch.float64))
    assert (wide[17:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 24:] == 7).all()         # rows behind the last sequence stay


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [2, 4, 8])
def test_conv_in_chunks_and_tokens_equals_one_pass(device, K):
    x, w, b, _, _, _, _ = conv_inputs(device, [40], 24, K, torch.bfloat16, seed=5)
    one, many = torch.zeros(2, 24, K - 1, device=device), torch.zeros(2, 24, K - 1, device=device)
    cu = lambda *n: torch.tensor(n, dtype=torch.int32, device=device)
    row = torch.tensor([1], device=device)
    whole = ops.causal_conv(x, w, b, cu_seqlens=cu(0, 40), state=one, rows=row)
    parts = [ops.causal_conv(x[:1], w, b, cu_seqlens=cu(0, 1), state=many, rows=row), ops.causal_conv(x[1:3], w, b, cu_seqlens=cu(0, 2), state=many, rows=row),
             ops.causal_conv(x[3:30], w, b, cu_seqlens=cu(0, 27), state=many, rows=row)]
    parts += [ops.causal_conv_step(x[t: t + 1], w, b, state=many, rows=row) for t in range(30, 40)]
    assert torch.equal(whole, torch.cat(parts)) and torch.equal(one, many) and not one[0].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", range(2, 9))
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_conv_of_every_number_of_taps(device, K, dtype):
    """Whole-word rows, sequences shorter and longer than the window, fresh and old; a pool on a 16-byte boundary and one four bytes behind it."""
    lens, C = [1, 2, 5, 9, 0, 20], 64
    x, w, b, state, rows, fresh, cu = conv_inputs(device, lens, C, K, TYPES[dtype], seed=K)
    want = conv_oracle(x, w, b, state, spans(cu, fresh, rows.tolist()), 1)
    for offset in (0, 1):
        pool = torch.empty(state.numel() + 1, device=device)[offset:offset + state.numel()].view_as(state).copy_(state)
        out = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device), state=pool, rows=rows.to(device),
                              fresh=fresh.to(device))
        check_conv(out, pool, *want)
        one = torch.empty(state.numel() + 1, device=device)[offset:offset + state.numel()].view_as(state).copy_(state)
        step = conv_oracle(x[:6], w, b, state, [(i, 1, r, False) for i, r in enumerate(rows.tolist())], 1)
        check_conv(ops.causal_conv_step(x[:6], w, b, state=one, rows=rows.to(device)), one, *step)


SSM_CASES = [
    ([1], 1, 1, "fp32", {}), ([3], 8, 16, "bf16", {}), ([33, 1, 0, 40], 40, 16, "bf16", {"tail": 5}), ([70], 33, 16, "fp16", {}),
    ([5, 66], 24, 8, "fp32", {}), ([31, 7], 16, 24, "bf16", {}), ([65], 48, 64, "bf16", {"bc": torch.float32}), ([20, 9], 17, 128, "fp16", {}),
    ([129], 8, 5, "bf16", {"dt_type": torch.float32}), ([0, 0, 3], 64, 16, "bf16", {"tail": 70}), ([64, 32, 96], 136, 32, "bf16", {}),
    ([17], 9, 100, "fp32", {}),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,C,N,dtype,kw", SSM_CASES)
def test_scan_of_ragged_prompts(device, lens, C, N, dtype, kw):
    p = ssm_inputs(device, lens, C, N, TYPES[dtype], **kw)
    out, state = run_ssm(p, device)
    assert out.dtype == p["x"].dtype
    check_ssm(out, state, want_ssm(p))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("use", ["plain", "D", "z", "bias", "all", "no pool"])
def test_scan_options(device, use):
    """Every optional input on its own; without softplus dt is the step itself, here of both signs (the state may grow)."""
    p = ssm_inputs(device, [37, 12], 24, 16, torch.bfloat16, seed=2)
    dt = (p["dt"].float() * 0.05).to(torch.bfloat16)
    D, z = (p[n] if use in (n, "all") else None for n in ("D", "z"))
    bias = p["dt_bias"] * 0.01 if use in ("bias", "all") else None
    cu = torch.tensor(p["cu"], dtype=torch.int32, device=device)
    pool = None if use == "no pool" else p["state"].clone()
    out = ops.ssm_scan(p["x"], dt, p["A"], p["Bm"], p["Cm"], cu_seqlens=cu, state=pool, rows=None if pool is None else p["rows"].to(device), D=D, z=z,
                       dt_bias=bias, out_dtype=torch.float32)
    rows, fresh = (p["rows"].tolist(), [False] * 2) if pool is not None else ([0, 1], [True] * 2)
    want = ssm_oracle(p["x"], dt, p["A"], p["Bm"], p["Cm"], D, z, bias, False, p["state"], spans(p["cu"], fresh, rows))
    check_ssm(out, want[2] if pool is None else pool, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("C,N,dtype", [(8, 16, "bf16"), (7, 16, "fp16"), (130, 8, "bf16"), (64, 64, "fp32"), (33, 5, "bf16"), (24, 128, "bf16"), (10, 30, "fp32"), (12, 36, "bf16")])
def test_scan_of_single_tokens(device, C, N, dtype):
    p = ssm_inputs(device, [6], C, N, TYPES[dtype], seed=4)
    state = gen(8, device)(9, C, N)
    rows = torch.tensor([4, -1, 0, 8, -3, 2])
    want = ssm_oracle(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], p["D"], p["z"], p["dt_bias"], True, state, [(i, 1, r, False) for i, r in enumerate(rows.tolist())])
    out = ops.ssm_step(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], state=state, rows=rows.to(device), D=p["D"], z=p["z"], dt_bias=p["dt_bias"], dt_softplus=True)
    check_ssm(out, state, want)
    assert not out[1].any() and not out[4].any()


@pytest.mark.parametrize("device", DEVICES)
def test_scan_with_extreme_steps(device):
    """Softplus far on both sides, a step that empties the state, and one that leaves it alone."""
    p = ssm_inputs(device, [9], 16, 16, torch.float32, seed=6)
    p["dt"] = torch.tensor([-100.0, -30.0, -9.0, 0.0, 9.0, 30.0, 88.0, 200.0, -5.0], device=device)[:, None].expand(9, 16).contiguous()
    p["dt_bias"] = torch.zeros(16, device=device)
    out, state = run_ssm(p, device)
    assert torch.isfinite(out).all()
    y, err, st, st_err = want_ssm(p)
    # exponents of a few thousand: their rounding multiplies factors that are below 2^-1000 and vanish either way
    check_ssm(out, state, (y, err, st, st_err + 1e-30))


def test_refusals_of_the_state_operators():
    """The same checks in the CPU path and in the binding (which looks at shapes and types before it asks for a GPU)."""
    from metal_marlin_b200 import _build
    x, w, b, state, rows, fresh, cu = conv_inputs("cpu", [3, 4], 8, 4, torch.bfloat16)
    cu = torch.tensor(cu, dtype=torch.int32)
    conv = dict(x=x, w=w, bias=b, cu_seqlens=cu, state=state, rows=rows, fresh=fresh, act=1)
    bad = [dict(x=x.double()), dict(x=x[0]), dict(x=x.t().contiguous().t()), dict(w=w[:, :1].contiguous()), dict(w=w.repeat(1, 3)), dict(w=w[:4]), dict(w=w.double()),
           dict(w=w.t().contiguous().t()), dict(bias=b[:3]), dict(bias=b.float()), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:0]), dict(state=state.half()),
           dict(state=state[:, :, :2]), dict(state=state[0]), dict(state=state.transpose(0, 1).contiguous().transpose(0, 1)), dict(rows=rows.int()), dict(rows=rows[:1]),
           dict(rows=None, state=state[:1]), dict(state=None), dict(fresh=fresh[:1]), dict(fresh=fresh.int()), dict(act=2)]
    assert ops.causal_conv(**conv).shape == x.shape
    native = _build.load()
    for change in bad:
        kw = dict(conv, **change)
        with pytest.raises(ValueError):
            ops.causal_conv(**kw)
        if native and kw["x"].dim() == 2:
            with pytest.raises(ValueError):
                torch.ops.mmb200.causal_conv(kw["x"], kw["w"], kw["bias"], torch.empty_like(kw["x"]), kw["state"], kw["rows"], kw["fresh"], kw["cu_seqlens"], kw["act"], True)
    with pytest.raises(ValueError):
        ops.causal_conv(x, w, b, cu_seqlens=cu, out=x)
    with pytest.raises(ValueError):
        ops.causal_conv(x, w, b, cu_seqlens=cu, out=torch.empty(7, 8), out_dtype=torch.bfloat16)
    wide = torch.zeros(7, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.causal_conv(wide[:, :8], w, b, cu_seqlens=cu, out=wide[:, 4:12])
    assert ops.causal_conv(wide[:, :8], w, b, cu_seqlens=cu, out=wide[:, 8:]) is not None          # side by side in one buffer
    with pytest.raises(ValueError):
        ops.causal_conv_step(x, w, b, state=None)
    with pytest.raises(ValueError):
        ops.causal_conv_step(x, w, b, state=state[:5])
    p = ssm_inputs("cpu", [3, 4], 8, 16, torch.bfloat16)
    cu = torch.tensor(p["cu"], dtype=torch.int32)
    scan = dict(x=p["x"], dt=p["dt"], A=p["A"], Bm=p["Bm"], Cm=p["Cm"], D=p["D"], z=p["z"], dt_bias=p["dt_bias"], state=p["state"], rows=p["rows"], fresh=p["fresh"], cu_seqlens=cu)
    bad = [dict(dt=p["dt"][:, :4]), dict(A=p["A"].half()), dict(A=p["A"][:, :8]), dict(A=p["A"].repeat(1, 9)), dict(Bm=p["Bm"][:3]), dict(Cm=p["Cm"].float()),
           dict(Bm=p["Bm"].double(), Cm=p["Cm"].double()), dict(D=p["D"].half()), dict(D=p["D"][:3]), dict(z=p["z"][:2]), dict(dt_bias=p["dt_bias"].double()),
           dict(state=p["state"][:, :4]), dict(rows=None, state=p["state"][:1]), dict(state=None), dict(cu_seqlens=cu.float()), dict(x=p["x"].long())]
    assert ops.ssm_scan(dt_softplus=True, **scan).shape == (7, 8)
    for change in bad:
        kw = dict(scan, **change)
        with pytest.raises(ValueError):
            ops.ssm_scan(**kw)
        if native:
            with pytest.raises(ValueError):
                torch.ops.mmb200.ssm(kw["x"], kw["dt"], kw["A"], kw["Bm"], kw["Cm"], kw["D"], kw["z"], kw["dt_bias"], torch.empty(7, 8), kw["state"], kw["rows"], kw["fresh"],
                                     kw["cu_seqlens"], True, True)
    with pytest.raises(ValueError):
        ops.ssm_step(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], state=p["state"], rows=p["rows"])


# the launchers choose other tiles, splits of a channel and rows a block for large calls: the same definitions at sizes that reach them
@pytest.mark.gpu
@pytest.mark.parametrize("lens,C,dtype,out", [([2500, 0, 100], 4096, "bf16", None), ([700, 8000, 3], 4096, "fp16", "fp32"), ([4000, 300], 2050, "bf16", "bf16"),
                                              ([90] * 40, 4096, "fp32", None)])
def test_conv_of_large_batches(lens, C, dtype, out):
    x, w, b, state, rows, fresh, cu = conv_inputs("cuda", lens, C, 4, TYPES[dtype], tail=5)
    want = conv_oracle(x, w, b, state, spans(cu, fresh, rows.tolist()), 1)
    got = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), state=state, rows=rows.to("cuda"), fresh=fresh.to("cuda"),
                          out_dtype=TYPES[out] if out else None)
    check_conv(got, state, *want)


@pytest.mark.gpu
def test_conv_of_many_short_sequences():
    """More sequences than the kernel keeps starts of in shared memory."""
    lens = [1 + i % 3 for i in range(1500)]
    x, w, b, state, rows, fresh, cu = conv_inputs("cuda", lens, 12, 4, torch.bfloat16)
    want = conv_oracle(x, w, b, state, spans(cu, fresh, rows.tolist()), 1)
    got = ops.causal_conv(x, w, b, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), state=state, rows=rows.to("cuda"), fresh=fresh.to("cuda"))
    check_conv(got, state, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("C,K", [(8192, 4), (4100, 5)])
def test_conv_of_a_large_decode_batch(C, K):
    B = 257
    x, w, b, _, _, _, _ = conv_inputs("cuda", [B], C, K, torch.bfloat16)
    state = gen(9, "cuda")(B + 3, C, K - 1)
    rows = torch.randperm(B + 3, generator=torch.Generator().manual_seed(2))[:B]
    rows[5], rows[200] = -1, -1
    want = conv_oracle(x, w, b, state, [(i, 1, r, False) for i, r in enumerate(rows.tolist())], 1)
    check_conv(ops.causal_conv_step(x, w, b, state=state, rows=rows.to("cuda")), state, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,C,N,dtype", [([45, 3], 2104, 16, "bf16"), ([33], 4160, 16, "fp16"), ([40, 31], 2056, 7, "bf16"), ([35], 4100, 8, "fp32"),
                                            ([37], 4104, 64, "bf16"), ([40, 9], 1032, 16, "bf16"), ([70], 4096, 30, "bf16"), ([33], 4104, 50, "fp32"), ([34], 1500, 16, "fp32")])
def test_scan_of_wide_layers(lens, C, N, dtype):
    p = ssm_inputs("cuda", lens, C, N, TYPES[dtype], tail=3)
    out, state = run_ssm(p, "cuda")
    check_ssm(out, state, want_ssm(p))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,C,N,dtype", [([70], 4600, 16, "bf16"), ([131], 4744, 16, "fp16"), ([65], 5919, 13, "fp32"), ([64], 5928, 16, "bf16"), ([130], 7101, 10, "fp32"),
                                            ([33, 0, 66], 2760, 16, "bf16"), ([129], 7112, 16, "bf16"), ([1, 67], 4140, 16, "fp16"), ([66], 8288, 9, "fp16"),
                                            ([40], 8280, 16, "fp32"), ([129], 1192, 64, "fp32"), ([70], 1775, 50, "fp32"), ([66], 1400, 64, "bf16"),
                                            ([70], 1185, 16, "bf16"), ([97], 2368, 16, "fp32")])
def test_scan_where_wider_blocks_fill_the_sms(lens, C, N, dtype):
    """Channel counts on both sides of the launcher's choices of five, six and seven scanning warps; tiles of 64 tokens that end inside."""
    p = ssm_inputs("cuda", lens, C, N, TYPES[dtype], tail=2, seed=C)
    out, state = run_ssm(p, "cuda")
    check_ssm(out, state, want_ssm(p))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[3, 0, 40, 40, 1, 33, 0, 66], [5] * 16, [20, 1] * 8, [7] * 17])
def test_scan_of_sequences_in_order_of_length(lens):
    """Equal and empty ones among them; one more than are ordered."""
    p = ssm_inputs("cuda", lens, 2560, 16, torch.bfloat16, tail=3, seed=len(lens))
    out, state = run_ssm(p, "cuda")
    check_ssm(out, state, want_ssm(p))


@pytest.mark.gpu
@pytest.mark.parametrize("C,N,dtype,bc,dt_type", [(8288, 16, "bf16", None, torch.float32), (8280, 12, "fp16", torch.float32, torch.float32), (5928, 16, "bf16", torch.float32, None),
                                                  (7100, 16, "fp32", torch.bfloat16, None), (4744, 16, "fp32", None, torch.float16), (2400, 16, "bf16", torch.float32, torch.float32),
                                                  (1300, 64, "fp32", torch.bfloat16, None), (2000, 16, "fp16", torch.float32, None)])
def test_scan_of_mixed_types_in_every_width(C, N, dtype, bc, dt_type):
    p = ssm_inputs("cuda", [67], C, N, TYPES[dtype], tail=1, seed=C, bc=bc, dt_type=dt_type)
    out, state = run_ssm(p, "cuda")
    check_ssm(out, state, want_ssm(p))


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,N", [(80, 4100, 16), (300, 2048, 16), (70, 1000, 64), (90, 600, 128)])
def test_scan_of_a_large_decode_batch(B, C, N):
    p = ssm_inputs("cuda", [B], C, N, torch.bfloat16, seed=4)
    state = gen(8, "cuda")(B + 2, C, N)
    rows = torch.randperm(B + 2, generator=torch.Generator().manual_seed(2))[:B]
    rows[3], rows[B - 1] = -1, -1
    want = ssm_oracle(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], p["D"], p["z"], p["dt_bias"], True, state, [(i, 1, r, False) for i, r in enumerate(rows.tolist())])
    out = ops.ssm_step(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], state=state, rows=rows.to("cuda"), D=p["D"], z=p["z"], dt_bias=p["dt_bias"], dt_softplus=True)
    check_ssm(out, state, want)


# ----------------------------------------------------------------------------------------------------------- attention with sinks
ATTENTION_CASES = [
    # contexts, query heads, KV heads, head size, block, window, sinks
    ([1], 1, 1, 64, 16, 1, 1), ([0, 1, 2, 5], 4, 2, 64, 16, 2, 1), ([40, 7, 300, 64], 8, 2, 128, 16, 33, 4), ([90, 17], 9, 1, 128, 16, 64, 3),
    ([200, 15, 16], 6, 6, 256, 64, 100, 65), ([130], 24, 4, 256, 16, 17, 40), ([77, 500], 16, 1, 64, 24, 48, 5), ([333], 20, 1, 128, 32, 200, 1),
    ([64, 65, 66], 32, 4, 128, 7, 31, 31), ([1200], 4, 4, 64, 128, 1000, 190), ([50, 33], 12, 1, 256, 16, 1, 1), ([31], 5, 1, 64, 1, 10, 100),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ctx,Hq,Hkv,D,bs,window,sinks", ATTENTION_CASES)
def test_attention_with_sinks(device, ctx, Hq, Hkv, D, bs, window, sinks):
    """What the new token may not see is NaN: pages between the sinks and the window, slots behind the context, blocks of no sequence."""
    a = attention_inputs(device, ctx, Hq, Hkv, D, bs)
    seen = torch.zeros(a[1].shape[0], dtype=torch.bool)
    for b, n in enumerate(ctx):
        for p in range(n):
            if p < sinks or p >= n - window:
                seen[int(a[3][b, p // bs]) * bs + p % bs] = True
    a[1][~seen.to(device)] = float("nan")
    a[2][~seen.to(device)] = float("nan")
    got = run_attention(a, ctx, Hq, Hkv, D, bs, window, sinks, device)
    check_attention(got, attention_oracle(a[0], a[4], a[5], a[3], ctx, Hkv, bs, D ** -0.5, window, sinks))
    for b, n in enumerate(ctx):
        assert n or not got[b].any()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp8", "int8", "fp4", "int4"])
@pytest.mark.parametrize("ctx,Hq,Hkv,D,bs,window,sinks", [([40, 7, 300], 8, 2, 128, 16, 65, 4), ([90, 17], 9, 1, 64, 16, 64, 3), ([200, 15], 6, 2, 256, 64, 101, 33),
                                                          ([150, 1], 20, 2, 256, 16, 77, 5), ([64, 190], 4, 2, 64, 24, 100, 9), ([99], 16, 1, 128, 16, 50, 2)])
def test_attention_with_sinks_over_quantized_pools(fmt, ctx, Hq, Hkv, D, bs, window, sinks):
    a = attention_inputs("cuda", ctx, Hq, Hkv, D, bs, fmt)
    got = run_attention(a, ctx, Hq, Hkv, D, bs, window, sinks, "cuda")
    check_attention(got, attention_oracle(a[0], a[4], a[5], a[3], ctx, Hkv, bs, D ** -0.5, window, sinks))


@pytest.mark.parametrize("fmt", ["fp8", "int4"])
def test_attention_with_sinks_over_quantized_pools_on_the_cpu(fmt):
    """The CPU path rounds the de-quantized rows to bf16 first: 2^-8 more on scores and values."""
    ctx, Hq, Hkv, D, bs = [40, 7], 4, 2, 64, 16
    a = attention_inputs("cpu", ctx, Hq, Hkv, D, bs, fmt)
    got = run_attention(a, ctx, Hq, Hkv, D, bs, 20, 3, "cpu").double()
    o, _ = attention_oracle(a[0], a[4], a[5], a[3], ctx, Hkv, bs, D ** -0.5, 20, 3)
    assert float((got - o).abs().max() / o.abs().max()) < 4 * 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,splits", [("bf16", s) for s in range(1, 9)] + [("fp8", 1), ("fp8", 3), ("int4", 5)])
def test_every_split_gives_the_same(fmt, splits):
    ctx, Hq, Hkv, D, bs = [700, 1, 333, 0], 16, 2, 128, 16
    a = attention_inputs("cuda", ctx, Hq, Hkv, D, bs, fmt)
    out = torch.full((4, Hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    k, v = (a[1], a[2]) if fmt == "bf16" else (a[1].data, a[2].data)
    ks, vs = (None, None) if fmt == "bf16" else (a[1].scale, a[2].scale)
    torch.ops.mmb200.sink_decode(a[0], k, v, ks, vs, a[3].cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), out, Hq, Hkv, D, bs, D ** -0.5, 500, 20,
                                 -1 if fmt == "bf16" else a[1].fmt_code, splits)
    check_attention(out, attention_oracle(a[0], a[4], a[5], a[3], ctx, Hkv, bs, D ** -0.5, 500, 20))


@pytest.mark.gpu
def test_value_scales_that_grow_along_the_sequence():
    """Rows of one cache differ by many powers of two: small rows in front, large ones behind, and the other way round."""
    Hq, Hkv, D, bs, n = 8, 1, 128, 16, 200
    for flip in (False, True):
        rn = gen(5, "cuda")
        mag = torch.logspace(-3, 3, n, device="cuda")[:, None, None]
        mag = mag.flip(0) if flip else mag
        pools, exact = [], []
        for m in (torch.ones_like(mag), mag):
            pool = ops.FP8KV(208, (Hkv, D), "cuda", "fp8")
            pool.store(torch.arange(n, device="cuda"), rn(n, Hkv, D) * m)
            pools.append(pool)
            exact.append((pool._decode(pool.data).double() * pool.scale.double()[..., None]).cpu())
        q = rn(1, Hq, D).to(torch.bfloat16)
        tables = torch.arange(13, dtype=torch.int32)[None]
        got = run_attention((q, pools[0], pools[1], tables), [n], Hq, Hkv, D, bs, 150, 8, "cuda")
        check_attention(got, attention_oracle(q, exact[0], exact[1], tables, [n], Hkv, bs, D ** -0.5, 150, 8))


@pytest.mark.gpu
def test_attention_with_sharp_and_flat_scores():
    """Scores of hundreds (one key takes all), a zero and a negative scale."""
    ctx, Hq, Hkv, D, bs = [300, 222], 8, 2, 128, 16
    a = attention_inputs("cuda", ctx, Hq, Hkv, D, bs, sharp=30.0)
    for scale in (D ** -0.5, 0.0, -0.1):
        got = run_attention(a, ctx, Hq, Hkv, D, bs, 150, 4, "cuda", scale=scale)
        check_attention(got, attention_oracle(a[0], a[4], a[5], a[3], ctx, Hkv, bs, scale, 150, 4))


def test_refusals_of_attention_with_sinks():
    from metal_marlin_b200 import _build
    ctx, Hq, Hkv, D, bs = [40, 7], 4, 2, 64, 16
    a = attention_inputs("cpu", ctx, Hq, Hkv, D, bs)
    base = dict(Hq=Hq, Hkv=Hkv, dqk=D, dv=D, block_size=bs, scale=0.1, window=8, sinks=2)
    lens = torch.tensor(ctx, dtype=torch.int32)
    for change in (dict(sinks=-1), dict(window=-4), dict(dqk=32), dict(dqk=32, dv=32), dict(Hkv=3), dict(w_uv=torch.zeros(4, 8, 64))):
        with pytest.raises(ValueError):
            ops.paged_attention(a[0], a[1], a[2], a[3], lens, **dict(base, **change))
    with pytest.raises(ValueError):
        ops.paged_attention(a[0], a[1], None, a[3], lens, **base)
    with pytest.raises(ValueError):
        ops.paged_attention(a[0], ops.FP8KV(64, (2, 64), "cpu", "fp8"), ops.FP8KV(64, (2, 64), "cpu", "int8"), a[3], lens, **base)
    # without a window everything is visible and sinks change nothing
    got = ops.paged_attention(a[0], a[1], a[2], a[3], lens, **dict(base, window=0))
    assert torch.equal(got, ops.paged_attention(a[0], a[1], a[2], a[3], lens, **dict(base, window=0, sinks=0)))
    if not _build.load():
        return
    out = torch.empty_like(a[0])
    call = dict(q=a[0], k=a[1], v=a[2], ks=None, vs=None, tables=a[3], ctx=lens, out=out, Hq=Hq, Hkv=Hkv, D=D, bs=bs, scale=0.1, window=8, sinks=2, fmt=-1, splits=0)
    odd = torch.zeros(out.numel() + 1, dtype=torch.bfloat16)[1:].view(2, 4, 64)
    for change in (dict(window=0), dict(window=2 ** 31), dict(sinks=-1), dict(D=32), dict(Hkv=3), dict(Hkv=0), dict(bs=0), dict(splits=9), dict(q=a[0].float()), dict(q=a[0][:1]),
                   dict(out=out.float()), dict(out=odd), dict(q=odd), dict(tables=a[3].long()), dict(tables=a[3][:1]), dict(ctx=lens.long()), dict(fmt=0), dict(fmt=5),
                   dict(k=a[1][:16]), dict(k=a[1].float(), v=a[2].float()), dict(k=a[1].view(torch.uint8)[..., :64].contiguous(), v=a[2].view(torch.uint8)[..., :64].contiguous(), fmt=0)):
        with pytest.raises(ValueError):
            torch.ops.mmb200.sink_decode(*dict(call, **change).values())


@pytest.mark.gpu
def test_blocks_and_rows_outside_the_pools_are_hidden_and_reported():
    """A bad table entry inside the context hides its tokens; a pool row that does not exist skips its sequence.  Both are reported."""
    dev = torch.device("cuda")
    ctx, Hq, Hkv, D, bs = [48], 4, 2, 64, 16
    a = attention_inputs("cuda", ctx, Hq, Hkv, D, bs)
    ops.clear_status(dev)
    tables = a[3].clone()
    tables[0, 1] = 10 ** 6
    got = run_attention((*a[:3], tables), ctx, Hq, Hkv, D, bs, 40, 2, "cuda")
    assert ops.check_status(dev) == 131
    ops.clear_status(dev)
    run_attention((*a[:3], a[3][:, :2].contiguous()), ctx, Hq, Hkv, D, bs, 40, 2, "cuda")            # 48 tokens, a table for 32
    assert ops.check_status(dev) == 131
    ops.clear_status(dev)
    pos = [p for p in range(48) if (p < 2 or p >= 8) and p // bs != 1]
    slots = torch.tensor([int(a[3][0, p // bs]) * bs + p % bs for p in pos])
    q = a[0][0].double().cpu().view(Hkv, 2, D)
    p = torch.softmax(torch.einsum("hgd,thd->hgt", q, a[4][slots]) * D ** -0.5, -1)
    want = torch.einsum("hgt,thd->hgd", p, a[5][slots]).reshape(1, Hq, D)
    assert float((got.double().cpu() - want).abs().max()) < 2.0 ** -8 * float(want.abs().max()) + 1e-4
    s = ssm_inputs("cuda", [5, 6], 8, 16, torch.bfloat16)
    s["rows"] = torch.tensor([1, 99])
    out, state = run_ssm(s, "cuda")
    assert ops.check_status(dev) == 130
    ops.clear_status(dev)
    check_ssm(out, state, want_ssm(s))
    assert not out[5:].any()


# ----------------------------------------------------------------------------------------------- streams, graphs, sizes (GPU only)
@pytest.mark.gpu
def test_other_streams_and_captured_graphs():
    """Two graphs over the same pools, replayed in turn, and a side stream, give what the same calls give one after the other."""
    dev = "cuda"
    p = ssm_inputs(dev, [4], 64, 16, torch.bfloat16, seed=3)
    x, w, b, cstate, _, _, _ = conv_inputs(dev, [4], 64, 4, torch.bfloat16, seed=4)
    ctx, Hq, Hkv, D, bs = [900, 30, 411, 65], 8, 2, 128, 16
    a = attention_inputs(dev, ctx, Hq, Hkv, D, bs)
    tables, lens = a[3].to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev)
    rows = [torch.tensor([0, 1, 2, -1], device=dev), torch.tensor([3, -1, 1, 0], device=dev)]

    def step(cs, ss, r):
        y = ops.causal_conv_step(x, w, b, state=cs, rows=r)
        h = ops.ssm_step(y, p["dt"], p["A"], p["Bm"], p["Cm"], state=ss, rows=r, D=p["D"], z=p["z"], dt_bias=p["dt_bias"], dt_softplus=True)
        o = ops.paged_attention(a[0], a[1], a[2], tables, lens, Hq=Hq, Hkv=Hkv, dqk=D, dv=D, block_size=bs, scale=D ** -0.5, window=256, sinks=4)
        return h, o

    pools = lambda: (gen(1, dev)(5, 64, 3), gen(2, dev)(5, 64, 16))
    cs, ss = pools()
    want = [tuple(t.clone() for t in step(cs, ss, rows[i % 2])) for i in range(4)]
    want_pools = (cs, ss)
    cs, ss = pools()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(cs, ss, rows[i % 2]) for i in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for g, h in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(g, h))
    assert torch.equal(cs, want_pools[0]) and torch.equal(ss, want_pools[1])
    cs, ss = pools()
    keep = cs.clone(), ss.clone()
    graphs, outs = [], []
    for r in rows:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(cs, ss, r))
        graphs.append(g)
    cs.copy_(keep[0])
    ss.copy_(keep[1])
    for i in range(4):
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(outs[i % 2], want[i]))
    assert torch.equal(cs, want_pools[0]) and torch.equal(ss, want_pools[1])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pools of more than 2^31 values, the rows in use at their far end."""
    dev = "cuda"
    D, Hkv, bs = 128, 8, 16
    blocks = (2 ** 31) // (Hkv * D * bs) + 40
    k, v = (torch.empty(blocks * bs, Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    rn = gen(0, dev)
    ctx = [100]
    tables = torch.tensor([[blocks - 1, 0, blocks - 3, blocks - 7, blocks - 2, blocks - 9, 5]], dtype=torch.int32)
    for blk in tables[0].tolist():
        k[blk * bs: (blk + 1) * bs] = rn(bs, Hkv, D).to(torch.bfloat16)
        v[blk * bs: (blk + 1) * bs] = rn(bs, Hkv, D).to(torch.bfloat16)
    q = rn(1, 16, D).to(torch.bfloat16)
    got = run_attention((q, k, v, tables), ctx, 16, Hkv, D, bs, 80, 4, dev)
    near = torch.arange(7, dtype=torch.int32)[None]
    sel = torch.cat([torch.arange(b * bs, (b + 1) * bs) for b in tables[0].tolist()]).to(dev)
    check_attention(got, attention_oracle(q, k[sel].double().cpu(), v[sel].double().cpu(), near, ctx, Hkv, bs, D ** -0.5, 80, 4))
    del k, v
    C, N = 8192, 128
    pool = torch.empty(2 ** 31 // (C * N) + 4, C, N, device=dev)
    last = pool.shape[0] - 1
    p = ssm_inputs(dev, [2], C, N, torch.bfloat16)
    pool[last] = 0.5
    small = pool[last:].clone()
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    call = lambda st, r: ops.ssm_scan(p["x"], p["dt"], p["A"], p["Bm"], p["Cm"], cu_seqlens=cu, state=st, rows=torch.tensor([r], device=dev), dt_bias=p["dt_bias"], dt_softplus=True)
    assert torch.equal(call(pool, last), call(small, 0)) and torch.equal(pool[last], small[0])
    one = lambda st, r: ops.ssm_step(p["x"][:1], p["dt"][:1], p["A"], p["Bm"][:1], p["Cm"][:1], state=st, rows=torch.tensor([r], device=dev), dt_bias=p["dt_bias"], dt_softplus=True)
    assert torch.equal(one(pool, last), one(small, 0)) and torch.equal(pool[last], small[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_unaligned_and_strided_inputs_give_the_same(dtype):
    """Slices that start inside a vector of the fast path against contiguous copies."""
    dev, t = "cuda", TYPES[dtype]
    p = ssm_inputs(dev, [50, 30], 64, 16, t, seed=1)
    out, state = run_ssm(p, dev)
    off = dict(p)
    for name in ("x", "z", "dt", "Bm", "Cm"):
        wide = torch.zeros(p[name].shape[0], p[name].shape[1] + 3, dtype=t, device=dev)
        wide[:, 1:-2] = p[name]
        off[name] = wide[:, 1:-2]
    into = torch.zeros(80, 67, dtype=t, device=dev)
    out2, state2 = run_ssm(off, dev, out=into[:, 1:65])
    assert torch.equal(out, out2) and torch.equal(state, state2)
    x, w, b, cs, rows, fresh, cu = conv_inputs(dev, [50, 30], 64, 4, t)
    wide = torch.zeros(80, 67, dtype=t, device=dev)
    wide[:, 3:] = x
    cu, c2 = torch.tensor(cu, dtype=torch.int32, device=dev), cs.clone()
    y = ops.causal_conv(x, w, b, cu_seqlens=cu, state=cs, rows=rows.to(dev), fresh=fresh.to(dev))
    y2 = ops.causal_conv(wide[:, 3:], w, b, cu_seqlens=cu, state=c2, rows=rows.to(dev), fresh=fresh.to(dev))
    assert torch.equal(y, y2) and torch.equal(cs, c2)


# ----------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("device", DEVICES)
def test_a_stream_through_all_of_them(device):
    """A prompt in two chunks, then tokens: convolution, scan and windowed attention with sinks of one layer stack, the state carried in
    pools and pages, against one pass over the whole sequence in 64 bits."""
    C, N, Hq, Hkv, D, bs, window, sinks, T = 64, 16, 2, 1, 64, 16, 24, 3, 60
    rn = gen(11, device)
    x, w, b, _, _, _, _ = conv_inputs(device, [T], C, 4, torch.bfloat16, seed=12)
    p = ssm_inputs(device, [T], C, N, torch.bfloat16, seed=13)
    cpool, spool = torch.full((3, C, 3), float("nan"), device=device), torch.full((3, C, N), float("nan"), device=device)
    row = torch.tensor([2], device=device)
    k, v, q = (rn(T, 1, D).to(torch.bfloat16) for _ in range(3))
    q = torch.cat([q, q.flip(0)], 1)
    kp, vp = (torch.full((5 * bs, 1, D), float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2))
    table = torch.tensor([[3, 0, 4, 1]], dtype=torch.int32, device=device)
    ys, hs, os_ = [], [], []

    def args(lo, hi):
        return p["dt"][lo:hi], p["A"], p["Bm"][lo:hi], p["Cm"][lo:hi]

    for lo, hi in [(0, 7), (7, 40)] + [(t, t + 1) for t in range(40, T)]:
        for t in range(lo, hi):
            slot = int(table[0, t // bs]) * bs + t % bs
            kp[slot], vp[slot] = k[t], v[t]
        if hi - lo > 1:
            cu, fresh = torch.tensor([0, hi - lo], dtype=torch.int32, device=device), torch.tensor([lo == 0], device=device)
            y = ops.causal_conv(x[lo:hi], w, b, cu_seqlens=cu, state=cpool, rows=row, fresh=fresh, out_dtype=torch.float32)
            h = ops.ssm_scan(y, *args(lo, hi), cu_seqlens=cu, state=spool, rows=row, fresh=fresh, D=p["D"], z=p["z"][lo:hi], dt_bias=p["dt_bias"], dt_softplus=True)
        else:
            y = ops.causal_conv_step(x[lo:hi], w, b, state=cpool, rows=row, out_dtype=torch.float32)
            h = ops.ssm_step(y, *args(lo, hi), state=spool, rows=row, D=p["D"], z=p["z"][lo:hi], dt_bias=p["dt_bias"], dt_softplus=True)
            os_.append(ops.paged_attention(q[lo:hi], kp, vp, table, torch.tensor([hi], dtype=torch.int32, device=device), Hq=Hq, Hkv=Hkv, dqk=D, dv=D, block_size=bs,
                                           scale=D ** -0.5, window=window, sinks=sinks))
        ys.append(y)
        hs.append(h)
    y = torch.cat(ys)
    check_conv(y, cpool[2:], *conv_oracle(x, w, b, torch.zeros(1, C, 3), [(0, T, 0, True)], 1))
    want = ssm_oracle(y, p["dt"], p["A"], p["Bm"], p["Cm"], p["D"], p["z"], p["dt_bias"], True, torch.zeros(1, C, N), [(0, T, 0, True)])
    check_ssm(torch.cat(hs), spool[2:], want)
    assert torch.isnan(cpool[:2]).all() and torch.isnan(spool[:2]).all()
    order = torch.cat([torch.arange(int(i) * bs, int(i) * bs + bs) for i in table[0]])
    for t, o in zip(range(40, T), os_):
        check_attention(o, attention_oracle(q[t: t + 1], kp.double().cpu()[order], vp.double().cpu()[order], torch.arange(4)[None], [t + 1], Hkv, bs, D ** -0.5, window, sinks))


def test_refusals_of_calls_that_are_too_large_or_write_a_row_twice():
    """Expanded tensors: nothing of that size is allocated."""
    from metal_marlin_b200 import _build
    native = _build.load()
    x, w = torch.zeros(1, 4).expand(65536, 4), torch.zeros(4, 2)
    state = torch.zeros(1, 4, 1)
    rows = torch.full((65536,), -1)
    with pytest.raises(ValueError):
        ops.causal_conv_step(x, w, state=state, rows=rows)
    A, bc = torch.zeros(4, 3), torch.zeros(1, 3).expand(65536, 3)
    with pytest.raises(ValueError):
        ops.ssm_step(x, x, A, bc, bc, state=torch.zeros(1, 4, 3), rows=rows)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.causal_conv(x[:5].clone(), w, cu_seqlens=cu, out=torch.zeros(1, 4).expand(5, 4))
    wide = torch.zeros(8)
    with pytest.raises(ValueError):
        ops.causal_conv(x[:5].clone(), w, cu_seqlens=cu, out=wide.as_strided((5, 4), (1, 1)))
    pool, q = torch.zeros(16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    base = dict(Hq=1, Hkv=1, dqk=64, dv=64, scale=1.0, window=8, sinks=2)
    lens = torch.zeros(1, dtype=torch.int32)
    for bs, n in ((2 ** 30, 2), (2 ** 31 - 1, 1), (16, 2 ** 26 + 1)):
        tables = torch.zeros(1, n, dtype=torch.int32) if n < 100 else torch.zeros(1, 1, dtype=torch.int32).expand(1, n)
        with pytest.raises(ValueError):
            ops.paged_attention(q, pool, pool, tables, lens, block_size=bs, **base)
        if native and n < 100:
            with pytest.raises(ValueError):
                torch.ops.mmb200.sink_decode(q, pool, pool, None, None, tables, lens, q.clone(), 1, 1, 64, bs, 1.0, 8, 2, -1, 0)
    many = torch.zeros(65536, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention(q.expand(65536, 1, 64), pool, pool, torch.zeros(65536, 1, dtype=torch.int32), many, block_size=16, **base)
    if native:
        with pytest.raises(ValueError):
            torch.ops.mmb200.causal_conv(x, w, None, torch.empty(65536, 4), state, rows, None, None, 1, True)
        with pytest.raises(ValueError):
            torch.ops.mmb200.sink_decode(q.expand(65536, 1, 64).contiguous(), pool, pool, None, None, torch.zeros(65536, 1, dtype=torch.int32), many,
                                         torch.empty(65536, 1, 64, dtype=torch.bfloat16), 1, 1, 64, 16, 1.0, 8, 2, -1, 0)
