"""What is measured of the operators that keep a sequence going at constant cost per token: the short causal convolution over a pool
of per-sequence windows, the selective state space scan over a pool of states, and attention of one new token over a paged cache
with a sliding window and sinks.  ``run`` computes each in elementary torch operations, or, where ``own`` is set, through the
framework's entry points; ``exact`` gives the values of the definitions in 64 bits."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
RANGE = {"fp8": 448.0, "int8": 127.0}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request of a small hybrid model decodes a token: nothing but latency
        {"name": "conv step, 1 row", "op": "conv_step", "rows": 1, "dead": 0, "channels": 512, "taps": 4, "dtype": "bf16", "bias": True},
        # a full decode batch, bucketed (padding rows behind the live ones), of a wide linear-attention mixer
        {"name": "conv step, 256 rows", "op": "conv_step", "rows": 256, "dead": 19, "channels": 10240, "taps": 4, "dtype": "bf16", "bias": False},
        # a prefill batch of ragged prompts, half of them continued chunks, convolution in front of a linear-attention mixer
        {"name": "conv prompts, ragged", "op": "conv", "tokens": 8111, "seqs": 9, "tail": 81, "channels": 10240, "taps": 4, "dtype": "bf16", "bias": False},
        # one request of a small hybrid model decodes a token
        {"name": "scan step, 1 row", "op": "scan_step", "rows": 1, "dead": 0, "channels": 512, "states": 16, "dtype": "bf16"},
        # a full decode batch of a large hybrid model, bucketed
        {"name": "scan step, 256 rows", "op": "scan_step", "rows": 256, "dead": 19, "channels": 8192, "states": 16, "dtype": "bf16"},
        # one long prompt of a large hybrid model
        {"name": "scan prompt, 4096", "op": "scan", "tokens": 4096, "seqs": 1, "tail": 0, "channels": 8192, "states": 16, "dtype": "bf16"},
        # a prefill batch of ragged prompts and continued chunks, padded behind the last one
        {"name": "scan prompts, ragged", "op": "scan", "tokens": 5003, "seqs": 11, "tail": 117, "channels": 4096, "states": 16, "dtype": "fp16"},
        # one prompt of a small model with a large state, in 32 bits
        {"name": "scan prompt, 64 states", "op": "scan", "tokens": 1531, "seqs": 1, "tail": 0, "channels": 1536, "states": 64, "dtype": "fp32"},
        # one chat request, its context still shorter than the window
        {"name": "window decode, 1 row", "op": "attention", "rows": 1, "longest": 701, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 4096,
         "sinks": 4, "block": 16, "kv": "bf16"},
        # a decode batch of streams far past their window
        {"name": "window decode, 64 rows", "op": "attention", "rows": 64, "longest": 12345, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 4096,
         "sinks": 4, "block": 16, "kv": "bf16"},
        # long streams of a hybrid model with wide heads over an 8-bit cache
        {"name": "window decode, 8-bit cache", "op": "attention", "rows": 16, "longest": 50021, "heads": 24, "kv_heads": 4, "head_dim": 256, "window": 8192,
         "sinks": 64, "block": 64, "kv": "fp8"},
        # many short-window layers of a small model: an odd window whose ends lie inside pages
        {"name": "window decode, small heads", "op": "attention", "rows": 33, "longest": 1999, "heads": 4, "kv_heads": 2, "head_dim": 64, "window": 509,
         "sinks": 3, "block": 16, "kv": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_step", "conv", "scan_step", "scan", "scan", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "conv_step":
        rows = _log(rng, 1, 256)
        return {"op": op, "rows": rows, "dead": rng.randrange(rows), "channels": _log(rng, 64, 10240), "taps": rng.choice([2, 3, 4, 4, 5, 8]), "dtype": dtype,
                "bias": rng.random() < 0.5}
    if op == "conv":
        channels = _log(rng, 64, 10240)
        tokens = _log(rng, 1, min(16384, 83000000 // channels))
        return {"op": op, "tokens": tokens, "seqs": rng.randint(1, min(16, tokens)), "tail": rng.choice([0, 0, rng.randint(1, 64)]), "channels": channels,
                "taps": rng.choice([2, 3, 4, 4, 5, 8]), "dtype": dtype, "bias": rng.random() < 0.5}
    if op == "scan_step":
        rows = _log(rng, 1, 256)
        return {"op": op, "rows": rows, "dead": rng.randrange(rows), "channels": _log(rng, 64, 8192), "states": rng.choice([8, 16, 16]), "dtype": dtype}
    if op == "scan":
        states = rng.choice([8, 16, 16, 16, 24, 64, 128])
        channels = _log(rng, 64, 8192)
        tokens = _log(rng, 1, min(8192, 500000000 // (channels * states)))
        return {"op": op, "tokens": tokens, "seqs": rng.randint(1, min(16, tokens)), "tail": rng.choice([0, 0, rng.randint(1, 64)]), "channels": channels,
                "states": states, "dtype": dtype}
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    rows = _log(rng, 1, 64)
    longest = _log(rng, 1, min(60000, 6000000000 // (rows * kv_heads * head_dim * 4)))
    window = _log(rng, 1, 8192)
    return {"op": op, "rows": rows, "longest": longest, "heads": kv_heads * rng.randint(1, 16), "kv_heads": kv_heads, "head_dim": head_dim,
            "window": min(window, 33000000 // (rows * kv_heads * head_dim // 8)), "sinks": _log(rng, 1, 128), "block": rng.choice([16, 16, 32, 64]),
            "kv": rng.choice(["bf16", "bf16", "fp8", "int8"])}


def _lengths(case):
    """Lengths of the prompts of a ragged batch: spread over the logarithm, one of them empty where there are many."""
    rng = random.Random(case["tokens"] * 131 + case["seqs"])
    n = case["seqs"]
    weights = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(n)]
    if n >= 6:
        weights[n // 2] = 0.0
    total = sum(weights)
    ends = [int(round(sum(weights[: i + 1]) / total * case["tokens"])) for i in range(n)]
    ends[-1] = case["tokens"]
    return [e - s for s, e in zip([0] + ends[:-1], ends)]


def _contexts(case):
    """Tokens in the cache of each sequence of a decode batch, the longest first."""
    rng = random.Random(case["longest"] * 257 + case["rows"])
    return [case["longest"]] + [rng.randint(max(1, case["longest"] // 3), case["longest"]) for _ in range(case["rows"] - 1)]


def _visible(case):
    return [min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in _contexts(case)]


# --------------------------------------------------------------------------------------------------------------- inputs
def _made(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device="cuda")


def _rows_of_pool(seed, count, dead, pool):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randperm(pool, generator=g)[:count]
    if dead:
        rows[count - dead:] = -1
    return rows.to("cuda")


def prepare(case, seed):
    rn = _made(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "attention":
        return _prepare_attention(case, seed, rn, s)
    dtype, C = DTYPES[case["dtype"]], case["channels"]
    if op in ("conv", "scan"):
        lens = _lengths(case)
        ends = torch.tensor([0] + lens).cumsum(0)
        rows_in, live = case["tokens"] + case["tail"], case["seqs"]
        s["cu_seqlens"] = ends.to(torch.int32).to("cuda")
        s["fresh"] = (torch.arange(live) % 2 == 0).to("cuda")
        s["rows"] = _rows_of_pool(seed, live, 0, live + 5)
        pool = live + 5
    else:
        rows_in, pool = case["rows"], case["rows"] + 3
        s["rows"] = _rows_of_pool(seed, rows_in, case["dead"], pool)
    if op in ("conv", "conv_step"):
        s["x"] = rn(rows_in, C).to(dtype)
        s["w"] = (rn(C, case["taps"]) * case["taps"] ** -0.5).to(dtype)
        s["bias"] = (rn(C) * 0.1).to(dtype) if case["bias"] else None
        s["state"] = rn(pool, C, case["taps"] - 1)
        return s
    N = case["states"]
    xz = rn(rows_in, 2 * C).to(dtype)                       # the in-projection gives both halves side by side
    s["x"], s["z"] = xz[:, :C], xz[:, C:]
    step = torch.exp(math.log(1e-3) + torch.sigmoid(rn(C) * 1.5) * math.log(100.0))         # time steps from 0.001 to 0.1
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["dt"] = (rn(rows_in, C) * 0.5).to(dtype)
    s["A"] = -torch.arange(1, N + 1, device="cuda").float() * torch.exp(rn(C, N) * 0.1)
    bc = rn(rows_in, 2 * N).to(dtype)
    s["B"], s["C"] = bc[:, :N], bc[:, N:]
    s["D"] = rn(C)
    s["state"] = rn(pool, C, N) * 0.1
    return s


def _prepare_attention(case, seed, rn, s):
    Hk, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    ctx = _contexts(case)
    need = [(n + bs - 1) // bs for n in ctx]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need), generator=g).to(torch.int32)
    tables = torch.full((case["rows"], max(need)), 0, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at: at + n]
        at += n
    s["tables"], s["ctx"] = tables.to("cuda"), torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["q"] = rn(case["rows"], case["heads"], D).to(torch.bfloat16)
    slots = sum(need) * bs
    if case["kv"] == "bf16":
        s["k"], s["v"] = rn(slots, Hk, D).to(torch.bfloat16), rn(slots, Hk, D).to(torch.bfloat16)
        return s
    for name in ("k", "v"):
        codes = torch.empty(slots, Hk, D, dtype=torch.uint8, device="cuda")
        scales = torch.empty(slots, Hk, device="cuda")
        for lo in range(0, slots, 65536):
            hi = min(slots, lo + 65536)
            x = rn(hi - lo, Hk, D)
            scale = x.abs().amax(-1) / RANGE[case["kv"]]
            x = x / scale[..., None]
            codes[lo:hi] = x.to(torch.float8_e4m3fn).view(torch.uint8) if case["kv"] == "fp8" else x.round().to(torch.int8).view(torch.uint8)
            scales[lo:hi] = scale
        s[name + "_codes"], s[name + "_scale"] = codes, scales
        if own:
            from metal_marlin_b200 import ops
            pool = ops.FP8KV(0, (Hk, D), "cuda", case["kv"])     # the handle of the cache: its codes and row scales
            pool.data, pool.scale = codes, scales
            s[name] = pool
    return s


# ------------------------------------------------------------------------------------------------------------ operators
def run(s):
    op = s["case"]["op"]
    return {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "attention": _attention}[op](s)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _places(cu, total):
    """For every row of a ragged batch: its sequence and its place in it, and whether it belongs to one at all."""
    t = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    inside = seq < cu.numel() - 1
    seq = seq.clamp(max=cu.numel() - 2)
    return seq, t - cu.long()[seq], inside


def _conv(s):
    if own:
        from metal_marlin_b200 import ops
        out = ops.causal_conv(s["x"], s["w"], s["bias"], cu_seqlens=s["cu_seqlens"], state=s["state"], rows=s["rows"], fresh=s["fresh"])
        return out, s["state"]
    x, w, cu, state, rows = s["x"].float(), s["w"].float(), s["cu_seqlens"].long(), s["state"], s["rows"]
    T, K, S = x.shape[0], w.shape[1], rows.numel()
    old = state[rows].transpose(1, 2) * (~s["fresh"])[:, None, None]                       # [S, K - 1, C]
    seq, _, inside = _places(cu, T)
    lens, pads = cu[1:] - cu[:-1], torch.arange(S, device=x.device) * (K - 1)
    line = torch.zeros(T + S * (K - 1), x.shape[1], device=x.device)                       # every sequence behind its window
    head = (cu[:-1] + pads)[:, None] + torch.arange(K - 1, device=x.device)
    line[head] = old
    place = torch.arange(T, device=x.device) + (seq + 1) * (K - 1)
    line[place] = x
    near = place[:, None] + torch.arange(1 - K, 1, device=x.device)                        # the K inputs that a row sees
    y = (line[near] * w.t()).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = torch.where(inside[:, None], _silu(y), torch.zeros_like(y))
    last = (cu[1:] + pads)[:, None] + torch.arange(K - 1, device=x.device)
    new = line[last].transpose(1, 2)
    state[rows] = torch.where((lens > 0)[:, None, None], new, state[rows])
    return y.to(s["x"].dtype), state


def _conv_step(s):
    if own:
        from metal_marlin_b200 import ops
        out = ops.causal_conv_step(s["x"], s["w"], s["bias"], state=s["state"], rows=s["rows"])
        return out, s["state"]
    live = s["case"]["rows"] - s["case"]["dead"]
    rows, state, out = s["rows"][:live], s["state"], torch.zeros_like(s["x"])
    seen = torch.cat([state[rows], s["x"][:live].float()[..., None]], -1)                  # [B, C, K]
    y = (seen * s["w"].float()).sum(-1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out[:live] = _silu(y).to(out.dtype)
    state[rows] = seen[..., 1:]
    return out, state


def _all_states(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, by doubling."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _scan(s):
    if own:
        from metal_marlin_b200 import ops
        out = ops.ssm_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], cu_seqlens=s["cu_seqlens"], state=s["state"], rows=s["rows"], fresh=s["fresh"], D=s["D"],
                           z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
        return out, s["state"]
    tokens, cu, state, rows = s["case"]["tokens"], s["cu_seqlens"].long(), s["state"], s["rows"]
    x, z = s["x"][:tokens].float(), s["z"][:tokens].float()
    dt = _softplus(s["dt"][:tokens].float() + s["dt_bias"])
    a = torch.exp(dt[..., None] * s["A"])                                                  # [T, C, N]
    b = (dt * x)[..., None] * s["B"][:tokens].float()[:, None, :]
    seq, place, _ = _places(cu, tokens)
    first = torch.nonzero(place == 0)[:, 0]                                                # rows at which a sequence begins
    b[first] += a[first] * state[rows[seq[first]]] * (~s["fresh"])[seq[first], None, None]
    a[first] = 0
    h = _all_states(a, b)
    y = (h * s["C"][:tokens].float()[:, None, :]).sum(-1) + s["D"] * x
    out = torch.zeros(s["x"].shape, dtype=s["x"].dtype, device=x.device)
    out[:tokens] = (y * _silu(z)).to(out.dtype)
    last = torch.cat([first[1:] - 1, first.new_tensor([tokens - 1])])
    state[rows[seq[last]]] = h[last]
    return out, state


def _scan_step(s):
    if own:
        from metal_marlin_b200 import ops
        out = ops.ssm_step(s["x"], s["dt"], s["A"], s["B"], s["C"], state=s["state"], rows=s["rows"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                           dt_softplus=True)
        return out, s["state"]
    live = s["case"]["rows"] - s["case"]["dead"]
    rows, state = s["rows"][:live], s["state"]
    x, z = s["x"][:live].float(), s["z"][:live].float()
    dt = _softplus(s["dt"][:live].float() + s["dt_bias"])
    h = torch.exp(dt[..., None] * s["A"]) * state[rows] + (dt * x)[..., None] * s["B"][:live].float()[:, None, :]
    y = (h * s["C"][:live].float()[:, None, :]).sum(-1) + s["D"] * x
    out = torch.zeros(s["x"].shape, dtype=s["x"].dtype, device=x.device)
    out[:live] = (y * _silu(z)).to(out.dtype)
    state[rows] = h
    return out, state


def _seen_slots(case, tables, ctx):
    """Cache slots that each sequence's new token sees, as a rectangle, and which of its places hold one."""
    most = max(_visible(case))
    j = torch.arange(most, device=tables.device)
    lo = (ctx.long() - case["window"]).clamp(min=0)[:, None]
    sinks = lo.clamp(max=case["sinks"])
    at = torch.where(j < sinks, j, lo + j - sinks)
    ok = at < ctx.long()[:, None]
    at = torch.where(ok, at, torch.zeros_like(at))
    return tables.long().gather(1, at // case["block"]) * case["block"] + at % case["block"], ok


def _values(s, name, slots, kind):
    """Cached rows of the given slots in a floating type."""
    if s["case"]["kv"] == "bf16":
        return s[name][slots].to(kind)
    codes = s[name + "_codes"][slots]
    codes = codes.view(torch.float8_e4m3fn if s["case"]["kv"] == "fp8" else torch.int8).to(kind)
    return codes * s[name + "_scale"][slots].to(kind)[..., None]


def _attention(s):
    c = s["case"]
    B, H, Hk, D = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    if own:
        from metal_marlin_b200 import ops
        return ops.paged_attention(s["q"], s["k"], s["v"], s["tables"], s["ctx"], Hq=H, Hkv=Hk, dqk=D, dv=D, block_size=c["block"], scale=D ** -0.5,
                                   window=c["window"], sinks=c["sinks"])
    slots, ok = _seen_slots(c, s["tables"], s["ctx"])
    q = s["q"].float().view(B, Hk, H // Hk, D) * D ** -0.5
    score = q @ _values(s, "k", slots, torch.float32).permute(0, 2, 3, 1)                  # [B, Hk, g, M]
    score = torch.where(ok[:, None, None, :], score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p @ _values(s, "v", slots, torch.float32).transpose(1, 2)) / p.sum(-1, keepdim=True)
    return o.reshape(B, H, D).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------- floors
def work(case):
    op = case["op"]
    if op == "attention":
        seen, row = sum(_visible(case)), case["kv_heads"] * case["head_dim"]
        kv = seen * (2 * row * 2 if case["kv"] == "bf16" else 2 * (row + 4 * case["kv_heads"]))
        return {"bytes": kv + 2 * case["rows"] * case["heads"] * case["head_dim"] * 2, "flops": 4 * seen * case["heads"] * case["head_dim"]}
    e, C = BYTES[case["dtype"]], case["channels"]
    tokens = case["tokens"] if op in ("conv", "scan") else case["rows"] - case["dead"]
    live = case["seqs"] if op in ("conv", "scan") else tokens
    kept = (live + 1) // 2 if op in ("conv", "scan") else live                             # states that are read: fresh ones are not
    if op in ("conv", "conv_step"):
        K = case["taps"]
        return {"bytes": 2 * tokens * C * e + C * (K + case["bias"]) * e + (live + kept) * C * (K - 1) * 4, "flops": tokens * C * (2 * K + 4)}
    N = case["states"]
    return {"bytes": tokens * (4 * C + 2 * N) * e + C * (N + 2) * 4 + (live + kept) * C * N * 4, "flops": tokens * C * (7 * N + 14)}


# ----------------------------------------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "conv_step": _exact_conv, "scan": _exact_scan, "scan_step": _exact_scan, "attention": _exact_attention}[case["op"]](case, s)


def _sequences(case, s):
    """(first row, length, row of the pool, starts anew) of every live sequence; a decode step is a batch of one-token prompts."""
    rows = s["rows"].tolist()
    if "cu_seqlens" in s:
        cu, fresh = s["cu_seqlens"].tolist(), s["fresh"].tolist()
        return [(cu[i], cu[i + 1] - cu[i], rows[i], fresh[i]) for i in range(len(rows)) if cu[i + 1] > cu[i]]
    return [(i, 1, r, False) for i, r in enumerate(rows) if r >= 0]


def _exact_conv(case, s):
    x, w, K = s["x"].double(), s["w"].double(), case["taps"]
    state, out = s["state"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    for at, n, row, fresh in _sequences(case, s):
        before = torch.zeros_like(state[row]) if fresh else state[row]
        line = torch.cat([before.t(), x[at: at + n]])
        y = sum(line[k: k + n] * w[:, k] for k in range(K))
        if s["bias"] is not None:
            y = y + s["bias"].double()
        out[at: at + n] = y * torch.sigmoid(y)
        state[row] = line[n:].t()
    return out, state


def _exact_scan(case, s):
    x, z, dt, Bm, Cm = (s[k].double() for k in ("x", "z", "dt", "B", "C"))
    A, D, state = s["A"].double(), s["D"].double(), s["state"].double()
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    delta = torch.logaddexp(dt + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    todo = sorted(_sequences(case, s), key=lambda q: -q[1])                                # the longest first: the live ones stay in front
    at, row = (torch.tensor([q[k] for q in todo], device="cuda") for k in (0, 2))
    h = state[row] * torch.tensor([0.0 if q[3] else 1.0 for q in todo], dtype=torch.float64, device="cuda")[:, None, None]
    for t in range(todo[0][1]):
        n = sum(q[1] > t for q in todo)
        i = at[:n] + t
        d, u = delta[i], x[i]
        h[:n] = torch.exp(d[..., None] * A) * h[:n] + (d * u)[..., None] * Bm[i][:, None, :]
        out[i] = (torch.einsum("bcn,bn->bc", h[:n], Cm[i]) + D * u) * z[i] * torch.sigmoid(z[i])
    state[row] = h
    return out, state


def _exact_attention(case, s):
    Hk, D, bs, g = case["kv_heads"], case["head_dim"], case["block"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_contexts(case)):
        pos = torch.arange(n, device="cuda")
        pos = pos[(pos < case["sinks"]) | (pos >= n - case["window"])]
        slots = s["tables"][b].long()[pos // bs] * bs + pos % bs
        k, v = (_values(s, name, slots, torch.float64) for name in ("k", "v"))
        q = s["q"][b].double().view(Hk, g, D)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(D), -1)
        out[b] = torch.einsum("hgt,thd->hgd", p, v).reshape(-1, D)
    return out
