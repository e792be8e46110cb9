"""The serving operators around KDA prefill, as measurable cases: short causal convolution, selective state space scan and the KDA
state's single-token step, each over packed batches and slot pools, and the upkeep of the pools' slots.

A case is one call of a public entry point on one batch:

    op        "conv" = `short_conv`, "conv_step" = `short_conv_step`, "scan" = `selective_scan`, "scan_step" =
              `selective_scan_step`, "kda_step" = `kda_step` (raw = 1) or `kda_step_plain` (raw = 0), "fork" = `pool_fork` and
              `pool_free`, "compact" = `pool_compact`
    dtype     type of the token tensors
    lengths, low, high, rows, layout
              prompts: `rows` sequence lengths, drawn from `layout` by the rule "one" (a single one of `high` tokens), "uniform" in
              [low, high] or "lognormal" around 1024 (sigma 0.8) clipped to [low, high]; steps: `rows` tokens, one a sequence
    pad       steps: trailing rows of the batch that belong to no sequence (slot -1)
    channels  channels of the convolution or the scan
    width     taps of the convolution
    state     state values a channel of the scan
    groups    groups of channels that share B and C
    gate      1: the scan's output is gated by z
    heads     KDA heads
    slots     slots of the pool
    fresh     fork: trailing new sequences without a parent
    live      compact: slots in use
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False
D = 128
DEV = "cuda:0"
LOWER = -5.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # q, k and v of a short user turn, 16 heads on this GPU: latency counts
        dict(name="conv_turn", op="conv", dtype="bf16", lengths="one", low=1, high=77, rows=1, layout=0, channels=6144, width=4, slots=8),
        # q, k and v of a serving batch of 48 prompts, 16 heads
        dict(name="conv_serving", op="conv", dtype="bf16", lengths="lognormal", low=16, high=8192, rows=48, layout=2, channels=6144, width=4, slots=256),
        # one token for each of 48 sequences, q, k and v of 64 heads
        dict(name="conv_step_48", op="conv_step", dtype="bf16", rows=48, pad=0, channels=24576, width=4, slots=256),
        # a padded decode batch of a small fp32 model with an odd number of channels
        dict(name="conv_step_odd", op="conv_step", dtype="fp32", rows=13, pad=3, channels=1539, width=3, slots=32),
        # a packed batch of ragged prompts through a gated scan layer
        dict(name="scan_ragged", op="scan", dtype="bf16", lengths="uniform", low=1, high=2048, rows=8, layout=11, channels=4096, state=16, groups=1, gate=1, slots=32),
        # one long prompt on an eighth of the channels: few rows, a long axis
        dict(name="scan_long", op="scan", dtype="fp16", lengths="one", low=1, high=32768, rows=1, layout=0, channels=512, state=16, groups=1, gate=1, slots=4),
        # a decode batch of 256 sequences
        dict(name="scan_step_256", op="scan_step", dtype="bf16", rows=256, pad=0, channels=4096, state=16, groups=1, gate=1, slots=512),
        # the next token of a single sequence, odd channel count
        dict(name="scan_step_1", op="scan_step", dtype="fp32", rows=1, pad=0, channels=1000, state=16, groups=1, gate=0, slots=8),
        # a decode batch over 64 heads, raw gates
        dict(name="kda_step_48", op="kda_step", raw=1, rows=48, pad=0, heads=64, slots=64),
        # the next token of a single sequence, 16 heads, activated inputs
        dict(name="kda_step_1", op="kda_step", raw=0, rows=1, pad=0, heads=16, slots=8),
        # eight sequences forked off running ones, one started from nothing, all ended again (16 heads, with its convolution)
        dict(name="fork_9", op="fork", dtype="bf16", rows=9, fresh=1, heads=16, channels=6144, width=4, slots=64),
        # a pool of 256 slots, half of them in use, moved to its front
        dict(name="compact_256", op="compact", dtype="bf16", rows=128, live=128, heads=16, channels=6144, width=4, slots=256),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan_step", "kda_step", "fork", "compact"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    odd = rng.random() < 0.3
    if op in ("conv", "scan"):
        how = rng.choice(["one", "uniform", "uniform", "lognormal"])
        rows = 1 if how == "one" else rng.randint(2, 48)
        channels = _spread(rng, 64, 16384 if op == "conv" else 8192) if odd else 128 * _spread(rng, 1, 96 if op == "conv" else 48)
        c = dict(op=op, dtype=kind, lengths=how, low=1, high=_spread(rng, 16, 32768 if how == "one" else 4096), rows=rows, layout=rng.randrange(1 << 20),
                 channels=channels, slots=rows + rng.randint(0, 16))
        if op == "conv":
            c["width"] = rng.randint(2, 4)
            most = 30_000 * 6144
        else:
            c.update(state=rng.choice([4, 8, 13, 16, 16, 16, 32, 64]), groups=1 if channels % 4 else rng.choice([1, 1, 2, 4]), gate=rng.randint(0, 1))
            most = 6000 * 4096 * 16 // c["state"]
        while sum(_lengths(c)) * channels > most and c["high"] > 1:
            c["high"] = max(1, c["high"] * 2 // 3)
        return c
    if op in ("conv_step", "scan_step"):
        rows = _spread(rng, 1, 512)
        channels = _spread(rng, 64, 8192) if odd else 128 * _spread(rng, 1, 64)
        c = dict(op=op, dtype=kind, rows=rows, pad=rng.choice([0, 0, 1, 5]), channels=channels, slots=rows + rng.randint(0, 64))
        if op == "conv_step":
            c["width"] = rng.randint(2, 4)
        else:
            c.update(state=rng.choice([4, 8, 13, 16, 16, 16, 32, 64]), groups=1 if channels % 4 else rng.choice([1, 1, 2, 4]), gate=rng.randint(0, 1))
            while c["rows"] * channels * c["state"] > 256 * 4096 * 16:
                c["rows"] = max(1, c["rows"] // 2)
                c["slots"] = c["rows"] + 7
        return c
    heads = rng.choice([4, 8, 12, 16, 24, 32, 48, 64])
    if op == "kda_step":
        rows = _spread(rng, 1, max(1, 2048 // heads))
        return dict(op=op, raw=rng.randint(0, 1), rows=rows, pad=rng.choice([0, 0, 1, 5]), heads=heads, slots=rows + rng.randint(0, 15))
    slots = _spread(rng, 8, max(9, 4096 // heads))
    channels = rng.choice([128 * heads, 64 * heads, 101 * heads])
    if op == "fork":
        rows = rng.randint(1, max(1, slots // 3))
        return dict(op=op, dtype=kind, rows=rows, fresh=rng.randint(0, min(rows, 2)), heads=heads, channels=channels, width=rng.randint(2, 4), slots=slots)
    live = rng.randint(1, slots)
    return dict(op=op, dtype=kind, rows=live, live=live, heads=heads, channels=channels, width=rng.randint(2, 4), slots=slots)


def _lengths(case):
    rng, n, low, high = random.Random(case["layout"]), case["rows"], case["low"], case["high"]
    if case["lengths"] == "one":
        return [high]
    if case["lengths"] == "uniform":
        return [rng.randint(min(low, high), high) for _ in range(n)]
    return [int(round(min(high, max(low, 1024.0 * math.exp(0.8 * rng.gauss(0.0, 1.0)))))) for _ in range(n)]


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op, rows = case["op"], case["rows"]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    s = {"op": op}
    if op in ("conv", "scan"):
        lens = _lengths(case)
        T = sum(lens)
        s["cu"] = _cu(lens)
    else:
        T = rows + case.get("pad", 0)
    if op not in ("fork", "compact"):
        s["rows"] = rows
        ids = torch.randperm(case["slots"], generator=host)[:rows].tolist() + [-1] * case.get("pad", 0)
        s["slots"] = torch.tensor(ids, dtype=torch.int32, device=DEV)
    if op in ("conv", "conv_step"):
        dt, C, W = TYPES[case["dtype"]], case["channels"], case["width"]
        s.update(x=randn(1, T, C, dtype=dt), weight=randn(C, W, dtype=dt, scale=W ** -0.5), bias=randn(C, dtype=dt, scale=0.1),
                 pool=randn(case["slots"], W - 1, C, dtype=dt))
    elif op in ("scan", "scan_step"):
        dt, Dm, Ns, G = TYPES[case["dtype"]], case["channels"], case["state"], case["groups"]
        s.update(u=randn(1, T, Dm, dtype=dt), dt=randn(1, T, Dm, dtype=dt, scale=0.5), B=randn(1, T, G, Ns, dtype=dt), C=randn(1, T, G, Ns, dtype=dt),
                 z=randn(1, T, Dm, dtype=dt) if case["gate"] else None, D=randn(Dm), pool=randn(case["slots"], Dm, Ns))
        # decay rates 1 .. Ns, jittered, and step sizes even over the logarithm in [0.001, 0.1]
        s["A"] = -torch.arange(1, Ns + 1, device=DEV) * torch.exp(randn(Dm, Ns, scale=0.3))
        step = torch.exp(torch.rand(Dm, generator=gen, device=DEV) * math.log(100.0) + math.log(0.001))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    elif op == "kda_step":
        H, raw, bf = case["heads"], case["raw"], torch.bfloat16
        s.update(raw=raw, scale=D ** -0.5, v=randn(1, T, H, D, dtype=bf), pool=randn(case["slots"], H, D, D, scale=0.25))
        q, k = randn(1, T, H, D), randn(1, T, H, D)
        if raw:
            s.update(q=(q * 0.5).to(bf), k=(k * 0.5).to(bf), g=randn(1, T, H, D, dtype=bf, scale=0.5), beta=randn(1, T, H, dtype=bf, scale=0.5),
                     A_log=torch.log(torch.rand(H, generator=gen, device=DEV) * 15.0 + 1.0), dt_bias=torch.rand(H * D, generator=gen, device=DEV) * 4.0 - 6.0)
        else:
            s.update(q=torch.nn.functional.normalize(q, dim=-1).to(bf), k=torch.nn.functional.normalize(k, dim=-1).to(bf),
                     g=torch.nn.functional.logsigmoid(randn(1, T, H, D)), beta=torch.sigmoid(randn(1, T, H)))
    else:
        H, P, dt = case["heads"], case["slots"], TYPES[case["dtype"]]
        s["pools"] = [randn(P, H, D, D), randn(P, case["width"] - 1, case["channels"], dtype=dt)]
        order = torch.randperm(P, generator=host)
        live = case["live"] if op == "compact" else max(1, P - rows - int(torch.randint(0, P // 4 + 1, (1,), generator=host)))
        live = max(1, min(live, P if op == "compact" else P - rows))
        used = torch.zeros(P, dtype=torch.bool)
        used[order[:live]] = True
        s["used"] = used.to(DEV)
        if op == "fork":
            parents = order[torch.randint(0, live, (rows,), generator=host)]
            parents[rows - case["fresh"]:] = -1
            s["parents"] = parents.to(torch.int32).to(DEV)
        else:
            s["table"] = order[:live].to(torch.int32).to(DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _conv(s):
    x, w, cu, slots, pool = s["x"][0].float(), s["weight"].float(), s["cu"], s["slots"].long(), s["pool"]
    T, W = x.shape[0], w.shape[1]
    at = torch.arange(T, device=x.device)
    seq = torch.searchsorted(cu, at, right=True) - 1
    into = at - cu[seq]                                                     # tokens of the sequence in front of this one
    # history and tokens in one table of rows: row r < S (W - 1) is history, the tokens follow
    hist = pool[slots].float().reshape(-1, x.shape[1])
    rows = torch.cat([hist, x])
    y = s["bias"].float().expand(T, -1)
    for j in range(W):
        back = W - 1 - j
        y = y + rows[torch.where(into >= back, hist.shape[0] + at - back, (seq + 1) * (W - 1) + into - back)] * w[:, j]
    out = _silu(y).to(s["x"].dtype)[None]
    n, j = torch.arange(slots.numel(), device=x.device)[:, None], torch.arange(W - 1, device=x.device)
    length, left = (cu[1:] - cu[:-1])[:, None], W - 1 - j
    src = torch.where(length >= left, hist.shape[0] + cu[1:, None] - left, n * (W - 1) + length + j)
    pool[slots] = rows[src].to(pool.dtype)
    return out, pool


def _conv_step(s):
    n, pool, w = s["rows"], s["pool"], s["weight"].float()
    slots = s["slots"][:n].long()
    window = torch.cat([pool[slots], s["x"][0, :n, None]], 1)               # [n, W, C]
    out = torch.zeros_like(s["x"])
    out[0, :n] = _silu((window.float() * w.t()).sum(1) + s["bias"].float()).to(out.dtype)
    pool[slots] = window[:, 1:]
    return out, pool


def _per_channel(t, channels):
    """[T, G, Ns] of B or C as [T, channels, Ns] (a view where there is one group)."""
    T, G, Ns = t.shape
    return t.float()[:, :, None].expand(T, G, channels // G, Ns).reshape(T, channels, Ns) if G > 1 else t.float().expand(T, channels, Ns)


def _scan(s):
    u, cu, slots, pool = s["u"][0].float(), s["cu"], s["slots"].long(), s["pool"]
    T, Dm = u.shape
    step = _softplus(s["dt"][0].float() + s["dt_bias"])
    a = torch.exp(step[:, :, None] * s["A"])
    h = (step * u)[:, :, None] * _per_channel(s["B"][0], Dm)
    # the entering states join the first tokens' terms; an empty sequence writes behind the last row
    first = torch.where(cu[1:] > cu[:-1], cu[:-1], T)
    begins = torch.zeros(T + 1, dtype=torch.bool, device=u.device).index_fill_(0, first, True)[:T]
    seq = torch.searchsorted(cu, torch.arange(T, device=u.device), right=True) - 1
    at = cu[:-1].clamp(max=T - 1)
    entering = torch.where((cu[1:] > cu[:-1])[:, None, None], a[at] * pool[slots], torch.zeros_like(a[at]))
    h.index_add_(0, at, entering)
    a.masked_fill_(begins[:, None, None], 0.0)
    k = 1
    while k < T:                                                            # prefix products by doubling
        h = torch.cat([h[:k], torch.addcmul(h[k:], a[k:], h[:-k])])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    y = (h * _per_channel(s["C"][0], Dm)).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * _silu(s["z"][0].float())
    last = (cu[1:] - 1).clamp(min=0)
    pool[slots] = torch.where((cu[1:] > cu[:-1])[:, None, None], h[last], pool[slots])
    return y.to(s["u"].dtype)[None], pool


def _scan_step(s):
    n, pool = s["rows"], s["pool"]
    slots, u = s["slots"][:n].long(), s["u"][0, :n].float()
    step = _softplus(s["dt"][0, :n].float() + s["dt_bias"])
    h = torch.exp(step[:, :, None] * s["A"]) * pool[slots] + (step * u)[:, :, None] * _per_channel(s["B"][0, :n], u.shape[1])
    y = (h * _per_channel(s["C"][0, :n], u.shape[1])).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * _silu(s["z"][0, :n].float())
    pool[slots] = h
    out = torch.zeros_like(s["u"])
    out[0, :n] = y.to(out.dtype)
    return out, pool


def _kda_step(s):
    n, pool = s["rows"], s["pool"]
    slots = s["slots"][:n].long()
    q, k, v, g, beta = (s[name][0, :n].float() for name in ("q", "k", "v", "g", "beta"))
    if s["raw"]:
        q = q / q.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-6)
        k = k / k.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-6)
        x = torch.exp(s["A_log"])[:, None] * (g + s["dt_bias"].view(-1, D))
        g = LOWER / (1.0 + torch.exp(-x))
        beta = 1.0 / (1.0 + torch.exp(-beta))
    S = pool[slots]                                                         # raw: [n, H, V, K]; plain: [n, H, K, V]
    key = (lambda t: t[:, :, None, :]) if s["raw"] else (lambda t: t[:, :, :, None])
    val = (lambda t: t[:, :, :, None]) if s["raw"] else (lambda t: t[:, :, None, :])
    axis = 3 if s["raw"] else 2
    S = S * torch.exp(key(g))
    S = S + key(k) * val(beta[:, :, None] * (v - (S * key(k)).sum(axis)))
    out = torch.zeros_like(s["q"])
    out[0, :n] = (s["scale"] * (S * key(q)).sum(axis)).to(out.dtype)
    pool[slots] = S
    return out, pool


def _fork(s):
    used, parents = s["used"], s["parents"].long()
    slots = torch.argsort(used.to(torch.int8), stable=True)[:parents.numel()]
    for pool in s["pools"]:
        rows = pool[parents.clamp(min=0)]
        pool[slots] = torch.where((parents >= 0).view(-1, *[1] * (pool.dim() - 1)), rows, torch.zeros_like(rows))
    forked = used.index_fill(0, slots, True)
    freed = forked.index_fill(0, slots, False)
    return [slots.to(torch.int32), forked, freed, *s["pools"]]


def _compact(s):
    used, P = s["used"], s["used"].numel()
    at = torch.arange(P, device=used.device)
    front = at < used.sum()
    mover, hole = used & ~front, ~used & front
    holes = torch.argsort((~hole).to(torch.int8), stable=True)              # the holes first, ascending
    movers = torch.argsort((~mover).to(torch.int8), stable=True)
    remap = torch.where(mover, holes[(torch.cumsum(mover, 0) - 1).clamp(min=0)], torch.where(used, at, -1))
    source = torch.where(hole, movers[(torch.cumsum(hole, 0) - 1).clamp(min=0)], at)
    for pool in s["pools"]:
        pool.copy_(pool[source])
    return [remap.to(torch.int32), front, remap[s["table"].long()].to(torch.int32), *s["pools"]]


def _framework():
    if "kda_b200" not in sys.modules:
        sys.path.insert(0, str(Path("eat-kernels_b200").resolve()))
    import kda_b200
    return kda_b200


def run(s):
    op = s["op"]
    if not own:
        return {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "kda_step": _kda_step, "fork": _fork,
                "compact": _compact}[op](s)
    kda = _framework()
    if op == "conv":
        return kda.short_conv(s["x"], s["weight"], s["bias"], s["pool"], s["cu"], ssm_state_indices=s["slots"])
    if op == "conv_step":
        return kda.short_conv_step(s["x"], s["weight"], s["bias"], s["pool"], s["slots"])
    if op == "scan":
        return kda.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], s["pool"], s["cu"], ssm_state_indices=s["slots"])
    if op == "scan_step":
        return kda.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], s["pool"], s["slots"])
    if op == "kda_step" and s["raw"]:
        return kda.kda_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["A_log"], s["dt_bias"], s["scale"], s["pool"], s["slots"])
    if op == "kda_step":
        return kda.kda_step_plain(s["q"], s["k"], s["v"], s["g"], s["beta"], s["scale"], s["pool"], s["slots"])
    used = s["used"].clone()                                                # the scheduler's table of this moment
    if op == "fork":
        slots = kda.pool_fork(s["pools"], used, s["parents"])
        forked = used.clone()
        kda.pool_free(used, slots)
        return [slots, forked, used, *s["pools"]]
    table = s["table"].clone()
    remap = kda.pool_compact(s["pools"], used, [table])
    return [remap, used, table, *s["pools"]]


def work(case):
    """Every token tensor read or written once, every state row that the call touches read and written once (fork and
    compact: every moved row, with the expected number of moves)."""
    op, rows = case["op"], case["rows"]
    size = 4 if case.get("dtype") == "fp32" else 2
    T = sum(_lengths(case)) if op in ("conv", "scan") else rows
    if op in ("conv", "conv_step"):
        C, W = case["channels"], case["width"]
        return {"bytes": size * C * (2 * T + 2 * rows * (W - 1) + W + 1), "flops": T * C * (2 * W + 5)}
    if op in ("scan", "scan_step"):
        Dm, Ns = case["channels"], case["state"]
        return {"bytes": size * T * ((3 + case["gate"]) * Dm + 2 * case["groups"] * Ns) + 8 * rows * Dm * Ns + 4 * Dm * (Ns + 2),
                "flops": T * Dm * (7 * Ns + 12)}
    state = case["heads"] * D * D * 4
    if op == "kda_step":
        return {"bytes": rows * (2 * state + case["heads"] * (D * (10 if case["raw"] else 12) + 2)), "flops": rows * case["heads"] * D * D * 7}
    row = state + size * (case["width"] - 1) * case["channels"]
    if op == "fork":
        return {"bytes": row * (2 * (rows - case["fresh"]) + case["fresh"]), "flops": 0}
    return {"bytes": max(1, round(2 * row * case["live"] * (case["slots"] - case["live"]) / case["slots"])) + case["slots"], "flops": 0}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    """The definitions, token by token, in 64 bits."""
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    op, f = case["op"], torch.float64
    if op in ("fork", "compact"):
        used, pools = s["used"].tolist(), [p.to(f) for p in s["pools"]]
        P = len(used)
        if op == "fork":
            free = [i for i in range(P) if not used[i]][:case["rows"]]
            before = [p.clone() for p in pools]
            for slot, parent in zip(free, s["parents"].tolist()):
                for p, b in zip(pools, before):
                    p[slot] = b[parent] if parent >= 0 else 0.0
            return [None, None, None, *pools]
        n = sum(used)
        moves = list(zip([i for i in range(n) if not used[i]], [i for i in range(n, P) if used[i]]))
        for hole, mover in moves:
            for p in pools:
                p[hole] = p[mover]
        return [None, None, None, *pools]
    pool, slots = s["pool"].to(f), s["slots"].tolist()
    if op in ("conv", "scan"):
        bounds = s["cu"].tolist()
        spans = [(bounds[i], bounds[i + 1]) for i in range(case["rows"])]
    else:
        spans = [(i, i + 1) for i in range(case["rows"])]
    if op in ("conv", "conv_step"):
        x, w, b, W = s["x"][0].to(f), s["weight"].to(f), s["bias"].to(f), case["width"]
        out = torch.zeros_like(x)
        for (t0, t1), slot in zip(spans, slots):
            full = torch.cat([pool[slot], x[t0:t1]])
            acc = b + torch.nn.functional.conv1d(full.t()[None], w[:, None], groups=w.shape[0])[0].t()
            out[t0:t1] = acc * torch.sigmoid(acc)
            pool[slot] = full[full.shape[0] - (W - 1):]
        return out[None], pool
    if op in ("scan", "scan_step"):
        u, A, Dm, G = s["u"][0].to(f), s["A"].to(f), case["channels"], case["groups"]
        delta = torch.nn.functional.softplus(s["dt"][0].to(f) + s["dt_bias"].to(f), threshold=200.0)
        B, C = (s[n][0].to(f).repeat_interleave(Dm // G, 1) if G > 1 else s[n][0].to(f) for n in "BC")
        out, longest = torch.zeros_like(u), max(t1 - t0 for t0, t1 in spans)
        h = pool[slots[:len(spans)]]
        for j in range(longest):                                            # token j of every sequence that has one
            on = [i for i, (t0, t1) in enumerate(spans) if t0 + j < t1]
            t = [spans[i][0] + j for i in on]
            i0 = slice(None) if len(on) == len(spans) else on
            new = torch.exp(delta[t][:, :, None] * A) * h[i0] + (delta[t] * u[t])[:, :, None] * B[t]
            h[i0] = new
            out[t] = torch.einsum("idn,idn->id", new, C[t].expand(len(t), Dm, -1)) + s["D"].to(f) * u[t]
        pool[slots[:len(spans)]] = h
        if s["z"] is not None:
            out = out * torch.nn.functional.silu(s["z"][0].to(f))
            if op == "scan_step":
                out[case["rows"]:] = 0.0
        return out[None], pool
    q, k, v, g, beta = (s[n][0].to(f) for n in ("q", "k", "v", "g", "beta"))
    if s["raw"]:
        q, k = (torch.nn.functional.normalize(t, dim=-1, eps=1e-6) for t in (q, k))
        g = LOWER * torch.sigmoid(s["A_log"].to(f).exp().view(-1, 1) * (g + s["dt_bias"].to(f).view(-1, D)))
        beta = torch.sigmoid(beta)
    out = torch.zeros_like(v)
    for i, (_, slot) in enumerate(zip(spans, slots)):
        S = pool[slot].transpose(1, 2) if s["raw"] else pool[slot]          # [H, K, V]
        S = S * g[i].exp()[:, :, None]
        S = S + torch.einsum("hk,hv->hkv", k[i], beta[i][:, None] * (v[i] - torch.einsum("hk,hkv->hv", k[i], S)))
        out[i] = s["scale"] * torch.einsum("hk,hkv->hv", q[i], S)
        pool[slot] = S.transpose(1, 2) if s["raw"] else S
    return out[None], pool
