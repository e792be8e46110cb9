"""The gated linear recurrence and the output norm of recurrent layers, as measurable cases: prompts and single tokens over slot
pools, and training passes with all gradients.

A case is one pass through a public entry point on one batch:

    op        "scan" = `gated_scan` over prompts in a pool, "step" = `gated_scan_step`, "train" = `gated_scan` of a packed batch
              with the gradients of everything it takes, "norm" = `group_norm`, "norm_train" = `group_norm` with its gradients
    dtype     type of the token tensors
    lengths, low, high, rows, layout
              packed sequences: `rows` lengths, drawn from `layout` by the rule "one" (a single one of `high` tokens), "uniform" in
              [low, high] or "lognormal" around 1024 (sigma 0.8) clipped to [low, high]; steps and norms: `rows` tokens
    pad       steps: trailing rows of the batch that belong to no sequence (slot -1)
    channels  channels of the recurrence
    form      "power": decay exp(-8 softplus(rate) sigmoid(r)), input scaled by sqrt(1 - decay^2); "logistic": decay sigmoid(r),
              input scaled by 1 - decay
    gated     1: the input has a gate i of its own
    slots     slots of the pool
    groups, width
              groups of a token's channels that are normalised, channels of each
    act       activation of the norm ("silu", "sigmoid" or "" for none)
    z         1: the activation is that of a gate z, 0: that of the normalised value
    center    1: the group's mean is taken off
    shared    1: weight and bias are one group's, used by all
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
C_RATE = 8.0
EPS = 1e-5


def listed():
    return [
        # a short user turn through one recurrent layer: latency counts
        dict(name="scan_turn", op="scan", dtype="bf16", lengths="one", low=1, high=77, rows=1, layout=0, channels=2560, form="power", gated=1, slots=8),
        # a serving batch of ragged prompts
        dict(name="scan_serving", op="scan", dtype="bf16", lengths="lognormal", low=16, high=8192, rows=20, layout=4, channels=4096, form="power", gated=1, slots=64),
        # one long prompt on a quarter of the channels, the form without a gate of the input
        dict(name="scan_long", op="scan", dtype="fp16", lengths="one", low=1, high=65537, rows=1, layout=0, channels=1024, form="logistic", gated=0, slots=4),
        # the next token of a single sequence, odd channel count
        dict(name="step_1", op="step", dtype="fp32", rows=1, pad=0, channels=2561, form="logistic", gated=1, slots=8),
        # a padded decode batch
        dict(name="step_256", op="step", dtype="bf16", rows=251, pad=5, channels=4096, form="power", gated=1, slots=512),
        # a training batch of packed documents
        dict(name="train_packed", op="train", dtype="bf16", lengths="uniform", low=1, high=2048, rows=8, layout=11, channels=4096, form="power", gated=1),
        # one long document in 32 bits, few channels
        dict(name="train_long", op="train", dtype="fp32", lengths="one", low=1, high=16384, rows=1, layout=0, channels=512, form="logistic", gated=1),
        # a small batch of a small model, odd channel count
        dict(name="train_odd", op="train", dtype="fp16", lengths="uniform", low=1, high=300, rows=5, layout=3, channels=771, form="power", gated=0),
        # output norm of a KDA layer of 64 heads, a decode batch: one weight for all heads, gated by a sigmoid
        dict(name="norm_decode", op="norm", dtype="bf16", rows=48, groups=64, width=128, act="sigmoid", z=1, center=0, shared=1),
        # the same layer with 32 heads behind a prefill
        dict(name="norm_prompt", op="norm", dtype="bf16", rows=20000, groups=32, width=128, act="sigmoid", z=1, center=0, shared=1),
        # a training pass over centred heads gated by silu
        dict(name="norm_train", op="norm_train", dtype="bf16", rows=8192, groups=16, width=256, act="silu", z=1, center=1, shared=0),
        # groups of an odd width behind an odd number of tokens, activation on the value itself
        dict(name="norm_train_odd", op="norm_train", dtype="fp32", rows=1021, groups=7, width=67, act="silu", z=0, center=1, shared=0),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan", "step", "train", "norm", "norm_train"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    odd = rng.random() < 0.3
    size = 2 if kind == "fp32" else 1
    if op in ("norm", "norm_train"):
        width = _spread(rng, 8, 1024) if odd else rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 160, 192, 256, 256, 512])
        groups = _spread(rng, 1, max(1, 12288 // width))
        most = (80_000_000 if op == "norm" else 32_000_000) // (size * width * groups)
        rows = min(_spread(rng, 1, 30000), most)
        return dict(op=op, dtype=kind, rows=rows, groups=groups, width=width, act=rng.choice(["silu", "silu", "sigmoid", ""]), z=rng.randint(0, 1),
                    center=rng.randint(0, 1), shared=rng.randint(0, 1))
    channels = _spread(rng, 64, 8192) if odd else 128 * _spread(rng, 1, 64)
    c = dict(op=op, dtype=kind, channels=channels, form=rng.choice(["power", "power", "logistic"]), gated=rng.randint(0, 1))
    if op == "step":
        rows = min(_spread(rng, 1, 512), max(1, 1_000_000 // channels))
        return dict(c, rows=rows, pad=rng.choice([0, 0, 1, 5]), slots=rows + rng.randint(0, 64))
    how = rng.choice(["one", "uniform", "uniform", "lognormal"])
    rows = 1 if how == "one" else rng.randint(2, 40)
    c.update(lengths=how, low=1, high=_spread(rng, 16, 65536 if how == "one" else 4096), rows=rows, layout=rng.randrange(1 << 20))
    if op == "scan":
        c["slots"] = rows + rng.randint(0, 16)
    most = (90_000_000 if op == "scan" else 32_000_000) // size
    while sum(_lengths(c)) * channels > most and c["high"] > 1:
        c["high"] = max(1, c["high"] * 2 // 3)
    return c


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
    op, rows, dt = case["op"], case["rows"], TYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    s = {"op": op}
    if op in ("norm", "norm_train"):
        G, W = case["groups"], case["width"]
        n = W if case["shared"] else G * W
        s.update(groups=G, act=case["act"] or None, center=bool(case["center"]), x=randn(1, rows, G * W, dtype=dt, scale=0.7), weight=1.0 + randn(n, scale=0.2),
                 bias=randn(n, scale=0.1) if case["center"] else None, z=randn(1, rows, G * W, dtype=dt) if case["z"] else None)
        if op == "norm_train":
            s["dy"] = randn(1, rows, G * W, dtype=dt)
        return s
    C = case["channels"]
    if op == "step":
        T = rows + case["pad"]
        s["rows"] = rows
    else:
        lens = _lengths(case)
        T = sum(lens)
        s["cu"] = _cu(lens)
    s.update(x=randn(1, T, C, dtype=dt), r=randn(1, T, C, dtype=dt), i=randn(1, T, C, dtype=dt) if case["gated"] else None,
             i_bias=randn(C, scale=0.1) if case["gated"] else None, rate=None)
    if case["form"] == "power":                                             # decays of 0.9 to 0.999 where the gate is open
        a = 0.9 + 0.099 * rand(C)
        s.update(rate=torch.log(torch.expm1(-torch.log(a) / C_RATE)), r_bias=randn(C, scale=0.1))
    else:
        s["r_bias"] = 1.0 + 4.0 * rand(C)                                   # decays around 0.73 to 0.99
    if op == "train":
        s.update(state=randn(rows, C, scale=0.5), dy=randn(1, T, C, dtype=dt), dfinal=randn(rows, C, scale=0.5))
    else:
        s["pool"] = randn(case["slots"], C, scale=0.5)
        ids = torch.randperm(case["slots"], generator=host)[:rows].tolist() + [-1] * case.get("pad", 0)
        s["slots"] = torch.tensor(ids, dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _sigmoid(x):
    """1 / (1 + e^-x) and 1 minus it, each to its own last digits."""
    e = torch.exp(-x.abs())
    small, large = e / (1.0 + e), 1.0 / (1.0 + e)
    return torch.where(x >= 0, large, small), torch.where(x >= 0, small, large)


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _gates(s, n):
    """Of the first n rows: x, s, 1 - s, log decay (or None), decay f, gain, g, 1 - g."""
    x, r = s["x"][0, :n].float(), s["r"][0, :n].float() + s["r_bias"]
    sr, nr = _sigmoid(r)
    if s["rate"] is not None:
        log = -C_RATE * _softplus(s["rate"]) * sr
        f, gain = torch.exp(log), torch.sqrt(-torch.expm1(2.0 * log))
    else:
        log, f, gain = None, sr, nr
    if s["i"] is not None:
        g, ng = _sigmoid(s["i"][0, :n].float() + s["i_bias"])
    else:
        g, ng = 1.0, 0.0
    return x, sr, nr, log, f, gain, g, ng


def _prefixes(f, u, T):
    """h[t] = f[t] h[t-1] + u[t] from h[-1] = 0, by doubling."""
    k = 1
    while k < T:
        u = torch.cat([u[:k], torch.addcmul(u[k:], f[k:], u[:-k])])
        f = torch.cat([f[:k], f[k:] * f[:-k]])
        k *= 2
    return u


def _starts(cu, T):
    """Truth value of each token: the first of its sequence."""
    first = torch.where(cu[1:] > cu[:-1], cu[:-1], T)
    return torch.zeros(T + 1, dtype=torch.bool, device=cu.device).index_fill_(0, first, True)[:T]


def _recurrence(f, u, cu, entering):
    """States of every token; the entering states [N, C] join the first tokens' terms."""
    T, some = f.shape[0], (cu[1:] > cu[:-1])[:, None]
    at = cu[:-1].clamp(max=T - 1)
    u = u.index_add(0, at, torch.where(some, f[at] * entering, torch.zeros_like(entering)))
    h = _prefixes(f.masked_fill(_starts(cu, T)[:, None], 0.0), u, T)
    return h, torch.where(some, h[(cu[1:] - 1).clamp(min=0)], entering)


def _scan(s):
    x, _, _, _, f, gain, g, _ = _gates(s, s["x"].shape[1])
    slots, pool = s["slots"].long(), s["pool"]
    h, final = _recurrence(f, gain * g * x, s["cu"], pool[slots])
    pool[slots] = final
    return h.to(s["x"].dtype)[None], pool


def _step(s):
    n, pool = s["rows"], s["pool"]
    x, _, _, _, f, gain, g, _ = _gates(s, n)
    slots = s["slots"][:n].long()
    h = f * pool[slots] + gain * g * x
    pool[slots] = h
    out = torch.zeros_like(s["x"])
    out[0, :n] = h.to(out.dtype)
    return out, pool


def _train(s):
    cu, dt = s["cu"], s["x"].dtype
    T = s["x"].shape[1]
    x, sr, nr, log, f, gain, g, ng = _gates(s, T)
    h, final = _recurrence(f, gain * g * x, cu, s["state"])
    # backward: the same recurrence from the last token to the first
    some, starts = (cu[1:] > cu[:-1])[:, None], _starts(cu, T)
    last = (cu[1:] - 1).clamp(min=0)
    d = s["dy"][0].float().index_add(0, last, torch.where(some, s["dfinal"], torch.zeros_like(s["dfinal"])))
    follow = torch.cat([f[1:].masked_fill(starts[1:, None], 0.0), torch.zeros_like(f[:1])])
    d = _prefixes(follow.flip(0), d.flip(0), T).flip(0)
    first = cu[:-1].clamp(max=T - 1)
    dstate = torch.where(some, f[first] * d[first], s["dfinal"])
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]]).masked_fill(starts[:, None], 0.0)
    before = before.index_add(0, first, torch.where(some, s["state"], torch.zeros_like(s["state"])))
    dx = d * gain * g
    grads = [dx]
    if log is not None:
        dlog = d * before * f - d * g * x * f * f / gain
        dr = dlog * log * nr
        rate = s["rate"]
        grads += [dr, (dlog * log).sum(0) * _sigmoid(rate)[0] / _softplus(rate)]
    else:
        dr = (d * before - d * g * x) * sr * nr
        grads += [dr]
    grads.append(dr.sum(0))
    if s["i"] is not None:
        di = d * gain * x * g * ng
        grads += [di, di.sum(0)]
    grads.append(dstate)
    return [h.to(dt)[None], final] + [t.to(dt)[None] if t.shape == h.shape else t for t in grads[:-1]] + grads[-1:]


def _act(v, act):
    """act(v) and its slope."""
    if act is None:
        return v, torch.ones_like(v)
    p, q = _sigmoid(v)
    return (p, p * q) if act == "sigmoid" else (v * p, p * (1.0 + v * q))


def _norm(s, train):
    x, G, dt = s["x"][0].float(), s["groups"], s["x"].dtype
    T, C = x.shape
    x = x.view(T, G, C // G)
    mean = x.mean(-1, keepdim=True) if s["center"] else 0.0
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    xh = (x - mean) * rstd
    w, b = s["weight"].view(-1, C // G), s["bias"].view(-1, C // G) if s["bias"] is not None else 0.0
    n = xh * w + b
    z = s["z"][0].float().view_as(x) if s["z"] is not None else None
    a, slope = _act(n if z is None else z, s["act"])
    y = (a if z is None else n * a).to(dt).view(1, T, C)
    if not train:
        return y
    dy = s["dy"][0].float().view_as(x)
    dn = dy * (slope if z is None else a)
    k = dn * w
    dx = k - xh * (k * xh).mean(-1, keepdim=True)
    if s["center"]:
        dx = dx - k.mean(-1, keepdim=True)

    def total(t):
        return t.sum(0).view(-1) if w.shape[0] == G and w.numel() == C else t.sum((0, 1))

    out = [y, (dx * rstd).to(dt).view(1, T, C), total(dn * xh)]
    if s["bias"] is not None:
        out.append(total(dn))
    if z is not None:
        out.append((dy * n * slope).to(dt).view(1, T, C))
    return out


def _framework():
    if "kda_b200" not in sys.modules:
        sys.path.insert(0, str(Path("eat-kernels_b200").resolve()))
    import kda_b200
    return kda_b200


def _leaves(s, *names):
    return [s[n].detach().requires_grad_() if s[n] is not None else None for n in names]


def run(s):
    op = s["op"]
    if not own:
        return {"scan": _scan, "step": _step, "train": _train}[op](s) if op in ("scan", "step", "train") else _norm(s, op == "norm_train")
    kda = _framework()
    if op == "scan":
        return kda.gated_scan(s["x"], s["r"], s["i"], s["rate"], s["r_bias"], s["i_bias"], s["pool"], s["cu"], ssm_state_indices=s["slots"])
    if op == "step":
        return kda.gated_scan_step(s["x"], s["r"], s["i"], s["rate"], s["r_bias"], s["i_bias"], s["pool"], s["slots"])
    if op == "norm":
        return kda.group_norm(s["x"], s["groups"], s["weight"], s["bias"], s["z"], activation=s["act"], eps=EPS, center=s["center"])
    if op == "train":
        x, r, i, rate, r_bias, i_bias, state = _leaves(s, "x", "r", "i", "rate", "r_bias", "i_bias", "state")
        y, final = kda.gated_scan(x, r, i, rate, r_bias, i_bias, state, s["cu"])
        wanted = [t for t in (x, r, rate, r_bias, i, i_bias, state) if t is not None]
        return [y.detach(), final.detach(), *torch.autograd.grad((y, final), wanted, (s["dy"], s["dfinal"]))]
    x, weight, bias, z = _leaves(s, "x", "weight", "bias", "z")
    y = kda.group_norm(x, s["groups"], weight, bias, z, activation=s["act"], eps=EPS, center=s["center"])
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, weight, bias, z) if t is not None], s["dy"])]


def work(case):
    """Every token tensor read or written once, every state row and parameter too; a training pass reads its inputs for the
    forward and again, with the outputs' gradients, for the backward pass."""
    op, rows = case["op"], case["rows"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op in ("norm", "norm_train"):
        n, z = rows * case["groups"] * case["width"], case["z"]
        params = 8 * (1 if case["shared"] else case["groups"]) * case["width"]
        if op == "norm":
            return {"bytes": size * n * (2 + z) + params, "flops": 12 * n}
        return {"bytes": size * n * (5 + 3 * z) + 3 * params, "flops": 40 * n}
    C, g = case["channels"], case["gated"]
    T = rows if op == "step" else sum(_lengths(case))
    if op in ("scan", "step"):
        return {"bytes": size * T * C * (3 + g) + 8 * rows * C + 12 * C, "flops": 20 * T * C}
    return {"bytes": size * T * C * (8 + 3 * g) + 16 * rows * C + 36 * C, "flops": 60 * T * C}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, the recurrence token by token, gradients of what is elementwise by differentiation."""
    s = prepare(case, seed)
    f64 = torch.float64
    op = case["op"]
    names = ("x", "weight", "bias", "z") if op in ("norm", "norm_train") else ("x", "r", "i", "rate", "r_bias", "i_bias")
    v = {n: None if s[n] is None else s[n].to(f64) for n in names}
    if op in ("train", "norm_train"):
        v = {n: t if t is None else t.requires_grad_() for n, t in v.items()}
    if op in ("norm", "norm_train"):
        G, W, T = case["groups"], case["width"], case["rows"]
        x = v["x"].reshape(T * G, 1, W)
        if case["center"]:
            n = torch.nn.functional.group_norm(x.reshape(T, G * W, 1), G, eps=EPS).reshape(T, G, W)
        else:
            n = torch.nn.functional.rms_norm(x.reshape(T, G, W), (W,), eps=EPS)
        n = (n * v["weight"].view(-1, W) + (v["bias"].view(-1, W) if v["bias"] is not None else 0.0)).reshape(1, T, G * W)
        act = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "": lambda t: t}[case["act"]]
        y = act(n) if v["z"] is None else n * act(v["z"])
        if op == "norm":
            return y
        return [y.detach(), *torch.autograd.grad(y, [t for t in v.values() if t is not None], s["dy"].to(f64))]
    r = torch.sigmoid(v["r"][0] + v["r_bias"])
    if v["rate"] is not None:
        log = -C_RATE * torch.nn.functional.softplus(v["rate"], threshold=200.0) * r
        decay, gain = log.exp(), (-(2.0 * log).expm1()).sqrt()
    else:
        decay, gain = r, torch.sigmoid(-(v["r"][0] + v["r_bias"]))
    u = gain * v["x"][0]
    if v["i"] is not None:
        u = u * torch.sigmoid(v["i"][0] + v["i_bias"])
    f, b = decay.detach(), u.detach()
    if op == "step":
        n, pool = case["rows"], s["pool"].to(f64)
        slots = s["slots"][:n].long()
        out = torch.zeros_like(b)
        out[:n] = f[:n] * pool[slots] + b[:n]
        pool[slots] = out[:n]
        return out[None], pool
    bounds = s["cu"].tolist()
    spans = list(zip(bounds[:-1], bounds[1:]))
    if op == "scan":
        pool = s["pool"].to(f64)
        entering = pool[s["slots"].long()]
    else:
        entering = s["state"].to(f64)
    h, final = torch.empty_like(b), entering.clone()
    for k, (t0, t1) in enumerate(spans):
        state = entering[k]
        for t in range(t0, t1):
            state = torch.addcmul(b[t], f[t], state, out=h[t])
        if t1 > t0:
            final[k] = h[t1 - 1]
    if op == "scan":
        pool[s["slots"].long()] = final
        return h[None], pool
    d, back = s["dy"][0].to(f64), s["dfinal"].to(f64).clone()
    before = torch.empty_like(h)
    for k, (t0, t1) in enumerate(spans):
        if t1 == t0:
            continue
        before[t0] = entering[k]
        before[t0 + 1:t1] = h[t0:t1 - 1]
        d[t1 - 1] += back[k]
        for t in range(t1 - 2, t0 - 1, -1):
            d[t].addcmul_(f[t + 1], d[t + 1])
        back[k] = f[t0] * d[t0]
    wanted = [v[n] for n in ("x", "r", "rate", "r_bias", "i", "i_bias") if v[n] is not None]
    return [h[None], final, *torch.autograd.grad((decay, u), wanted, (d * before, d)), back]
