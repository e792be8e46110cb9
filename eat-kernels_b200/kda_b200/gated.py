"""The gated linear recurrence and the norm of groups of channels, for serving and for training.

    y, final = gated_scan(x, r, i, rate, r_bias, i_bias, initial_state, cu_seqlens)                # differentiable
    y, pool = gated_scan(x, r, i, rate, r_bias, i_bias, pool, cu_seqlens, ssm_state_indices=slots)
    y, pool = gated_scan_step(x, r, i, rate, r_bias, i_bias, pool, slots)
    y = group_norm(x, groups, weight, bias, z, activation="silu")                                  # differentiable

Tokens, sequences, slots, `out` and `status` are those of the operators in `serving.py` (`status`: also the bit 64 = a wait inside
the kernel ran out, results are wrong; a recorded call's backward pass reports into the same tensor, and without one nothing does).

Gradients: with grad mode on, a call without `ssm_state_indices` and `out` whose tensors ask for some is recorded; calls that work on a
pool or write the caller's `out` are serving calls and record nothing.  Backward passes return the same bits whenever they run, can be
captured in a CUDA graph (while no eager graph of the same leaves lives, as torch wants it) and are differentiable once.  Forward-mode
derivatives are refused."""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _cabi, _err, _reject_aliasing
from .serving import (INT32_MAX, TYPES, _call, _cuda, _is, _layout, _lead, _out, _pool_rows, _ptr, _Ready, _rows, _sequences, _states, _status,
                      _step_pool, _step_slots, _vector)

ACTIVATIONS = {None: _cabi.ACT_NONE, "silu": _cabi.ACT_SILU, "sigmoid": _cabi.ACT_SIGMOID}


def _recorded(*tensors):
    return torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in tensors)


def _no_tangents(*tensors):
    """A launch by address would lose the tangents of forward-mode derivatives, which counts as zero."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _err("forward-mode derivatives are not supported")


# ------------------------------------------------------------------------------------------------ gated linear recurrence
def _gated_inputs(x, r, i, rate, r_bias, i_bias):
    """Checks of the tensors that all passes have; returns (T, device, channels, rate, r_bias, i_bias)."""
    T = _lead(x, "x", 1)
    dev, channels = x.device, x.shape[2]
    if x.dtype not in TYPES:
        raise _err(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if channels > INT32_MAX // 2:
        raise _err(f"x has more than {INT32_MAX // 2} channels")
    if r is None:
        raise _err("r is required")
    if i_bias is not None and i is None:
        raise _err("i_bias needs i")
    _cuda(dev, r=r, i=i, rate=rate, r_bias=r_bias, i_bias=i_bias)
    _is(r, "r", (1, T, channels), x.dtype)
    if i is not None:
        _is(i, "i", (1, T, channels), x.dtype)
    return T, dev, channels, _vector(rate, "rate", channels), _vector(r_bias, "r_bias", channels), _vector(i_bias, "i_bias", channels)


F32 = torch.finfo(torch.float32)


def _scale(rate_scale):
    scale = float(rate_scale)
    if not F32.tiny <= scale <= F32.max:               # the kernels take it in 32 bits
        raise _err(f"rate_scale must be a positive number of fp32's range, got {rate_scale!r}")
    return scale


def _scan(x, r, i, rate, r_bias, i_bias, state, cu_seqlens, slots, out, status, rate_scale, step, keep):
    T, dev, channels, rate, r_bias, i_bias = _gated_inputs(x, r, i, rate, r_bias, i_bias)
    _cuda(dev, out=out)
    inner = (channels,)
    if step:
        cu, N = None, T
        _step_pool(dev, state, inner, torch.float32)
        src = dst = state
        src_stride = dst_stride = _pool_rows(state, "the pool", inner)
        n_slots, slots = state.shape[0], _step_slots(dev, slots, N, state)
    else:
        cu, N = _layout(dev, cu_seqlens)
        src, src_stride, dst, dst_stride, n_slots, slots = _states(dev, state, slots, N, inner, torch.float32, "the pool")
    (x, ldx), (r, ldr) = _rows(x), _rows(r)
    i, ldi = _rows(i) if i is not None else (None, 0)
    y = _out(out, x)
    in_place = src is dst
    if in_place or out is not None or status is not None:
        _reject_aliasing([("out", y), ("the pool", dst), _status(dev, status)],
                         [("x", x), ("r", r), ("i", i), ("rate", rate), ("r_bias", r_bias), ("i_bias", i_bias), ("cu_seqlens", cu),
                          ("ssm_state_indices", slots), ("initial_state", None if in_place else src)])
    tiles = torch.empty(((T + _cabi.GATED_SCAN_TILE - 1) // _cabi.GATED_SCAN_TILE, channels), dtype=torch.float32, device=dev) if keep else None
    args = _cabi.KdaGatedScanArgs(_ptr(x), _ptr(r), _ptr(i), _ptr(y), _ptr(rate), _ptr(r_bias), _ptr(i_bias), _ptr(src), _ptr(dst), _ptr(tiles),
                                  ldx, ldr, ldi, _rows(y)[1], src_stride, dst_stride, _sequences(T, N, cu, slots, n_slots, status, int(out is None)),
                                  rate_scale, channels, TYPES[x.dtype])
    given = {k: [f] for k, f in enumerate(("x", "r", "i", "rate", "r_bias", "i_bias"))}
    given.update({7: ["seq.cu_seqlens"], 8: ["seq.slots"], 9: ["out"], 10: ["seq.status"]})
    given[6] = ["src", "dst"] if in_place else ["src"]
    fresh = ([(y, ["out"])] if out is None else []) + ([] if in_place else [(dst, ["dst"])])
    result = (9 if out is not None else -1, 6 if in_place else -len(fresh))
    if keep:
        fresh.append((tiles, ["tiles"]))
        result += (-len(fresh),)
    name = None if step and not T else "kda_gated_scan_step_launch" if step else "kda_gated_scan_launch"
    return _Ready(name, dev, args, given, fresh, result, [9, 10] + [6] * in_place, keep=(x, r, i, rate, r_bias, i_bias, src, cu, slots))


def _scan_grad(x, r, i, rate, r_bias, i_bias, state, cu, tiles, dy, dfinal, status, rate_scale, wants):
    T, dev, channels, rate, r_bias, i_bias = _gated_inputs(x, r, i, rate, r_bias, i_bias)
    N = 1 if cu is None else cu.numel() - 1
    cu, _ = _layout(dev, cu)
    dx, dr, di = (torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None else None for t in (x, r, i))
    state, dfinal = (t.contiguous() if t is not None else None for t in (state, dfinal))
    (x, ldx), (r, ldr) = _rows(x), _rows(r)
    i, ldi = _rows(i) if i is not None else (None, 0)
    dy, lddy = _rows(dy) if dy is not None else (None, 0)
    sums = [torch.empty(channels, dtype=torch.float32, device=dev) if wanted else None for wanted in wants[:3]]
    dsrc = torch.empty((N, channels), dtype=torch.float32, device=dev) if wants[3] else None
    if status is not None:
        _reject_aliasing([_status(dev, status)], [("x", x), ("r", r), ("i", i), ("rate", rate), ("r_bias", r_bias), ("i_bias", i_bias),
                                                  ("initial_state", state), ("cu_seqlens", cu), ("dy", dy), ("dfinal", dfinal)])
    args = _cabi.KdaGatedScanGradArgs(_ptr(x), _ptr(r), _ptr(i), _ptr(dy), _ptr(dx), _ptr(dr), _ptr(di), _ptr(rate), _ptr(r_bias), _ptr(i_bias),
                                      _ptr(tiles), _ptr(state), _ptr(dfinal), _ptr(dsrc), *map(_ptr, sums), ldx, ldr, ldi, lddy, channels, channels,
                                      channels, _sequences(T, N, cu, None, N, status, 1), rate_scale, channels, TYPES[x.dtype])
    given = {k: [f] for k, f in enumerate(("x", "r", "i", "rate", "r_bias", "i_bias", "src", "seq.cu_seqlens", "tiles", "dy", "dfinal", "seq.status"))}
    fresh, result = [], []
    for t, field in ((dx, "dx"), (dr, "dr"), (di, "di"), *zip(sums, ("drate", "dr_bias", "di_bias")), (dsrc, "dsrc")):
        if t is not None:
            fresh.append((t, [field]))
            result.append(-len(fresh))
    return _Ready("kda_gated_scan_grad_launch", dev, args, given, fresh, tuple(result), [11], keep=(x, r, i, rate, r_bias, i_bias, state, cu, tiles, dy, dfinal))


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, rate, r_bias, i_bias, state, cu_seqlens, status, rate_scale):
        y, final, tiles = _call(_scan, (x, r, i, rate, r_bias, i_bias, state, cu_seqlens, None, None, status), rate_scale, False, True)
        ctx.set_materialize_grads(False)
        ctx.rate_scale, ctx.status = rate_scale, status          # not a saved tensor: calls write it
        ctx.save_for_backward(x, r, i, rate, r_bias, i_bias, state, cu_seqlens, tiles)
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        tensors, need = ctx.saved_tensors, ctx.needs_input_grad
        if dy is None and dfinal is None:
            return (None,) * 10
        wants = (need[3], need[4], need[5], need[6])
        grads = iter(_call(_scan_grad, (*tensors, dy, dfinal, ctx.status), ctx.rate_scale, wants))
        dx, dr = next(grads), next(grads)
        di = next(grads) if tensors[2] is not None else None
        params = [next(grads).view_as(tensors[3 + k]) if wants[k] else None for k in range(3)]
        return (dx if need[0] else None, dr if need[1] else None, di if need[2] else None, *params, next(grads) if wants[3] else None, None, None, None)


def gated_scan(x, r, i=None, rate=None, r_bias=None, i_bias=None, initial_state=None, cu_seqlens=None, *, rate_scale=8.0,
               ssm_state_indices=None, out=None, status=None):
    """Gated linear recurrence over prompts: per channel h = f h + gain g x, y = h, with s = sigmoid(r + r_bias), g = sigmoid(i + i_bias)
    (1 without i) and, with `rate`, f = exp(-rate_scale softplus(rate) s), gain = sqrt(1 - f^2); without it f = s, gain = 1 - s.  The gain
    holds for every token, a sequence's first one too: models that leave it out there (gain 1 behind a reset) get another first state.
    Of 16-bit tokens an input gate below 2^-64 counts as shut.

    x, r, i [1, T, C] of one type (bf16, fp16 or fp32; any token strides); rate, r_bias, i_bias [C] fp32, each may be None.  State
    fp32: a pool [P, C] with `ssm_state_indices`, else [N, C].  Returns (y, pool or final state); without pool and `out` both are
    differentiable with respect to everything but cu_seqlens (rows behind the last sequence get zero gradients)."""
    scale = _scale(rate_scale)
    _no_tangents(x, r, i, rate, r_bias, i_bias, initial_state)
    if ssm_state_indices is None and out is None and _recorded(x, r, i, rate, r_bias, i_bias, initial_state):
        return _GatedScan.apply(x, r, i, rate, r_bias, i_bias, initial_state, cu_seqlens, status, scale)
    return _call(_scan, (x, r, i, rate, r_bias, i_bias, initial_state, cu_seqlens, ssm_state_indices, out, status), scale, False, False)


def gated_scan_step(x, r, i, rate, r_bias, i_bias, pool, ssm_state_indices=None, *, rate_scale=8.0, out=None, status=None):
    """The recurrence of the next token of each row, x, r, i [1, N, C]; records no gradients; equal to a prompt's tokens but for last digits.
    Returns (y, pool)."""
    _no_tangents(x, r, i, rate, r_bias, i_bias, pool)
    return _call(_scan, (x, r, i, rate, r_bias, i_bias, pool, None, ssm_state_indices, out, status), _scale(rate_scale), True, False)


# ------------------------------------------------------------------------------------------------ norm of groups of channels
def _norm_inputs(x, groups, weight, bias, z, activation):
    """Returns (T, device, groups, width, whether the groups share weight and bias, weight, bias)."""
    if not torch.is_tensor(x) or not x.is_cuda:
        raise _err("x must be a CUDA tensor")
    T = _lead(x, "x", 2 if x.dim() == 4 else 1)
    dev = x.device
    if x.dtype not in TYPES:
        raise _err(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise _err(f"activation must be 'silu', 'sigmoid' or None, got {activation!r}")
    channels = math.prod(x.shape[2:])
    if x.dim() == 4:
        if groups not in (None, x.shape[2]):
            raise _err(f"x [1, T, {x.shape[2]}, {x.shape[3]}] has {x.shape[2]} groups, got groups = {groups!r}")
        groups = x.shape[2]
    if groups is None or groups < 1 or channels % groups:
        raise _err(f"groups must divide the {channels} channels, got {groups!r}")
    width = channels // groups
    if width > _cabi.GROUP_NORM_MAX_WIDTH:
        raise _err(f"groups of {width} channels: the most is {_cabi.GROUP_NORM_MAX_WIDTH}")
    if channels > INT32_MAX // 2:
        raise _err(f"x has more than {INT32_MAX // 2} channels")
    _cuda(dev, weight=weight, bias=bias, z=z)
    if z is not None:
        _is(z, "z", tuple(x.shape), x.dtype)
    shared = False
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or t.numel() not in (channels, width)):
            raise _err(f"{name} must be fp32 with {channels} entries, or the {width} that all groups share, got {t.dtype} {list(t.shape)}")
        shared = shared or (t is not None and t.numel() == width and groups > 1)
    if weight is not None and bias is not None and weight.numel() != bias.numel():
        raise _err(f"weight and bias must be of one size, got {list(weight.shape)} and {list(bias.shape)}")
    return T, dev, groups, width, shared, *(t.contiguous() if t is not None else None for t in (weight, bias))


def _norm(x, weight, bias, z, out, groups, activation, eps, center):
    T, dev, groups, width, shared, weight, bias = _norm_inputs(x, groups, weight, bias, z, activation)
    _cuda(dev, out=out)
    x, ldx = _rows(x)
    z, ldz = _rows(z) if z is not None else (None, 0)
    y = _out(out, x)
    if out is not None:
        _reject_aliasing([("out", y)], [("x", x), ("z", z), ("weight", weight), ("bias", bias)])
    args = _cabi.KdaGroupNormArgs(_ptr(x), _ptr(z), None, _ptr(y), None, _ptr(weight), _ptr(bias), None, None, None, 0, T, ldx, ldz, 0, _rows(y)[1], 0,
                                  eps, groups, width, ACTIVATIONS[activation], int(center), int(shared), TYPES[x.dtype])
    given = {k: [f] for k, f in enumerate(("x", "weight", "bias", "z", "out"))}
    fresh = [(y, ["out"])] if out is None else []
    return _Ready("kda_group_norm_launch", dev, args, given, fresh, (4 if out is not None else -1,), [4], keep=(x, z, weight, bias))


def _norm_grad(x, weight, bias, z, dy, groups, activation, eps, center, wants):
    T, dev, groups, width, shared, weight, bias = _norm_inputs(x, groups, weight, bias, z, activation)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dz = torch.empty(x.shape, dtype=x.dtype, device=dev) if z is not None else None
    (x, ldx), (dy, lddy) = _rows(x), _rows(dy)
    z, ldz = _rows(z) if z is not None else (None, 0)
    cols = width if shared else groups * width
    sums = [torch.empty(cols, dtype=torch.float32, device=dev) if wanted else None for wanted in wants]
    ws_bytes = _cabi.lib().kda_group_norm_workspace_bytes(T, groups, width, TYPES[x.dtype], int(shared)) if any(wants) else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    args = _cabi.KdaGroupNormArgs(_ptr(x), _ptr(z), _ptr(dy), _ptr(dx), _ptr(dz), _ptr(weight), _ptr(bias), *map(_ptr, sums), _ptr(ws), ws_bytes, T, ldx, ldz,
                                  lddy, groups * width, groups * width, eps, groups, width, ACTIVATIONS[activation], int(center), int(shared),
                                  TYPES[x.dtype])
    given = {k: [f] for k, f in enumerate(("x", "weight", "bias", "z", "dy"))}
    fresh, result = [], []
    for t, field in ((dx, "out"), (dz, "dz"), *zip(sums, ("dweight", "dbias")), (ws, "workspace")):
        if t is not None:
            fresh.append((t, [field]))
            result.append(-len(fresh))
    return _Ready("kda_group_norm_grad_launch", dev, args, given, fresh, tuple(result[:-1] if ws is not None else result), keep=(x, z, dy, weight, bias))


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, z, groups, activation, eps, center):
        ctx.save_for_backward(x, weight, bias, z)
        ctx.options = groups, activation, eps, center
        return _call(_norm, (x, weight, bias, z, None), groups, activation, eps, center)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = iter(_call(_norm_grad, (x, weight, bias, z, dy), *ctx.options, (need[1], need[2])))
        dx = next(grads)
        dz = next(grads) if z is not None else None
        dweight = next(grads).view_as(weight) if need[1] else None
        dbias = next(grads).view_as(bias) if need[2] else None
        return dx if need[0] else None, dweight, dbias, dz if need[3] else None, None, None, None, None


def group_norm(x, groups=None, weight=None, bias=None, z=None, *, activation=None, eps=1e-5, center=True, out=None):
    """Norm of each group of channels of a token, with an activation: xh = (x - mean) / sqrt(mean((x - mean)^2) + eps) over the group
    (center=False: mean = 0), n = xh weight + bias, and y = n act(z), or act(n) without z.  The output norm of recurrent layers: of
    KDA's, x is the prefill's output, center=False, weight [128], z the gate's logits, activation "sigmoid".

    x, z [1, T, C] of one type (bf16, fp16 or fp32; any token strides) with `groups` dividing C, or [1, T, groups, D]; groups of up to
    16384 channels.  weight, bias fp32 with C entries, or with the C / groups that all groups share; each may be None.  activation
    "silu", "sigmoid" or None.  Returns y like x; without `out` it is differentiable with respect to all tensors."""
    if groups is not None and (isinstance(groups, bool) or not isinstance(groups, int)):
        raise _err(f"groups must be a whole number, got {groups!r}")
    eps = float(eps)
    if not 0.0 <= eps <= F32.max:
        raise _err(f"eps must be a number of zero or more in fp32's range, got {eps!r}")
    _no_tangents(x, weight, bias, z)
    if out is None and _recorded(x, weight, bias, z):
        return _GroupNorm.apply(x, weight, bias, z, groups, activation, eps, bool(center))
    return _call(_norm, (x, weight, bias, z, out), groups, activation, eps, bool(center))[0]
