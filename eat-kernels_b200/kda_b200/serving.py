"""The operators around KDA prefill in a recurrent layer, for prompts and for single tokens.

    y, pool = short_conv(x, weight, bias, pool, cu_seqlens, ssm_state_indices=slots)      # depthwise causal convolution
    y, pool = short_conv_step(x, weight, bias, pool, slots)
    y, pool = selective_scan(u, dt, A, B, C, D, z, dt_bias, pool, cu_seqlens, ssm_state_indices=slots)
    y, pool = selective_scan_step(u, dt, A, B, C, D, z, dt_bias, pool, slots)
    o, pool = kda_step(q, k, v, g, beta, A_log, dt_bias, scale, pool, slots)              # the prefill's next token
    o, pool = kda_step_plain(q, k, v, g, beta, scale, pool, slots)                        # that of `chunk_kda`

Tokens are packed as in the prefill, [1, T, ...].  Prompts: sequences by `cu_seqlens` (None: one); with `ssm_state_indices` the
state buffer is a pool of slots that is updated in place and returned, without it `initial_state` has one entry a sequence (or is
None: zeros), is left alone, and a new final state is returned.  Steps: row i is the next token of a sequence of its own, in slot
`ssm_state_indices[i]` (None: slot i); a negative entry marks a row of padding, of which nothing is used or stored.

Tables are read on the device where they lie; every call enqueues its launches on the current stream of the tensors' device, reads
nothing on the host and can be captured in a CUDA graph.  Rows of the output that no sequence owns (behind the last sequence,
padding) are zeros, or stay as they are in a caller's `out`.  `status`: an int32 CUDA tensor, apart from every other operand, whose
first entry collects (ORs) the bits 1 = rejected cu_seqlens (all sequences taken as empty, output rows zero) and 2 = slot out of
range or named before (that sequence starts from zeros and its state is not stored)."""
from __future__ import annotations

import ctypes as C

import torch

from . import D, LOWER_BOUND, _byte_interval, _cabi, _err, _reject_aliasing, _table

TYPES = {torch.bfloat16: _cabi.TYPE_BF16, torch.float16: _cabi.TYPE_FP16, torch.float32: _cabi.TYPE_FP32}
INT32_MAX = 0x7fffffff


class _Ready:
    """A checked call: the argument block, where the pointers of the caller's tensors and of the ones made for this call go in it,
    and what it returns."""

    def __init__(self, name, dev, args, given, fresh, result, written=(), aligned=(), keep=()):
        self.name, self.dev, self.args = name, dev, args
        self.keep = keep              # what the block points to, copies of the caller's tensors among it, until the launch
        self.given = given            # {index among the caller's tensors: names of pointer fields}
        self.fresh = fresh            # [(tensor made for this call, names of pointer fields)]
        self.result = result          # indices among the caller's tensors, or -1 - index in `fresh`
        self.written = written        # caller's tensors that the call writes
        self.aligned = aligned        # caller's tensors that must lie on 16 bytes


def _offset(block, field):
    """Byte offset of a field, "a.b" in a nested block and "a[i]" in an array."""
    at = 0
    for part in field.split("."):
        part, _, i = part.partition("[")
        f = getattr(block, part)
        at += f.offset
        kind = dict(block._fields_)[part]
        if i:
            at += int(i[:-1]) * C.sizeof(kind._type_)
        block = kind
    return at


class _Plan:
    """What the checks of a call found, for later calls whose tensors have the same types, shapes, strides and devices: the argument
    block without its pointers.  Nothing of the tensors themselves is kept."""

    def __init__(self, ready, tensors):
        block = type(ready.args)
        self.words = C.c_uint64 * (C.sizeof(block) // 8)
        self.template = bytes(ready.args)
        self.given = [(_offset(block, f) // 8, i) for i, fields in ready.given.items() if tensors[i] is not None for f in fields]
        # a tensor made for each call: like one of the caller's where that is a dense one (the cheaper way to ask for it)
        self.fresh = []
        for t, fields in ready.fresh:
            like = [i for i, g in enumerate(tensors) if g is not None and g.shape == t.shape and g.dtype == t.dtype and g.is_contiguous()
                    and type(g) is torch.Tensor]
            self.fresh.append(([_offset(block, f) // 8 for f in fields], t.shape, t.dtype, like[0] if like else -1))
        self.result, self.written, self.aligned = ready.result, [i for i in ready.written if tensors[i] is not None], ready.aligned
        self.present = [i for i, t in enumerate(tensors) if t is not None]
        spans = [_byte_interval(t) for t in tensors]
        self.reach = [0 if s is None else s[1] - s[0] for s in spans]
        self.name, self.dev = ready.name, ready.dev
        self.entry = _cabi.raw(ready.name)

    def run(self, tensors):
        """The call's results, or None where the tensors' addresses need another look."""
        at = [0] * len(tensors)
        for i in self.present:
            at[i] = tensors[i].data_ptr()
        for i in self.aligned:
            if at[i] & 15:
                return None
        reach = self.reach
        for w in self.written:
            lo, hi = at[w], at[w] + reach[w]
            for i in self.present:
                if i != w and at[i] < hi and lo < at[i] + reach[i]:
                    return None
        args, dev = self.words.from_buffer_copy(self.template), self.dev
        for word, i in self.given:
            args[word] = at[i]
        fresh = []
        for words, shape, dtype, like in self.fresh:
            t = torch.empty_like(tensors[like]) if like >= 0 else torch.empty(shape, dtype=dtype, device=dev)
            fresh.append(t)
            for word in words:
                args[word] = t.data_ptr()
        _launch(self.entry, self.name, args, dev)
        return tuple([tensors[i] if i >= 0 else fresh[-1 - i] for i in self.result])


_plans = {}
PLANS_MAX = 1024          # layouts remembered; a program that has more starts over


def _stream(index):
    """Handle of the device's current stream."""
    return torch.cuda.current_stream(index).cuda_stream


_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)       # the same without a Stream object (2 us a call)


def _launch(entry, name, args, dev):
    if torch.cuda.current_device() == dev.index:
        rc = entry(args, _stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = entry(args, _stream(dev.index))
    if rc:
        _cabi.check(rc, name)


def _call(check, tensors, *options):
    """Runs `check`, which returns a _Ready, and what it found; a layout that has been checked before goes straight to the launch."""
    try:
        key = (check, options, *[t if t is None else (t.dtype, t.shape, t.stride(), t.device) for t in tensors])
        plan = _plans.get(key)
    except (AttributeError, TypeError, RuntimeError):  # not tensors, or without strides: the checks say so
        key = plan = None
    if plan is not None:
        result = plan.run(tensors)
        if result is not None:
            return result
    ready = check(*tensors, *options)
    if ready.name is not None:
        _launch(_cabi.raw(ready.name), ready.name, C.byref(ready.args), ready.dev)
        block = type(ready.args)
        raw = bytes(ready.args)
        same = all(int.from_bytes(raw[o:o + 8], "little") == tensors[i].data_ptr() for i, fields in ready.given.items()
                   if tensors[i] is not None for o in (_offset(block, f) for f in fields))
        if key is not None and same:                   # nothing was copied on the way
            if len(_plans) >= PLANS_MAX:
                _plans.clear()
            _plans[key] = _Plan(ready, tensors)
    return tuple([tensors[i] if i >= 0 else ready.fresh[-1 - i][0] for i in ready.result])


def _cuda(dev, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if not torch.is_tensor(t) or not t.is_cuda:
            raise _err(f"{name} must be a CUDA tensor")
        if t.device != dev:
            raise _err(f"all CUDA tensors must be on one device ({dev}), got {name} on {t.device}")


def _is(t, name, shape, dtype=None):
    if tuple(t.shape) != shape or (dtype is not None and t.dtype != dtype):
        want = f"{dtype} " if dtype is not None else ""
        raise _err(f"{name} must be {want}{list(shape)}, got {t.dtype} {list(t.shape)}")


def _lead(t, name, width_dims):
    """Rows of a packed token tensor [1, T, ...]."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise _err(f"{name} must be a CUDA tensor")
    if t.dim() != 2 + width_dims or t.shape[0] != 1 or 0 in t.shape[2:]:
        raise _err(f"{name} must be a packed token tensor [1, T{', .' * width_dims}], got {list(t.shape)}")
    if t.shape[1] > INT32_MAX:
        raise _err(f"{name} has more than 2^31 - 1 tokens")
    if t.shape[2:].numel() > INT32_MAX:                # argument blocks hold 32 bits
        raise _err(f"{name} has more than 2^31 - 1 channels")
    return t.shape[1]


def _rows(t):
    """(tensor whose rows are dense and do not overlap, elements between rows): a view that is not like that is copied."""
    width = 1
    for n, s in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if n > 1 and s != width:
            t = t.contiguous()
            break
        width *= n
    width = t[0, 0].numel() if t.shape[1] else 1
    if t.shape[1] <= 1:
        return t, width
    if t.stride(1) < width:
        t = t.contiguous()
    return t, t.stride(1)


def _vector(t, name, n, dtype=torch.float32):
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != n:
        raise _err(f"{name} must be {dtype} with {n} entries, got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def _out(out, like, name="out"):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _is(out, name, tuple(like.shape), like.dtype)
    kept, _ = _rows(out)
    if kept is not out:
        raise _err(f"{name} must have dense rows that do not overlap")
    return out


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _pool_rows(t, name, inner):
    """Slots are dense blocks that do not overlap; returns the stride between them."""
    n = 1
    for extent, stride in zip(reversed(inner), reversed(t.stride()[1:])):
        if extent > 1 and stride != n:
            raise _err(f"{name} must have dense slots {list(inner)}")
        n *= extent
    if t.shape[0] > 1 and t.stride(0) < n:
        raise _err(f"{name} must have slots that do not overlap")
    return t.stride(0) if t.shape[0] > 1 else n


def _status(dev, status):
    """Checks `status`; returns the bytes of it that a call writes, named."""
    if status is None:
        return "status", None
    if not (torch.is_tensor(status) and status.dtype == torch.int32 and status.device == dev and status.numel() >= 1):
        raise _err(f"status must be an int32 tensor on {dev}")
    return "status", (status.data_ptr(), status.data_ptr() + 4)


def _sequences(T, N, cu, slots, n_slots, status, zero_rest):
    return _cabi.KdaSequences(_ptr(cu), _ptr(slots), n_slots, T, _ptr(status), int(cu is not None and cu.dtype == torch.int64),
                              int(slots is not None and slots.dtype == torch.int64), N, zero_rest)


def _layout(dev, cu_seqlens):
    """(cu_seqlens on the device or None, sequences)."""
    if cu_seqlens is None:
        return None, 1
    if not (torch.is_tensor(cu_seqlens) and cu_seqlens.dim() == 1 and cu_seqlens.dtype in (torch.int32, torch.int64)):
        raise _err("cu_seqlens must be a 1-D int32 / int64 tensor")
    if cu_seqlens.numel() < 2:
        raise _err("cu_seqlens must describe at least one sequence")
    if cu_seqlens.is_cuda and cu_seqlens.device != dev:
        raise _err(f"all CUDA tensors must be on one device ({dev}), got cu_seqlens on {cu_seqlens.device}")
    return cu_seqlens.to(dev).contiguous(), cu_seqlens.numel() - 1


def _states(dev, state, slots, N, inner, dtype, what):
    """Source and destination of a prompt call: (source, its slot stride, destination, its slot stride, slots, table)."""
    if slots is not None:
        if state is None:
            raise _err("initial_state (the pool) is required with ssm_state_indices")
        _step_pool(dev, state, inner, dtype, what)
        stride = _pool_rows(state, what, inner)
        return state, stride, state, stride, state.shape[0], _slots(dev, slots, N)
    final = torch.empty((N, *inner), dtype=dtype, device=dev)
    if state is not None:
        _cuda(dev, initial_state=state)
        _is(state, "initial_state", (N, *inner), dtype)
        state = state.contiguous()
    size = final[0].numel()
    return state, size, final, size, N, None


def _step_pool(dev, pool, inner, dtype, what="the pool"):
    _cuda(dev, **{what: pool})
    if pool is None or pool.dim() != 1 + len(inner) or tuple(pool.shape[1:]) != inner or pool.dtype != dtype or pool.shape[0] < 1:
        got = "None" if pool is None else f"{pool.dtype} {list(pool.shape)}"
        raise _err(f"{what} must be {dtype} [P, {', '.join(map(str, inner))}], got {got}")


def _slots(dev, slots, N):
    _cuda(dev, ssm_state_indices=slots)
    return _table(slots, "ssm_state_indices", N, False)


def _step_slots(dev, slots, N, pool):
    if slots is None:
        if pool.shape[0] < N:
            raise _err(f"the pool has {pool.shape[0]} slots for {N} rows: without ssm_state_indices row i uses slot i")
        return None
    return _slots(dev, slots, N)


# ------------------------------------------------------------------------------------------------ short convolution
def _conv(x, weight, bias, state, cu_seqlens, slots, out, status, activation, step):
    T = _lead(x, "x", 1)
    dev, channels = x.device, x.shape[2]
    if x.dtype not in TYPES:
        raise _err(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if activation not in ("silu", None):
        raise _err(f"activation must be 'silu' or None, got {activation!r}")
    _cuda(dev, weight=weight, bias=bias, out=out)
    if weight is not None and weight.dim() == 3 and weight.shape[1] == 1:           # a depthwise Conv1d's weight
        weight = weight[:, 0]
    if weight is None or weight.dim() != 2 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 4 or weight.dtype not in TYPES:
        got = "None" if weight is None else f"{weight.dtype} {list(weight.shape)}"
        raise _err(f"weight must be bf16, fp16 or fp32 [{channels}, W] with W of 2 to 4, got {got}")
    W = weight.shape[1]
    weight, bias = weight.contiguous(), _vector(bias, "bias", channels, weight.dtype)
    inner = (W - 1, channels)
    if step:
        cu, N = None, T
        _step_pool(dev, state, inner, x.dtype)
        src = dst = state
        src_stride = dst_stride = _pool_rows(state, "the pool", inner)
        n_slots, slots = state.shape[0], _step_slots(dev, slots, N, state)
    else:
        cu, N = _layout(dev, cu_seqlens)
        src, src_stride, dst, dst_stride, n_slots, slots = _states(dev, state, slots, N, inner, x.dtype, "the pool")
    x, ldx = _rows(x)
    y = _out(out, x)
    in_place = src is dst
    if in_place or out is not None or status is not None:
        _reject_aliasing([("out", y), ("the pool", dst), _status(dev, status)], [("x", x), ("weight", weight), ("bias", bias), ("cu_seqlens", cu),
                         ("ssm_state_indices", slots), ("initial_state", None if in_place else src)])
    args = _cabi.KdaConvArgs(_ptr(x), _ptr(weight), _ptr(bias), _ptr(y), _ptr(src), _ptr(dst), ldx, _rows(y)[1], src_stride, dst_stride,
                             _sequences(T, N, cu, slots, n_slots, status, int(out is None)), channels, W, TYPES[x.dtype],
                             TYPES[weight.dtype], int(activation is not None))
    given = {0: ["x"], 1: ["weight"], 2: ["bias"], 4: ["seq.cu_seqlens"], 5: ["seq.slots"], 6: ["out"], 7: ["seq.status"]}
    given[3] = ["src", "dst"] if in_place else ["src"]
    fresh = ([(y, ["out"])] if out is None else []) + ([] if in_place else [(dst, ["dst"])])
    result = (6 if out is not None else -1, 3 if in_place else -len(fresh))
    name = None if step and not T else "kda_short_conv_step_launch" if step else "kda_short_conv_launch"
    return _Ready(name, dev, args, given, fresh, result, [6, 7] + [3] * in_place, keep=(x, weight, bias, src, cu, slots))


def short_conv(x, weight, bias=None, initial_state=None, cu_seqlens=None, *, activation="silu", ssm_state_indices=None, out=None,
               status=None):
    """Depthwise causal convolution in front of q, k, v (or u): y[t] = act(bias + sum_j weight[:, j] x[t - W + 1 + j]).

    x [1, T, C] bf16, fp16 or fp32 (any token stride); weight [C, W] or [C, 1, W], W of 2 to 4, in any of these types, bias [C] in
    weight's type; activation "silu" or None.  State: the last W - 1 rows of a sequence, oldest first, in x's type: a pool
    [P, W - 1, C] with `ssm_state_indices`, else [N, W - 1, C].  Returns (y, pool or final state)."""
    return _call(_conv, (x, weight, bias, initial_state, cu_seqlens, ssm_state_indices, out, status), activation, False)


def short_conv_step(x, weight, bias, pool, ssm_state_indices=None, *, activation="silu", out=None, status=None):
    """The convolution of the next token of each row, x [1, N, C]; the pool's slots move on by a row.  Returns (y, pool)."""
    return _call(_conv, (x, weight, bias, pool, None, ssm_state_indices, out, status), activation, True)


# ------------------------------------------------------------------------------------------------ selective scan
def _scan(u, dt, A, B, C_, skip, z, dt_bias, state, cu_seqlens, slots, out, status, softplus, step):
    T = _lead(u, "u", 1)
    dev, channels = u.device, u.shape[2]
    if u.dtype not in TYPES:
        raise _err(f"u must be bf16, fp16 or fp32, got {u.dtype}")
    if dt is None or A is None or B is None or C_ is None:
        raise _err("dt, A, B and C are required")
    _cuda(dev, dt=dt, A=A, B=B, C=C_, D=skip, z=z, dt_bias=dt_bias, out=out)
    if A.dim() != 2 or A.shape[0] != channels or not 1 <= A.shape[1] <= _cabi.SCAN_MAX_STATE or A.dtype != torch.float32:
        raise _err(f"A must be fp32 [{channels}, Ns] with Ns of 1 to {_cabi.SCAN_MAX_STATE}, got {A.dtype} {list(A.shape)}")
    size = A.shape[1]
    groups = B.shape[2] if B.dim() == 4 else 0
    if groups < 1 or channels % groups:
        raise _err(f"B must be [1, T, groups, {size}] with groups dividing {channels}, got {list(B.shape)}")
    _is(dt, "dt", (1, T, channels), u.dtype)
    _is(B, "B", (1, T, groups, size), u.dtype)
    _is(C_, "C", (1, T, groups, size), u.dtype)
    if z is not None:
        _is(z, "z", (1, T, channels), u.dtype)
    A, skip, dt_bias = A.contiguous(), _vector(skip, "D", channels), _vector(dt_bias, "dt_bias", channels)
    inner = (channels, size)
    if step:
        cu, N = None, T
        _step_pool(dev, state, inner, torch.float32)
        src = dst = state
        src_stride = dst_stride = _pool_rows(state, "the pool", inner)
        n_slots, slots = state.shape[0], _step_slots(dev, slots, N, state)
    else:
        cu, N = _layout(dev, cu_seqlens)
        src, src_stride, dst, dst_stride, n_slots, slots = _states(dev, state, slots, N, inner, torch.float32, "the pool")
    u, ldu = _rows(u)
    dt, lddt = _rows(dt)
    B, ldb = _rows(B)
    C_, ldc = _rows(C_)
    ldz = 0
    if z is not None:
        z, ldz = _rows(z)
    y = _out(out, u)
    in_place = src is dst
    if in_place or out is not None or status is not None:
        _reject_aliasing([("out", y), ("the pool", dst), _status(dev, status)], [("u", u), ("dt", dt), ("A", A), ("B", B), ("C", C_), ("D", skip), ("z", z),
                         ("dt_bias", dt_bias), ("cu_seqlens", cu), ("ssm_state_indices", slots), ("initial_state", None if in_place else src)])
    ws_bytes = 0 if step else _cabi.lib().kda_selective_scan_workspace_bytes(T, N, channels, size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    args = _cabi.KdaScanArgs(_ptr(u), _ptr(dt), _ptr(B), _ptr(C_), _ptr(z), _ptr(y), _ptr(A), _ptr(skip), _ptr(dt_bias), _ptr(src), _ptr(dst),
                             ldu, lddt, ldb, ldc, ldz, _rows(y)[1], src_stride, dst_stride,
                             _sequences(T, N, cu, slots, n_slots, status, int(out is None)), channels, size, groups, TYPES[u.dtype],
                             int(bool(softplus)), _ptr(ws), ws_bytes)
    given = {i: [f] for i, f in enumerate(("u", "dt", "A", "B", "C", "D", "z", "dt_bias"))}
    given.update({9: ["seq.cu_seqlens"], 10: ["seq.slots"], 11: ["out"], 12: ["seq.status"]})
    given[8] = ["src", "dst"] if in_place else ["src"]
    fresh = ([(y, ["out"])] if out is None else []) + ([] if in_place else [(dst, ["dst"])])
    result = (11 if out is not None else -1, 8 if in_place else -len(fresh))
    if ws is not None:
        fresh.append((ws, ["workspace"]))
    name = None if step and not T else "kda_selective_scan_step_launch" if step else "kda_selective_scan_launch"
    return _Ready(name, dev, args, given, fresh, result, [11, 12] + [8] * in_place, keep=(u, dt, A, B, C_, skip, z, dt_bias, src, cu, slots))


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, initial_state=None, cu_seqlens=None, *, dt_softplus=True,
                   ssm_state_indices=None, out=None, status=None):
    """Selective state space scan: with s = softplus(dt + dt_bias), per channel d,
    h[n] = exp(s A[d, n]) h[n] + s u B[n];  y = sum_n C[n] h[n] + D[d] u;  y *= silu(z).

    u, dt, z [1, T, channels] and B, C [1, T, groups, Ns] of one type (bf16, fp16 or fp32; any token strides), channel d in group
    d // (channels / groups); A [channels, Ns] (Ns up to 128), D and dt_bias [channels] fp32; D, z and dt_bias may be None, and
    dt_softplus=False takes s = dt + dt_bias.  State fp32: a pool [P, channels, Ns] with `ssm_state_indices`, else
    [N, channels, Ns].  Returns (y, pool or final state)."""
    return _call(_scan, (u, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens, ssm_state_indices, out, status), bool(dt_softplus), False)


def selective_scan_step(u, dt, A, B, C, D, z, dt_bias, pool, ssm_state_indices=None, *, dt_softplus=True, out=None, status=None):
    """The scan of the next token of each row: u, dt, z [1, N, channels], B, C [1, N, groups, Ns].  Returns (y, pool)."""
    return _call(_scan, (u, dt, A, B, C, D, z, dt_bias, pool, None, ssm_state_indices, out, status), bool(dt_softplus), True)


# ------------------------------------------------------------------------------------------------ KDA, one token
def _kda(q, k, v, g, beta, A_log, dt_bias, pool, slots, out, status, scale, raw):
    N = _lead(q, "q", 2)
    dev, H = q.device, q.shape[2]
    if q.shape[3] != D:
        raise _err(f"expected q of shape [1, N, H, 128], got {list(q.shape)}")
    if any(t is None for t in (k, v, g, beta)):
        raise _err("k, v, g and beta are required")
    _cuda(dev, k=k, v=v, g=g, beta=beta, A_log=A_log, dt_bias=dt_bias, out=out)
    for name, t in (("k", k), ("v", v), ("g", g)):
        _is(t, name, (1, N, H, D))
    _is(beta, "beta", (1, N, H))
    bf, gate = torch.bfloat16, torch.bfloat16 if raw else torch.float32
    q, k, v, g, beta = q.to(bf), k.to(bf), v.to(bf), g.to(gate), beta.to(gate)      # as the prefill reads them
    if raw:
        if A_log is None or A_log.numel() != H or dt_bias is None or dt_bias.numel() != H * D:
            raise _err(f"A_log must have {H} and dt_bias {H * D} entries")
        A_log, dt_bias = A_log.to(torch.float32).contiguous(), dt_bias.to(torch.float32).contiguous()
    _step_pool(dev, pool, (H, D, D), torch.float32)
    stride = _pool_rows(pool, "the pool", (H, D, D))
    if stride % 4 or pool.data_ptr() % 16:
        raise _err("pool slots must be 16-byte aligned")
    slots = _step_slots(dev, slots, N, pool)
    (q, ldq), (k, ldk), (v, ldv), (g, ldg), (beta, ldbeta) = map(_rows, (q, k, v, g, beta))
    y = _out(out, q)
    _reject_aliasing([("out", y), ("the pool", pool), _status(dev, status)], [("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta), ("A_log", A_log),
                     ("dt_bias", dt_bias), ("ssm_state_indices", slots)])
    args = _cabi.KdaStepArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(y), _ptr(A_log), _ptr(dt_bias), _ptr(pool), ldq, ldk, ldv,
                             ldg, ldbeta, _rows(y)[1], stride, _sequences(N, N, None, slots, pool.shape[0], status, int(out is None)),
                             float(scale), LOWER_BOUND, _cabi.FRONTEND_RAW if raw else _cabi.FRONTEND_PLAIN, H)
    given = {i: [f] for i, f in enumerate(("q", "k", "v", "g", "beta", "A_log", "dt_bias", "pool", "seq.slots", "out", "seq.status"))}
    fresh = [(y, ["out"])] if out is None else []
    return _Ready("kda_step_launch" if N else None, dev, args, given, fresh, (9 if out is not None else -1, 7), [9, 10, 7], [7],
                  keep=(q, k, v, g, beta, A_log, dt_bias, slots))


def kda_step(q, k, v, g, beta, A_log, dt_bias, scale, pool, ssm_state_indices=None, *, out=None, status=None):
    """The next token of each row after `kda_prefill`, on the same pool (fp32 [P, H, 128 (V), 128 (K)]): q, k, v, g [1, N, H, 128]
    and beta [1, N, H] bf16 with the gate, beta's sigmoid and the L2 norm of q, k computed in the kernel (other types are cast, as
    there).  Returns (o [1, N, H, 128] bf16, pool)."""
    return _call(_kda, (q, k, v, g, beta, A_log, dt_bias, pool, ssm_state_indices, out, status), float(scale), True)


def kda_step_plain(q, k, v, g, beta, scale, pool, ssm_state_indices=None, *, out=None, status=None):
    """The next token of each row after `chunk_kda`: g the fp32 log-decay, beta fp32 in (0, 1), q, k normalised, the pool key-first
    [P, H, 128 (K), 128 (V)].  Returns (o [1, N, H, 128] bf16, pool)."""
    return _call(_kda, (q, k, v, g, beta, None, None, pool, ssm_state_indices, out, status), D ** -0.5 if scale is None else float(scale), False)
