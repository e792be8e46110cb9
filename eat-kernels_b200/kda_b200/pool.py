"""Upkeep of state pools: copying, forking, freeing and compacting slots on the device.

A pool is a tensor [P, ...] with a dense block for each slot: KDA or scan states, convolution histories, whatever type.  Several
pools that one table of slots addresses (`ssm_state_indices` of the layers) are given together.  `used` [P] bool says which slots
are taken; the calls keep it up to date.

    slots = pool_fork([states, histories], used, parents)     # a new slot for each entry, filled with its parent's rows
    pool_free(used, slots)
    remap = pool_compact([states, histories], used, [table])  # the slots in use move to the front, tables follow
    pool_copy([states, histories], src, dst)

Nothing is read on the host: the calls can be captured, and a replay follows the tables.  `status`: an int32 CUDA tensor whose
first entry collects (ORs) the bits 2 = an entry was left out (each call says which) and 32 = no free slot was left."""
from __future__ import annotations

import torch

from . import _cabi, _err, _reject_aliasing
from .serving import _call, _pool_rows, _ptr, _Ready, _status


def _index(t, name, dev=None):
    if not (torch.is_tensor(t) and t.is_cuda and t.dim() == 1 and t.dtype in (torch.int32, torch.int64) and t.is_contiguous()):
        got = f"{t.dtype} {list(t.shape)}" if torch.is_tensor(t) else type(t)
        raise _err(f"{name} must be a contiguous 1-D int32 / int64 CUDA tensor, got {got}")
    if dev is not None and t.device != dev:
        raise _err(f"all CUDA tensors must be on one device ({dev}), got {name} on {t.device}")
    return t


def _args(pools, used, status, dev, slots, written, read):
    """Argument block of a call: pools, `used` and status checked and filled in."""
    a = _cabi.KdaPoolArgs()
    for i, t in enumerate(pools):
        if not (torch.is_tensor(t) and t.is_cuda and t.dim() >= 1):
            raise _err(f"pools[{i}] must be a CUDA tensor [P, ...]")
        dev = t.device if dev is None else dev
        slots = t.shape[0] if slots is None else slots
        if t.device != dev:
            raise _err(f"all CUDA tensors must be on one device ({dev}), got pools[{i}] on {t.device}")
        if t.shape[0] != slots or t.numel() == 0:
            raise _err(f"pools[{i}] must have {slots} slots and no empty dimension, got {list(t.shape)}")
        size = t.element_size()
        a.base[i], a.stride[i] = t.data_ptr(), _pool_rows(t, f"pools[{i}]", tuple(t.shape[1:])) * size
        a.bytes[i] = t.numel() // slots * size
    if slots is None or slots < 1:
        raise _err("at least one pool with at least one slot is needed")
    if used is not None:
        if not (used.dtype == torch.bool and used.is_contiguous()):
            raise _err(f"used must be a contiguous bool tensor [{slots}], got {used.dtype} {list(used.shape)}")
        a.used = used.data_ptr()
    a.slots, a.n_pools = slots, len(pools)
    _reject_aliasing(_extents(a) + [("used", used), _status(dev, status)] + written, read)
    a.status = _ptr(status)
    return a, dev


def _extents(a):
    """Named byte intervals of the pools.  Pools may lie interleaved in one buffer (rows of several layers in one page): with one
    slot stride, and rows that do not overlap within it, they count as one interval."""
    merged = []                                      # [lo, hi, name, [(base, bytes, stride), ...]]
    for i in range(a.n_pools):
        base, size, stride = a.base[i], a.bytes[i], a.stride[i]
        one = [base, base + (a.slots - 1) * stride + size, f"pools[{i}]", [(base, size, stride)]]
        for other in [m for m in merged if m[0] < one[1] and one[0] < m[1]]:
            if all(stride == s and (base - b) % s >= n and (base - b) % s + size <= s for b, n, s in other[3]):
                merged.remove(other)
                one = [min(one[0], other[0]), max(one[1], other[1]), one[2], one[3] + other[3]]
        merged.append(one)
    return [(name, (lo, hi)) for lo, hi, name, _ in merged]


def _used(used):
    if not (torch.is_tensor(used) and used.is_cuda and used.dim() == 1 and used.numel() >= 1):
        raise _err("used must be a CUDA tensor [P]")
    return used.device, used.numel()


def _workspace(a, n, dev):
    nbytes = _cabi.lib().kda_pool_workspace_bytes(n, a.slots)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes, a.n = ws.data_ptr(), nbytes, n
    return ws


def _ready(name, dev, a, first, given, fresh, result, n_pools, written):
    """The pools are the caller's tensors from `first` on."""
    given.update({first + i: [f"base[{i}]"] for i in range(n_pools)})
    return _Ready(name, dev, a, given, fresh, result, [*written, *range(first, first + n_pools)])


def _pools(pools):
    if not isinstance(pools, (list, tuple)) or len(pools) > _cabi.MAX_POOLS:
        raise _err(f"pools must be a list of at most {_cabi.MAX_POOLS} tensors")
    return tuple(pools)


def _copy(src, dst, status, *pools):
    _index(src, "src")
    _index(dst, "dst", src.device)
    if src.numel() != dst.numel():
        raise _err(f"src and dst must have the same number of entries, got {src.numel()} and {dst.numel()}")
    a, dev = _args(pools, None, status, src.device, None, [], [("src", src), ("dst", dst)])
    ws = _workspace(a, src.numel(), dev)
    a.src, a.src_is64, a.dst, a.dst_is64 = _ptr(src), src.dtype == torch.int64, _ptr(dst), dst.dtype == torch.int64
    return _ready("kda_pool_copy_launch" if src.numel() else None, dev, a, 3, {0: ["src"], 1: ["dst"], 2: ["status"]}, [(ws, ["workspace"])], (),
                  len(pools), [2])


def pool_copy(pools, src, dst, *, status=None):
    """Row dst[i] of every pool <- row src[i] (a negative source: zeros; a negative destination: padding).  Left out, with bit 2: an
    entry out of range, a destination that an earlier entry names, and one that any entry reads (the result would depend on the
    order)."""
    _call(_copy, (src, dst, status, *_pools(pools)))


def _fork(used, parents, status, *pools):
    dev, P = _used(used)
    _index(parents, "parents", dev)
    slots = torch.empty(parents.numel(), dtype=torch.int32, device=dev)
    a, dev = _args(pools, used, status, dev, P, [], [("parents", parents)])
    ws = _workspace(a, parents.numel(), dev)
    a.src, a.src_is64, a.slots_out = _ptr(parents), parents.dtype == torch.int64, _ptr(slots)
    return _ready("kda_pool_fork_launch" if parents.numel() else None, dev, a, 3, {0: ["used"], 1: ["src"], 2: ["status"]},
                  [(slots, ["slots_out"]), (ws, ["workspace"])], (-1,), len(pools), [0, 2])


def pool_fork(pools, used, parents, *, status=None):
    """A slot for each entry of `parents`, in order the lowest free ones: marked used, and filled with the parent's row of every
    pool (a negative parent: a new sequence, zeros).  Returns the slots, int32; -1 where the parent is out of range or was not in
    use before the call (bit 2) and where no slot was left (bit 32)."""
    return _call(_fork, (used, parents, status, *_pools(pools)))[0]


def _free(used, slots, status):
    dev, P = _used(used)
    _index(slots, "slots", dev)
    a, dev = _args([], used, status, dev, P, [], [("slots", slots)])
    a.n, a.src, a.src_is64 = slots.numel(), _ptr(slots), slots.dtype == torch.int64
    return _ready("kda_pool_free_launch" if slots.numel() else None, dev, a, 3, {0: ["used"], 1: ["src"], 2: ["status"]}, [], (), 0, [0, 2])


def pool_free(used, slots, *, status=None):
    """Marks slots free (negative entries: padding).  Bit 2: one is out of range, free already or named twice."""
    _call(_free, (used, slots, status))


def _compact(*tensors):
    used, status, *rest = tensors[:-1]
    tables, pools = rest[:tensors[-1]], rest[tensors[-1]:]
    dev, P = _used(used)
    remap = torch.empty(P, dtype=torch.int32, device=dev)
    for i, t in enumerate(tables):
        _index(t, f"tables[{i}]", dev)
    a, dev = _args(pools, used, status, dev, P, [(f"tables[{i}]", t) for i, t in enumerate(tables)], [])
    for i, t in enumerate(tables):
        a.tables[i], a.table_n[i], a.table_is64[i] = _ptr(t), t.numel(), t.dtype == torch.int64
    a.n_tables, a.remap = len(tables), remap.data_ptr()
    ws = _workspace(a, 0, dev)
    given = {0: ["used"], 1: ["status"], **{2 + i: [f"tables[{i}]"] for i in range(len(tables))}}
    return _ready("kda_pool_compact_launch", dev, a, 2 + len(tables), given, [(remap, ["remap"]), (ws, ["workspace"])], (-1,), len(pools),
                  [0, 1, *range(2, 2 + len(tables))])


def pool_compact(pools, used, tables=(), *, status=None):
    """With m slots in use, moves those behind the first m, in order, into the holes among them: `used` becomes m ones and then
    zeros, and the entries of `tables` (slot tables, at most 8; negative entries: padding) follow.  An entry that names no slot in
    use becomes -1 (bit 2).  Returns where each slot went, int32 [P], -1 for those that were free."""
    if not isinstance(tables, (list, tuple)) or len(tables) > _cabi.MAX_TABLES:
        raise _err(f"tables must be a list of at most {_cabi.MAX_TABLES} tensors")
    return _call(_compact, (used, status, *tables, *_pools(pools)), len(tables))[0]
