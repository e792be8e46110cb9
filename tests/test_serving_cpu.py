"""What the operators around the prefill refuse, without a device: argument errors of the Python entry points and error codes of
the C entry points (nothing is launched)."""
import ctypes as C

import pytest
import torch

import __graft_entry__ as entry

AT = 0x10000


@pytest.fixture(scope="module")
def lib():
    entry.build()
    from kda_b200 import _cabi
    return _cabi.lib()


def test_struct_layouts_match(lib):
    from kda_b200 import _cabi
    for i, block in enumerate(_cabi.STRUCTS):
        assert lib.kda_abi_struct_bytes(i) == C.sizeof(block)
    assert lib.kda_abi_struct_bytes(len(_cabi.STRUCTS)) == 0
    for name in _cabi.EXPORTS:
        assert hasattr(lib, name)


def _seq(N, T, **more):
    from kda_b200 import _cabi
    s = _cabi.KdaSequences()
    s.N, s.T, s.n_slots = N, T, N
    for name, value in more.items():
        setattr(s, name, value)
    return s


def _conv():
    from kda_b200 import _cabi
    a = _cabi.KdaConvArgs()
    a.x = a.weight = a.out = a.src = a.dst = AT
    a.ldx = a.ldo = a.C = 64
    a.W, a.src_slot_stride, a.dst_slot_stride = 4, 192, 192
    a.seq = _seq(2, 2, cu_seqlens=AT)
    return a


def _scan():
    from kda_b200 import _cabi
    a = _cabi.KdaScanArgs()
    a.u = a.dt = a.B = a.C = a.out = a.A = a.src = a.dst = AT
    a.ldu = a.lddt = a.ldo = a.Dm = 64
    a.ldb = a.ldc = a.Ns = 16
    a.groups, a.src_slot_stride, a.dst_slot_stride = 1, 1024, 1024
    a.seq = _seq(2, 2, cu_seqlens=AT)
    return a


def _step():
    from kda_b200 import _cabi
    a = _cabi.KdaStepArgs()
    a.q = a.k = a.v = a.g = a.beta = a.out = a.A_log = a.dt_bias = a.pool = AT
    a.ldq = a.ldk = a.ldv = a.ldg = a.ldo = 256
    a.ldbeta = a.H = 2
    a.slot_stride = 2 * 16384
    a.seq = _seq(2, 2)
    return a


def _pool():
    from kda_b200 import _cabi
    a = _cabi.KdaPoolArgs()
    a.base[0], a.stride[0], a.bytes[0] = AT, 64, 64
    a.slots, a.n_pools, a.n = 8, 1, 2
    a.used = a.src = a.dst = a.slots_out = a.remap = a.workspace = AT
    a.workspace_bytes = 1 << 20
    return a


CASES = [(_conv, ["kda_short_conv_launch", "kda_short_conv_step_launch"],
          [dict(C=0), dict(W=1), dict(W=5), dict(type=3), dict(weight_type=-1), dict(x=None), dict(out=None), dict(weight=None), dict(ldx=63), dict(ldo=63),
           dict(src_slot_stride=191), dict(dst_slot_stride=191), dict(x=AT + 1), dict(out=AT + 1), dict(src=AT + 1, dst=AT + 1), dict(bias=AT + 1)]),
         (_scan, ["kda_selective_scan_launch", "kda_selective_scan_step_launch"],
          [dict(Dm=0), dict(Ns=0), dict(groups=0), dict(groups=3), dict(type=7), dict(A=None), dict(u=None), dict(dt=None), dict(B=None), dict(C=None),
           dict(out=None), dict(ldu=63), dict(ldb=15), dict(ldc=15), dict(z=AT, ldz=63), dict(dst_slot_stride=1023), dict(A=AT + 2), dict(u=AT + 1)]),
         (_step, ["kda_step_launch"],
          [dict(H=0), dict(frontend=2), dict(A_log=None), dict(dt_bias=None), dict(q=None), dict(beta=None), dict(pool=None), dict(pool=AT + 8),
           dict(slot_stride=2 * 16384 + 2), dict(slot_stride=16384), dict(ldq=255), dict(ldbeta=1), dict(out=AT + 1), dict(frontend=1, g=AT + 2)]),
         (_pool, ["kda_pool_copy_launch"], [dict(slots=0), dict(n=-1), dict(src=None), dict(dst=None), dict(n_pools=9), dict(workspace=None), dict(workspace=AT + 2),
                                            dict(src=AT + 2), dict(src=AT + 4, src_is64=1)]),
         (_pool, ["kda_pool_fork_launch"], [dict(used=None), dict(src=None), dict(slots_out=None), dict(slots_out=AT + 1)]),
         (_pool, ["kda_pool_free_launch"], [dict(used=None), dict(src=None), dict(slots=0)]),
         (_pool, ["kda_pool_compact_launch"], [dict(used=None), dict(remap=None), dict(n_tables=9), dict(remap=AT + 2)])]


@pytest.mark.parametrize("make,names,bad", CASES, ids=[names[0] for _, names, _ in CASES])
def test_bad_argument_blocks(lib, make, names, bad):
    for name in names:
        call = getattr(lib, name)
        assert call(None, None) == -1
        for change in bad:
            a = make()
            for field, value in change.items():
                setattr(a, field, value)
            assert call(a, None) == -1, (name, change)


def test_bad_sequences_and_limits(lib):
    for make, prompt, step in ((_conv, "kda_short_conv_launch", "kda_short_conv_step_launch"), (_scan, "kda_selective_scan_launch", "kda_selective_scan_step_launch")):
        for seq in (_seq(0, 2, cu_seqlens=AT), _seq(2, 2), _seq(1, -1), _seq(2, 2, cu_seqlens=AT, n_slots=1), _seq(2, 2, cu_seqlens=AT + 4, cu_is64=1),
                    _seq(1, 2, slots=AT + 2), _seq(1, 2, status=AT + 1)):
            a = make()
            a.seq = seq
            assert getattr(lib, prompt)(a, None) == -1
        for seq in (_seq(2, 3), _seq(2, 2, n_slots=1)):
            a = make()
            a.seq = seq
            assert getattr(lib, step)(a, None) == -1
        a = make()
        a.seq = _seq(1, 1 << 31)
        assert getattr(lib, prompt)(a, None) == -4
        a = make()
        a.seq, a.dst = _seq(2, 2), AT + 64                           # a step works in place
        assert getattr(lib, step)(a, None) == -1
    a = _scan()
    a.Ns = 129
    assert lib.kda_selective_scan_launch(a, None) == -4
    a = _scan()
    a.seq = _seq(262141, 262141)
    assert lib.kda_selective_scan_step_launch(a, None) == -4
    a = _step()
    a.H = 65536
    assert lib.kda_step_launch(a, None) == -4
    for make, name in ((_conv, "kda_short_conv_step_launch"), (_scan, "kda_selective_scan_step_launch"), (_step, "kda_step_launch")):
        a = make()
        a.seq = _seq(2, 2, n_slots=1 << 31)
        assert getattr(lib, name)(a, None) == -4
    a = _scan()                                                      # a long axis on few channels needs a workspace
    a.seq = _seq(1, 4096)
    need = lib.kda_selective_scan_workspace_bytes(4096, 1, 64, 16)
    assert need > 0 and lib.kda_selective_scan_launch(a, None) == -1
    a.workspace, a.workspace_bytes = AT, need - 1
    assert lib.kda_selective_scan_launch(a, None) == -2
    a.workspace, a.workspace_bytes = AT + 8, need
    assert lib.kda_selective_scan_launch(a, None) == -1
    assert lib.kda_selective_scan_workspace_bytes(100, 1, 64, 16) == lib.kda_selective_scan_workspace_bytes(4096, 0, 64, 16) == 0
    a = _pool()
    a.workspace_bytes = lib.kda_pool_workspace_bytes(2, 8) - 1
    assert lib.kda_pool_copy_launch(a, None) == -2
    assert lib.kda_pool_workspace_bytes(-1, 8) == 0 and lib.kda_pool_workspace_bytes(3, 0) == 0
    a = _pool()
    a.stride[0] = 32
    assert lib.kda_pool_copy_launch(a, None) == -1
    a = _pool()
    a.slots = 1 << 31
    assert lib.kda_pool_copy_launch(a, None) == -4
    # nothing to do is no launch
    a = _pool()
    a.n = 0
    assert lib.kda_pool_copy_launch(a, None) == lib.kda_pool_fork_launch(a, None) == lib.kda_pool_free_launch(a, None) == 0
    for make, step in ((_conv, "kda_short_conv_step_launch"), (_scan, "kda_selective_scan_step_launch"), (_step, "kda_step_launch")):
        a = make()
        a.seq = _seq(0, 0)
        assert getattr(lib, step)(a, None) == 0


def test_host_tensors_are_refused():
    import kda_b200
    x, w, pool = torch.zeros(1, 4, 64), torch.zeros(64, 4), torch.zeros(4, 3, 64)
    t = torch.zeros(1, 4, 2, 128)
    for call in (lambda: kda_b200.short_conv(x, w), lambda: kda_b200.short_conv_step(x, w, None, pool), lambda: kda_b200.selective_scan(x, x, w, x, x),
                 lambda: kda_b200.selective_scan_step(x, x, w, x, x, None, None, None, pool),
                 lambda: kda_b200.kda_step(t, t, t, t, t[..., 0], w, w, 0.1, pool), lambda: kda_b200.kda_step_plain(t, t, t, t, t[..., 0], None, pool),
                 lambda: kda_b200.pool_copy([pool], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
                 lambda: kda_b200.pool_fork([pool], torch.zeros(4, dtype=torch.bool), torch.zeros(1, dtype=torch.int32)),
                 lambda: kda_b200.pool_free(torch.zeros(4, dtype=torch.bool), torch.zeros(1, dtype=torch.int32)),
                 lambda: kda_b200.pool_compact([pool], torch.zeros(4, dtype=torch.bool))):
        with pytest.raises(ValueError, match="KDA kernel"):
            call()


def test_registers_of_the_convolution_fit():
    """No type or width spills more than a few registers in the prompt kernel (one cap for all types left 296 bytes in fp32)."""
    import re
    import subprocess

    from kda_b200 import _build
    r = subprocess.run([_build.nvcc_path(), *_build.NVCC_FLAGS, "-Xptxas", "-v", "-cubin", "-o", "/dev/null", str(_build.CSRC / "kda_conv.cu")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    spills = re.findall(r"Function properties for \S*kda_short_conv_kernel\S*\n.*?(\d+) bytes spill loads", r.stderr)
    assert len(spills) == 18 and max(map(int, spills)) <= 64, spills
