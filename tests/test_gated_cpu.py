"""What the gated linear recurrence and the group norm refuse without a device, and the oracle's own gradients."""
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


def _seq(N, T, **more):
    from kda_b200 import _cabi
    s = _cabi.KdaSequences()
    s.N, s.T, s.n_slots = N, T, N
    for name, value in more.items():
        setattr(s, name, value)
    return s


def _scan():
    from kda_b200 import _cabi
    a = _cabi.KdaGatedScanArgs()
    a.x = a.r = a.i = a.out = a.rate = a.r_bias = a.i_bias = a.src = a.dst = AT
    a.ldx = a.ldr = a.ldi = a.ldo = a.C = a.src_slot_stride = a.dst_slot_stride = 64
    a.rate_scale, a.seq = 8.0, _seq(2, 2, cu_seqlens=AT)
    return a


def _grad():
    from kda_b200 import _cabi
    a = _cabi.KdaGatedScanGradArgs()
    a.x = a.r = a.i = a.dy = a.dx = a.dr = a.di = a.rate = a.r_bias = a.i_bias = a.tiles = a.src = a.dfinal = a.dsrc = a.drate = a.dr_bias = a.di_bias = AT
    a.ldx = a.ldr = a.ldi = a.lddy = a.lddx = a.lddr = a.lddi = a.C = 64
    a.rate_scale, a.seq = 8.0, _seq(2, 2, cu_seqlens=AT)
    return a


def _norm():
    from kda_b200 import _cabi
    a = _cabi.KdaGroupNormArgs()
    a.x = a.z = a.dy = a.out = a.dz = a.weight = a.bias = a.dweight = a.dbias = a.workspace = AT
    a.T, a.G, a.D, a.workspace_bytes = 2, 2, 32, 1 << 30
    a.ldx = a.ldz = a.lddy = a.ldo = a.lddz = 64
    return a


CASES = [(_scan, ["kda_gated_scan_launch", "kda_gated_scan_step_launch"],
          [dict(C=0), dict(type=3), dict(type=-1), dict(x=None), dict(r=None), dict(out=None), dict(ldx=63), dict(ldr=63), dict(ldi=63), dict(ldo=63), dict(i=None),
           dict(src_slot_stride=63), dict(dst_slot_stride=63), dict(x=AT + 1), dict(i=AT + 1), dict(rate=AT + 2), dict(src=AT + 2, dst=AT + 2)]),
         (_grad, ["kda_gated_scan_grad_launch"],
          [dict(C=0), dict(type=3), dict(x=None), dict(r=None), dict(dx=None), dict(dr=None), dict(di=None), dict(i=None), dict(tiles=None), dict(ldx=63), dict(ldr=63),
           dict(ldi=63), dict(lddy=63), dict(lddx=63), dict(lddr=63), dict(lddi=63), dict(rate=None), dict(dx=AT + 1), dict(tiles=AT + 2), dict(drate=AT + 1)]),
         (_norm, ["kda_group_norm_launch", "kda_group_norm_grad_launch"],
          [dict(T=-1), dict(G=0), dict(D=0), dict(type=3), dict(act=3), dict(act=-1), dict(x=None), dict(out=None), dict(ldx=63), dict(ldz=63), dict(ldo=63), dict(x=AT + 1),
           dict(z=AT + 1), dict(weight=AT + 2), dict(bias=AT + 1)]),
         (_norm, ["kda_group_norm_grad_launch"], [dict(dy=None), dict(dz=None), dict(lddy=63), dict(lddz=63), dict(workspace=None), dict(workspace=AT + 8), dict(dweight=AT + 2)])]


@pytest.mark.parametrize("make,names,bad", CASES, ids=[names[-1] + str(len(names)) for _, names, _ in CASES])
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
    for make, name in ((_scan, "kda_gated_scan_launch"), (_grad, "kda_gated_scan_grad_launch")):
        for seq in (_seq(0, 2, cu_seqlens=AT), _seq(2, 2), _seq(1, -1), _seq(2, 2, cu_seqlens=AT + 4, cu_is64=1), _seq(1, 2, status=AT + 1)):
            a = make()
            a.seq = seq
            assert getattr(lib, name)(a, None) == -1
        a = make()
        a.seq = _seq(1, 1 << 31)
        assert getattr(lib, name)(a, None) == -4
    a = _grad()
    a.seq = _seq(2, 2, cu_seqlens=AT, slots=AT)                      # gradients belong to states of their own
    assert lib.kda_gated_scan_grad_launch(a, None) == -1
    for seq in (_seq(2, 3), _seq(2, 2, n_slots=1)):
        a = _scan()
        a.seq = seq
        assert lib.kda_gated_scan_step_launch(a, None) == -1
    a = _scan()
    a.seq, a.dst = _seq(2, 2), AT + 64                               # a step works in place
    assert lib.kda_gated_scan_step_launch(a, None) == -1
    a = _scan()
    a.seq = _seq(0, 0)
    assert lib.kda_gated_scan_step_launch(a, None) == 0
    for change, code in ((dict(D=16385, ldx=1 << 20, ldz=1 << 20, lddy=1 << 20, ldo=1 << 20, lddz=1 << 20), -4), (dict(T=1 << 31), -4), (dict(G=1 << 30), -4)):
        for name in ("kda_group_norm_launch", "kda_group_norm_grad_launch"):
            a = _norm()
            for field, value in change.items():
                setattr(a, field, value)
            assert getattr(lib, name)(a, None) == code
    a = _norm()
    a.workspace_bytes = lib.kda_group_norm_workspace_bytes(2, 2, 32, 0, 0) - 1
    assert lib.kda_group_norm_grad_launch(a, None) == -2
    a = _norm()
    a.T = 0
    assert lib.kda_group_norm_launch(a, None) == 0
    bad = [(-1, 2, 32, 0, 0), (2, 0, 32, 0, 0), (2, 2, 0, 0, 0), (2, 2, 16385, 0, 0), (2, 2, 32, 3, 0)]
    assert all(lib.kda_group_norm_workspace_bytes(*v) == 0 for v in bad)
    for T in (1, 7, 1000, 1 << 20):                                  # a workspace never has to hold more than the card's blocks leave
        for G, D in ((1, 8), (7, 67), (64, 128), (300, 16), (2, 2500), (1, 16384)):
            for shared in (0, 1):
                assert 0 < lib.kda_group_norm_workspace_bytes(T, G, D, 0, shared) <= 64 << 20


def test_host_tensors_are_refused():
    import kda_b200
    x, pool = torch.zeros(1, 4, 64), torch.zeros(4, 64)
    for call in (lambda: kda_b200.gated_scan(x, x), lambda: kda_b200.gated_scan(x.requires_grad_(), x), lambda: kda_b200.gated_scan_step(x, x, None, None, None, None, pool),
                 lambda: kda_b200.group_norm(x, 4), lambda: kda_b200.group_norm(x.requires_grad_(), 4), lambda: kda_b200.group_norm(None, 4)):
        with pytest.raises(ValueError, match="KDA kernel"):
            call()
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="rate_scale"):
            kda_b200.gated_scan(x, x, rate_scale=bad)
    for bad in (-1e-5, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            kda_b200.group_norm(x, 4, eps=bad)


def test_the_oracles_formulas_are_the_definitions_gradients(monkeypatch):
    import gated_testlib as g
    gen = torch.Generator().manual_seed(1)
    lens, T, Ch = [7, 0, 1, 12], 20, 3
    for form, gated in (("power", 1), ("power", 0), ("logistic", 1), ("logistic", 0)):
        rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
        tensors = [rn(T, Ch), rn(T, Ch), rn(T, Ch) if gated else None, rn(Ch) - 4.0 if form == "power" else None, rn(Ch), rn(Ch) if gated else None]
        states, dy, dfinal = rn(4, Ch), rn(T, Ch), rn(4, Ch)
        for w, a in zip(g.gradients64(lens, tensors, states, dy, dfinal), g.autograd64(lens, tensors, states, dy, dfinal)):
            assert (w is None) == (a is None)
            if w is not None:
                torch.testing.assert_close(w[0], a, rtol=1e-10, atol=1e-12)
                assert (w[1] >= 0).all()
