"""Arguments of the gated linear recurrence and the group norm that 32-bit fields of the entry points cannot hold, and tangents."""
import pytest
import torch

from test_gated_cpu import _grad, _scan, _seq, lib  # noqa: F401


def test_channels_that_index_arithmetic_cannot_hold(lib):  # noqa: F811
    """Refused before anything is launched: blocks and channels are counted in 32 bits, with a block's width on top."""
    wide = 1 << 31
    for make, names in ((_scan, ["kda_gated_scan_launch", "kda_gated_scan_step_launch"]), (_grad, ["kda_gated_scan_grad_launch"])):
        for name in names:
            for C in ((1 << 30) + 1, (1 << 31) - 1):
                a = make()
                a.C = C
                for field, _ in a._fields_:
                    if field.startswith("ld") or field.endswith("_stride"):
                        setattr(a, field, wide)
                a.seq = _seq(2, 2) if "step" in name else a.seq
                assert getattr(lib, name)(a, None) == -4, (name, C)


def test_numbers_that_32_bits_do_not_hold():
    """A positive number must still be one in 32 bits: 1e39 would be infinite there and 1e-50 zero."""
    import kda_b200
    x = torch.zeros(1, 4, 64)
    for bad in (1e39, 1e-50):
        with pytest.raises(ValueError, match="rate_scale"):
            kda_b200.gated_scan(x, x, rate_scale=bad)
        with pytest.raises(ValueError, match="rate_scale"):
            kda_b200.gated_scan_step(x, x, None, None, None, None, x[0], rate_scale=bad)
    with pytest.raises(ValueError, match="eps"):
        kda_b200.group_norm(x, 4, eps=1e39)


def test_tangents_are_refused():
    """Forward-mode derivatives are not offered; without a word they would be lost, which counts as zero."""
    import torch.autograd.forward_ad as fwd

    import kda_b200
    x = torch.zeros(1, 4, 64)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: kda_b200.gated_scan(d, x), lambda: kda_b200.gated_scan(x, d), lambda: kda_b200.gated_scan(x, x, initial_state=d[0]),
                     lambda: kda_b200.gated_scan_step(x, x, d, None, None, None, x[0]), lambda: kda_b200.gated_scan_step(x, x, None, None, None, None, d[0]),
                     lambda: kda_b200.group_norm(d, 4), lambda: kda_b200.group_norm(x, 4, z=d), lambda: kda_b200.group_norm(x, 4, d[0, 0])):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA tensor"):           # others go on to the other checks
            kda_b200.gated_scan(x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        kda_b200.group_norm(x, 4)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda t: kda_b200.group_norm(t, 4), (x,), (torch.ones_like(x),))
