"""Gates that are shut: what stands behind an infinitely low gate does not count, and a low one counts with its own value."""
import pytest
import torch

from gated_testlib import forward64
from serving_testlib import DEV, assert_within, cu_of, generator, randn
from test_gpu_gated_scan import inputs, rows

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
LOW = float("-inf")


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form", ["power", "logistic"])
def test_tokens_behind_a_shut_input_gate_do_not_count(dtype, form):
    import kda_b200
    for C in (64, 33):
        gen, lens = generator(41 + C), [30, 1, 160]
        x, r, i, rate, rb, ib = inputs(gen, sum(lens), C, dtype, form, 1)
        shut = torch.rand(i.shape, generator=gen, device=DEV) < 0.3
        shut[0, :31], shut[..., :3] = True, True                   # whole sequences, whole channels
        states = randn(gen, 3, C)
        none, masked = x.masked_fill(shut, 0.0), i.masked_fill(shut, LOW)
        for h0 in (states, torch.zeros_like(states)):
            y, final = kda_b200.gated_scan(x, r, masked, rate, rb, ib, h0, cu_of(lens))
            want, wf = kda_b200.gated_scan(none, r, i, rate, rb, ib, h0, cu_of(lens))
            assert torch.equal(y, want) and torch.equal(final, wf)
        pool, other = randn(gen, 191, C), None
        other = pool.clone()
        y, _ = kda_b200.gated_scan_step(x, r, masked, rate, rb, ib, pool)
        want, _ = kda_b200.gated_scan_step(none, r, i, rate, rb, ib, other)
        assert torch.equal(y, want) and torch.equal(pool, other)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_low_input_gates_count_with_their_own_value(dtype):
    """Down to 2^-63, where nothing larger covers them: no states, and gates as low in all of a channel."""
    import kda_b200
    gen, lens, C = generator(43), [70, 40], 64
    x, r, i, rate, rb, _ = inputs(gen, 110, C, dtype, "power", 1)
    i = (-torch.linspace(20.0, 43.5, C, device=DEV).to(dtype).expand_as(i)).contiguous()
    states = torch.zeros(2, C, device=DEV)
    y, final = kda_b200.gated_scan(x, r, i, rate, rb, None, states, cu_of(lens))
    want, e, wf, fe = forward64(lens, x[0], r[0], rows(i), rate, rb, None, states)
    assert_within(y[0], want, e, "y")
    assert_within(final, wf, fe, "final state")


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
def test_a_shut_output_gate_gives_zeros(dtype):
    import kda_b200
    for G, D in ((6, 128), (3, 45), (1, 1500)):
        gen = generator(44 + D)
        x, z, dy = (randn(gen, 1, 9, G * D, dtype=dtype) for _ in range(3))
        shut = torch.rand(z.shape, generator=gen, device=DEV) < 0.3
        z = z.masked_fill(shut, LOW).requires_grad_()
        y = kda_b200.group_norm(x, G, None, None, z, activation="sigmoid")
        open_, dz = kda_b200.group_norm(x, G, None, None, z.detach().masked_fill(shut, 0.5), activation="sigmoid"), torch.autograd.grad(y, z, dy)[0]
        assert (y[shut] == 0).all() and (dz[shut] == 0).all() and torch.equal(y[~shut], open_[~shut])


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form", ["power", "logistic"])
def test_nothing_flows_back_through_a_shut_input_gate(dtype, form):
    """Its token gets zeros and so does the gate; everything else is as for a token of zeros there."""
    import kda_b200
    for C in (64, 33):
        gen, lens = generator(45 + C), [30, 1, 160]
        x, r, i, rate, rb, ib = inputs(gen, sum(lens), C, dtype, form, 1)
        shut = torch.rand(i.shape, generator=gen, device=DEV) < 0.3
        states, dy, dfinal, got = randn(gen, 3, C), randn(gen, *x.shape, dtype=dtype), randn(gen, 3, C), []
        for xs, gate in ((x, i.masked_fill(shut, LOW)), (x.masked_fill(shut, 0.0), i)):
            v = [t.detach().requires_grad_() for t in (xs, r, gate, *(t for t in (rate, rb, ib, states) if t is not None))]
            it = iter(v[3:])
            out = kda_b200.gated_scan(*v[:3], next(it) if rate is not None else None, *it, cu_of(lens))
            got.append(torch.autograd.grad(out, v, (dy, dfinal)))
        masked, none = got
        assert (masked[0][shut] == 0).all() and (masked[2][shut] == 0).all()
        assert torch.equal(masked[0][~shut], none[0][~shut]) and all(torch.equal(a, b) for a, b in zip(masked[1:], none[1:]))
