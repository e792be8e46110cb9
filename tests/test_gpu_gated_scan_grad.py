"""Gradients of the gated linear recurrence: against the formulas in 64 bits with their bounds, against differences, through autograd."""
import pytest
import torch

from gated_testlib import autograd64, gradients64
from serving_testlib import DEV, assert_within, cu_of, generator, randn
from test_gpu_gated_scan import inputs, rows

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ["dx", "dr", "di", "drate", "dr_bias", "di_bias", "dstate"]


def leaves(*tensors):
    return [t.detach().requires_grad_() if t is not None else None for t in tensors]


def grads_of(tensors, cu, dy, dfinal, scale=8.0):
    """Gradients of everything given, in place of it."""
    import kda_b200
    v = leaves(*tensors)
    out = kda_b200.gated_scan(*v, cu, rate_scale=scale)
    pairs = [(o, g) for o, g in zip(out, (dy, dfinal)) if g is not None]
    got = iter(torch.autograd.grad([o for o, _ in pairs], [t for t in v if t is not None], [g for _, g in pairs]))
    return [next(got) if t is not None else None for t in v]


def case(lens, C, dtype, form, gated, seed, biases=True):
    gen, T, N = generator(seed), sum(lens), len(lens)
    return [*inputs(gen, T, C, dtype, form, gated, biases), randn(gen, N, C)], randn(gen, 1, T, C, dtype=dtype), randn(gen, N, C)


def check(lens, C, dtype, form, gated, seed, biases=True):
    tensors, dy, dfinal = case(lens, C, dtype, form, gated, seed, biases)
    got = grads_of(tensors, cu_of(lens), dy, dfinal)
    want = gradients64(lens, [rows(t) for t in tensors[:3]] + tensors[3:6], tensors[6], dy[0], dfinal)
    for name, g, w, t in zip(NAMES, got, want, tensors):
        assert (g is None) == (w is None)
        if g is not None:
            assert g.dtype == t.dtype
            assert_within(g.reshape(w[0].shape), w[0], w[1], name)
    again = grads_of(tensors, cu_of(lens, torch.int32), dy, dfinal)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, again))


LAYOUTS = {"one token": [1], "slice": [6], "borders": [47, 48, 49, 95, 97, 1, 0, 5, 7], "empty ones": [0, 0, 5, 0, 130, 0, 0], "ragged": [70, 1, 2, 300, 3, 64], "nothing": [0],
           "rounds": [1700]}


@pytest.mark.parametrize("lens", LAYOUTS.values(), ids=LAYOUTS.keys())
@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form,gated", [("power", 1), ("power", 0), ("logistic", 1), ("logistic", 0)])
def test_gradients(lens, dtype, form, gated):
    for C in (64, 72, 33):
        check(lens, C, dtype, form, gated, seed=sum(lens) + C)


def test_many_short_sequences_and_no_biases():
    check([(7 * k) % 4 for k in range(700)], 40, BF, "power", 1, seed=5)
    check([100, 30], 64, BF, "power", 1, seed=6, biases=False)
    check([100, 30], 33, F32, "logistic", 0, seed=7, biases=False)


@pytest.mark.parametrize("form,gated", [("power", 1), ("logistic", 0)])
def test_formulas_are_the_definitions_gradients(form, gated):
    lens = [9, 0, 1, 14]
    tensors, dy, dfinal = case(lens, 5, F32, form, gated, 8)
    plain = [rows(t) for t in tensors[:3]] + tensors[3:6]
    for w, a in zip(gradients64(lens, plain, tensors[6], dy[0], dfinal), autograd64(lens, plain, tensors[6], dy[0], dfinal)):
        assert (w is None) == (a is None)
        if w is not None:
            torch.testing.assert_close(w[0], a, rtol=1e-9, atol=1e-11)


def test_differences():
    """L(v + h d) - L(v - h d) of the kernel's own outputs in 32 bits over 2 h, h = 2^-7, against the gradient along d.  What third
    derivatives leave is h^2 / 6 of them, some 1e-5 of the terms' magnitude; the outputs' own errors, 2^-20 of them, over 2 h: 2^-14."""
    import kda_b200
    lens = [40, 1, 130]
    for form, gated in (("power", 1), ("logistic", 1)):
        tensors, dy, dfinal = case(lens, 48, F32, form, gated, 9)
        grads, gen, h = grads_of(tensors, cu_of(lens), dy, dfinal), generator(10), 2.0 ** -7

        def loss(ts):
            y, final = kda_b200.gated_scan(*ts, cu_of(lens))
            return (y.double() * dy).sum() + (final.double() * dfinal).sum(), (y.double() * dy).abs().sum() + (final.double() * dfinal).abs().sum()

        for k, t in enumerate(tensors):
            if t is None:
                continue
            d = randn(gen, *t.shape)
            up, down = ([t + s * h * d if q == k else v for q, v in enumerate(tensors)] for s in (1, -1))
            (a, mag), (b, _) = loss(up), loss(down)
            along = (grads[k].double() * d).sum()
            allowed = 2.0 ** -14 * mag + 1e-3 * (grads[k].double() * d).abs().sum()
            assert ((a - b) / (2 * h) - along).abs() <= allowed, (form, NAMES[k])


def test_parts_of_the_outputs_and_of_the_inputs():
    import kda_b200
    lens = [30, 50]
    tensors, dy, dfinal = case(lens, 64, BF, "power", 1, 11)
    cu = cu_of(lens)
    both, only_y, only_f = (grads_of(tensors, cu, a, b) for a, b in ((dy, dfinal), (dy, torch.zeros_like(dfinal)), (torch.zeros_like(dy), dfinal)))
    for got, want in ((grads_of(tensors, cu, dy, None), only_y), (grads_of(tensors, cu, None, dfinal), only_f)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for k in range(7):                                       # one leaf at a time
        v = [t.detach() for t in tensors]
        v[k].requires_grad_()
        y, final = kda_b200.gated_scan(*v, cu)
        g, = torch.autograd.grad([y, final], [v[k]], [dy, dfinal])
        assert torch.equal(g, both[k]), NAMES[k]
    v = leaves(*tensors)
    y, _ = kda_b200.gated_scan(*v, cu)
    y.sum().backward()                                       # a gradient without strides of its own
    assert all(torch.equal(t.grad, g) for t, g in zip(v, grads_of(tensors, cu, torch.ones_like(dy), None)))
    # rows behind the last sequence: nothing comes from them or goes there
    more = [torch.cat([t, t[:, :7] * float("nan")], 1) for t in tensors[:3]] + tensors[3:]
    got = grads_of(more, cu, torch.cat([dy, dy[:, :7]], 1), dfinal)
    assert all((g[:, 80:] == 0).all() and torch.equal(g[:, :80], w) for g, w in zip(got[:3], both[:3])) and all(torch.equal(a, b) for a, b in zip(got[3:], both[3:]))
    # without initial states, and one sequence without a table
    got = grads_of(tensors[:6] + [None], None, dy, dfinal[:1])
    want = grads_of(tensors[:6] + [torch.zeros(1, 64, device=DEV)], cu_of([80]), dy, dfinal[:1])
    assert all(torch.equal(a, b) for a, b in zip(got[:6], want[:6]))


def test_rejected_layouts_have_no_gradients():
    tensors, dy, dfinal = case([30, 50], 64, F32, "power", 1, 12)
    got = grads_of(tensors, torch.tensor([0, 90, 80], device=DEV), dy, dfinal)
    assert all((g == 0).all() for g in got[:6]) and torch.equal(got[6], dfinal)
    empty = [t[:, :0] for t in tensors[:3]] + tensors[3:]
    got = grads_of(empty, cu_of([0, 0]), dy[:, :0], dfinal)
    assert all((g == 0).all() for g in got[3:6]) and got[0].shape == (1, 0, 64) and torch.equal(got[6], dfinal)


def test_views_give_the_same_gradients():
    for dtype in (BF, F32):
        tensors, dy, dfinal = case([60, 90], 64, dtype, "power", 1, 13)
        want = grads_of(tensors, cu_of([60, 90]), dy, dfinal)
        for shift in (1, 8):
            room = torch.zeros(1, 150, 4 * 72 + shift, dtype=dtype, device=DEV)
            v = [room[..., shift + k * 72:][..., :64] for k in range(4)]
            for a, b in zip(v, (*tensors[:3], dy)):
                a.copy_(b)
            got = grads_of([*v[:3], *tensors[3:]], cu_of([60, 90]), v[3], dfinal)
            for a, b in zip(got[:3], want[:3]):
                torch.testing.assert_close(a, b, rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
            for a, b in zip(got[3:], want[3:]):               # other sums of the same terms
                torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


def test_far_gates_have_finite_gradients():
    for dtype in (BF, F32):
        tensors, dy, dfinal = case([120], 64, dtype, "power", 1, 14)
        x, r, i, rate = tensors[:4]
        r[0, :, :8], r[0, :, 8:16], i[0, :, 16:24], i[0, :, 24:32] = -300.0, 80.0, 80.0, -300.0
        rate[32:40], rate[40:48], rate[48:56] = -200.0, -60.0, 80.0
        for g in grads_of(tensors, cu_of([120]), dy, dfinal):
            assert g is None or torch.isfinite(g).all()
        tensors, dy, dfinal = case([120], 64, dtype, "logistic", 1, 15)
        tensors[1][0, :, :8], tensors[1][0, :, 8:16] = -300.0, 80.0
        for g in grads_of(tensors, cu_of([120]), dy, dfinal):
            assert g is None or torch.isfinite(g).all()


def test_recorded_only_where_gradients_can_flow():
    import kda_b200
    tensors, dy, dfinal = case([30], 64, BF, "power", 1, 16)
    v = leaves(*tensors)
    y, final = kda_b200.gated_scan(*v)
    plain, pf = kda_b200.gated_scan(*tensors)
    assert y.requires_grad and final.requires_grad and torch.equal(y, plain) and torch.equal(final, pf) and not plain.requires_grad
    with torch.no_grad():
        assert not kda_b200.gated_scan(*v)[0].requires_grad
    pool = tensors[6].clone()
    assert not kda_b200.gated_scan(*v[:6], pool, ssm_state_indices=torch.tensor([0], device=DEV))[0].requires_grad
    assert not kda_b200.gated_scan(*v, out=torch.empty_like(dy))[0].requires_grad
    assert not kda_b200.gated_scan_step(*(t[:, :1] for t in v[:3]), *v[3:6], pool)[0].requires_grad
    g, = torch.autograd.grad(y, [v[0]], [torch.ones_like(y).requires_grad_()], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.float().sum().backward()
    y, _ = kda_b200.gated_scan(*v)
    with torch.no_grad():
        v[1].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified"):
        y.float().sum().backward()


def test_captured_training_passes():
    """Forward and backward in one graph, replayed on other values; no eager graph of the leaves lives meanwhile."""
    import kda_b200
    lens = [30, 200]
    tensors, dy, dfinal = case(lens, 72, BF, "power", 1, 17)
    cu = cu_of(lens)
    grads_of(tensors, cu, dy, dfinal)
    torch.cuda.synchronize()
    v, graph = leaves(*tensors), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kda_b200.gated_scan(*v, cu)
        got = torch.autograd.grad(out, v, (dy, dfinal))
    for k in range(2):
        graph.replay()
        torch.cuda.synchronize()
        want = grads_of([t.detach() for t in v], cu, dy, dfinal)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.no_grad():
            for t in (*v, dy):
                t.mul_(0.5)
