"""Group norm with an activation and its gradients against the definition in 64 bits; and a layer of it behind the recurrence."""
import pytest
import torch

from gated_testlib import U, norm64, norm_bounds
from serving_testlib import DEV, assert_within, cu_of, generator, randn

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def case(T, G, D, dtype, z, shared, seed, scale=1.0, shift=0.0):
    gen, n = generator(seed), D if shared else G * D
    x = (randn(gen, 1, T, G * D) * scale + shift).to(dtype)
    return x, 1.0 + randn(gen, n, scale=0.3), randn(gen, n, scale=0.3), randn(gen, 1, T, G * D, dtype=dtype) if z else None, randn(gen, 1, T, G * D, dtype=dtype)


def check(T, G, D, dtype, act="silu", z=True, center=True, shared=False, seed=0, eps=1e-5, weight=True, bias=True, **more):
    import kda_b200
    x, w, b, zz, dy = case(T, G, D, dtype, z, shared, seed, **more)
    w, b = w if weight else None, b if bias else None
    v = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, zz)]
    y = kda_b200.group_norm(v[0], G, *v[1:], activation=act, eps=eps, center=center)
    plain = kda_b200.group_norm(x, G, w, b, zz, activation=act, eps=eps, center=center)
    assert torch.equal(y, plain) and y.dtype == dtype and y.shape == x.shape
    some = [t for t in v if t is not None]
    grads = torch.autograd.grad(y, some, dy)
    d = [t.detach().double().requires_grad_() if t is not None else None for t in (x[0], w, b, zz[0] if z else None)]
    want = norm64(d[0], G, *d[1:], act, eps, center)
    wants = torch.autograd.grad(want, [t for t in d if t is not None], dy[0].double())
    bounds = norm_bounds(x[0], G, w, b, zz[0] if z else None, act, eps, center, dy[0])
    assert_within(y[0], want.detach(), bounds[0], "y")
    for name, g, ref, e in zip(["d" + n for n, t in zip(("x", "weight", "bias", "z"), v) if t is not None], grads, wants, bounds[1:]):
        assert_within(g.reshape(ref.shape), ref, e.reshape(ref.shape), name)
    v = [t.detach().requires_grad_() for t in some]          # the same bits again
    it = iter(v)
    v = [next(it) if t is not None else None for t in (x, w, b, zz)]
    again = torch.autograd.grad(kda_b200.group_norm(v[0], G, *v[1:], activation=act, eps=eps, center=center), [t for t in v if t is not None], dy)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


SHAPES = [(1, 1, 8), (5, 3, 67), (100, 64, 128), (33, 7, 80), (700, 16, 64), (9, 1, 1000), (50, 40, 8), (17, 3, 700), (301, 5, 24), (2, 300, 16), (40, 2, 1024), (7, 33, 1),
          (3, 1, 2500), (11, 2, 1030), (64, 130, 3)]


@pytest.mark.parametrize("T,G,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
def test_shapes(T, G, D, dtype):
    check(T, G, D, dtype, seed=T + D, center=D > 1)


@pytest.mark.parametrize("act", ["silu", "sigmoid", None])
@pytest.mark.parametrize("z,center,shared", [(0, 1, 0), (1, 1, 1), (1, 0, 1), (0, 0, 0), (1, 0, 0)])
def test_forms(act, z, center, shared):
    for T, G, D in ((37, 6, 128), (20, 3, 45), (5, 2, 1500)):
        for dtype in (BF, F32):
            check(T, G, D, dtype, act, bool(z), bool(center), bool(shared), seed=3)


def test_without_weight_or_bias():
    check(40, 8, 64, BF, weight=False, bias=False, seed=4)
    check(40, 8, 64, F32, bias=False, shared=True, seed=5)
    check(40, 3, 37, F32, weight=False, seed=6)
    check(6, 2, 1500, BF, weight=False, bias=False, seed=7)


def test_means_far_from_zero_and_small_values():
    check(40, 8, 64, F32, seed=8, shift=100.0)
    check(40, 3, 45, F32, seed=9, shift=-30.0)
    check(4, 2, 2000, F32, seed=10, shift=50.0)
    check(40, 8, 64, F32, seed=11, scale=1e-3, eps=1e-6)
    check(40, 8, 64, BF, seed=12, scale=1e3)


def test_constant_groups_and_many_rows():
    import kda_b200
    x = torch.full((1, 3, 256), 7.0, device=DEV)
    y = kda_b200.group_norm(x, 2)
    assert (y == 0).all()                                     # sums of 128 sevens and their mean are whole
    check(20000, 2, 64, BF, seed=13)
    check(5000, 3, 50, F32, seed=14, shared=True)


def test_widest_groups():
    check(3, 1, 16384, BF, seed=15)
    check(2, 2, 16383, F32, seed=16, shared=True)


def test_head_layout_views_and_out():
    import kda_b200
    for dtype, T, G, D in ((BF, 30, 6, 128), (F32, 20, 3, 45), (BF, 9, 2, 1500)):
        x, w, b, z, dy = case(T, G, D, dtype, True, False, 17)
        want = kda_b200.group_norm(x, G, w, b, z, activation="silu")
        heads = x.view(1, T, G, D)
        assert torch.equal(kda_b200.group_norm(heads, None, w.view(G, D), b, z.view(1, T, G, D), activation="silu").view_as(want), want)
        for shift in (0, 1):
            room = torch.zeros(1, T, 2 * G * D + 16 + shift, dtype=dtype, device=DEV)
            v = [room[..., shift + k * (G * D + 8):][..., :G * D] for k in range(2)]
            v[0].copy_(x)
            v[1].copy_(z)
            out = torch.zeros(1, T, G * D + 8, dtype=dtype, device=DEV)
            got = kda_b200.group_norm(v[0], G, w, b, v[1], activation="silu", out=out[..., :G * D])
            assert got.data_ptr() == out.data_ptr() and (out[..., G * D:] == 0).all()
            torch.testing.assert_close(got, want, rtol=2 * torch.finfo(dtype).eps, atol=64 * U)
            leaves = [t.detach().requires_grad_() for t in (v[0], w, b, v[1])]
            a = torch.autograd.grad(kda_b200.group_norm(leaves[0], G, *leaves[1:], activation="silu"), leaves, dy)
            leaves = [t.detach().requires_grad_() for t in (x, w, b, z)]
            for p, q in zip(a, torch.autograd.grad(kda_b200.group_norm(leaves[0], G, *leaves[1:], activation="silu"), leaves, dy)):
                torch.testing.assert_close(p, q, rtol=max(2 * torch.finfo(p.dtype).eps, 1e-5), atol=1e-4)


def test_no_rows_and_rows_behind_2_to_the_31_elements():
    import kda_b200
    x, w, b, z, dy = case(4, 2, 64, F32, True, False, 18)
    v = [t.detach().requires_grad_() for t in (x[:, :0], w, b, z[:, :0])]
    y = kda_b200.group_norm(v[0], 2, *v[1:])
    grads = torch.autograd.grad(y, v, dy[:, :0])
    assert y.shape == (1, 0, 128) and (grads[1] == 0).all() and (grads[2] == 0).all()
    ld, T = 1 << 27, 20
    room = torch.empty(ld * (T - 1) + 256, dtype=BF, device=DEV)
    x, w, b, z, dy = case(T, 2, 64, BF, True, False, 19)
    far = [room.as_strided((1, T, 128), (0, ld, 1), k * 128) for k in range(2)]
    far[0].copy_(x)
    far[1].copy_(z)
    want = kda_b200.group_norm(x, 2, w, b, z, activation="silu")
    assert torch.equal(kda_b200.group_norm(far[0], 2, w, b, far[1], activation="silu"), want)
    kda_b200.group_norm(x, 2, w, b, z, activation="silu", out=far[0])
    assert torch.equal(far[0], want)


def test_infinities_stay_in_their_group():
    import kda_b200
    x, w, b, z, dy = case(6, 4, 128, BF, True, False, 20)
    clean = kda_b200.group_norm(x, 4, w, b, z, activation="sigmoid")
    x[0, 2, 130], x[0, 4, 5], z[0, 5, 300] = float("inf"), float("nan"), float("nan")
    y = kda_b200.group_norm(x, 4, w, b, z, activation="sigmoid")
    hit = torch.zeros(6, 512, dtype=torch.bool, device=DEV)
    hit[2, 128:256], hit[4, :128], hit[5, 300] = True, True, True
    assert torch.equal(torch.isnan(y[0]), hit) and torch.equal(y[0][~hit], clean[0][~hit])


def test_differences():
    """Of the kernel's own outputs in 32 bits, along random directions (as for the recurrence)."""
    import kda_b200
    for act, z, center, shared in (("silu", 1, 1, 0), ("sigmoid", 1, 0, 1), ("silu", 0, 1, 1)):
        x, w, b, zz, dy = case(30, 5, 48, F32, z, shared, 21)
        ts = [t for t in (x, w, b, zz) if t is not None]

        def loss(v):
            y = kda_b200.group_norm(v[0], 5, v[1], v[2], v[3] if z else None, activation=act, center=bool(center)).double() * dy
            return y.sum(), y.abs().sum()

        v = [t.detach().requires_grad_() for t in ts]
        grads = torch.autograd.grad(kda_b200.group_norm(v[0], 5, v[1], v[2], v[3] if z else None, activation=act, center=bool(center)), v, dy)
        gen, h = generator(22), 2.0 ** -7
        for k, t in enumerate(ts):
            d = randn(gen, *t.shape)
            (p, mag), (q, _) = (loss([u + s * h * d if j == k else u for j, u in enumerate(ts)]) for s in (1, -1))
            along = (grads[k].double() * d).sum()
            assert ((p - q) / (2 * h) - along).abs() <= 2.0 ** -14 * mag + 1e-3 * (grads[k].double() * d).abs().sum()


def test_captured_training_passes_and_streams():
    import kda_b200
    x, w, b, z, dy = case(60, 8, 64, BF, True, True, 23)

    def grads(ts):
        y = kda_b200.group_norm(ts[0], 8, *ts[1:], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, ts, dy)]

    want = grads([t.detach().requires_grad_() for t in (x, w, b, z)])
    torch.cuda.synchronize()
    v, graph = [t.detach().requires_grad_() for t in (x, w, b, z)], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads(v)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = grads([t.detach().requires_grad_() for t in (x, w, b, z)])
    stream.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other, want))


def test_a_layer_trains_and_generates():
    """Convolution, recurrence and gated norm as a layer runs them: gradients through both differentiable parts against the same layer of
    plain operations, and token by token the prompt's outputs."""
    import kda_b200
    gen, lens, C, G = generator(24), [33, 1, 90], 128, 4
    T = sum(lens)
    xin, r, i, z = (randn(gen, 1, T, C) for _ in range(4))
    cw, rate, rb, w = randn(gen, C, 4, scale=0.5), randn(gen, C) - 5.0, randn(gen, C), 1.0 + randn(gen, C // G, scale=0.2)
    cu = cu_of(lens)
    x, _ = kda_b200.short_conv(xin, cw, None, None, cu)
    v = [t.detach().requires_grad_() for t in (x, r, i, rate, rb, z, w)]
    h, final = kda_b200.gated_scan(v[0], v[1], v[2], v[3], v[4], None, None, cu)
    y = kda_b200.group_norm(h, G, v[6], None, v[5], activation="sigmoid", center=False)
    dy = randn(gen, 1, T, C)
    grads = torch.autograd.grad(y, v, dy)
    d = [t.detach().double().requires_grad_() for t in (x, r, i, rate, rb, z, w)]
    log = -8.0 * torch.nn.functional.softplus(d[3]) * torch.sigmoid(d[1][0] + d[4])
    f, u = log.exp(), (-(2 * log).expm1()).sqrt() * torch.sigmoid(d[2][0]) * d[0][0]
    out, at = [], 0
    for n in lens:
        s = torch.zeros(C, dtype=torch.float64, device=DEV)
        for t in range(at, at + n):
            s = f[t] * s + u[t]
            out.append(s)
        at += n
    want = norm64(torch.stack(out), G, d[6], None, d[5][0], "sigmoid", 1e-5, False)
    torch.testing.assert_close(y[0].double(), want, rtol=2e-4, atol=2e-4)
    for g, e in zip(grads, torch.autograd.grad(want, d, dy[0].double())):
        torch.testing.assert_close(g.double(), e, rtol=2e-3, atol=2e-3 * e.abs().max().item())
    pool, hist = torch.zeros(3, C, device=DEV), torch.zeros(3, 3, C, device=DEV)
    for t in range(90):                                       # the last sequence, one token at a time, in slot 2
        rows = slice(34 + t, 35 + t)
        slot = torch.tensor([2], device=DEV)
        x1, _ = kda_b200.short_conv_step(xin[:, rows], cw, None, hist, slot)
        h1, _ = kda_b200.gated_scan_step(x1, r[:, rows], i[:, rows], rate, rb, None, pool, slot)
        y1 = kda_b200.group_norm(h1, G, w, None, z[:, rows], activation="sigmoid", center=False)
        torch.testing.assert_close(y1, y[:, rows].detach(), rtol=1e-3, atol=1e-4)
    torch.testing.assert_close(pool[2], final[2].detach(), rtol=1e-4, atol=1e-4)
