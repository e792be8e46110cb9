"""selective_scan and selective_scan_step against the definition in 64 bits, with a running error bound: types, state sizes, groups,
odd channels, strides, lengths from none to long, tables that are wrong, padding, captured calls."""
import math

import pytest
import torch

from serving_testlib import DEV, assert_within, cu_of, generator, randn, scan64

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def make(gen, T, Dm, Ns, G, dtype, gate=True, slow=False):
    A = -torch.arange(1, Ns + 1, device=DEV) * torch.exp(randn(gen, Dm, Ns, scale=0.3))
    step = torch.exp(torch.rand(Dm, generator=gen, device=DEV) * math.log(100.0) + math.log(1e-4 if slow else 1e-3))
    return dict(u=randn(gen, 1, T, Dm, dtype=dtype), dt=randn(gen, 1, T, Dm, dtype=dtype, scale=0.5), A=A, B=randn(gen, 1, T, G, Ns, dtype=dtype),
                C=randn(gen, 1, T, G, Ns, dtype=dtype), D=randn(gen, Dm), z=randn(gen, 1, T, Dm, dtype=dtype) if gate else None,
                dt_bias=step + torch.log(-torch.expm1(-step)))


def at(a, rows):
    return {n: t[:, rows] if t is not None and n in ("u", "dt", "B", "C", "z") else t for n, t in a.items()}


def check(a, init, lens, y, final, softplus=True, what=""):
    t = 0
    for i, n in enumerate(lens):
        s = at(a, slice(t, t + n))
        want, bound, h, E = scan64(s["u"][0], s["dt"][0], a["A"], s["B"][0], s["C"][0], a["D"], s["z"][0] if s["z"] is not None else None,
                                   a["dt_bias"], init[i], softplus)
        assert_within(y[0, t:t + n], want, bound, f"{what} sequence {i}")
        assert_within(final[i], h, E, f"{what} state {i}")
        t += n


@pytest.mark.parametrize("dtype,Dm,Ns,G,lens,gate", [
    (BF, 256, 16, 1, [77], True), (BF, 200, 16, 2, [1, 0, 33, 64, 65, 2], True), (HF, 129, 13, 1, [40, 0, 3], False), (F, 64, 4, 4, [1], True),
    (F, 96, 8, 1, [130, 31], False), (BF, 64, 32, 2, [70, 5], True), (F, 36, 64, 1, [50], True), (HF, 24, 128, 3, [35, 1], True),
    (F, 1, 16, 1, [300], True), (BF, 1000, 16, 1, [1] * 20, True), (F, 33, 1, 1, [0, 9, 0], True), (F, 40, 100, 1, [20], False)])
@pytest.mark.parametrize("pooled", [False, True])
def test_prompts(dtype, Dm, Ns, G, lens, gate, pooled):
    import kda_b200
    gen, N = generator(Dm + Ns), len(lens)
    a = make(gen, sum(lens), Dm, Ns, G, dtype, gate)
    if pooled:
        pool = randn(gen, N + 3, Dm, Ns)
        slots = torch.randperm(N + 3, generator=torch.Generator().manual_seed(3))[:N].to(DEV)
        before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
        y, got = kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu_of(lens), ssm_state_indices=slots, status=status)
        assert got is pool and int(status) == 0
        check(a, before[slots], lens, y, pool[slots])
        rest = [i for i in range(N + 3) if i not in slots.tolist()]
        assert torch.equal(pool[rest], before[rest])
    else:
        init = randn(gen, N, Dm, Ns)
        keep = init.clone()
        y, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of(lens, torch.int32))
        assert torch.equal(init, keep)
        check(a, init, lens, y, final)
        y, final = kda_b200.selective_scan(**a, cu_seqlens=cu_of(lens))
        check(a, torch.zeros_like(init), lens, y, final)


@pytest.mark.parametrize("Dm,T,dtype", [(16, 5000, F), (512, 3000, HF), (96, 2049, BF), (7, 4097, F)])
@pytest.mark.parametrize("slow", [False, True])
def test_long_axes_on_few_channels(Dm, T, dtype, slow):
    import kda_b200
    gen = generator(T)
    a = make(gen, T, Dm, 16, 1, dtype, True, slow)
    lens = [T - 700, 1, 0, 699]
    init = randn(gen, 4, Dm, 16)
    y, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of(lens))
    check(a, init, lens, y, final)
    y, final = kda_b200.selective_scan(**a, initial_state=init[:1])
    check(a, init[:1], [T], y, final)


@pytest.mark.parametrize("Dm,Ns,G,lens,dtype", [(40, 24, 2, [900, 0, 1, 350, 127, 129], BF), (36, 16, 4, [513], F), (64, 100, 1, [600, 5], HF),
                                                (130, 3, 1, [640, 128], BF), (24, 33, 3, [256, 256, 256], F), (256, 8, 1, [1000, 200], HF)])
def test_pieces_over_a_pool(Dm, Ns, G, lens, dtype):
    """Long axes on few channels are cut into pieces: the slots in place, groups, odd state sizes, empty sequences, a repeated slot, rows
    behind the last sequence."""
    import kda_b200
    gen, N, rest = generator(Ns), len(lens), 40
    a = make(gen, sum(lens) + rest, Dm, Ns, G, dtype)
    for n in ("u", "dt", "B", "C", "z"):
        a[n][:, sum(lens):] = float("nan")
    pool = randn(gen, N + 2, Dm, Ns)
    slots = torch.randperm(N + 2, generator=torch.Generator().manual_seed(3))[:N].to(DEV)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, _ = kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu_of(lens), ssm_state_indices=slots, status=status)
    assert int(status) == 0 and bool((y[:, sum(lens):] == 0).all())
    check(a, before[slots], lens, y, pool[slots])
    free = [i for i in range(N + 2) if i not in slots.tolist()]
    assert torch.equal(pool[free], before[free])
    if N > 1:                                                         # the last sequence names the first one's slot
        slots[-1] = slots[0]
        again = before.clone()
        y2, _ = kda_b200.selective_scan(**a, initial_state=again, cu_seqlens=cu_of(lens), ssm_state_indices=slots, status=status)
        init = before[slots].clone()
        init[-1] = 0
        assert int(status) == 2
        want = [again[slots[i]] for i in range(N - 1)] + [kda_b200.selective_scan(**at(a, slice(sum(lens) - lens[-1], sum(lens))))[1][0]]
        check(a, init, lens, y2, torch.stack(want))
    status.zero_()
    bad, keep = torch.tensor([0, *[5] * (N - 1), sum(lens) + rest + 1], device=DEV), before.clone()
    y, _ = kda_b200.selective_scan(**a, initial_state=keep, cu_seqlens=bad, ssm_state_indices=torch.arange(N, device=DEV), status=status)
    assert int(status) == 1 and bool((y == 0).all()) and torch.equal(keep, before)


@pytest.mark.parametrize("N", [129, 300])
def test_many_sequences(N):
    import kda_b200
    gen = generator(N)
    lens = [(7 * i) % 23 for i in range(N)]
    a, init = make(gen, sum(lens), 96, 16, 1, BF), randn(gen, N, 96, 16)
    y, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of(lens))
    check(a, init, lens, y, final)


@pytest.mark.parametrize("leave", ["D", "z", "dt_bias", "all"])
def test_what_may_be_left_out(leave):
    import kda_b200
    gen = generator(12)
    a = make(gen, 50, 72, 16, 1, BF)
    for n in ("D", "z", "dt_bias"):
        if leave in (n, "all"):
            a[n] = None
    y, final = kda_b200.selective_scan(**a)
    check(a, torch.zeros(1, 72, 16, device=DEV), [50], y, final)


@pytest.mark.parametrize("step", [False, True])
def test_step_sizes_as_given_growing_states_and_hard_decays(step):
    """Without the softplus a step may be negative (the state grows); step sizes and rates whose decay underflows; none at all."""
    import kda_b200
    gen = generator(13)
    a = make(gen, 40, 48, 16, 1, F)
    a["dt"] = a["dt"] * 0.3
    a["dt_bias"] = None
    a["A"][:4] = -1e4
    a["dt"][:, 10:14] = 0.0
    init = randn(gen, 40 if step else 1, 48, 16)
    if step:
        pool = init.clone()
        y, _ = kda_b200.selective_scan_step(**{n: a[n] for n in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")}, pool=pool, dt_softplus=False)
        keep = torch.ones(48, dtype=torch.bool, device=DEV)
        keep[:4] = False                                              # those overflow where the step is negative
        part = {n: (t[..., keep] if n in ("u", "dt", "z") else t[keep] if n in ("A", "D") else t) if t is not None else None for n, t in a.items()}
        check(part, init[:, keep], [1] * 40, y[..., keep], pool[:, keep], False)
        return
    a["dt"][..., :4] = a["dt"][..., :4].abs()
    y, final = kda_b200.selective_scan(**a, initial_state=init, dt_softplus=False)
    check(a, init, [40], y, final, False)


def test_large_and_small_step_logits():
    """softplus over its whole range: e^x far below fp32's step at one, x itself far above."""
    import kda_b200
    gen = generator(14)
    a = make(gen, 64, 32, 16, 1, F)
    a["dt"] = torch.linspace(-80.0, 40.0, 64 * 32, device=DEV).view(1, 64, 32)[:, torch.randperm(64, generator=torch.Generator().manual_seed(1)).to(DEV)]
    a["dt_bias"] = None
    y, final = kda_b200.selective_scan(**a)
    check(a, torch.zeros(1, 32, 16, device=DEV), [64], y, final)


@pytest.mark.parametrize("off", [0, 1, 8])
def test_views_are_read_and_written_in_place(off):
    import kda_b200
    gen, lens = generator(15), [40, 25]
    a = make(gen, 65, 256, 16, 1, BF)
    wide = randn(gen, 1, 65, 1200, dtype=BF)
    a["u"], a["z"], a["dt"] = wide[:, :, off:off + 256], wide[:, :, 300 + off:556 + off], wide[:, :, 600 + off:856 + off] * 0.5
    xbc = randn(gen, 1, 65, 1, 50, dtype=BF)
    a["B"], a["C"] = xbc[..., off:off + 16], xbc[..., 20 + off:36 + off]
    target = torch.full((1, 70, 512), 7.0, dtype=BF, device=DEV)
    y, final = kda_b200.selective_scan(**a, cu_seqlens=cu_of(lens), out=target[:, 2:67, off:off + 256])
    check(a, torch.zeros(2, 256, 16, device=DEV), lens, y, final)
    rest = target.clone()
    rest[:, 2:67, off:off + 256] = 7.0
    assert bool((rest == 7.0).all())


def test_rows_behind_the_last_sequence():
    import kda_b200
    gen, lens = generator(16), [10, 60]
    a = make(gen, 100, 136, 16, 1, BF)
    for n in ("u", "dt", "B", "C", "z"):
        a[n][:, 70:] = float("nan")
    y, final = kda_b200.selective_scan(**a, cu_seqlens=cu_of(lens))
    check(a, torch.zeros(2, 136, 16, device=DEV), lens, y, final)
    assert bool((y[:, 70:] == 0).all())
    out = torch.full_like(y, 3.0)
    kda_b200.selective_scan(**a, cu_seqlens=cu_of(lens), out=out)
    assert torch.equal(out[:, :70], y[:, :70]) and bool((out[:, 70:] == 3.0).all())


def test_a_neighbour_that_is_not_a_number_stays_there():
    import kda_b200
    gen, lens = generator(17), [32, 33, 31]
    a = make(gen, 96, 40, 16, 1, F)
    pool = randn(gen, 5, 40, 16)
    for n in ("u", "dt", "B", "C", "z"):
        a[n][:, :32] = float("nan")
    pool[[0, 2]] = float("inf")
    before, slots = pool.clone(), torch.tensor([0, 3, 1], device=DEV)
    y, _ = kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu_of(lens), ssm_state_indices=slots)
    check(at(a, slice(32, 96)), before[slots[1:]], lens[1:], y[:, 32:], pool[slots[1:]])
    assert bool(torch.isinf(pool[2]).all()) and torch.equal(pool[4], before[4])


@pytest.mark.parametrize("bad", [[0, 40, 30, 60], [1, 20, 40, 60], [0, 20, 40, 61]])
def test_a_rejected_layout(bad):
    import kda_b200
    gen = generator(18)
    a = make(gen, 60, 64, 16, 1, BF)
    pool = randn(gen, 3, 64, 16)
    before, status, out = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1, 60, 64), 3.0, dtype=BF, device=DEV)
    cu = torch.tensor(bad, device=DEV)
    kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu, ssm_state_indices=torch.arange(3, device=DEV), out=out, status=status)
    assert int(status) == 1 and bool((out == 0).all()) and torch.equal(pool, before)
    _, final = kda_b200.selective_scan(**a, initial_state=before, cu_seqlens=cu)
    assert torch.equal(final, before)


def test_slots_out_of_range_or_named_twice():
    import kda_b200
    gen, n = generator(19), 6
    a = make(gen, 5 * n, 64, 16, 1, F)
    pool = randn(gen, n, 64, 16)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    slots = torch.tensor([0, n, -1, 0, 4, 5], device=DEV, dtype=torch.int32)
    y, _ = kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu_of([5] * n), ssm_state_indices=slots, status=status)
    assert int(status) == 2 and torch.equal(pool[1:4], before[1:4])
    init = before.clone()
    init[1:4] = 0
    _, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of([5] * n))
    final[[0, 4, 5]] = pool[[0, 4, 5]]
    check(a, init, [5] * n, y, final)


@pytest.mark.parametrize("dtype,Dm,Ns,G,rows", [(BF, 4096, 16, 1, 3), (F, 1000, 16, 1, 1), (HF, 72, 13, 2, 40), (BF, 64, 64, 1, 7), (F, 24, 128, 3, 5),
                                                (BF, 100, 8, 4, 9), (F, 3, 1, 1, 2), (HF, 256, 32, 1, 300)])
@pytest.mark.parametrize("pad", [0, 2])
def test_single_tokens(dtype, Dm, Ns, G, rows, pad):
    import kda_b200
    gen, N = generator(rows + Dm), rows + pad
    a = make(gen, N, Dm, Ns, G, dtype)
    pool = randn(gen, N + 2, Dm, Ns)
    before = pool.clone()
    slots = torch.randperm(N + 2, generator=torch.Generator().manual_seed(3))[:N].to(torch.int32).to(DEV)
    if pad:
        slots[1 if rows > 1 else 0] = -1
        slots[-1] = -7
        a["u"][0, -1] = float("nan")
    live = [i for i in range(N) if int(slots[i]) >= 0]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y, got = kda_b200.selective_scan_step(**a, pool=pool, ssm_state_indices=slots, status=status)
    assert got is pool and int(status) == 0
    ids = slots[live].long()
    some = live[:12]
    check(at(a, some), before[ids[:12]], [1] * len(some), y[:, some], pool[ids[:12]])
    whole = before.clone()
    y2, final = kda_b200.selective_scan(**at(a, live), initial_state=whole[ids].contiguous(), cu_seqlens=cu_of([1] * len(live)))
    torch.testing.assert_close(y[:, live].float(), y2.float(), rtol=2 ** -7, atol=1e-4)
    torch.testing.assert_close(pool[ids], final, rtol=1e-5, atol=1e-5)
    dead = [i for i in range(N) if i not in live]
    assert bool((y[0, dead] == 0).all())
    rest = [i for i in range(N + 2) if i not in ids.tolist()]
    assert torch.equal(pool[rest], before[rest])
    out, again = torch.full_like(y, 3.0), before.clone()
    kda_b200.selective_scan_step(**a, pool=again, ssm_state_indices=slots, out=out)
    assert torch.equal(out[0, live], y[0, live]) and bool((out[0, dead] == 3.0).all()) and torch.equal(again, pool)


def test_single_tokens_with_a_slot_named_twice():
    import kda_b200
    gen = generator(20)
    a, pool = make(gen, 4, 64, 16, 1, F), randn(gen, 3, 64, 16)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, _ = kda_b200.selective_scan_step(**a, pool=pool, ssm_state_indices=torch.tensor([2, 0, 2, 3], device=DEV), status=status)
    assert int(status) == 2 and torch.equal(pool[1], before[1])
    init = torch.stack([before[2], before[0], torch.zeros_like(before[0]), torch.zeros_like(before[0])])
    _, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of([1] * 4))
    check(a, init, [1] * 4, y, torch.stack([pool[2], pool[0], final[2], final[3]]))


def test_captured_calls_follow_their_tables():
    import kda_b200
    gen, N, T = generator(21), 6, 90
    a, pool = make(gen, T, 96, 16, 1, BF), randn(gen, 9, 96, 16)
    tok = make(gen, N, 96, 16, 1, BF)
    tok["A"], tok["D"], tok["dt_bias"] = a["A"], a["D"], a["dt_bias"]
    cu, slots, step_slots = cu_of([15] * N), torch.arange(N, device=DEV), torch.arange(N, device=DEV)
    kda_b200.selective_scan(**a, initial_state=pool.clone(), cu_seqlens=cu, ssm_state_indices=slots)
    torch.cuda.synchronize()
    prompt, token = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(prompt):
        y, _ = kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu, ssm_state_indices=slots)
    with torch.cuda.graph(token):
        ys, _ = kda_b200.selective_scan_step(**tok, pool=pool, ssm_state_indices=step_slots)
    for lens, ids in (([15] * N, [0, 1, 2, 3, 4, 5]), ([1, 0, 40, 2, 30, 0], [8, 2, 7, 1, 0, 5]), ([90, 0, 0, 0, 0, 0], [3, 4, 5, 6, 7, 8])):
        cu.copy_(cu_of(lens))
        slots.copy_(torch.tensor(ids))
        step_slots.copy_(torch.tensor(ids[:4] + [-1, -1]))
        a["u"].normal_()
        before = pool.clone()
        prompt.replay()
        check(a, before[slots], lens, y, pool[slots])
        middle = pool.clone()
        token.replay()
        check(at(tok, slice(0, 4)), middle[slots[:4]], [1] * 4, ys[:, :4], pool[slots[:4]])
        assert bool((ys[:, 4:] == 0).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z, final = kda_b200.selective_scan(**a, cu_seqlens=cu)
    side.synchronize()
    check(a, torch.zeros(N, 96, 16, device=DEV), [90, 0, 0, 0, 0, 0], z, final)


def test_captured_pieces_follow_their_tables():
    """A long axis on few channels is cut by its size alone: a replay may have any layout of as many sequences."""
    import kda_b200
    gen, N, T = generator(23), 5, 1200
    a, pool = make(gen, T, 48, 16, 1, BF), randn(gen, 8, 48, 16)
    cu, slots = cu_of([240] * N), torch.arange(N, device=DEV)
    kda_b200.selective_scan(**a, initial_state=pool.clone(), cu_seqlens=cu, ssm_state_indices=slots)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(kda_b200.selective_scan(**a, initial_state=pool, cu_seqlens=cu, ssm_state_indices=slots)[0])
    for lens, ids in (([1200, 0, 0, 0, 0], [4, 1, 2, 3, 0]), ([1, 128, 129, 0, 942], [7, 0, 3, 5, 6]), ([240] * N, [0, 1, 2, 3, 4]), ([0, 0, 0, 0, 300], [5, 6, 7, 0, 1])):
        cu.copy_(cu_of(lens))
        slots.copy_(torch.tensor(ids))
        for graph, y in zip(graphs, outs):
            before = pool.clone()
            graph.replay()
            check(a, before[slots], lens, y, pool[slots])
            assert bool((y[:, sum(lens):] == 0).all())


def test_states_and_rates_in_other_orders():
    import kda_b200
    gen, lens = generator(24), [30, 20]
    a = make(gen, 50, 64, 16, 1, F)
    init = randn(gen, 2, 16, 64).transpose(1, 2)
    a["A"] = a["A"].t().contiguous().t()
    for _ in range(2):
        y, final = kda_b200.selective_scan(**a, initial_state=init, cu_seqlens=cu_of(lens).cpu())
        check(a, init, lens, y, final)


def test_offsets_behind_32_bits():
    import kda_b200
    Dm, T = 8192, 270_000
    gen = generator(22)
    a = make(gen, 40, Dm, 16, 1, BF)
    far = {n: torch.zeros(1, T, *t.shape[2:], dtype=BF, device=DEV) for n, t in a.items() if n in ("u", "dt", "B", "C")}
    for n in far:
        far[n][:, -40:] = a[n]
    big = dict(a, **far, z=None)
    lens = [T - 40, 40]
    y, final = kda_b200.selective_scan(**big, cu_seqlens=cu_of(lens))
    check(dict(a, z=None), torch.zeros(1, Dm, 16, device=DEV), [40], y[:, -40:], final[1:])
    assert bool((y[:, :100] == 0).all())
    del big, far, y
    pool = torch.zeros(17_000, Dm, 16, device=DEV)                   # slots up to 2.2e9 values
    tok = at(a, slice(0, 2))
    y, _ = kda_b200.selective_scan_step(**tok, pool=pool, ssm_state_indices=torch.tensor([16_999, 3], device=DEV))
    check(tok, torch.zeros(2, Dm, 16, device=DEV), [1, 1], y, pool[[16_999, 3]])
    assert int((pool != 0).any(-1).any(-1).sum()) == 2


def same(got, want, what):
    """Equal where `want` is infinite or not a number; nothing is said about the rest."""
    got, want = got.double(), want.to(got.device)
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(torch.where(want.isinf(), want, 0.0), torch.where(got.isinf(), got, 0.0)), what


@pytest.mark.parametrize("dtype,Ns", [(F, 1), (BF, 3), (HF, 13), (BF, 16), (F, 24), (BF, 24), (F, 33), (HF, 100)])
@pytest.mark.parametrize("how", ["whole", "pieces", "step"])
def test_infinite_tokens_reach_no_state_that_does_not_exist(dtype, Ns, how):
    """An infinite u (channel 0) or dt (channel 1) makes the states and outputs from there on infinite, not NaN, whatever the number of
    state values (B, C, D positive, so that no infinities cancel); the other channels stay as they are."""
    import kda_b200
    gen, T = generator(30 + Ns), 600 if how == "pieces" else 40
    a = make(gen, T, 24, Ns, 1, dtype, gate=False)
    for n in "BC":
        a[n] = a[n].abs() + 0.5
    a["A"] = a["A"] / Ns                                              # no single step's decay is zero in fp32
    a["u"][..., :2] = a["u"][..., :2].abs()
    a["D"][:2] = 1.0
    a["u"][0, 21, 0] = a["dt"][0, 9, 1] = float("inf")
    lens = [1] * T if how == "step" else [T]
    init = torch.zeros(len(lens), 24, Ns, device=DEV)
    if how == "step":
        final = init.clone()
        y, _ = kda_b200.selective_scan_step(**a, pool=final)
    else:
        y, final = kda_b200.selective_scan(**a, initial_state=init)
    rest = {n: t[..., 2:] if n in ("u", "dt") else t[2:] if n in ("A", "D", "dt_bias") else t for n, t in a.items() if t is not None}
    check(dict(rest, z=None), init[:, 2:], lens, y[..., 2:], final[:, 2:])
    t = 0
    for i, n in enumerate(lens):
        s = at(a, slice(t, t + n))
        want, _, h, _ = scan64(s["u"][0], s["dt"][0], a["A"], s["B"][0], s["C"][0], a["D"], None, a["dt_bias"], init[i], True)
        assert not bool(want.isnan().any()) and not bool(h.isnan().any())
        same(y[0, t:t + n, :2], want[:, :2], f"sequence {i}")
        same(final[i, :2], h[:2], f"state {i}")
        t += n


@pytest.mark.parametrize("step", [False, True])
def test_without_a_skip_an_infinite_token_is_not_multiplied_by_it(step):
    """D left out adds nothing, also where u is infinite: the output is the infinite sum of C h (B, C positive)."""
    import kda_b200
    gen, T = generator(31), 40
    a = make(gen, T, 64, 16, 1, BF, gate=False)
    a.update(D=None, B=a["B"].abs() + 0.5, C=a["C"].abs() + 0.5)
    a["u"][0, 21, 0] = float("inf")
    a["u"][0, 33, 1] = -float("inf")
    lens = [1] * T if step else [T]
    init = torch.zeros(len(lens), 64, 16, device=DEV)
    if step:
        y, _ = kda_b200.selective_scan_step(**a, pool=init.clone())
    else:
        y, _ = kda_b200.selective_scan(**a)
    t = 0
    for n in lens:
        s = at(a, slice(t, t + n))
        want = scan64(s["u"][0], s["dt"][0], a["A"], s["B"][0], s["C"][0], None, None, a["dt_bias"], init[0], True)[0]
        assert not bool(want.isnan().any())
        same(y[0, t:t + n], want, f"token {t}")
        t += n


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_rates_that_are_infinite(step, sign):
    """A of -inf forgets the state at every positive step and keeps it at a step of zero, for prompts (of a length that ends inside a
    tile) as for single tokens; +inf does so with negative steps.  In 64 bits: a rate of 1e30, since exp(-1e30 s) is 0 for every step
    here but zero."""
    import kda_b200
    gen, T = generator(32), 41
    a = make(gen, T, 48, 16, 1, F)
    a.update(dt=-sign * (a["dt"].abs() + 0.01), dt_bias=None)
    a["dt"][:, 10:14] = 0.0
    a["dt"][:, -1] = 0.0
    a["A"][:4] = sign * float("inf")
    a["dt"][..., 4:] = a["dt"][..., 4:].abs()
    finite = dict(a, A=a["A"].clamp(-1e30, 1e30))
    lens = [1] * T if step else [T]
    init = randn(gen, len(lens), 48, 16)
    if step:
        final = init.clone()
        y, _ = kda_b200.selective_scan_step(**a, pool=final, dt_softplus=False)
    else:
        y, final = kda_b200.selective_scan(**a, initial_state=init, dt_softplus=False)
    check(finite, init, lens, y, final, False)


def test_pieces_with_states_and_growth_that_fp32_products_do_not_hold():
    """What a piece leaves of the state in front of it is one exponential of many steps: it may be beyond fp32's range where the state
    is zero or small, and zero where the state is infinite.  Channels 0-1: a zero state that nothing enters, growing; 2-3: 1e-30 times
    e^96 within the first piece; 4-5: an infinite state that decays (B, C positive); the rest as ever."""
    import kda_b200
    gen, T = generator(33), 3000
    a = make(gen, T, 16, 16, 1, F, gate=False)
    a.update(B=a["B"].abs() + 0.5, C=a["C"].abs() + 0.5, dt=a["dt"].abs() * 0.1, dt_bias=None)
    a["A"][:4], a["A"][4:6] = 1.0, -1.0
    a["u"][..., :4] = 0.0
    a["dt"][..., :2] = 1.0
    a["dt"][..., 2:4] = 0.0
    a["dt"][:, :128, 2:4] = 0.75
    a["dt"][..., 4:6] = 1.0
    init = randn(gen, 1, 16, 16)
    init[:, :2], init[:, 2:4], init[:, 4:6] = 0.0, 1e-30, float("inf")
    y, final = kda_b200.selective_scan(**a, initial_state=init, dt_softplus=False)
    assert bool((final[0, :2] == 0).all()) and bool((y[..., :2] == 0).all())
    assert bool((final[0, 4:6] == float("inf")).all()) and bool((y[..., 4:6] == float("inf")).all())
    keep = [2, 3, *range(6, 16)]
    part = {n: t[..., keep] if n in ("u", "dt") else t[keep] if n in ("A", "D") else t for n, t in a.items()}
    check(part, init[:, keep], [T], y[..., keep], final[:, keep], False)


@pytest.mark.parametrize("dtype,Dm,Ns", [(BF, 256, 16), (F, 72, 13), (HF, 40, 64), (F, 24, 128)])
@pytest.mark.parametrize("fill", ["nan", "inf", "-inf"])
def test_nothing_of_a_row_of_padding_is_used(dtype, Dm, Ns, fill):
    """Four rows of a step share a block: whatever lies in the rows of padding among them, in every tensor, the others, the pool and a
    caller's output rows of padding stay bit for bit."""
    import kda_b200
    gen, N = generator(25), 13
    a, pool = make(gen, N, Dm, Ns, 1, dtype), randn(gen, 11, Dm, Ns)
    dead = [1, 2, 3, 6, 12]
    slots = torch.tensor([5, -1, -9, -1, 0, 10, -2, 3, 4, 1, 2, 8, -1], device=DEV)
    outs, pools = [], []
    for value in (0.0, float(fill)):
        for n in ("u", "dt", "B", "C", "z"):
            a[n][:, dead] = value
        pools.append(pool.clone())
        outs.append(torch.full((1, N, Dm), 3.0, dtype=dtype, device=DEV))
        kda_b200.selective_scan_step(**a, pool=pools[-1], ssm_state_indices=slots, out=outs[-1])
    assert torch.equal(outs[0], outs[1]) and torch.equal(pools[0], pools[1])
    assert bool((outs[1][0, dead] == 3.0).all()) and bool(torch.isfinite(outs[1]).all()) and torch.equal(pools[1][[6, 7, 9]], pool[[6, 7, 9]])
