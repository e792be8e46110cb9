"""The gated linear recurrence against its definition in 64 bits: prompts in all types, forms and layouts, slots and tables, single tokens."""
import pytest
import torch

from gated_testlib import U, forward64
from serving_testlib import DEV, assert_within, cu_of, generator, randn

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(gen, T, C, dtype, form, gated, biases=True):
    x, r = randn(gen, 1, T, C, dtype=dtype), randn(gen, 1, T, C, dtype=dtype)
    i = randn(gen, 1, T, C, dtype=dtype) if gated else None
    rate = randn(gen, C) - 5.0 if form == "power" else None
    r_bias = randn(gen, C) + (0.0 if form == "power" else 2.0) if biases else None
    return x, r, i, rate, r_bias, randn(gen, C) if gated and biases else None


def rows(t):
    return t[0] if t is not None else None


def check(lens, C, dtype, form, gated, seed, biases=True, scale=8.0):
    import kda_b200
    gen, T, N = generator(seed), sum(lens), len(lens)
    x, r, i, rate, rb, ib = inputs(gen, T, C, dtype, form, gated, biases)
    states = randn(gen, N, C)
    y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib, states, cu_of(lens), rate_scale=scale)
    want, e, wf, fe = forward64(lens, x[0], r[0], rows(i), rate, rb, ib, states, scale)
    assert y.dtype == dtype and final.dtype == F32
    assert_within(y[0], want, e, "y")
    assert_within(final, wf, fe, "final state")
    again, f2 = kda_b200.gated_scan(x, r, i, rate, rb, ib, states, cu_of(lens, torch.int32), rate_scale=scale)
    assert torch.equal(again, y) and torch.equal(f2, final)


LAYOUTS = {"one token": [1], "slice": [12], "borders": [47, 48, 49, 95, 96, 97, 1, 0, 11, 13], "empty ones": [0, 0, 5, 0, 130, 0, 0], "ragged": [70, 1, 2, 300, 3, 64],
           "nothing": [0], "rounds": [1700]}


@pytest.mark.parametrize("lens", LAYOUTS.values(), ids=LAYOUTS.keys())
@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form,gated", [("power", 1), ("power", 0), ("logistic", 1), ("logistic", 0)])
def test_prompts(lens, dtype, form, gated):
    for C in (64, 72, 33):                                   # a whole slab, the end of one, single values
        check(lens, C, dtype, form, gated, seed=sum(lens) + C)


@pytest.mark.parametrize("C", [1, 2, 31, 32, 63, 65, 130, 200, 1000])
def test_channel_counts(C):
    for dtype in (BF, F32):
        check([40, 9, 100], C, dtype, "power", 1, seed=C)


def test_many_short_sequences():
    """More entries than a block keeps in shared memory."""
    check([(7 * k) % 4 for k in range(700)], 40, BF, "power", 1, seed=5)
    check([1] * 900, 16, F32, "logistic", 0, seed=6)


def test_without_biases_and_with_another_scale():
    check([100, 30], 64, BF, "power", 1, seed=7, biases=False)
    check([100, 30], 33, F32, "power", 0, seed=8, biases=False, scale=0.5)
    check([100, 30], 64, FP, "logistic", 1, seed=9, biases=False)


def test_no_initial_state_and_one_sequence():
    import kda_b200
    gen = generator(10)
    x, r, i, rate, rb, ib = inputs(gen, 200, 64, BF, "power", 1)
    y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib)
    want = kda_b200.gated_scan(x, r, i, rate, rb, ib, torch.zeros(1, 64, device=DEV), cu_of([200]))
    assert torch.equal(y, want[0]) and torch.equal(final, want[1])


def test_views_and_odd_addresses():
    """Rows with other columns between them, tensors of one buffer, starts off 16 bytes: the same values whatever way they are read."""
    import kda_b200
    gen, T, C = generator(11), 150, 64
    for dtype in (BF, F32):
        x, r, i, rate, rb, ib = inputs(gen, T, C, dtype, "power", 1)
        y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib)
        for shift in (0, 1, 8):
            room = torch.zeros(1, T, 3 * C + 24 + shift, dtype=dtype, device=DEV)
            v = [room[..., shift + k * (C + 8):][..., :C] for k in range(3)]
            for a, b in zip(v, (x, r, i)):
                a.copy_(b)
            out = torch.zeros(1, T, C + 8, dtype=dtype, device=DEV)[..., :C]
            y2, f2 = kda_b200.gated_scan(*v, rate, rb, ib, out=out)
            assert y2 is out and torch.equal(f2, final) and torch.equal(y2, y)
        t = x.transpose(1, 2).contiguous().transpose(1, 2)                    # channels apart: copied
        assert torch.equal(kda_b200.gated_scan(t, r, i, rate, rb, ib)[0], y)


def test_rows_behind_2_to_the_31_elements():
    import kda_b200
    T, C, ld = 20, 64, 1 << 27
    room = torch.empty(ld * (T - 1) + 3 * C, dtype=BF, device=DEV)
    v = [room.as_strided((1, T, C), (0, ld, 1), k * C) for k in range(3)]
    gen = generator(12)
    x, r, i, rate, rb, ib = inputs(gen, T, C, BF, "power", 1)
    for a, b in zip(v, (x, r, i)):
        a.copy_(b)
    y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib)
    y2, f2 = kda_b200.gated_scan(*v, rate, rb, ib)
    assert torch.equal(y, y2) and torch.equal(final, f2)
    y2, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, out=v[0])
    assert torch.equal(y, y2)


@pytest.mark.parametrize("table", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_pools(table):
    import kda_b200
    gen, lens, C = generator(13), [30, 0, 200, 1], 72
    x, r, i, rate, rb, ib = inputs(gen, sum(lens) + 9, C, BF, "power", 1)
    store = randn(gen, 9, C + 5)
    pool, slots = store[:, 2:2 + C], torch.tensor([7, 0, 3, 5], dtype=table, device=DEV)
    before, status = store.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, got = kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, cu_of(lens), ssm_state_indices=slots, status=status)
    want, final = kda_b200.gated_scan(x[:, :sum(lens)], r[:, :sum(lens)], i[:, :sum(lens)], rate, rb, ib, before[slots.long(), 2:2 + C].contiguous(), cu_of(lens))
    assert got is pool and int(status) == 0
    assert torch.equal(y[:, :sum(lens)], want) and (y[:, sum(lens):] == 0).all() and torch.equal(pool[slots.long()], final)
    rest = store.clone()
    rest[slots.long(), 2:2 + C] = before[slots.long(), 2:2 + C]
    assert torch.equal(rest, before)                          # nothing else was written
    out = torch.full_like(x, 3.0)                             # rows behind the last sequence stay in a caller's buffer
    pool.copy_(before[:, 2:2 + C])
    kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, cu_of(lens), ssm_state_indices=slots, out=out)
    assert torch.equal(out[:, :sum(lens)], want) and (out[:, sum(lens):] == 3.0).all()


def test_bad_slots_and_tables_are_reported():
    import kda_b200
    gen, lens, C = generator(14), [20, 33, 10, 7], 64
    x, r, i, rate, rb, ib = inputs(gen, sum(lens), C, F32, "power", 1)
    pool = randn(gen, 6, C)
    before = pool.clone()
    for bad in ([2, 2, 0, 5], [2, 6, 0, 5], [2, -1, 0, 5]):   # a repeat, out of range, negative: zeros, and not stored
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        pool.copy_(before)
        y, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, cu_of(lens), ssm_state_indices=torch.tensor(bad, device=DEV), status=status)
        states = before[[2, 0, 0, 5]]
        states[1] = 0.0
        want, final = kda_b200.gated_scan(x, r, i, rate, rb, ib, states, cu_of(lens))
        assert int(status) == 2 and torch.equal(y, want)
        assert torch.equal(pool[[2, 0, 5]], final[[0, 2, 3]]) and torch.equal(pool[[1, 3, 4]], before[[1, 3, 4]])
    for bad in ([0, 20, 10, 63, 70], [1, 20, 53, 63, 70], [0, 20, 53, 63, 71], [0, -5, 53, 63, 70]):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        pool.copy_(before)
        y, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, torch.tensor(bad, device=DEV), ssm_state_indices=torch.tensor([0, 1, 2, 3], device=DEV), status=status)
        assert int(status) == 1 and (y == 0).all() and torch.equal(pool, before)
        y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib, before[:4], torch.tensor(bad, device=DEV))
        assert (y == 0).all() and torch.equal(final, before[:4])


def test_infinities_and_nan_stay_in_their_sequence():
    import kda_b200
    gen, lens, C = generator(15), [50, 150, 40, 0, 130], 64
    for dtype in (BF, F32):
        x, r, i, rate, rb, ib = inputs(gen, sum(lens), C, dtype, "power", 1)
        states = randn(gen, 5, C)
        clean, cf = kda_b200.gated_scan(x, r, i, rate, rb, ib, states, cu_of(lens))
        x[0, 60, 3], x[0, 70, 4], states[1, 5], r[0, 80, 6], i[0, 90, 7], x[0, 241, 8] = float("inf"), float("nan"), float("-inf"), float("nan"), float("nan"), float("inf")
        y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib, states, cu_of(lens))
        want, _, wf, _ = forward64(lens, x[0], r[0], i[0], rate, rb, ib, states)
        for got, ref in ((y[0], want), (final, wf)):
            for kind in (torch.isnan, torch.isposinf, torch.isneginf):
                assert torch.equal(kind(got), kind(ref))
        same = torch.isfinite(want)
        assert torch.equal(y[0][same], clean[0][same]) and torch.equal(final[torch.isfinite(wf)], cf[torch.isfinite(wf)])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_far_gates_and_rates(dtype):
    """Closed and open gates, rates that keep everything or nothing."""
    import kda_b200
    gen, C = generator(16), 64
    x, r, i, rate, _, _ = inputs(gen, 120, C, dtype, "power", 1, False)
    states = randn(gen, 1, C)
    r[0, :, :8], r[0, :, 8:16], i[0, :, 16:24] = -30.0, 30.0, 30.0
    i[0, :, 24:32], rate[32:40], rate[40:48], rate[48:52], rate[52:56] = -30.0, -60.0, 5.0, -200.0, 80.0
    y, final = kda_b200.gated_scan(x, r, i, rate, None, None, states)
    want, e, wf, fe = forward64([120], x[0], r[0], i[0], rate, None, None, states)
    assert_within(y[0], want, e + 1e-20, "y")
    assert_within(final, wf, fe + 1e-20, "final state")
    r[0, :, :32], i[0, :, 32:] = -300.0, -300.0               # behind the exponentials' range
    y, final = kda_b200.gated_scan(x, r, i, rate, None, None, states)
    assert torch.isfinite(y).all()
    assert (final[0, :32] - states[0, :32]).abs().max() < 1e-6 and (y[0, 60:, 53].abs() < 1e-9).all()


def test_captured_calls_and_other_streams():
    import kda_b200
    gen, lens, C = generator(17), [60, 300], 72
    x, r, i, rate, rb, ib = inputs(gen, 360, C, BF, "power", 1)
    pool, cu, slots = randn(gen, 4, C), cu_of(lens), torch.tensor([2, 1], device=DEV)
    one = pool.clone()
    want, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, one, cu, ssm_state_indices=slots)
    torch.cuda.synchronize()
    two, graph = pool.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, two, cu, ssm_state_indices=slots)
    for _ in range(2):
        two.copy_(pool)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(two, one)
    cu.copy_(cu_of([100, 260]))                               # tables are read at each replay
    two.copy_(pool)
    graph.replay()
    other = pool.clone()
    assert torch.equal(kda_b200.gated_scan(x, r, i, rate, rb, ib, other, cu, ssm_state_indices=slots)[0], y) and torch.equal(two, other)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z, _ = kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, cu_of(lens), ssm_state_indices=slots)
    stream.synchronize()
    assert torch.equal(z, want) and torch.equal(pool, one)


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form,gated", [("power", 1), ("power", 0), ("logistic", 1), ("logistic", 0)])
def test_steps_are_prompts_of_one_token(dtype, form, gated):
    import kda_b200
    for n, C in ((1, 64), (5, 1), (33, 130), (300, 36)):
        gen = generator(n + C)
        x, r, i, rate, rb, ib = inputs(gen, n + 2, C, dtype, form, gated)
        pool = randn(gen, n + 4, C)
        slots = torch.cat([torch.randperm(n + 4, device=DEV)[:n], torch.tensor([-1, -7], device=DEV)])
        one = pool.clone()
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        y, got = kda_b200.gated_scan_step(x, r, i, rate, rb, ib, one, slots, status=status)
        head = [t[:, :n] if t is not None else None for t in (x, r, i)]
        want, e, wf, fe = forward64([1] * n, *(rows(t) for t in head), rate, rb, ib, pool[slots[:n]])
        assert got is one and int(status) == 0 and (y[:, n:] == 0).all()
        assert_within(y[0, :n], want, e, "y")
        assert_within(one[slots[:n]], wf, fe, "state")
        rest = one.clone()
        rest[slots[:n]] = pool[slots[:n]]
        assert torch.equal(rest, pool)


def test_steps_with_repeats_without_slots_and_without_rows():
    import kda_b200
    gen, C = generator(21), 40
    x, r, i, rate, rb, ib = inputs(gen, 6, C, F32, "power", 1)
    pool = randn(gen, 8, C)
    one, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, _ = kda_b200.gated_scan_step(x, r, i, rate, rb, ib, one, torch.tensor([3, 1, 3, 8, 0, 1], device=DEV), status=status)
    states = pool[[3, 1, 0, 0, 0, 0]]
    states[[2, 3, 5]] = 0.0
    two = states.clone()
    want, _ = kda_b200.gated_scan_step(x, r, i, rate, rb, ib, two)
    assert int(status) == 2 and torch.equal(y, want)
    assert torch.equal(one[[3, 1, 0]], two[[0, 1, 4]]) and torch.equal(one[[2, 4, 5, 6, 7]], pool[[2, 4, 5, 6, 7]])
    out = torch.full((1, 6, C), 5.0, device=DEV)              # padding stays in a caller's buffer
    kda_b200.gated_scan_step(x, r, i, rate, rb, ib, one, torch.tensor([3, -1, 2, -1, 0, 1], device=DEV), out=out)
    assert (out[0, [1, 3]] == 5.0).all() and not (out[0, [0, 2, 4, 5]] == 5.0).any()
    empty = x[:, :0]
    y, got = kda_b200.gated_scan_step(empty, empty, empty, rate, rb, ib, pool)
    assert y.shape == (1, 0, C) and got is pool
    y, final = kda_b200.gated_scan(empty, empty, empty, rate, rb, ib, pool[:3], cu_of([0, 0, 0]))
    assert y.shape == (1, 0, C) and torch.equal(final, pool[:3])


def test_threads_with_calls_of_different_sizes():
    """Clusters of different sizes of one kernel, launched side by side."""
    import threading

    import kda_b200
    gen = generator(23)
    args = [inputs(gen, T, 64, BF, "power", 1) for T in (40, 150, 700, 3000)]
    want, got = [kda_b200.gated_scan(*a)[0] for a in args], [None] * 4
    torch.cuda.synchronize()

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got[k] = kda_b200.gated_scan(*args[k])[0]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_prompt_then_steps_is_the_whole_prompt():
    import kda_b200
    gen, C = generator(22), 128
    x, r, i, rate, rb, ib = inputs(gen, 140, C, F32, "logistic", 1)
    y, final = kda_b200.gated_scan(x, r, i, rate, rb, ib)
    head, pool = kda_b200.gated_scan(x[:, :130], r[:, :130], i[:, :130], rate, rb, ib)
    for t in range(130, 140):
        z, pool = kda_b200.gated_scan_step(x[:, t:t + 1], r[:, t:t + 1], i[:, t:t + 1], rate, rb, ib, pool)
        torch.testing.assert_close(z, y[:, t:t + 1], rtol=64 * U, atol=64 * U)
    torch.testing.assert_close(pool, final, rtol=64 * U, atol=64 * U)
