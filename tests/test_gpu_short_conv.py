"""short_conv and short_conv_step against the definition in 64 bits: types, widths, odd and unaligned channels, strides, lengths from
none to long, tables that are wrong, padding, captured calls."""
import pytest
import torch

from serving_testlib import DEV, assert_within, conv64, cu_of, generator, randn

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def check(x, w, b, hist, lens, y, final, act="silu", what=""):
    t = 0
    for i, n in enumerate(lens):
        want, bound, new = conv64(x[0, t:t + n], w, b, hist[i], act)
        assert_within(y[0, t:t + n], want, bound, f"{what} sequence {i}")
        assert torch.equal(final[i].double(), new), f"{what} history {i}"
        t += n


@pytest.mark.parametrize("dtype,W,C,lens,act,bias", [
    (BF, 4, 256, [77], "silu", True), (BF, 4, 264, [1, 2, 3, 4, 0, 33, 31, 32, 64], "silu", False), (HF, 3, 1539, [5, 0, 0, 100], None, True),
    (F, 2, 130, [1], "silu", True), (F, 4, 1, [3, 70], "silu", True), (BF, 2, 4096, [700, 1, 29], None, False), (F, 3, 1024, [65] * 9, "silu", True),
    (BF, 4, 8, [1] * 200, "silu", True), (BF, 4, 129, [0, 0, 0], "silu", True)])
@pytest.mark.parametrize("pooled", [False, True])
def test_prompts(dtype, W, C, lens, act, bias, pooled):
    import kda_b200
    gen, N = generator(len(lens) + C), len(lens)
    x, w = randn(gen, 1, sum(lens), C, dtype=dtype), randn(gen, C, W, dtype=dtype)
    b = randn(gen, C, dtype=dtype) if bias else None
    if pooled:
        pool = randn(gen, N + 3, W - 1, C, dtype=dtype)
        slots = torch.randperm(N + 3, generator=torch.Generator().manual_seed(3))[:N].to(DEV)
        before = pool.clone()
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        y, got = kda_b200.short_conv(x, w, b, pool, cu_of(lens), activation=act, ssm_state_indices=slots, status=status)
        assert got is pool and int(status) == 0
        check(x, w, b, before[slots], lens, y, pool[slots], act)
        rest = [i for i in range(N + 3) if i not in slots.tolist()]
        assert torch.equal(pool[rest], before[rest])
    else:
        init = randn(gen, N, W - 1, C, dtype=dtype)
        keep = init.clone()
        y, final = kda_b200.short_conv(x, w, b, init, cu_of(lens, torch.int32), activation=act)
        assert torch.equal(init, keep)
        check(x, w, b, init, lens, y, final, act)
        y0, final0 = kda_b200.short_conv(x, w, b, None, cu_of(lens), activation=act)
        check(x, w, b, torch.zeros_like(init), lens, y0, final0, act)


def test_one_sequence_without_a_table_and_a_conv1d_weight():
    import kda_b200
    gen = generator(1)
    x, w, b = randn(gen, 1, 50, 384, dtype=BF), randn(gen, 384, 1, 4, dtype=F), randn(gen, 384, dtype=F)
    y, final = kda_b200.short_conv(x, w, b)
    check(x, w[:, 0], b, torch.zeros(1, 3, 384, device=DEV), [50], y, final)
    empty, state = kda_b200.short_conv(x[:, :0], w, b, final)
    assert empty.shape == (1, 0, 384) and torch.equal(state, final)


@pytest.mark.parametrize("off", [0, 1, 8])
def test_views_are_read_and_written_in_place(off):
    """A slice of a wider projection, on 16 bytes or not, tokens in another order of strides, and a caller's output."""
    import kda_b200
    gen, lens = generator(2), [40, 25]
    wide = randn(gen, 1, 65, 700, dtype=BF)
    x = wide[:, :, off:off + 256]
    w, init = randn(gen, 256, 4, dtype=BF), randn(gen, 2, 3, 256, dtype=BF)
    target = torch.full((1, 70, 512), 7.0, dtype=BF, device=DEV)
    y, final = kda_b200.short_conv(x, w, None, init, cu_of(lens), out=target[:, 2:67, off:off + 256])
    check(x, w, None, init, lens, y, final)
    rest = target.clone()
    rest[:, 2:67, off:off + 256] = 7.0
    assert bool((rest == 7.0).all())
    turned = wide[0, :, :64].t().contiguous().t()[None]              # token stride 1
    y, final = kda_b200.short_conv(turned, w[:64], None, None, cu_of(lens))
    check(turned, w[:64], None, torch.zeros(2, 3, 64, device=DEV), lens, y, final)


def test_rows_behind_the_last_sequence():
    import kda_b200
    gen, lens = generator(3), [10, 60]
    x = randn(gen, 1, 100, 136, dtype=BF)
    x[:, 70:] = float("nan")
    w = randn(gen, 136, 4, dtype=BF)
    y, final = kda_b200.short_conv(x, w, None, None, cu_of(lens))
    check(x, w, None, torch.zeros(2, 3, 136, device=DEV), lens, y, final)
    assert bool((y[:, 70:] == 0).all())
    out = torch.full_like(x, 3.0)
    kda_b200.short_conv(x, w, None, None, cu_of(lens), out=out)
    assert torch.equal(out[:, :70], y[:, :70]) and bool((out[:, 70:] == 3.0).all())


def test_a_neighbour_that_is_not_a_number_stays_there():
    """Neither the row in front of a sequence nor the slot of another one reaches it."""
    import kda_b200
    gen, lens = generator(4), [32, 33, 31]
    x, w = randn(gen, 1, 96, 64, dtype=F), randn(gen, 64, 4)
    pool = randn(gen, 5, 3, 64)
    x[:, :32] = float("nan")
    pool[[0, 2]] = float("inf")
    before, slots = pool.clone(), torch.tensor([0, 3, 1], device=DEV)
    y, _ = kda_b200.short_conv(x, w, None, pool, cu_of(lens), ssm_state_indices=slots)
    check(x[:, 32:], w, None, before[slots[1:]], lens[1:], y[:, 32:], pool[slots[1:]])


@pytest.mark.parametrize("bad", [[0, 40, 30, 60], [1, 20, 40, 60], [0, 20, 40, 61], [-1, 20, 40, 60]])
def test_a_rejected_layout(bad):
    import kda_b200
    gen = generator(5)
    x, w, pool = randn(gen, 1, 60, 128, dtype=BF), randn(gen, 128, 4, dtype=BF), randn(gen, 3, 3, 128, dtype=BF)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(x, 3.0)
    cu = torch.tensor(bad, device=DEV)
    kda_b200.short_conv(x, w, None, pool, cu, ssm_state_indices=torch.arange(3, device=DEV), out=out, status=status)
    assert int(status) == 1 and bool((out == 0).all()) and torch.equal(pool, before)
    _, final = kda_b200.short_conv(x, w, None, before, cu)
    assert torch.equal(final, before)


@pytest.mark.parametrize("n", [4, 300])
def test_slots_out_of_range_or_named_twice(n):
    import kda_b200
    gen = generator(6)
    x, w, pool = randn(gen, 1, 5 * n, 64, dtype=BF), randn(gen, 64, 4, dtype=BF), randn(gen, n, 3, 64, dtype=BF)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    slots = torch.arange(n, device=DEV, dtype=torch.int32)
    slots[1], slots[2], slots[3] = n, -1, 0
    y, _ = kda_b200.short_conv(x, w, None, pool, cu_of([5] * n), ssm_state_indices=slots, status=status)
    assert int(status) == 2
    hist = before.clone()
    hist[1:4] = 0                                                    # those sequences start from zeros
    final = torch.stack([pool[i] if i not in (1, 2, 3) else conv64(x[0, 5 * i:5 * i + 5], w, None, hist[i], "silu")[2].to(BF) for i in range(n)])
    check(x, w, None, hist, [5] * n, y, final)
    assert torch.equal(pool[1:4], before[1:4])


@pytest.mark.parametrize("dtype,W,C,rows", [(BF, 4, 24576, 3), (F, 3, 1539, 10), (HF, 2, 72, 300), (BF, 4, 1, 1), (HF, 4, 1000, 33), (F, 4, 4, 2)])
@pytest.mark.parametrize("pad", [0, 2])
def test_single_tokens(dtype, W, C, rows, pad):
    import kda_b200
    gen = generator(rows + C)
    N = rows + pad
    x, w, b = randn(gen, 1, N, C, dtype=dtype), randn(gen, C, W, dtype=dtype), randn(gen, C, dtype=dtype)
    pool = randn(gen, N + 2, W - 1, C, dtype=dtype)
    before = pool.clone()
    slots = torch.randperm(N + 2, generator=torch.Generator().manual_seed(3))[:N].to(torch.int32).to(DEV)
    if pad:
        slots[1 if rows > 1 else 0] = -1
        slots[-1] = -7
        x[0, -1] = float("nan")
    live = [i for i in range(N) if int(slots[i]) >= 0]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y, got = kda_b200.short_conv_step(x, w, b, pool, slots, status=status)
    assert got is pool and int(status) == 0
    at = slots[live].long()
    check(x[:, live], w, b, before[at], [1] * len(live), y[:, live], pool[at])
    dead = [i for i in range(N) if i not in live]
    assert bool((y[0, dead] == 0).all())
    rest = [i for i in range(N + 2) if i not in at.tolist()]
    assert torch.equal(pool[rest], before[rest])
    out = torch.full_like(x, 3.0)
    again = before.clone()
    kda_b200.short_conv_step(x, w, b, again, slots, out=out)
    assert torch.equal(out[0, live], y[0, live]) and bool((out[0, dead] == 3.0).all()) and torch.equal(again, pool)


def test_single_tokens_with_a_slot_named_twice():
    import kda_b200
    gen = generator(8)
    x, w, pool = randn(gen, 1, 4, 64, dtype=BF), randn(gen, 64, 4, dtype=BF), randn(gen, 3, 3, 64, dtype=BF)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, _ = kda_b200.short_conv_step(x, w, None, pool, torch.tensor([2, 0, 2, 3], device=DEV), status=status)
    assert int(status) == 2 and torch.equal(pool[1], before[1])
    hist = torch.stack([before[2], before[0], torch.zeros_like(before[0]), torch.zeros_like(before[0])])
    final = torch.cat([hist[:, 1:], x[0][:, None]], 1)
    check(x, w, None, hist, [1] * 4, y, final)
    assert torch.equal(pool[2], final[0]) and torch.equal(pool[0], final[1])


def test_tokens_one_by_one_are_the_prompt():
    import kda_b200
    gen = generator(9)
    x, w = randn(gen, 1, 9, 320, dtype=BF), randn(gen, 320, 4, dtype=BF)
    whole, final = kda_b200.short_conv(x, w)
    pool = torch.zeros(1, 3, 320, dtype=BF, device=DEV)
    parts = [kda_b200.short_conv(x[:, :4], w, None, pool, ssm_state_indices=torch.zeros(1, dtype=torch.int32, device=DEV))[0]]
    parts += [kda_b200.short_conv_step(x[:, t:t + 1], w, None, pool)[0] for t in range(4, 9)]
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(pool, final)


def test_captured_calls_follow_their_tables():
    """Two captured graphs and an eager call, on a stream of their own; layout, slots and tokens change between replays."""
    import kda_b200
    gen, N, T = generator(10), 6, 90
    x, w, pool = randn(gen, 1, T, 96, dtype=BF), randn(gen, 96, 4, dtype=BF), randn(gen, 9, 3, 96, dtype=BF)
    cu, slots = cu_of([15] * N), torch.arange(N, device=DEV)
    steps, step_slots = randn(gen, 1, N, 96, dtype=BF), torch.arange(N, device=DEV)
    prompt, token = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    kda_b200.short_conv(x, w, None, pool.clone(), cu, ssm_state_indices=slots)
    torch.cuda.synchronize()
    with torch.cuda.graph(prompt):
        y, _ = kda_b200.short_conv(x, w, None, pool, cu, ssm_state_indices=slots)
    with torch.cuda.graph(token):
        ys, _ = kda_b200.short_conv_step(steps, w, None, pool, step_slots)
    for lens, ids in (([15] * N, [0, 1, 2, 3, 4, 5]), ([1, 0, 40, 2, 30, 0], [8, 2, 7, 1, 0, 5]), ([90, 0, 0, 0, 0, 0], [3, 4, 5, 6, 7, 8])):
        cu.copy_(cu_of(lens))
        slots.copy_(torch.tensor(ids))
        step_slots.copy_(torch.tensor(ids[:4] + [-1, -1]))
        x.normal_()
        before = pool.clone()
        prompt.replay()
        check(x, w, None, before[slots], lens, y, pool[slots])
        middle = pool.clone()
        token.replay()
        check(steps[:, :4], w, None, middle[slots[:4]], [1] * 4, ys[:, :4], pool[slots[:4]])
        assert bool((ys[:, 4:] == 0).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z, final = kda_b200.short_conv(x, w, None, None, cu)
    side.synchronize()
    check(x, w, None, torch.zeros(N, 3, 96, device=DEV), [90, 0, 0, 0, 0, 0], z, final)


def test_offsets_behind_32_bits():
    """Rows and slots further than 2^31 elements from the base."""
    import kda_b200
    C, T = 8192, 270_000
    x = torch.zeros(1, T, C, dtype=BF, device=DEV)
    gen = generator(11)
    x[:, -70:] = randn(gen, 1, 70, C, dtype=BF)
    w = randn(gen, C, 4, dtype=BF)
    lens = [T - 70, 70]
    y, final = kda_b200.short_conv(x, w, None, None, cu_of(lens))
    want, bound, new = conv64(x[0, -70:], w, None, torch.zeros(3, C, device=DEV), "silu")
    assert_within(y[0, -70:], want, bound, "far rows")
    assert torch.equal(final[1].double(), new) and bool((y[0, :1000] == 0).all())
    pool = x.view(-1, 3, C)
    y, _ = kda_b200.short_conv_step(x[:, -1:].clone(), w, None, pool, torch.tensor([pool.shape[0] - 1], device=DEV))
    assert bool(torch.isfinite(y).all())
    assert torch.equal(pool[-1, -1], pool.view(-1, C)[-1])


def test_single_tokens_in_slots_behind_32_bits():
    """Slots further than 2^31 elements from the base: values, new histories, and every other slot as it was."""
    import kda_b200
    gen, C, W = generator(12), 8192, 4
    P = 2 ** 31 // ((W - 1) * C) + 1000
    pool = torch.full((P, W - 1, C), 5.0, dtype=BF, device=DEV)
    ids = [P - 1, 3, 2 ** 31 // ((W - 1) * C) + 1, 0]
    at = torch.tensor(ids, device=DEV)
    x, w = randn(gen, 1, 4, C, dtype=BF), randn(gen, C, W, dtype=BF)
    pool[at] = randn(gen, 4, W - 1, C, dtype=BF)
    before = pool[at].clone()
    y, got = kda_b200.short_conv_step(x, w, None, pool, at)
    assert got is pool
    check(x, w, None, before, [1] * 4, y, pool[at])
    assert not torch.equal(pool[at], before)
    pool[at] = 5.0
    assert all(bool((part == 5.0).all()) for part in pool.split(4096))
