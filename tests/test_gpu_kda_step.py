"""kda_step and kda_step_plain against the recurrence in 64 bits and against the prefill, and a layer's serving loop: convolution,
prefill, forked slots, single tokens, freed and compacted slots."""
import pytest
import torch

import kda_oracle as ko
from serving_testlib import DEV, assert_within, cu_of, generator, kda_step64, randn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make(gen, N, H, raw):
    if raw:
        return dict(q=randn(gen, 1, N, H, 128, dtype=BF, scale=0.5), k=randn(gen, 1, N, H, 128, dtype=BF, scale=0.5), v=randn(gen, 1, N, H, 128, dtype=BF),
                    g=randn(gen, 1, N, H, 128, dtype=BF, scale=0.5), beta=randn(gen, 1, N, H, dtype=BF),
                    A_log=torch.log(torch.rand(H, generator=gen, device=DEV) * 15 + 1), dt_bias=torch.rand(H * 128, generator=gen, device=DEV) * 4 - 6)
    unit = lambda: torch.nn.functional.normalize(randn(gen, 1, N, H, 128), dim=-1).to(BF)  # noqa: E731
    return dict(q=unit(), k=unit(), v=randn(gen, 1, N, H, 128, dtype=BF), g=torch.nn.functional.logsigmoid(randn(gen, 1, N, H, 128)),
                beta=torch.sigmoid(randn(gen, 1, N, H)))


def call(a, raw, scale, pool, slots=None, **more):
    import kda_b200
    return (kda_b200.kda_step if raw else kda_b200.kda_step_plain)(**a, scale=scale, pool=pool, ssm_state_indices=slots, **more)


def check(a, raw, scale, before, rows, y, after):
    """Row i: state `before[i]`, output y[0, i], state `after[i]`."""
    for i in rows:
        S = before[i].transpose(1, 2) if raw else before[i]
        o, oE, new, E = kda_step64(a["q"][0, i], a["k"][0, i], a["v"][0, i], a["g"][0, i], a["beta"][0, i], a.get("A_log"), a.get("dt_bias"), scale, S, raw)
        assert_within(y[0, i], o, oE, f"output {i}")
        assert_within(after[i], new.transpose(1, 2) if raw else new, E.transpose(1, 2) if raw else E, f"state {i}")


@pytest.mark.parametrize("raw", [True, False])
@pytest.mark.parametrize("N,H,pad", [(1, 1, 0), (1, 16, 0), (3, 5, 2), (70, 2, 0), (9, 12, 1)])
def test_single_tokens(raw, N, H, pad):
    gen, scale = generator(N + H), 128 ** -0.5
    a, P = make(gen, N + pad, H, raw), N + pad + 2
    pool = randn(gen, P, H, 128, 128, scale=0.25)
    slots = torch.randperm(P, generator=torch.Generator().manual_seed(3))[:N + pad].to(torch.int64 if N > 5 else torch.int32).to(DEV)
    if pad:
        slots[1], slots[-1] = -1, -5
        a["v"][0, -1] = float("nan")
    live = [i for i in range(N + pad) if int(slots[i]) >= 0]
    dead = [i for i in range(N + pad) if i not in live]
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, got = call(a, raw, scale, pool, slots, status=status)
    assert got is pool and int(status) == 0
    check(a, raw, scale, before[slots.clamp(min=0).long()], live, y, pool[slots.clamp(min=0).long()])
    assert bool((y[0, dead] == 0).all())
    rest = [i for i in range(P) if i not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])
    out, again = torch.full_like(y, 3.0), before.clone()
    call(a, raw, scale, again, slots, out=out)
    assert torch.equal(out[0, live], y[0, live]) and bool((out[0, dead] == 3.0).all()) and torch.equal(again, pool)


@pytest.mark.parametrize("raw", [True, False])
def test_slots_out_of_range_or_named_twice(raw):
    gen = generator(30)
    a, pool = make(gen, 5, 3, raw), randn(gen, 4, 3, 128, 128, scale=0.25)
    before, status = pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    y, _ = call(a, raw, 0.1, pool, torch.tensor([2, 0, 2, 4, 0], device=DEV), status=status)
    assert int(status) == 2 and torch.equal(pool[[1, 3]], before[[1, 3]])
    zero = torch.zeros_like(before[0])
    init = torch.stack([before[2], before[0], zero, zero, zero])
    after = init.clone()
    y2, _ = call(a, raw, 0.1, after)
    assert torch.equal(y, y2) and torch.equal(pool[2], after[0]) and torch.equal(pool[0], after[1])
    check(a, raw, 0.1, init, range(5), y, after)


def test_strided_tokens_and_a_strided_pool():
    """Heads of a wider projection at an odd offset, slots further apart than a state."""
    gen, N, H = generator(31), 4, 3
    a = make(gen, N, H, True)
    wide = randn(gen, 1, N, 2000, dtype=BF)
    for i, n in enumerate("qkvg"):
        a[n] = wide[:, :, 1 + 400 * i:1 + 400 * i + H * 128].unflatten(2, (H, 128))
    a["beta"] = wide[:, :, 1700:1703]
    store = randn(gen, N, H + 2, 128, 128, scale=0.25)
    pool = store[:, 1:1 + H]
    before, keep = pool.clone(), store.clone()
    y, _ = call(a, True, 0.1, pool)
    check(a, True, 0.1, before, range(N), y, pool)
    assert torch.equal(store[:, 0], keep[:, 0]) and torch.equal(store[:, 4], keep[:, 4])


@pytest.mark.parametrize("raw", [True, False])
def test_hard_gates_and_empty_operands(raw):
    """Decay to nothing and none at all, keys and queries of zero norm, beta at its ends."""
    gen = generator(32)
    a, pool = make(gen, 4, 2, raw), randn(gen, 4, 2, 128, 128, scale=0.25)
    a["k"][0, 0] = 0
    a["q"][0, 1] = 0
    if raw:
        a["g"][0, 2], a["g"][0, 3] = 100.0, -100.0
        a["beta"][0, 2], a["beta"][0, 3] = 90.0, -90.0
    else:
        a["g"][0, 2], a["g"][0, 3] = -200.0, 0.0
        a["beta"][0, 2], a["beta"][0, 3] = 1.0, 0.0
    before = pool.clone()
    y, _ = call(a, raw, 128 ** -0.5, pool)
    check(a, raw, 128 ** -0.5, before, range(4), y, pool)


@pytest.mark.parametrize("raw", [True, False])
def test_the_token_after_a_prompt(raw):
    """A prefill of n + 1 tokens and one of n tokens with a step behind it."""
    import kda_b200
    gen, H, lens = generator(33), 4, [33, 1, 64, 7]
    T, cu = sum(lens) + len(lens), cu_of([n + 1 for n in lens])
    a, scale = make(gen, T, H, raw), 128 ** -0.5
    ends = (cu[1:] - 1).tolist()
    body = [t for t in range(T) if t not in ends]
    pick = lambda rows: {n: t[:, rows].contiguous() if n not in ("A_log", "dt_bias") else t for n, t in a.items()}  # noqa: E731
    init = randn(gen, 4, H, 128, 128, scale=0.25)
    if raw:
        whole, final = kda_b200.run(*a.values(), scale, init, cu)
        _, pool = kda_b200.run(*pick(body).values(), scale, init, cu_of(lens))
    else:
        whole, final = kda_b200.chunk_kda(**a, scale=scale, initial_state=init, output_final_state=True, cu_seqlens=cu)
        _, pool = kda_b200.chunk_kda(**pick(body), scale=scale, initial_state=init, output_final_state=True, cu_seqlens=cu_of(lens))
    y, _ = call(pick(ends), raw, scale, pool)
    ko.check_close(y, whole[:, ends], "output of the last token")
    ko.check_close(pool, final, "final state")


def test_other_types_are_cast_as_in_the_prefill():
    import kda_b200
    gen = generator(37)
    a, pool = make(gen, 3, 2, True), randn(gen, 3, 2, 128, 128, scale=0.25)
    one, two = pool.clone(), pool.clone()
    y, _ = kda_b200.kda_step(**a, scale=0.1, pool=one)
    z, _ = kda_b200.kda_step(**{n: t.double() if n in ("A_log", "dt_bias") else t.float() for n, t in a.items()}, scale=0.1, pool=two)
    assert torch.equal(y, z) and torch.equal(one, two) and z.dtype == BF


def test_captured_calls_follow_their_table():
    gen, N = generator(34), 4
    for raw in (True, False):
        a, pool = make(gen, N, 3, raw), randn(gen, 7, 3, 128, 128, scale=0.25)
        slots = torch.arange(N, device=DEV)
        call(a, raw, 0.1, pool.clone(), slots)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = call(a, raw, 0.1, pool, slots)
        for ids in ([0, 1, 2, 3], [6, -1, 2, 5], [-1, -1, -1, 1]):
            slots.copy_(torch.tensor(ids))
            a["v"].normal_()
            before = pool.clone()
            graph.replay()
            live, at = [i for i in range(N) if ids[i] >= 0], slots.clamp(min=0)
            check(a, raw, 0.1, before[at], live, y, pool[at])
            rest = [i for i in range(7) if i not in ids]
            assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("raw", [True, False])
def test_a_slot_behind_32_bits(raw):
    gen = generator(35)
    a, pool = make(gen, 2, 16, raw), torch.zeros(8300, 16, 128, 128, device=DEV)         # 2.2e9 values
    y, _ = call(a, raw, 0.1, pool, torch.tensor([8299, 5], device=DEV))
    at = [8299, 5]
    check(a, raw, 0.1, torch.zeros(2, 16, 128, 128, device=DEV), range(2), y, pool[at])
    assert int((pool.view(8300, -1) != 0).any(-1).sum()) == 2


def test_a_layer_served():
    """Prompts through convolution and prefill, sequences forked off them, tokens one by one, one sequence ended and the pools
    compacted: every output and state as if each sequence had been run whole."""
    import kda_b200
    gen, H, P, lens, more = generator(36), 2, 12, [40, 3, 70], 4
    C, scale, D = 3 * H * 128, 128 ** -0.5, 128
    weight = randn(gen, C, 4, dtype=BF, scale=0.5)
    A_log, dt_bias = torch.rand(H, generator=gen, device=DEV), torch.rand(H * D, generator=gen, device=DEV) * 4 - 6
    states, histories = torch.zeros(P, H, D, D, device=DEV), torch.zeros(P, 3, C, dtype=BF, device=DEV)
    used, status = torch.zeros(P, dtype=torch.bool, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    tokens = lambda n: (randn(gen, 1, n, C, dtype=BF), randn(gen, 1, n, H, D, dtype=BF, scale=0.5), randn(gen, 1, n, H, dtype=BF))  # noqa: E731
    qkv = lambda y: [t.unflatten(2, (H, D)) for t in y.split(H * D, 2)]  # noqa: E731
    # prompts
    slots = kda_b200.pool_fork([states, histories], used, torch.full((3,), -1, device=DEV), status=status)
    x, g, beta = tokens(sum(lens))
    cu = cu_of(lens)
    y, _ = kda_b200.short_conv(x, weight, None, histories, cu, ssm_state_indices=slots, status=status)
    kda_b200.kda_prefill(*qkv(y), g, beta, A_log, dt_bias, states, cu, ssm_state_indices=slots)
    streams = [[(x[:, a:b], g[:, a:b], beta[:, a:b])] for a, b in zip(cu[:-1].tolist(), cu[1:].tolist())]
    # two forks of the first, one of the third
    forks = kda_b200.pool_fork([states, histories], used, slots[[0, 0, 2]].contiguous(), status=status)
    table = torch.cat([slots, forks, torch.full((2,), -1, dtype=torch.int32, device=DEV)])
    streams += [list(streams[0]), list(streams[0]), list(streams[2])]
    outs = [[] for _ in range(6)]
    for j in range(more):
        x, g, beta = tokens(8)
        y, _ = kda_b200.short_conv_step(x, weight, None, histories, table, status=status)
        o, _ = kda_b200.kda_step(*qkv(y), g, beta, A_log, dt_bias, scale, states, table, status=status)
        for i in range(6):
            if int(table[i]) >= 0:
                streams[i].append((x[:, i:i + 1], g[:, i:i + 1], beta[:, i:i + 1]))
                outs[i].append(o[:, i:i + 1])
        if j == 1:                                                    # sequence 1 ends, the others move up
            kda_b200.pool_free(used, table[1:2], status=status)
            table[1] = -1
            kda_b200.pool_compact([states, histories], used, [table], status=status)
            assert used.tolist() == [True] * 5 + [False] * 7
    assert int(status) == 0 and sorted(table.tolist()) == [-1, -1, -1, 0, 1, 2, 3, 4]
    for i in (0, 2, 3, 4, 5):
        x, g, beta = (torch.cat(t, 1) for t in zip(*streams[i]))
        y, hist = kda_b200.short_conv(x, weight)
        o, final = kda_b200.kda_prefill(*qkv(y), g, beta, A_log, dt_bias, torch.zeros(1, H, D, D, device=DEV), None)
        ko.check_close(torch.cat(outs[i], 1), o[:, -len(outs[i]):], f"outputs of sequence {i}")
        ko.check_close(states[int(table[i])], final[0], f"state of sequence {i}")
        assert torch.equal(histories[int(table[i])], hist[0])
