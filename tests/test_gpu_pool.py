"""pool_copy, pool_fork, pool_free and pool_compact against the same steps on the CPU."""
import pytest
import torch

from serving_testlib import DEV, generator, randn

pytestmark = pytest.mark.gpu


def make(gen, P, shapes):
    return [randn(gen, P, *shape, dtype=dtype) if dtype.is_floating_point else torch.randint(0, 100, (P, *shape), generator=gen, device=DEV).to(dtype)
            for shape, dtype in shapes]


SHAPES = [[((2, 128, 128), torch.float32), ((3, 768), torch.bfloat16)], [((1, 5), torch.bfloat16), ((7,), torch.int8), ((3,), torch.float32)],
          [((5001,), torch.float16)], [((), torch.float32), ((4, 4), torch.float64)]]


@pytest.fixture
def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("P,seed", [(1, 0), (2, 1), (40, 2), (300, 3), (2050, 4)])
def test_fork_and_free(shapes, P, seed, status):
    import kda_b200
    gen, host = generator(seed), torch.Generator().manual_seed(seed)
    pools = make(gen, P, shapes if P < 1000 else SHAPES[1])
    used = torch.rand(P, generator=host) < 0.5
    live, free = [i for i in range(P) if used[i]], [i for i in range(P) if not used[i]]
    n = len(free)
    parents = [live[int(torch.randint(len(live), (1,), generator=host))] if live and i % 3 else -1 for i in range(n)]
    want = [p.clone() for p in pools]
    for slot, parent in zip(free, parents):
        for w, p in zip(want, pools):
            w[slot] = p[parent] if parent >= 0 else 0
    mask = used.to(DEV)
    slots = kda_b200.pool_fork(pools, mask, torch.tensor(parents, dtype=torch.int64, device=DEV), status=status)
    assert slots.tolist() == free and bool(mask.all()) and int(status) == 0
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    kda_b200.pool_free(mask, torch.cat([slots, torch.tensor([-1, -9], dtype=torch.int32, device=DEV)]), status=status)
    assert torch.equal(mask.cpu(), used) and int(status) == 0


def test_fork_of_bad_parents_and_a_full_pool(status):
    import kda_b200
    gen = generator(5)
    pools = make(gen, 8, SHAPES[0])
    used = torch.tensor([1, 0, 1, 1, 0, 1, 1, 0], dtype=torch.bool, device=DEV)
    before = [p.clone() for p in pools]
    slots = kda_b200.pool_fork(pools, used, torch.tensor([0, 1, 8, 2, -3, 5, 6], device=DEV), status=status)
    # 1 is free, 8 out of range; three slots for the five good entries
    assert slots.tolist() == [1, -1, -1, 4, 7, -1, -1] and int(status) == 2 | 32 and bool(used.all())
    for p, b in zip(pools, before):
        assert torch.equal(p[1], b[0]) and torch.equal(p[4], b[2]) and bool((p[7] == 0).all())
        assert torch.equal(p[[0, 2, 3, 5, 6]], b[[0, 2, 3, 5, 6]])
    status.zero_()
    assert kda_b200.pool_fork(pools, used, torch.tensor([0], device=DEV), status=status).tolist() == [-1] and int(status) == 32
    assert kda_b200.pool_fork(pools, used, torch.empty(0, dtype=torch.int32, device=DEV)).numel() == 0


def test_many_entries_over_a_full_pool(status):
    import kda_b200
    pools, used = [torch.arange(3000.0, device=DEV)[:, None]], torch.ones(3000, dtype=torch.bool, device=DEV)
    used[1::2] = False
    parents = torch.arange(0, 3000, device=DEV).repeat(2)             # half of them free, 3000 good ones for 1500 slots
    slots = kda_b200.pool_fork(pools, used, parents, status=status).tolist()
    good = [i for i in range(6000) if i % 2 == 0]
    assert [slots[i] for i in good[:1500]] == list(range(1, 3000, 2)) and set(slots) - set(range(1, 3000, 2)) == {-1} and int(status) == 34
    assert torch.equal(pools[0][1::2, 0], parents[good[:1500]].float())


def test_free_of_bad_slots(status):
    import kda_b200
    used = torch.tensor([1, 1, 0, 1, 1], dtype=torch.bool, device=DEV)
    kda_b200.pool_free(used, torch.tensor([0, 2, 5, 3, 0, -1], device=DEV, dtype=torch.int32), status=status)
    assert used.tolist() == [False, True, False, False, True] and int(status) == 2
    status.zero_()
    big = torch.ones(3000, dtype=torch.bool, device=DEV)
    kda_b200.pool_free(big, torch.cat([torch.arange(1500, device=DEV), torch.arange(5, device=DEV)]), status=status)
    assert int(big.sum()) == 1500 and bool(big[1500:].all()) and int(status) == 2


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("P,share,seed", [(1, 0.5, 1), (2, 0.5, 2), (64, 0.0, 3), (64, 1.0, 4), (64, 0.5, 5), (777, 0.3, 6), (777, 0.9, 7), (5000, 0.5, 8)])
def test_compact(shapes, P, share, seed, status):
    import kda_b200
    gen, host = generator(seed), torch.Generator().manual_seed(seed)
    pools = make(gen, P, shapes if P < 1000 else SHAPES[1])
    used = torch.rand(P, generator=host) < share
    live = [i for i in range(P) if used[i]]
    n = len(live)
    moves = dict(zip([i for i in live if i >= n], [i for i in range(n) if not used[i]]))
    want = [moves.get(i, i) if used[i] else -1 for i in range(P)]
    before = [p.clone() for p in pools]
    order = [live[i] for i in torch.randperm(n, generator=host).tolist()]
    tables = [torch.tensor(order + [-1], dtype=torch.int32, device=DEV), torch.tensor([-4] + order[:5], dtype=torch.int64, device=DEV)]
    mask = used.to(DEV)
    remap = kda_b200.pool_compact(pools, mask, tables, status=status)
    assert remap.tolist() == want and mask.tolist() == [i < n for i in range(P)] and int(status) == 0
    assert tables[0].tolist() == [want[i] for i in order] + [-1] and tables[1].tolist() == [-4] + [want[i] for i in order[:5]]
    for p, b in zip(pools, before):
        assert torch.equal(p[[want[i] for i in live]], b[live])


def test_compact_with_entries_of_free_slots(status):
    import kda_b200
    used = torch.tensor([0, 1, 0, 1], dtype=torch.bool, device=DEV)
    table = torch.tensor([3, 0, 4, 1, -2], device=DEV)
    remap = kda_b200.pool_compact([], used, [table], status=status)
    assert remap.tolist() == [-1, 1, -1, 0] and table.tolist() == [0, -1, -1, 1, -2] and int(status) == 2


@pytest.mark.parametrize("shapes", SHAPES)
def test_copy(shapes, status):
    import kda_b200
    gen = generator(9)
    pools = make(gen, 30, shapes)
    want = [p.clone() for p in pools]
    src, dst = [3, 7, 3, -1, 12, 29, 5], [0, 1, 2, 4, -1, 28, 5]
    for s, d in zip(src, dst):
        for w in want:
            if d >= 0:
                w[d] = w[s] if s >= 0 else 0
    kda_b200.pool_copy(pools, torch.tensor(src, dtype=torch.int32, device=DEV), torch.tensor(dst, device=DEV), status=status)
    assert int(status) == 0 and all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copies_that_depend_on_the_order_are_left_out(status):
    import kda_b200
    pool = torch.arange(10.0, device=DEV)[:, None].clone()
    #      into a source   repeated    out of range        fine
    src = [1, 2,           4, 5,       10, 6,              9]
    dst = [2, 3,           7, 7,       0, 11,              8]
    kda_b200.pool_copy([pool], torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV), status=status)
    assert int(status) == 2 and pool[:, 0].tolist() == [0, 1, 2, 2, 4, 5, 6, 4, 9, 9]


@pytest.mark.parametrize("n", [1, 1023, 1025, 2600])
def test_copies_by_long_tables(n, status):
    """Random tables against the rule entry by entry: repeats, chains, rows onto themselves, padding, entries out of range."""
    import kda_b200
    host = torch.Generator().manual_seed(n)
    P = 3 * n + 5
    pool = torch.arange(float(P), device=DEV)[:, None].clone()
    src, dst = torch.randint(-2, P + 2, (n,), generator=host), torch.randint(-2, P + 2, (n,), generator=host)
    some = torch.rand(n, generator=host) < 0.05
    dst[some] = src[some]
    want, seen, reads, bad = list(range(P)), set(), {s for s, d in zip(src.tolist(), dst.tolist()) if d >= 0}, False
    for s, d in zip(src.tolist(), dst.tolist()):
        if d < 0 or (d == s and d < P):
            seen |= {d}
            continue
        if d >= P or s >= P or d in seen or d in reads:
            bad = True
        else:
            want[d] = float(max(s, 0)) if s >= 0 else 0.0
        seen |= {d}
    kda_b200.pool_copy([pool], src.to(DEV), dst.to(torch.int32).to(DEV), status=status)
    assert pool[:, 0].tolist() == want and int(status) == (2 if bad else 0)


def test_strided_pools_keep_what_lies_between_their_slots():
    import kda_b200
    gen = generator(10)
    store = randn(gen, 20, 6, 64)
    keep = store.clone()
    kda_b200.pool_copy([store[:, 1:4], store[:, 5]], torch.tensor([0, 3], device=DEV), torch.tensor([10, 11], device=DEV))
    keep[[10, 11], 1:4], keep[[10, 11], 5] = keep[[0, 3], 1:4], keep[[0, 3], 5]
    assert torch.equal(store, keep)


def test_captured_calls_follow_their_tables(status):
    import kda_b200
    gen = generator(11)
    pools, used, parents = make(gen, 16, SHAPES[0]), torch.zeros(16, dtype=torch.bool, device=DEV), torch.full((3,), -1, device=DEV)
    kda_b200.pool_fork(pools, used.clone(), parents)
    torch.cuda.synchronize()
    fork, pack = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(fork):
        slots = kda_b200.pool_fork(pools, used, parents, status=status)
    table = torch.full((4,), -1, device=DEV)
    with torch.cuda.graph(pack):
        kda_b200.pool_compact(pools, used, [table], status=status)
    for live, ids in (([2, 9], [9, -1, 2]), ([0, 1, 2, 15], [15, 15, 0]), ([5], [5, 5, 5])):
        used.zero_()
        used[live] = True
        parents.copy_(torch.tensor(ids))
        before = [p.clone() for p in pools]
        fork.replay()
        free = [i for i in range(16) if i not in live][:3]
        assert slots.tolist() == free
        for p, b in zip(pools, before):
            for s, parent in zip(free, ids):
                assert torch.equal(p[s], b[parent] if parent >= 0 else torch.zeros_like(b[0]))
        table[:3] = slots
        middle = [p.clone() for p in pools]
        pack.replay()
        assert int(used.sum()) == len(live) + 3 and bool(used[:len(live) + 3].all())
        for p, m in zip(pools, middle):
            assert torch.equal(p[table[:3]], m[free])
    assert int(status) == 0


def test_offsets_behind_32_bits():
    import kda_b200
    pool = torch.zeros(9000, 16, 128, 128, device=DEV)                # 9.4e9 bytes, 2.4e9 values
    pool[8999] = 1.5
    pool[1] = 2.5
    kda_b200.pool_copy([pool], torch.tensor([8999, 1], device=DEV), torch.tensor([0, 8998], device=DEV))
    assert bool((pool[0] == 1.5).all()) and bool((pool[8998] == 2.5).all()) and bool((pool[8997] == 0).all())
