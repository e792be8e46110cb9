"""What the gated linear recurrence reports through `status` from its backward passes and of empty sequences."""
import pytest
import torch

from serving_testlib import DEV, cu_of, generator, randn
from test_gpu_gated_scan import inputs
from test_gpu_gated_scan_grad import case, leaves

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def fresh_status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_backward_passes_report_into_the_calls_status(dtype):
    """A rejected layout is found again by the backward pass (the caller has cleared the word meanwhile); twice, since the second call of a
    layout takes the remembered checks."""
    import kda_b200
    tensors, dy, dfinal = case([30, 50], 64, dtype, "power", 1, 31)
    for _ in range(2):
        status, v = fresh_status(), leaves(*tensors)
        out = kda_b200.gated_scan(*v, torch.tensor([0, 90, 80], device=DEV), status=status)
        assert int(status) == 1
        status.zero_()
        torch.autograd.grad(out, v, (dy, dfinal))
        assert int(status) == 1
        status.zero_()
        out = kda_b200.gated_scan(*v, cu_of([30, 50]), status=status)
        torch.autograd.grad(out, v, (dy, dfinal))
        assert int(status) == 0


def test_slots_of_empty_sequences_are_checked():
    """As by the convolution and the selective scan: out of range or a repeat is reported whether the sequence has tokens or not, and
    whether the layout is rejected or not; a sequence that names the slot of an empty one is a repeat."""
    import kda_b200
    gen, C = generator(32), 64
    for lens, slots, bits in (([3, 0], [0, 99], 2), ([3, 0], [1, 1], 2), ([0, 3], [1, 1], 2), ([0, 3, 0], [-1, 2, 3], 2), ([0, 0], [4, 4], 2), ([0, 0], [4, 5], 0),
                              ([0, 3, 0, 200, 0], [3, 0, 2, 1, 4], 0), ([0, 3, 0, 200, 0], [3, 0, 3, 1, 4], 2)):
        x, r, i, rate, rb, ib = inputs(gen, sum(lens), C, F32, "power", 1)
        pool, table = randn(gen, 6, C), torch.tensor(slots, device=DEV)
        before, status = pool.clone(), fresh_status()
        kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, cu_of(lens), ssm_state_indices=table, status=status)
        assert int(status) == bits, (lens, slots)
        kept = [s for s in range(6) if s not in [s for s, n in zip(slots, lens) if n > 0]]
        assert torch.equal(pool[kept], before[kept])
        other, word = randn(gen, 6, 3, C), fresh_status()
        kda_b200.short_conv(x, torch.ones(C, 4, device=DEV), None, other, cu_of(lens), ssm_state_indices=table, status=word)
        assert int(word) == bits
    x, r, i, rate, rb, ib = inputs(gen, 8, C, F32, "power", 1)
    for slots, bits in (([0, 1], 1), ([0, 6], 3), ([2, 2], 3)):
        pool, table, status, word = randn(gen, 6, C), torch.tensor(slots, device=DEV), fresh_status(), fresh_status()
        before = pool.clone()
        kda_b200.gated_scan(x, r, i, rate, rb, ib, pool, torch.tensor([0, 9, 8], device=DEV), ssm_state_indices=table, status=status)
        kda_b200.short_conv(x, torch.ones(C, 4, device=DEV), None, randn(gen, 6, 3, C), torch.tensor([0, 9, 8], device=DEV), ssm_state_indices=table, status=word)
        assert int(status) == bits and int(word) == bits and torch.equal(pool, before)


@pytest.mark.parametrize("C", [64, 33], ids=["copies", "one by one"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_a_wait_that_runs_out_is_reported(dtype, C):
    """The blocks of a cluster wait for each other's maps.  With the diagnostic switch under which they wait for one more than is sent,
    all run into the (shortened) bound: the call still ends, says so, and the next one is right.  Nothing faults or hangs."""
    import kda_b200
    from kda_b200 import _cabi
    lens = [1700, 1, 1299]
    tensors, dy, dfinal = case(lens, C, dtype, "power", 1, 33)
    v, cu, status = leaves(*tensors), cu_of(lens), fresh_status()
    want = kda_b200.gated_scan(*v, cu, status=status)
    grads = torch.autograd.grad(want, v, (dy, dfinal), retain_graph=True)
    assert int(status) == 0
    for back in (False, True):
        status.zero_()
        torch.cuda.synchronize()
        assert _cabi.lib().kda_debug_configure(200, 2, None) == 0             # 200 us
        try:
            if back:
                torch.autograd.grad(want, v, (dy, dfinal), retain_graph=True)
            else:
                kda_b200.gated_scan(*tensors, cu, status=status)
            torch.cuda.synchronize()
        finally:
            assert _cabi.lib().kda_debug_configure(0, 0, None) == 0
        assert int(status) == 64
    status.zero_()
    again = kda_b200.gated_scan(*v, cu, status=status)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, v, (dy, dfinal)), grads)) and int(status) == 0
