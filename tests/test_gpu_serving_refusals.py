"""Arguments that the operators around the prefill refuse on a device, before anything is launched."""
import pytest
import torch

from serving_testlib import DEV

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def conv(**change):
    import kda_b200
    a = dict(x=zeros(1, 8, 64), weight=zeros(64, 4), bias=None, initial_state=zeros(4, 3, 64), cu_seqlens=ints(0, 5, 8), ssm_state_indices=ints(0, 1))
    kda_b200.short_conv(**dict(a, **change))


def conv_step(**change):
    import kda_b200
    kda_b200.short_conv_step(**dict(dict(x=zeros(1, 2, 64), weight=zeros(64, 4), bias=None, pool=zeros(4, 3, 64), ssm_state_indices=ints(0, 1)), **change))


def scan(**change):
    import kda_b200
    a = dict(u=zeros(1, 8, 64), dt=zeros(1, 8, 64), A=zeros(64, 16), B=zeros(1, 8, 1, 16), C=zeros(1, 8, 1, 16), initial_state=zeros(4, 64, 16),
             cu_seqlens=ints(0, 5, 8), ssm_state_indices=ints(0, 1))
    kda_b200.selective_scan(**dict(a, **change))


def scan_step(**change):
    import kda_b200
    a = dict(u=zeros(1, 2, 64), dt=zeros(1, 2, 64), A=zeros(64, 16), B=zeros(1, 2, 1, 16), C=zeros(1, 2, 1, 16), D=None, z=None, dt_bias=None,
             pool=zeros(4, 64, 16), ssm_state_indices=ints(0, 1))
    kda_b200.selective_scan_step(**dict(a, **change))


def step(**change):
    import kda_b200
    t = zeros(1, 2, 3, 128, dtype=BF)
    a = dict(q=t, k=t, v=t, g=t, beta=zeros(1, 2, 3, dtype=BF), A_log=zeros(3), dt_bias=zeros(384), scale=0.1, pool=zeros(4, 3, 128, 128),
             ssm_state_indices=ints(0, 1))
    kda_b200.kda_step(**dict(a, **change))


def fork(**change):
    import kda_b200
    kda_b200.pool_fork(**dict(dict(pools=[zeros(4, 8)], used=zeros(4, dtype=torch.bool), parents=ints(-1)), **change))


def copy(**change):
    import kda_b200
    kda_b200.pool_copy(**dict(dict(pools=[zeros(4, 8)], src=ints(0), dst=ints(1)), **change))


def compact(**change):
    import kda_b200
    kda_b200.pool_compact(**dict(dict(pools=[zeros(4, 8)], used=zeros(4, dtype=torch.bool), tables=[ints(-1)]), **change))


CASES = [
    (conv, dict(x=lambda: zeros(2, 8, 64))), (conv, dict(x=lambda: zeros(1, 8, 64, dtype=torch.float64))), (conv, dict(weight=lambda: zeros(63, 4))),
    (conv, dict(weight=lambda: zeros(64, 5))), (conv, dict(weight=lambda: zeros(64, 1))), (conv, dict(bias=lambda: zeros(63))),
    (conv, dict(bias=lambda: zeros(64, dtype=BF))), (conv, dict(activation=lambda: "gelu")), (conv, dict(cu_seqlens=lambda: zeros(3))),
    (conv, dict(cu_seqlens=lambda: ints(0))), (conv, dict(initial_state=lambda: None)), (conv, dict(initial_state=lambda: zeros(4, 4, 64))),
    (conv, dict(initial_state=lambda: zeros(4, 3, 64, dtype=BF))), (conv, dict(initial_state=lambda: zeros(1, 3, 64).expand(4, 3, 64))),
    (conv, dict(ssm_state_indices=lambda: None)), (conv, dict(ssm_state_indices=lambda: ints(0, 1, 2))), (conv, dict(ssm_state_indices=lambda: ints(0, 9, 1, 9)[::2])),
    (conv, dict(out=lambda: zeros(1, 8, 65))), (conv, dict(out=lambda: zeros(1, 8, 64, dtype=BF))), (conv, dict(out=lambda: zeros(1, 1, 64).expand(1, 8, 64))),
    (conv, dict(status=lambda: zeros(1))),
    (conv_step, dict(pool=lambda: None)), (conv_step, dict(pool=lambda: zeros(4, 3, 63))), (conv_step, dict(ssm_state_indices=lambda: ints(0))),
    (conv_step, dict(pool=lambda: zeros(1, 3, 64), ssm_state_indices=lambda: None)),
    (scan, dict(dt=lambda: zeros(1, 8, 64, dtype=BF))), (scan, dict(dt=lambda: None)), (scan, dict(A=lambda: zeros(64, 129))), (scan, dict(A=lambda: zeros(64, 16, dtype=BF))),
    (scan, dict(B=lambda: zeros(1, 8, 3, 16))), (scan, dict(B=lambda: zeros(1, 8, 16))), (scan, dict(C=lambda: zeros(1, 8, 1, 15))), (scan, dict(D=lambda: zeros(63))),
    (scan, dict(z=lambda: zeros(1, 7, 64))), (scan, dict(dt_bias=lambda: zeros(64, dtype=BF))), (scan, dict(initial_state=lambda: zeros(4, 64, 16, dtype=BF))),
    (scan_step, dict(pool=lambda: zeros(4, 64, 15))), (scan_step, dict(ssm_state_indices=lambda: ints(0, 1, 2))),
    (step, dict(q=lambda: zeros(1, 2, 3, 64, dtype=BF))), (step, dict(k=lambda: zeros(1, 3, 3, 128, dtype=BF))), (step, dict(beta=lambda: zeros(1, 2, 4, dtype=BF))),
    (step, dict(A_log=lambda: zeros(4))), (step, dict(dt_bias=lambda: zeros(3))), (step, dict(pool=lambda: zeros(4, 3, 128, 128, dtype=BF))),
    (step, dict(pool=lambda: zeros(4 * 3 * 16384 + 1)[1:].view(4, 3, 128, 128))), (step, dict(pool=lambda: zeros(4, 3, 128, 128).transpose(2, 3))),
    (step, dict(pool=lambda: zeros(1, 3, 128, 128), ssm_state_indices=lambda: None)),
    (fork, dict(pools=lambda: [zeros(4, 8)] * 9)), (fork, dict(pools=lambda: [zeros(5, 8)])), (fork, dict(used=lambda: zeros(4))),
    (fork, dict(used=lambda: zeros(8, dtype=torch.bool)[::2])), (fork, dict(parents=lambda: zeros(1))), (fork, dict(pools=lambda: [zeros(4, 8).t().contiguous().t()])),
    (copy, dict(pools=lambda: [])), (copy, dict(src=lambda: ints(0, 1))), (copy, dict(pools=lambda: [zeros(1, 8).expand(4, 8)])), (copy, dict(pools=lambda: [zeros(4, 0)])),
    (compact, dict(tables=lambda: [ints(0)] * 9)), (compact, dict(tables=lambda: [zeros(1)])), (compact, dict(status=lambda: zeros(1))),
]


@pytest.mark.parametrize("call,change", CASES, ids=[f"{call.__name__}-{i}" for i, (call, _) in enumerate(CASES)])
def test_refused(call, change):
    call()
    with pytest.raises(ValueError, match="KDA kernel"):
        call(**{name: make() for name, make in change.items()})
    torch.cuda.synchronize()


def test_written_buffers_that_overlap_are_refused():
    import kda_b200
    x, pool = zeros(1, 8, 64), zeros(4, 3, 64)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.short_conv(x, zeros(64, 4), out=x)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.short_conv_step(pool.view(1, -1, 64)[:, :2], zeros(64, 4), None, pool)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.pool_fork([pool, pool], zeros(4, dtype=torch.bool), ints(-1))
    table = ints(0, 1)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.pool_compact([pool], zeros(4, dtype=torch.bool), [table, table])
    h = zeros(4, 64, 16)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.selective_scan_step(zeros(1, 2, 64), zeros(1, 2, 64), h[0], zeros(1, 2, 1, 16), zeros(1, 2, 1, 16), None, None, None, h)


def test_status_that_overlaps_an_operand_is_refused():
    """The kernels OR bits into it while other blocks read the tables.  Nothing is reported in these calls, so that they only write
    where they may."""
    import kda_b200
    cu, slots = ints(0, 5, 8), ints(0, 1)
    for call, operand in ((conv, dict(cu_seqlens=cu)), (conv, dict(ssm_state_indices=slots)), (conv_step, dict(ssm_state_indices=slots)),
                          (scan, dict(cu_seqlens=cu)), (scan_step, dict(ssm_state_indices=slots)), (step, dict(ssm_state_indices=slots))):
        for _ in range(2):
            call(**operand, status=ints(0))
            with pytest.raises(ValueError, match="overlap"):
                call(**operand, status=next(iter(operand.values()))[:1])
    src, used, slots = ints(0), zeros(4, dtype=torch.bool), ints(-1)
    for call, operand in ((lambda s: copy(src=src, status=s), src), (lambda s: fork(used=used, parents=slots, status=s), slots),
                          (lambda s: kda_b200.pool_free(used, slots, status=s), slots), (lambda s: compact(tables=[slots], status=s), slots)):
        for _ in range(2):
            call(ints(0))
            with pytest.raises(ValueError, match="overlap"):
                call(operand)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.short_conv(zeros(1, 8, 64), zeros(64, 4), None, None, cu, status=cu[1:])
    torch.cuda.synchronize()
