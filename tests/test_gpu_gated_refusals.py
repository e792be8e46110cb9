"""Arguments that the gated linear recurrence and the group norm refuse on a device, before anything is launched."""
import pytest
import torch

from test_gpu_serving_refusals import ints, zeros

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def scan(**change):
    import kda_b200
    a = dict(x=zeros(1, 8, 64), r=zeros(1, 8, 64), i=zeros(1, 8, 64), rate=zeros(64), r_bias=zeros(64), i_bias=zeros(64), initial_state=zeros(4, 64), cu_seqlens=ints(0, 5, 8),
             ssm_state_indices=ints(0, 1))
    kda_b200.gated_scan(**dict(a, **change))


def train(**change):
    import kda_b200
    a = dict(x=zeros(1, 8, 64).requires_grad_(), r=zeros(1, 8, 64), i=zeros(1, 8, 64), rate=zeros(64), r_bias=zeros(64), i_bias=zeros(64), initial_state=zeros(2, 64),
             cu_seqlens=ints(0, 5, 8))
    kda_b200.gated_scan(**dict(a, **change))


def step(**change):
    import kda_b200
    a = dict(x=zeros(1, 2, 64), r=zeros(1, 2, 64), i=None, rate=None, r_bias=None, i_bias=None, pool=zeros(4, 64), ssm_state_indices=ints(0, 1))
    kda_b200.gated_scan_step(**dict(a, **change))


def norm(**change):
    import kda_b200
    kda_b200.group_norm(**dict(dict(x=zeros(1, 8, 64), groups=4, weight=zeros(64), bias=zeros(64), z=zeros(1, 8, 64)), **change))


CASES = [
    (scan, dict(x=lambda: zeros(2, 8, 64))), (scan, dict(x=lambda: zeros(1, 8, 64, dtype=torch.float64))), (scan, dict(r=lambda: zeros(1, 8, 64, dtype=BF))),
    (scan, dict(r=lambda: None)), (scan, dict(r=lambda: zeros(1, 7, 64))), (scan, dict(i=lambda: zeros(1, 8, 63))), (scan, dict(i=lambda: None)),
    (scan, dict(rate=lambda: zeros(63))), (scan, dict(rate=lambda: zeros(64, dtype=BF))), (scan, dict(r_bias=lambda: zeros(65))), (scan, dict(i_bias=lambda: zeros(64, dtype=BF))),
    (scan, dict(initial_state=lambda: None)), (scan, dict(initial_state=lambda: zeros(4, 63))), (scan, dict(initial_state=lambda: zeros(4, 64, dtype=BF))),
    (scan, dict(initial_state=lambda: zeros(1, 64).expand(4, 64))), (scan, dict(initial_state=lambda: zeros(64, 4).t())), (scan, dict(cu_seqlens=lambda: zeros(3))),
    (scan, dict(cu_seqlens=lambda: ints(0))), (scan, dict(ssm_state_indices=lambda: ints(0))), (scan, dict(ssm_state_indices=lambda: None)),
    (scan, dict(out=lambda: zeros(1, 8, 65))), (scan, dict(out=lambda: zeros(1, 8, 64, dtype=BF))), (scan, dict(out=lambda: zeros(1, 1, 64).expand(1, 8, 64))),
    (scan, dict(status=lambda: zeros(1))), (scan, dict(rate_scale=lambda: 0.0)),
    (train, dict(initial_state=lambda: zeros(4, 64))), (train, dict(r=lambda: zeros(1, 8, 64, dtype=BF))), (train, dict(status=lambda: zeros(1))), (train, dict(i=lambda: None)),
    (step, dict(pool=lambda: None)), (step, dict(pool=lambda: zeros(4, 63))), (step, dict(ssm_state_indices=lambda: ints(0, 1, 2))),
    (step, dict(pool=lambda: zeros(1, 64), ssm_state_indices=lambda: None)), (step, dict(i_bias=lambda: zeros(64))),
    (norm, dict(x=lambda: zeros(8, 64))), (norm, dict(x=lambda: zeros(1, 8, 64, dtype=torch.float64))), (norm, dict(groups=lambda: 5)), (norm, dict(groups=lambda: 0)),
    (norm, dict(groups=lambda: None)), (norm, dict(groups=lambda: 4.0)), (norm, dict(weight=lambda: zeros(63))), (norm, dict(weight=lambda: zeros(64, dtype=BF))),
    (norm, dict(weight=lambda: zeros(16))), (norm, dict(bias=lambda: zeros(15))), (norm, dict(z=lambda: zeros(1, 8, 63))), (norm, dict(z=lambda: zeros(1, 8, 64, dtype=BF))),
    (norm, dict(activation=lambda: "gelu")), (norm, dict(eps=lambda: -1.0)), (norm, dict(out=lambda: zeros(1, 8, 65))), (norm, dict(out=lambda: zeros(1, 1, 64).expand(1, 8, 64))),
    (norm, dict(x=lambda: zeros(1, 2, 16385), groups=lambda: 1, weight=lambda: None, bias=lambda: None, z=lambda: None)),
    (norm, dict(x=lambda: zeros(1, 8, 4, 16), groups=lambda: 8)),
]


@pytest.mark.parametrize("call,change", CASES, ids=[f"{call.__name__}-{i}" for i, (call, _) in enumerate(CASES)])
def test_refused(call, change):
    call()
    with pytest.raises(ValueError, match="KDA kernel"):
        call(**{name: make() for name, make in change.items()})
    torch.cuda.synchronize()


def test_written_buffers_that_overlap_are_refused():
    import kda_b200
    x, pool = zeros(1, 8, 64), zeros(8, 64)
    for _ in range(2):
        kda_b200.gated_scan(x, x, out=zeros(1, 8, 64))
        with pytest.raises(ValueError, match="overlap"):
            kda_b200.gated_scan(x, x, out=x)
        with pytest.raises(ValueError, match="overlap"):
            kda_b200.gated_scan_step(pool.view(1, 8, 64), x, None, None, None, None, pool)
        with pytest.raises(ValueError, match="overlap"):
            kda_b200.group_norm(x, 4, out=x)
        cu = ints(0, 5, 8)
        with pytest.raises(ValueError, match="overlap"):
            kda_b200.gated_scan(x, x, None, None, None, None, zeros(2, 64), cu, status=cu[:1])
        with pytest.raises(ValueError, match="overlap"):
            train(cu_seqlens=cu, status=cu[:1])
    torch.cuda.synchronize()
