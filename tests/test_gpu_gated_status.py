"""What the gated linear recurrence reports through `status` from its backward passes."""
import pytest
import torch

from serving_testlib import DEV, cu_of
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
