"""Group norm at the widths where the forward pass and the gradients change from a warp's registers to a block's work."""
import pytest
import torch

from test_gpu_group_norm import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [256, 257, 260, 320, 384, 508, 512, 513, 516, 520, 640, 768, 1016, 1024, 1028, 1032])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_widths(D, dtype):
    check(45, 3, D, dtype, seed=D)
    check(9, 11, D, dtype, "sigmoid", shared=True, center=False, seed=D + 1)
    check(33, 1, D, dtype, None, z=False, weight=False, bias=False, seed=D + 2)
