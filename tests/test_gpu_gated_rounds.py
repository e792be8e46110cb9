"""The recurrence over several rounds of clusters of every size that layers have, one block alone among them, forward and backward, against
the definition in 64 bits.  A cluster's blocks work on 96 tokens each forward and on 48 backward; how many there are goes by the channels."""
import pytest
import torch

from gated_testlib import forward64, gradients64
from serving_testlib import assert_within, cu_of
from test_gpu_gated_scan import rows
from test_gpu_gated_scan_grad import NAMES, case, leaves

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

CASES = {
    "64 channels, 16 blocks": ([1, 4000, 0, 2500, 37, 1600, 96, 1], 64, BF, "power", 1),
    "33 channels one by one, 16 blocks": ([5000, 96, 0, 2304], 33, F32, "logistic", 1),
    "1024 channels": ([17, 3000, 1536, 0, 200], 1024, FP, "logistic", 0),
    "2560 channels": ([700, 1, 1200, 0, 96, 513], 2560, BF, "power", 1),
    "4096 channels": ([900, 0, 383, 1, 100, 60], 4096, BF, "power", 1),
    "8192 channels": ([191, 1, 0, 500, 250], 8192, FP, "power", 0),
    "20000 channels, blocks alone": ([95, 1, 0, 192, 130, 7], 20000, BF, "power", 1),
    "9001 channels one by one, blocks alone": ([300, 0, 5, 95, 48], 9001, BF, "power", 1),
    "5000 channels in 32 bits, blocks alone": ([100, 288, 0, 1, 50], 5000, F32, "logistic", 1),
}


@pytest.mark.parametrize("lens,C,dtype,form,gated", CASES.values(), ids=CASES.keys())
def test_rounds(lens, C, dtype, form, gated):
    import kda_b200
    tensors, dy, dfinal = case(lens, C, dtype, form, gated, seed=C)
    v = leaves(*tensors)
    y, final = kda_b200.gated_scan(*v, cu_of(lens))
    got = iter(torch.autograd.grad((y, final), [t for t in v if t is not None], (dy, dfinal)))
    got = [next(got) if t is not None else None for t in v]
    plain = [rows(t) for t in tensors[:3]] + tensors[3:6]
    want, e, wf, fe = forward64(lens, *plain, tensors[6])
    assert_within(y.detach()[0], want, e, "y")
    assert_within(final.detach(), wf, fe, "final state")
    del want, e
    for name, g, w in zip(NAMES, got, gradients64(lens, plain, tensors[6], dy[0], dfinal)):
        if g is not None:
            assert_within(g.reshape(w[0].shape), w[0], w[1], name)
