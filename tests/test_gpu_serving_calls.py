"""Calls with a layout that was checked before: other tensors, other addresses, other options, tensors that overlap or lie off 16 bytes,
threads, inference mode, more layouts than are remembered."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from serving_testlib import DEV, cu_of, generator, randn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_other_tensors_of_one_layout():
    import kda_b200
    gen = generator(1)
    outs = []
    for _ in range(3):
        x, w, pool, slots = randn(gen, 1, 6, 64, dtype=BF), randn(gen, 64, 4, dtype=BF), randn(gen, 8, 3, 64, dtype=BF), torch.randperm(8)[:6].to(DEV)
        one, two, status = pool.clone(), pool.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
        y, got = kda_b200.short_conv_step(x, w, None, one, slots, status=status)
        z = torch.empty_like(y)
        kda_b200.short_conv(x, w, None, two, cu_of([1] * 6), ssm_state_indices=slots, out=z)
        assert got is one and torch.equal(y, z) and torch.equal(one, two) and int(status) == 0
        slots[3] = slots[1]
        kda_b200.short_conv_step(x, w, None, one, slots, status=status)
        assert int(status) == 2
        outs.append(y)
    assert len({y.data_ptr() for y in outs}) == 3


def test_options_of_one_layout():
    import kda_b200
    gen = generator(2)
    x, w = randn(gen, 1, 6, 64), randn(gen, 64, 4)
    for _ in range(2):
        y, z = kda_b200.short_conv(x, w)[0], kda_b200.short_conv(x, w, activation=None)[0]
        torch.testing.assert_close(y, torch.nn.functional.silu(z), rtol=1e-5, atol=1e-6)
    q = torch.nn.functional.normalize(randn(gen, 1, 2, 3, 128), dim=-1).to(BF)
    g, beta, pool = -torch.rand(1, 2, 3, 128, device=DEV), torch.rand(1, 2, 3, device=DEV), randn(gen, 2, 3, 128, 128)
    a = [kda_b200.kda_step_plain(q, q, q, g, beta, s, pool.clone())[0].float() for s in (0.5, 1.0, torch.tensor(2.0), None)]
    assert torch.equal(a[1], 2 * a[0]) and torch.equal(a[2], 4 * a[0])
    torch.testing.assert_close(a[3], a[1] * 128 ** -0.5, rtol=2 ** -7, atol=0)


def test_tensors_that_overlap_or_lie_off_16_bytes_are_still_refused():
    import kda_b200
    gen = generator(3)
    x, w, store = randn(gen, 1, 4, 64, dtype=BF), randn(gen, 64, 4, dtype=BF), torch.zeros(4000, dtype=BF, device=DEV)
    pool, other = store[:4 * 192].view(4, 3, 64), store[192:192 + 256].view(1, 4, 64)
    kda_b200.short_conv_step(x, w, None, pool)
    kda_b200.short_conv_step(x, w, None, pool)
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.short_conv_step(other, w, None, pool)
    q, g, beta = randn(gen, 1, 1, 1, 128, dtype=BF), torch.zeros(1, 1, 1, 128, device=DEV), torch.zeros(1, 1, 1, device=DEV)
    room = torch.zeros(16384 + 8, device=DEV)
    kda_b200.kda_step_plain(q, q, q, g, beta, 1.0, room[:16384].view(1, 1, 128, 128))
    with pytest.raises(ValueError, match="16-byte"):
        kda_b200.kda_step_plain(q, q, q, g, beta, 1.0, room[1:16385].view(1, 1, 128, 128))
    used = torch.zeros(4, dtype=torch.bool, device=DEV)
    kda_b200.pool_fork([pool], used, torch.tensor([-1], device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        kda_b200.pool_fork([pool], store[10:12].view(torch.bool), torch.tensor([-1], device=DEV))


def test_threads_on_streams_of_their_own():
    import kda_b200
    gen = generator(4)
    x, w = [randn(gen, 1, 64, 512, dtype=BF) for _ in range(4)], randn(gen, 512, 4, dtype=BF)
    want, got = [kda_b200.short_conv(t, w)[0] for t in x], [None] * 4
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got[i] = kda_b200.short_conv(x[i], w)[0]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_parameters_and_inference_mode():
    import kda_b200
    gen = generator(5)
    layer = torch.nn.Conv1d(64, 64, 4, groups=64, padding=3, device=DEV)
    x = randn(gen, 1, 20, 64)
    want = torch.nn.functional.silu(layer(x.transpose(1, 2))[..., :20].transpose(1, 2))
    for _ in range(2):
        with torch.inference_mode():
            y, _ = kda_b200.short_conv(x, layer.weight, layer.bias)
        torch.testing.assert_close(y, want.detach(), rtol=1e-4, atol=1e-5)
        y, _ = kda_b200.short_conv(x, layer.weight, layer.bias)
        assert not y.requires_grad


def test_more_layouts_than_are_remembered(monkeypatch):
    import kda_b200
    from kda_b200 import serving
    monkeypatch.setattr(serving, "PLANS_MAX", 5)
    gen = generator(6)
    w = randn(gen, 16, 4)
    for n in list(range(1, 14)) * 2:
        x = randn(gen, 1, n, 16)
        y, _ = kda_b200.short_conv(x, w)
        padded = torch.cat([torch.zeros(3, 16, device=DEV), x[0]])
        want = torch.nn.functional.silu(sum(padded[j:j + n] * w[:, j] for j in range(4)))
        torch.testing.assert_close(y[0], want, rtol=1e-4, atol=1e-5)
        assert len(serving._plans) <= 5


FIRST_CALL = """
import sys
sys.path.insert(0, "eat-kernels_b200")
import torch, kda_b200
dev = "cuda:0"
x, w, h = torch.ones(1, 3000, 64, device=dev), torch.ones(64, 4, device=dev), torch.zeros(4, 3, 64, device=dev)
A, B, s = -torch.ones(64, 16, device=dev), torch.ones(1, 3000, 1, 16, device=dev), torch.zeros(4, 64, 16, device=dev)
q, g, b = torch.ones(1, 4, 2, 128, device=dev, dtype=torch.bfloat16), torch.zeros(1, 4, 2, 128, device=dev), torch.ones(1, 4, 2, device=dev)
S, used, none = torch.zeros(4, 2, 128, 128, device=dev), torch.zeros(4, dtype=torch.bool, device=dev), torch.tensor([-1, -1], device=dev)
def calls():
    slots = kda_b200.pool_fork([h, s, S], used, none)
    y, _ = kda_b200.short_conv(x, w)
    z, _ = kda_b200.selective_scan(y, x, A, B, B)
    kda_b200.short_conv_step(x[:, :4], w, None, h)
    kda_b200.selective_scan_step(x[:, :4], x[:, :4], A, B[:, :4], B[:, :4], None, None, None, s)
    o, _ = kda_b200.kda_step_plain(q, q, q, g, b, 1.0, S)
    kda_b200.pool_free(used, slots[:1])
    return z, o, kda_b200.pool_compact([h, s, S], used)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls()
graph.replay()
torch.cuda.synchronize()
first = [t.clone() for t in out] + [t.clone() for t in (h, s, S, used)]
for t in (h, s, S, used):
    t.zero_()
eager = list(calls()) + [h, s, S, used]
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, eager))
print("equal")
"""


def test_a_process_whose_first_calls_are_captured():
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]
