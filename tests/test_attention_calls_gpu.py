"""Calls of the attention operators that their documentation allows and that are easy to get wrong: plans used right after they are prepared, values that are not
finite in long caches, the largest scores, strides and batches."""
import pytest
import torch

import attentionutil as A
from oputil import E, close, randn

pytestmark = pytest.mark.gpu


def test_a_plan_is_ready_when_prepare_returns():
    """On a stream that waits for no other: calls right behind prepare, with frequencies that such a stream has just written."""
    rows, d = 64, 128
    s, pos = torch.cuda.Stream(), torch.arange(64, dtype=torch.int32, device="cuda") * 997
    x, out = randn(rows, 4, d, dtype=torch.float32, seed=1), torch.empty(rows, 4, d, dtype=torch.float32, device="cuda")
    slow = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    for i in range(20):
        f = torch.rand(d // 2, generator=torch.Generator().manual_seed(i))
        plan = E.Rotary(4, 0, d, dtype=E.f32)
        with torch.cuda.stream(s):
            for _ in range(10):
                slow.add_(1.0)
            given = f.to("cuda", non_blocking=True) + slow[0] * 0.0
        assert plan.prepare(given) == 0, E.last_error()
        assert plan.enqueue(out, None, x, None, pos, rows=rows, stream=s.cuda_stream) == 0, E.last_error()
        s.synchronize()
        want, err = A.turn64(x, pos, d, E.ROTARY_HALVES, f, 1.0)
        close(out, want, err + 1e-9, E.f32)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_frequencies_of_another_gpu():
    rows, d = 64, 128
    pos, x, out = torch.arange(64, dtype=torch.int32, device="cuda"), randn(rows, 2, d, dtype=torch.float32, seed=1), torch.empty(rows, 2, d, dtype=torch.float32, device="cuda")
    slow, s = torch.zeros(1 << 28, device="cuda:1"), torch.cuda.Stream(device=1)
    for i in range(3):
        torch.cuda.synchronize(0)
        torch.cuda.synchronize(1)
        f = torch.rand(d // 2, generator=torch.Generator().manual_seed(i))
        plan = E.Rotary(2, 0, d, dtype=E.f32, device=0)
        with torch.cuda.stream(s):
            for _ in range(20):
                slow.add_(1.0)
            given = f.to("cuda:1") + slow[0] * 0.0
        assert plan.prepare(given) == 0, E.last_error()
        assert plan.enqueue(out, None, x, None, pos, rows=rows) == 0, E.last_error()
        torch.cuda.synchronize(0)
        want, err = A.turn64(x, pos, d, E.ROTARY_HALVES, f, 1.0)
        close(out, want, err + 1e-9, E.f32)
