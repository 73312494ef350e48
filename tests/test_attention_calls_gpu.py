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


# ------------------------------------------------------------------------------------------- memory's full rate
@pytest.mark.parametrize("heads,kv_heads,d,dt", [(32, 8, 128, E.bf16), (16, 16, 64, E.f16)])
def test_the_same_bits_at_the_memory_s_full_rate(heads, kv_heads, d, dt):
    """A large batch of single tokens, whose copies come as fast as memory gives them, again and again: every tile is read before the next one takes its place."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    seqs, page = 64, 64
    lengths = [500 + (15501 * ((61 * i) % seqs)) // seqs for i in range(seqs)]
    held = [-(-n // page) for n in lengths]
    g = torch.Generator(device="cuda").manual_seed(3)
    order = torch.randperm(sum(held), generator=g, device="cuda").to(torch.int32)
    table = torch.full((seqs, max(held)), A.FAR_PAGE, dtype=torch.int32, device="cuda")
    for s, n in enumerate(held):
        table[s, :n] = order[sum(held[:s]):sum(held[:s]) + n]
    q = randn(seqs, heads, d, dtype=A.TORCH[dt], seed=1, scale=1.5)
    k, v = (randn(sum(held), kv_heads, page, d, dtype=A.TORCH[dt], seed=i) for i in (2, 3))
    plan, out = E.Attention(heads, kv_heads, d, dtype=dt, page_size=page), A.poisoned(seqs, heads, d, dt=dt)

    def call():
        assert plan.enqueue(out, q, k, v, table, A.ints(lengths), rows=seqs, seqs=seqs) == 0, E.last_error()
    call()
    torch.cuda.synchronize()
    first = out.clone()
    for s in (0, 17, 63):
        pages = table[s, :held[s]].long()
        ks, vs = (t[pages].permute(0, 2, 1, 3).flatten(0, 1)[:lengths[s]] for t in (k, v))
        want, err = A.attention64(q[s:s + 1], ks, vs, 1, True, d ** -0.5, dt)
        close(first[s:s + 1], want, err, dt, f"sequence {s}")
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        call()
        differ += (out != first).any()
    assert int(differ) == 0 and plan.device_status() == 0
