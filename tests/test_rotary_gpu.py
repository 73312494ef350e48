"""Rotary positions and appending to a cache of pages against the definitions in 64 bits."""
import pytest
import torch

import attentionutil as A
from oputil import E, POISON, TORCH, close, randn, strided, untouched

pytestmark = pytest.mark.gpu
LAYOUTS = [E.ROTARY_HALVES, E.ROTARY_NEIGHBOURS]


def positions(rows, far, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, far, (rows,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("rows", [1, 7, 1300])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dt", [E.bf16, E.f16, E.f32])
@pytest.mark.parametrize("heads,kv_heads,d,r", [(4, 2, 128, 128), (3, 1, 80, 32), (2, 2, 64, 48), (1, 1, 7, 6), (5, 0, 96, 96), (0, 3, 64, 2), (2, 1, 24, 20)])
def test_rotary(rows, layout, dt, heads, kv_heads, d, r):
    pos = positions(rows, 200000, rows)
    q, k = randn(rows, heads, d, dtype=TORCH[dt], seed=1), randn(rows, kv_heads, d, dtype=TORCH[dt], seed=2)
    plan = E.Rotary(heads, kv_heads, d, rotary_dim=r, dtype=dt, layout=layout, magnitude=1.25)
    assert plan.prepare() == 0, E.last_error()
    q_out, k_out = torch.full_like(q, POISON), torch.full_like(k, POISON)
    torch.cuda.synchronize()
    assert plan.enqueue(q_out, k_out, q, k, pos, rows=rows) == 0, E.last_error()
    assert plan.device_status() == 0
    for x, y in ((q, q_out), (k, k_out)):
        want, err = A.turn64(x, pos, r, layout, A.steps64(r), 1.25)
        close(y, want, err, dt)
        assert torch.equal(y[..., r:], x[..., r:])
    # in place
    assert plan.enqueue(q, k, q, k, pos, rows=rows) == 0
    torch.cuda.synchronize()
    assert torch.equal(q, q_out) and torch.equal(k, k_out)


@pytest.mark.parametrize("scaling", [E.SCALE_NONE, E.SCALE_LINEAR, E.SCALE_BY_PARTS])
@pytest.mark.parametrize("base", [100.0, 10000.0, 5e6])
def test_scaling_and_far_positions(scaling, base):
    """Positions up to the ends of their type: the 32-bit angle alone would have lost the turn."""
    pos = A.ints([0, 1, 2, 4095, 131072, 10 ** 6 + 7, 2 ** 24 + 1, 2 ** 31 - 1, -1, -(2 ** 31)])
    x = randn(len(pos), 2, 128, dtype=torch.float32, seed=1)
    plan = E.Rotary(2, 0, 128, dtype=E.f32, base=base, scaling=scaling, factor=8.0, slow=1.0, fast=4.0, original=8192)
    assert plan.prepare() == 0, E.last_error()
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    assert plan.enqueue(out, None, x, None, pos, rows=len(pos)) == 0, E.last_error()
    assert plan.device_status() == 0
    steps = A.steps64(128, base, scaling, 8.0)
    want, err = A.turn64(x, pos, 128, E.ROTARY_HALVES, steps, 1.0)
    # the definition's own angle in 64 bits is off by 2^-52 of itself, as is the frequency that it is made from
    err = err + (x.double().abs() + x.double().roll(64, -1).abs()) * (pos.double().abs()[:, None, None] * steps.max() * 2.0 ** -50)
    close(out, want, err, E.f32)


def test_frequencies_and_inverse():
    f = torch.tensor([1.0, 0.3, 7.5, 0.0, 1e-5, -2.0, 100.0, 0.25])
    pos = positions(50, 100000, 3)
    x = randn(50, 3, 16, dtype=torch.float32, seed=1)
    there, back = E.Rotary(3, 0, 16, dtype=E.f32), E.Rotary(3, 0, 16, dtype=E.f32, inverse=True)
    assert there.prepare(f) == 0 and back.prepare(f.cuda()) == 0, E.last_error()
    y, z = torch.empty_like(x), torch.empty_like(x)
    torch.cuda.synchronize()
    assert there.enqueue(y, None, x, None, pos, rows=50) == 0 and back.enqueue(z, None, y, None, pos, rows=50) == 0
    torch.cuda.synchronize()
    want, err = A.turn64(x, pos, 16, E.ROTARY_HALVES, f, 1.0)
    close(y, want, err + 1e-9, E.f32)
    assert float((z - x).abs().max()) <= 2.0 ** -18 * float(x.abs().max())        # two turns of |a| + |b| 2^-20 each
    want, err = A.turn64(x, pos, 16, E.ROTARY_HALVES, f, 1.0, inverse=True)
    assert back.enqueue(z, None, x, None, pos, rows=50) == 0
    torch.cuda.synchronize()
    close(z, want, err + 1e-9, E.f32)


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rotary_rows_apart(offset):
    rows, d = 33, 64
    q, _ = strided(rows, 2 * d, 200, torch.bfloat16, offset, source=randn(rows, 2 * d, dtype=torch.bfloat16, seed=1))
    out, buf = strided(rows, 2 * d, 136, torch.bfloat16, offset)
    pos = positions(rows, 1000, 1)
    plan = E.Rotary(2, 0, d, ld_q=200, ld_q_out=136)
    assert plan.prepare() == 0
    torch.cuda.synchronize()
    assert plan.enqueue(out, None, q, None, pos, rows=rows) == 0, E.last_error()
    assert plan.device_status() == 0
    want, err = A.turn64(q.reshape(rows, 2, d), pos, d, E.ROTARY_HALVES, A.steps64(d), 1.0)
    close(out.reshape(rows, 2, d), want, err, E.bf16)
    untouched(out, buf)


# ------------------------------------------------------------------------------------------- append
def run_append(b, heads, kv_heads, d, r, dt=E.bf16, layout=E.ROTARY_HALVES, order="heads", ld_extra=0, bad=(), status=0, **kw):
    """``bad``: rows that have no place"""
    k_cache, k_view, ld = A.cache(b, kv_heads, d, dt, order, ld_extra, fill=POISON)
    v_cache, v_view, _ = A.cache(b, kv_heads, d, dt, order, ld_extra, fill=POISON)
    q, k, v = (randn(b.rows, h, d, dtype=TORCH[dt], seed=i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    q_out = torch.full_like(q, POISON)
    plan = E.CacheAppend(heads, kv_heads, d, b.page_size, rotary_dim=r, dtype=dt, layout=layout, **ld, **kw)
    assert plan.prepare() == 0, E.last_error()
    torch.cuda.synchronize()
    assert plan.enqueue(q_out, k_cache, v_cache, q, k, v, b.table, b.lengths_t, b.starts_t, rows=b.rows, seqs=b.seqs) == 0, E.last_error()
    assert plan.device_status() == status
    at = torch.cat([torch.arange(m - n, m) for m, n in zip(b.lengths, b.new)] + [torch.zeros(b.rows - b.starts[-1], dtype=torch.int64)]).cuda()
    steps = A.steps64(max(r, 2), **{k: v for k, v in kw.items() if k != "magnitude"})
    (want_q, err_q), (want_k, err_k) = (A.turn64(x, at, r, layout, steps, kw.get("magnitude", 1.0)) if r else (x.double(), torch.zeros_like(x, dtype=torch.float64)) for x in (q, k))
    keep = torch.tensor([i not in bad and i < b.starts[-1] for i in range(b.rows)], device="cuda")
    close(q_out[keep], want_q[keep], err_q[keep], dt)
    assert bool((q_out[~keep] == POISON).all())
    left = torch.ones(b.pages, b.page_size, dtype=torch.bool)
    for s in range(b.seqs):
        for i in range(b.new[s]):
            row, place = b.starts[s] + i, b.lengths[s] - b.new[s] + i
            if row in bad:
                continue
            page, offset = int(b.table[s, place // b.page_size]), place % b.page_size
            left[page, offset] = False
            close(k_view[page, :, offset], want_k[row], err_k[row], dt, f"row {row}")
            assert torch.equal(v_view[page, :, offset], v[row])
    left = left.cuda()[:, None, :, None]
    assert bool((k_view.masked_fill(~left, POISON) == POISON).all()) and bool((v_view.masked_fill(~left, POISON) == POISON).all()), "other places"
    return plan


@pytest.mark.parametrize("dt", [E.bf16, E.f16, E.f32])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("heads,kv_heads,d,r,order", [(4, 2, 128, 128, "heads"), (3, 3, 80, 32, "tokens"), (2, 1, 10, 6, "heads"), (0, 2, 64, 0, "tokens")])
def test_append(dt, layout, heads, kv_heads, d, r, order):
    run_append(A.batch([1] * 5, [1, 16, 17, 300, 33], 16), heads, kv_heads, d, r, dt, layout, order)
    run_append(A.batch([5, 1, 0, 40, 16], [5, 64, 90, 60, 16], 16, behind=2), heads, kv_heads, d, r, dt, layout, order, ld_extra=8)


@pytest.mark.parametrize("page_size", [1, 5, 64, 200])
def test_append_pages(page_size):
    run_append(A.batch([70, 70], [70, 311], page_size), 4, 2, 64, 64, scaling=E.SCALE_BY_PARTS, factor=4.0, original=64, magnitude=1.5)


def test_append_many():
    new = [(7 * i) % 13 for i in range(300)]
    run_append(A.batch(new, [n + (5 * i) % 40 for i, n in enumerate(new)], 16), 2, 1, 32, 32)
    run_append(A.batch([2500], [3000], 16), 2, 1, 64, 64)


def test_rows_without_a_place_are_left_out():
    # more new tokens than the sequence holds; a page outside the pool
    run_append(A.batch([4, 1], [3, 20], 16), 2, 1, 32, 32, bad={0}, status=105)
    for page in (-1, 1 << 30, -2 ** 31):
        b = A.batch([1, 20], [5, 40], 16)
        b.table[1, 1] = page
        run_append(b, 2, 1, 32, 32, bad=set(range(1, 13)), status=105)
    b = A.batch([1], [5], 16)
    b.table[0, 0] = b.pages
    run_append(b, 2, 1, 32, 32, bad={0}, status=105)


def test_append_on_streams_and_in_a_graph():
    """A step that is captured once and replayed with lengths that grow, as a program that answers token by token does it."""
    b = A.batch([1, 1], [40, 40], 16)
    k_cache, v_cache = (torch.full((b.pages, 2, 16, 64), POISON, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    plan = E.CacheAppend(4, 2, 64, 16)
    assert plan.prepare() == 0
    q, k, v = (randn(2, h, 64, dtype=torch.bfloat16, seed=h) for h in (4, 2, 2))
    q_out, lengths, s, graph = torch.empty_like(q), A.ints([0, 0]), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        lengths.add_(1)
        assert plan.enqueue(q_out, k_cache, v_cache, q, k, v, b.table, lengths, rows=2, seqs=2, stream=s.cuda_stream) == 0, E.last_error()
    lengths.zero_()
    for i in range(40):
        x = randn(2, 2, 64, dtype=torch.bfloat16, seed=100 + i)
        k.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want, err = A.turn64(x, A.ints([i, i]), 64, E.ROTARY_HALVES, A.steps64(64), 1.0)
        got = torch.stack([k_cache[int(b.table[n, i // 16]), :, i % 16] for n in range(2)])
        close(got, want, err, E.bf16)
    assert plan.device_status() == 0
