"""Attention over a cache of pages and over dense tensors against the definition in 64 bits (attentionutil.py, which derives the bounds)."""
import math

import pytest
import torch

import attentionutil as A
from oputil import E, POISON, TORCH, close, randn, strided

pytestmark = pytest.mark.gpu


def check(plan):
    assert plan.device_status() == 0


def run_paged(b, heads, kv_heads, d, dt=E.bf16, causal=True, scale=0.0, order="heads", ld_extra=0, seed=1, size=1.0, stream=None):
    q, kv = A.inputs(b, heads, kv_heads, d, dt, seed, size)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, kv_heads, d, dt, order, ld_extra), A.cache(b, kv_heads, d, dt, order, ld_extra)
    for s, (ks, vs) in enumerate(kv):
        A.put(b, k_view, s, ks)
        A.put(b, v_view, s, vs)
    plan = E.Attention(heads, kv_heads, d, dtype=dt, page_size=b.page_size, causal=causal, scale=scale, **ld)
    out = A.poisoned(b.rows, heads, d, dt=dt)
    torch.cuda.synchronize()
    rc = plan.enqueue(out, q, k, v, b.table, b.lengths_t, b.starts_t, rows=b.rows, seqs=b.seqs)
    assert rc == E.ELB_OK, E.last_error()
    check(plan)
    want, err, rows = A.wanted(b, q, kv, causal, scale or 1.0 / math.sqrt(d), dt)
    close(out[:rows], want[:rows], err[:rows], dt, f"attention of {heads} over {kv_heads} heads of {d}")
    assert bool((out[rows:] == POISON).all()), "rows behind the last sequence"
    return plan


def run_dense(new, lengths, width, heads, kv_heads, d, dt=E.bf16, causal=False, given=True, behind=0, size=1.0):
    b = A.batch(new, lengths, 16, behind=behind)
    q, kv = A.inputs(b, heads, kv_heads, d, dt, 3, size)
    k = torch.full((b.seqs, width, kv_heads, d), A.NAN, dtype=TORCH[dt], device="cuda")
    v = k.clone()
    for s, (ks, vs) in enumerate(kv):
        k[s, :lengths[s]], v[s, :lengths[s]] = ks, vs
    plan = E.Attention(heads, kv_heads, d, dtype=dt, causal=causal)
    out = A.poisoned(b.rows, heads, d, dt=dt)
    torch.cuda.synchronize()
    rc = plan.enqueue(out, q, k, v, lengths=b.lengths_t if given else None, starts=b.starts_t, rows=b.rows, seqs=b.seqs)
    assert rc == E.ELB_OK, E.last_error()
    check(plan)
    want, err, rows = A.wanted(b, q, kv, causal, 1.0 / math.sqrt(d), dt)
    close(out[:rows], want[:rows], err[:rows], dt, "dense attention")
    assert bool((out[rows:] == POISON).all())


# ------------------------------------------------------------------------------------------- one token each, and a few
@pytest.mark.parametrize("lengths", [[1], [2], [15, 16, 17], [63, 64, 65, 0, 128, 129], [1000], [0], [700, 1, 0, 2500, 64], [4097] * 3], ids=str)
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (4, 4, 64), (7, 1, 96), (10, 2, 80)])
def test_token(lengths, heads, kv_heads, d):
    run_paged(A.batch([1] * len(lengths), lengths, 16), heads, kv_heads, d)


@pytest.mark.parametrize("page_size", [1, 5, 8, 16, 24, 32, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("dt", [E.bf16, E.f16])
def test_token_pages(page_size, dt):
    lengths = [1, page_size, page_size + 1, 3 * page_size - 1, 411]
    run_paged(A.batch([1] * 5, lengths, page_size), 8, 2, 128, dt)
    run_paged(A.batch([1] * 5, lengths, page_size), 6, 2, 64, dt, order="tokens")


@pytest.mark.parametrize("new", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (4, 4, 64), (16, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_tokens(new, heads, kv_heads, d, causal):
    run_paged(A.batch([new] * 4, [new, 200, 65, 1], 16), heads, kv_heads, d, causal=causal)


def test_many_sequences():
    lengths = [(37 * i) % 301 for i in range(700)]
    run_paged(A.batch([1] * 700, lengths, 16), 4, 1, 64)


def test_long_sequence_on_one_head():
    run_paged(A.batch([1], [70001], 64), 4, 1, 128)
    run_paged(A.batch([2, 2], [50000, 3], 64), 8, 1, 64, E.f16)


# ------------------------------------------------------------------------------------------- prompts
@pytest.mark.parametrize("n,length", [(1, 1), (17, 17), (64, 64), (100, 300), (127, 127), (128, 128), (129, 129), (255, 700), (256, 256), (257, 1100), (500, 500), (40, 3)])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (6, 2, 96)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt(n, length, heads, kv_heads, d, causal):
    run_paged(A.batch([n], [length], 16), heads, kv_heads, d, causal=causal)


@pytest.mark.parametrize("page_size", [1, 8, 16, 24, 32, 40, 64, 96, 128, 136, 256, 1000])
@pytest.mark.parametrize("dt", [E.bf16, E.f16])
def test_prompt_pages(page_size, dt):
    run_paged(A.batch([150, 150], [290, 777], page_size), 6, 2, 128, dt)
    run_paged(A.batch([150, 150], [290, 777], page_size), 6, 2, 64, dt, order="tokens", causal=False)


@pytest.mark.parametrize("new,lengths", [([5, 1, 0, 300, 64], [5, 700, 90, 300, 1000]), ([1, 1, 1], [400, 2, 77]), ([0, 0, 9], [5, 0, 9]), ([130] * 3, [0, 130, 131]),
                                         ([1, 600, 2], [1, 600, 2000])])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (3, 3, 64), (14, 2, 80)])
def test_ragged(new, lengths, heads, kv_heads, d):
    run_paged(A.batch(new, lengths, 16, ragged=True), heads, kv_heads, d)
    run_paged(A.batch(new, lengths, 16, behind=3), heads, kv_heads, d, causal=False)


@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 8), (2, 1, 16), (3, 1, 24), (12, 4, 32), (9, 3, 40), (128, 1, 64), (130, 1, 64), (66, 2, 56), (4, 2, 104), (5, 5, 120), (2, 1, 7),
                                              (4, 2, 100), (2, 2, 136), (4, 2, 192), (2, 1, 256), (3, 1, 1)])
def test_heads(heads, kv_heads, d):
    run_paged(A.batch([1] * 3, [33, 300, 1], 16), heads, kv_heads, d)
    run_paged(A.batch([90], [170], 16), heads, kv_heads, d)


def test_many_short_prompts():
    new = [(7 * i) % 23 for i in range(400)]
    run_paged(A.batch(new, [n + (11 * i) % 50 for i, n in enumerate(new)], 16), 4, 2, 64)


def test_piece_of_a_prompt_behind_a_long_cache():
    run_paged(A.batch([70], [9000], 32), 4, 1, 128)
    run_paged(A.batch([70, 3, 20], [9000, 20, 5001], 32), 8, 2, 64)


# ------------------------------------------------------------------------------------------- dense keys and values
@pytest.mark.parametrize("new,lengths,width", [([1] * 4, [1, 50, 0, 77], 77), ([30] * 3, [200, 1, 131], 200), ([200], [64], 64), ([3, 400, 1], [128, 129, 5], 129), ([1], [5000], 5000)])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (4, 2, 72), (2, 2, 20)])
@pytest.mark.parametrize("causal", [False, True])
def test_dense(new, lengths, width, heads, kv_heads, d, causal):
    run_dense(new, lengths, width, heads, kv_heads, d, causal=causal)


def test_dense_without_lengths():
    run_dense([1] * 2, [333] * 2, 333, 6, 3, 64, E.f16, given=False)
    run_dense([50] * 2, [333] * 2, 333, 6, 3, 64, E.f16, given=False, behind=2)


def test_no_keys():
    plan = E.Attention(4, 2, 64)
    q, out, k = randn(6, 4, 64, dtype=torch.bfloat16, seed=1), A.poisoned(6, 4, 64, dt=E.bf16), torch.empty(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert plan.enqueue(out, q, k, k, rows=6, seqs=2) == 0, E.last_error()
    check(plan)
    assert bool((out == 0).all())
    out.fill_(POISON)
    assert plan.enqueue(out, q, k, k, rows=0, seqs=2) == 0 and plan.enqueue(out, q, k, k, rows=6, seqs=0) == 0
    check(plan)
    assert bool((out == POISON).all())


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("n", [1, 70])
def test_rows_apart_and_unaligned(offset, n):
    """Rows of q and out that lie apart, k and v with heads in front of tokens, tensors that start anywhere."""
    heads, kv_heads, d, width, dt = 4, 2, 64, 150, E.bf16
    q, q_buf = strided(n, heads * d, 300, TORCH[dt], offset, source=randn(n, heads * d, dtype=TORCH[dt], seed=5))
    out, out_buf = strided(n, heads * d, 264, TORCH[dt], offset)
    k, v = (torch.empty(offset + kv_heads * width * 72, dtype=TORCH[dt], device="cuda")[offset:].view(1, kv_heads, width, 72)[..., :d] for _ in range(2))
    ks, vs = randn(width, kv_heads, d, dtype=TORCH[dt], seed=6), randn(width, kv_heads, d, dtype=TORCH[dt], seed=7)
    k[0], v[0] = ks.permute(1, 0, 2), vs.permute(1, 0, 2)
    plan = E.Attention(heads, kv_heads, d, causal=True, ld_input=300, ld_output=264, ld_head=width * 72, ld_token=72, ld_page=kv_heads * width * 72)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, rows=n, seqs=1) == 0, E.last_error()
    check(plan)
    want, err = A.attention64(q.view(n, heads, d), ks, vs, n, True, d ** -0.5, dt)
    close(out.reshape(n, heads, d), want, err, dt)
    from oputil import untouched
    untouched(out, out_buf)


# ------------------------------------------------------------------------------------------- values
@pytest.mark.parametrize("n", [1, 3, 90])
@pytest.mark.parametrize("size,dt", [(0.0, E.bf16), (8.0, E.bf16), (8.0, E.f16), (40.0, E.bf16)])
def test_sizes_of_scores(n, size, dt):
    """Scores that are all equal, and scores that are far apart and rise along the keys."""
    run_paged(A.batch([n], [600], 16), 4, 2, 64, dt, size=size)


@pytest.mark.parametrize("n", [1, 90])
def test_rising_scores(n):
    """The largest score moves on with every tile, so that every sum is scaled again."""
    heads, d, length, dt = 2, 64, 1500, E.bf16
    q = torch.ones(n, heads, d, dtype=TORCH[dt], device="cuda")
    k = (torch.arange(length, device="cuda") / 16.0).to(TORCH[dt])[:, None, None].expand(length, heads, d).contiguous()
    v = randn(length, heads, d, dtype=TORCH[dt], seed=4)
    for flip in (False, True):
        kk = k.flip(0).contiguous() if flip else k
        plan = E.Attention(heads, heads, d, causal=False, scale=0.5)
        out = A.poisoned(n, heads, d, dt=dt)
        torch.cuda.synchronize()
        assert plan.enqueue(out, q, kk[None], v[None], rows=n, seqs=1) == 0, E.last_error()
        check(plan)
        want, err = A.attention64(q, kk, v, n, False, 0.5, dt)
        close(out, want, err, dt)


@pytest.mark.parametrize("n", [1, 90])
def test_negative_scale_and_lowest_scores(n):
    run_paged(A.batch([n], [200], 16), 4, 2, 64, scale=-0.3)
    heads, d, length = 2, 64, 100
    q = torch.full((n, heads, d), 2.0 ** 60, dtype=torch.bfloat16, device="cuda")
    k = torch.full((1, length, heads, d), -2.0 ** 60, dtype=torch.bfloat16, device="cuda")
    v = randn(1, length, heads, d, dtype=torch.bfloat16, seed=4)
    plan, out = E.Attention(heads, heads, d, causal=False, scale=1.0), A.poisoned(n, heads, d, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, rows=n, seqs=1) == 0          # all scores -2^126
    check(plan)
    mean = v[0].double().mean(0).expand(n, -1, -1)
    close(out, mean, (2.0 ** -8 + 2.0 ** -15) * v[0].double().abs().mean(0).expand(n, -1, -1), E.bf16)


@pytest.mark.parametrize("n", [1, 90])
def test_nan_and_infinity_stay_in_their_rows(n):
    """A query that is NaN spoils its own row and head alone."""
    b = A.batch([n], [150], 16)
    q, kv = A.inputs(b, 4, 2, 64, E.bf16)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, 2, 64, E.bf16), A.cache(b, 2, 64, E.bf16)
    A.put(b, k_view, 0, kv[0][0])
    A.put(b, v_view, 0, kv[0][1])
    want, err, _ = A.wanted(b, q, kv, True, 0.125, E.bf16)
    q[n // 2, 1, 5] = A.NAN
    plan, out = E.Attention(4, 2, 64, page_size=16, **ld), A.poisoned(n, 4, 64, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, b.table, b.lengths_t, rows=n, seqs=1) == 0
    check(plan)
    assert bool(out[n // 2, 1].isnan().all())
    out[n // 2, 1], want[n // 2, 1] = 0, 0
    close(out, want, err, E.bf16)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, "pages", 2 ** 31 - 1])
def test_pages_outside_the_pool_count_as_zeros(n, bad):
    b = A.batch([n, n], [150, 200], 16)
    q, kv = A.inputs(b, 4, 2, 64, E.bf16)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, 2, 64, E.bf16), A.cache(b, 2, 64, E.bf16)
    for s in range(2):
        A.put(b, k_view, s, kv[s][0])
        A.put(b, v_view, s, kv[s][1])
    b.table[1, 3] = b.pages if bad == "pages" else bad
    kv[1][0][48:64], kv[1][1][48:64] = 0, 0
    plan, out = E.Attention(4, 2, 64, page_size=16, **ld), A.poisoned(2 * n, 4, 64, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, b.table, b.lengths_t, rows=2 * n, seqs=2) == 0
    assert plan.device_status() == 105
    want, err, _ = A.wanted(b, q, kv, True, 0.125, E.bf16)
    close(out, want, err, E.bf16)


@pytest.mark.parametrize("n", [1, 70])
def test_lengths_and_starts_are_held_in_bounds(n):
    """Lengths below zero or past the table count as the nearest that it can hold; starts past the rows end with them."""
    b = A.batch([n, n], [160, 160], 16, ragged=True)
    q, kv = A.inputs(b, 4, 2, 64, E.bf16)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, 2, 64, E.bf16), A.cache(b, 2, 64, E.bf16)
    for s in range(2):
        A.put(b, k_view, s, kv[s][0])
        A.put(b, v_view, s, kv[s][1])
    want, err, _ = A.wanted(b, q, kv, True, 0.125, E.bf16)
    plan, out = E.Attention(4, 2, 64, page_size=16, **ld), A.poisoned(2 * n, 4, 64, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, b.table, A.ints([1 << 30, 161]), A.ints([0, n, 1 << 30]), rows=2 * n, seqs=2) == 0
    check(plan)
    close(out, want, err, E.bf16)
    assert plan.enqueue(out, q, k, v, b.table, A.ints([-5, 160]), A.ints([0, n, 2 * n]), rows=2 * n, seqs=2) == 0
    check(plan)
    assert bool((out[:n] == 0).all())
    close(out[n:], want[n:], err[n:], E.bf16)


# ------------------------------------------------------------------------------------------- calls
@pytest.mark.parametrize("n", [1, 3, 200])
def test_same_bits_again_on_streams_and_in_graphs(n):
    """Calls of one plan on several streams at once and captured calls give the same bits; a graph is replayed on new inputs."""
    lengths = [900, 5, 2100]
    b = A.batch([n] * 3, [max(m, n) for m in lengths], 16)
    heads, kv_heads, d, dt = 8, 2, 128, E.bf16
    q, kv = A.inputs(b, heads, kv_heads, d, dt)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, kv_heads, d, dt), A.cache(b, kv_heads, d, dt)
    for s in range(3):
        A.put(b, k_view, s, kv[s][0])
        A.put(b, v_view, s, kv[s][1])
    plan = E.Attention(heads, kv_heads, d, page_size=16, **ld)
    out = A.poisoned(b.rows, heads, d, dt=dt)

    def call(o, stream=None):
        assert plan.enqueue(o, q, k, v, b.table, b.lengths_t, rows=b.rows, seqs=3, stream=stream) == 0, E.last_error()
    torch.cuda.synchronize()
    call(out)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(4)], [A.poisoned(b.rows, heads, d, dt=dt) for _ in range(12)]
    torch.cuda.synchronize()
    for i in range(12):
        call(outs[i], streams[i % 4].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)
    s, graph, again = torch.cuda.Stream(), torch.cuda.CUDAGraph(), A.poisoned(b.rows, heads, d, dt=dt)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        call(again, s.cuda_stream)
    for _ in range(3):
        again.fill_(POISON)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, out)
    q.copy_(randn(*q.shape, dtype=q.dtype, seed=77))
    b.lengths = [min(m, max(n, 33)) for m in b.lengths]
    b.lengths_t.copy_(A.ints(b.lengths))
    graph.replay()
    torch.cuda.synchronize()
    check(plan)
    want, err, _ = A.wanted(b, q, [(kk[:m], vv[:m]) for (kk, vv), m in zip(kv, b.lengths)], True, d ** -0.5, dt)
    close(again, want, err, dt)


def test_shared_pages():
    """Sequences whose tables name the same pages."""
    b = A.batch([1, 1], [160, 0], 16)
    q, kv = A.inputs(b, 4, 2, 64, E.bf16)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, 2, 64, E.bf16), A.cache(b, 2, 64, E.bf16)
    A.put(b, k_view, 0, kv[0][0])
    A.put(b, v_view, 0, kv[0][1])
    b.table[1] = b.table[0]
    b.lengths = [160, 100]
    plan, out = E.Attention(4, 2, 64, page_size=16, **ld), A.poisoned(2, 4, 64, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, b.table, A.ints(b.lengths), rows=2, seqs=2) == 0
    check(plan)
    want, err, _ = A.wanted(b, q, [kv[0], (kv[0][0][:100], kv[0][1][:100])], True, 0.125, E.bf16)
    close(out, want, err, E.bf16)


@pytest.mark.parametrize("n", [1, 40])
def test_offsets_past_32_bits(n):
    """The only pages in use lie behind 2^32 bytes and 2^31 elements of a pool."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    pages, page_size, kv_heads, d = 140000, 128, 1, 128              # 2.3e9 elements, 4.6 GB each
    k, v = (torch.empty(pages, kv_heads, page_size, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    length = 500
    ks, vs = randn(length, 1, d, dtype=torch.bfloat16, seed=1), randn(length, 1, d, dtype=torch.bfloat16, seed=2)
    table = A.ints([[pages - 1, 3, pages - 2, pages - 7]])
    for p in range(4):
        part = slice(p * 128, min(length, p * 128 + 128))
        at = int(table[0, p])
        k[at, 0, :part.stop - part.start], v[at, 0, :part.stop - part.start] = ks[part, 0], vs[part, 0]
    q, out = randn(n, 2, d, dtype=torch.bfloat16, seed=3), A.poisoned(n, 2, d, dt=E.bf16)
    plan = E.Attention(2, 1, d, page_size=page_size)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, table, A.ints([length]), rows=n, seqs=1) == 0
    check(plan)
    want, err = A.attention64(q, ks, vs, n, True, d ** -0.5, E.bf16)
    close(out, want, err, E.bf16)
