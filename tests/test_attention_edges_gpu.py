"""Calls of the attention operators at the edges of what they take: values that are not finite behind a mask, sequences without new tokens, lengths past the
table, many streams, plans and graphs, refused arguments."""
import math

import pytest
import torch

import attentionutil as A
from oputil import E, POISON, close, randn

pytestmark = pytest.mark.gpu


def paged(b, heads, kv_heads, d, dt=E.bf16, seed=1, **kw):
    """(plan, q, k, v, keys and values of each sequence)"""
    q, kv = A.inputs(b, heads, kv_heads, d, dt, seed)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, kv_heads, d, dt), A.cache(b, kv_heads, d, dt)
    for s, (ks, vs) in enumerate(kv):
        A.put(b, k_view, s, ks)
        A.put(b, v_view, s, vs)
    return E.Attention(heads, kv_heads, d, dtype=dt, page_size=b.page_size, **ld, **kw), q, k, v, kv


def run(plan, b, out, q, k, v, stream=None):
    assert plan.enqueue(out, q, k, v, b.table, b.lengths_t, b.starts_t, rows=b.rows, seqs=b.seqs, stream=stream) == E.ELB_OK, E.last_error()


@pytest.mark.parametrize("what", [A.NAN, math.inf, -math.inf])
@pytest.mark.parametrize("new,length,heads,kv_heads,d", [(3, 40, 8, 2, 128), (8, 500, 4, 4, 64), (90, 150, 8, 2, 128), (300, 300, 6, 2, 64), (130, 4000, 2, 1, 96), (40, 60, 2, 2, 20)])
@pytest.mark.parametrize("place", ["value", "key"])
def test_what_a_token_does_not_see_does_not_enter_its_result(what, new, length, heads, kv_heads, d, place):
    b = A.batch([new, new], [length, length + 5], 16)
    plan, q, k, v, kv = paged(b, heads, kv_heads, d)
    want, err, _ = A.wanted(b, q, kv, True, d ** -0.5, E.bf16)
    # of the last sequence, a token that the first half of its new ones do not see; one channel of the last key head
    at, channel, h = length + 5 - new + new // 2, d - 3, kv_heads - 1
    cache = v if place == "value" else k
    cache[int(b.table[1, at // 16]), h, at % 16, channel] = what
    out = A.poisoned(b.rows, heads, d, dt=E.bf16)
    torch.cuda.synchronize()
    run(plan, b, out, q, k, v)
    assert plan.device_status() == 0
    see = slice(new + new // 2, 2 * new)
    rows = out[see, h * (heads // kv_heads):]
    if place == "value":
        assert not bool(rows[..., channel].isfinite().any())
        keep = torch.arange(d, device="cuda") != channel
        close(rows[..., keep], want[see, h * (heads // kv_heads):][..., keep], err[see, h * (heads // kv_heads):][..., keep], E.bf16, "other channels")
    elif what != what:
        assert bool(rows.isnan().all())
    rows.zero_()
    want[see, h * (heads // kv_heads):] = 0
    close(out, want, err, E.bf16, "tokens that do not see it")


@pytest.mark.parametrize("seqs", [4, 31, 32, 33, 70])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128)])
def test_sequences_without_new_tokens(seqs, heads, kv_heads, d):
    """Few rows of a call among many places of a batch, the others of any length: what has no new tokens has no results, and its pages may be anyone's."""
    new = [1 if i in (1, seqs - 2) else 0 for i in range(seqs)]
    b = A.batch(new, [40 + 37 * (i % 30) for i in range(seqs)], 16)
    plan, q, k, v, kv = paged(b, heads, kv_heads, d)
    want, err, _ = A.wanted(b, q, kv, True, d ** -0.5, E.bf16)
    out = A.poisoned(b.rows, heads, d, dt=E.bf16)
    torch.cuda.synchronize()
    run(plan, b, out, q, k, v)
    assert plan.device_status() == 0
    close(out, want, err, E.bf16)


@pytest.mark.parametrize("new", [130, 257])
@pytest.mark.parametrize("causal", [True, False])
def test_a_long_cache_and_few_rows(new, causal):
    """Keys split over all SMs; the same bits again."""
    b = A.batch([new], [20000], 16)
    plan, q, k, v, kv = paged(b, 4, 1, 128, causal=causal)
    want, err, _ = A.wanted(b, q, kv, causal, 128 ** -0.5, E.bf16)
    out, again = A.poisoned(b.rows, 4, 128, dt=E.bf16), A.poisoned(b.rows, 4, 128, dt=E.bf16)
    torch.cuda.synchronize()
    run(plan, b, out, q, k, v)
    run(plan, b, again, q, k, v)
    assert plan.device_status() == 0
    close(out, want, err, E.bf16)
    assert torch.equal(out, again)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("scale", [1e-38, -1e-38, 2.0 ** -120])
def test_a_scale_near_zero_gives_means(new, scale):
    b = A.batch([new], [300], 16)
    plan, q, k, v, kv = paged(b, 4, 2, 64, scale=scale)
    out = A.poisoned(new, 4, 64, dt=E.bf16)
    torch.cuda.synchronize()
    run(plan, b, out, q, k, v)
    vs = kv[0][1].double().repeat_interleave(2, 1)
    seen = [vs[:300 - new + i + 1] for i in range(new)]
    want, size = (torch.stack([f(x).mean(0) for x in seen]) for f in (lambda x: x, torch.abs))
    # the terms are 1 as far as 16 bits go; their sums of at most 300 in 32 bits
    close(out, want, (2.0 ** -17 + (4 * math.sqrt(300) + 8) * 2.0 ** -23) * 2 * size, E.bf16)


@pytest.mark.parametrize("longer", [1, 40, 1 << 30])
def test_tokens_past_the_table_are_left_out(longer):
    """The table holds 64 tokens; of the sequence's 20 new ones those behind that have no place, the others stand where they belong."""
    b = A.batch([20], [64], 16)
    k, v = (torch.full((b.pages, 2, 16, 32), POISON, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, nk, nv = (randn(20, h, 32, dtype=torch.bfloat16, seed=h) for h in (4, 2, 2))
    q_out, plan = torch.full_like(q, POISON), E.CacheAppend(4, 2, 32, 16, rotary_dim=0)
    assert plan.prepare() == 0
    length = 64 + longer
    torch.cuda.synchronize()
    assert plan.enqueue(q_out, k, v, q, nk, nv, b.table, A.ints([length]), rows=20, seqs=1) == 0
    assert plan.device_status() == 105
    left = 0
    for i in range(20):
        place = length - 20 + i
        if place >= 64:
            assert bool((q_out[i] == POISON).all())
            continue
        left += 1
        page = int(b.table[0, place // 16])
        assert torch.equal(q_out[i], q[i]) and torch.equal(k[page, :, place % 16], nk[i]) and torch.equal(v[page, :, place % 16], nv[i])
    assert int((k != POISON).any(-1).sum()) == int((v != POISON).any(-1).sum()) == 2 * left


@pytest.mark.parametrize("new", [1, 200])
def test_plans_and_graphs_beside_one_another(new):
    """Three plans on three streams at once, and two captured calls of one plan replayed one after the other, give what single calls give."""
    cases = []
    for i, (heads, kv_heads, d, length) in enumerate([(8, 2, 128, 3000), (4, 4, 64, 900), (8, 1, 96, 5000)]):
        b = A.batch([new] * 3, [length, new, length // 2 + new], 16, seed=i)
        plan, q, k, v, _ = paged(b, heads, kv_heads, d, seed=5 * i + 1)
        out = A.poisoned(b.rows, heads, d, dt=E.bf16)
        torch.cuda.synchronize()
        run(plan, b, out, q, k, v)
        torch.cuda.synchronize()
        cases.append((plan, b, q, k, v, out, torch.cuda.Stream()))
    outs = [[torch.full_like(c[5], POISON) for _ in range(6)] for c in cases]
    torch.cuda.synchronize()
    for j in range(6):
        for (plan, b, q, k, v, _, s), o in zip(cases, outs):
            run(plan, b, o[j], q, k, v, s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, c[5]) for c, o in zip(cases, outs) for x in o)
    plan, b, q, k, v, out, s = cases[0]
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.full_like(out, POISON) for _ in range(2)]
    torch.cuda.synchronize()
    for g, r in zip(graphs, results):
        with torch.cuda.graph(g, stream=s):
            run(plan, b, r, q, k, v, s.cuda_stream)
    with torch.cuda.stream(s):
        for _ in range(3):
            for g, r in zip(graphs, results):
                r.fill_(POISON)
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(r, out) for r in results) and all(c[0].device_status() == 0 for c in cases)


@pytest.mark.parametrize("d", [96, 104, 56])
def test_what_lay_in_tensor_memory_does_not_matter(d):
    """Calls behind ones whose results are NaN in all of their channels give the bits that they give behind others."""
    b = A.batch([200] * 3, [700, 900, 800], 16)
    before, q0, k0, v0, _ = paged(b, 8, 2, 128 if d > 64 else 64)
    plan, q, k, v, _ = paged(b, 8, 2, d, seed=9)
    outs, rest = [A.poisoned(b.rows, 8, d, dt=E.bf16) for _ in range(2)], torch.empty_like(q0)
    torch.cuda.synchronize()
    for out in outs:
        for _ in range(3):
            run(before, b, rest, q0, k0, v0)
        run(plan, b, out, q, k, v)
        torch.cuda.synchronize()
        q0.fill_(A.NAN)
    assert bool(rest.isnan().all()) and torch.equal(*outs)
    assert plan.device_status() == before.device_status() == 0


def test_refused_calls():
    """Arguments that a call refuses, with the code and a word of the message; nothing is written."""
    b = A.batch([1, 1], [20, 20], 16)
    plan, q, k, v, _ = paged(b, 4, 2, 64)
    dense = E.Attention(4, 2, 64, causal=False)
    rotary, append = E.Rotary(4, 2, 64), E.CacheAppend(4, 2, 64, 16)
    out, at = A.poisoned(2, 4, 64, dt=E.bf16), torch.zeros(2, dtype=torch.int32, device="cuda")
    kd = randn(2, 30, 2, 64, dtype=torch.bfloat16, seed=3)
    L, p = E.lib, lambda t: t.data_ptr()                                                                                # noqa: E731

    def attend(op=plan, out=p(out), q=p(q), k=p(k), v=p(v), table=p(b.table), lengths=p(b.lengths_t), starts=None, rows=2, seqs=2, pages=b.pages, width=b.width):
        return L.elb_attention_enqueue(op.h, out, q, k, v, table, lengths, starts, rows, seqs, pages, width, None)
    assert rotary.enqueue(q, kd[0], q, kd[0], at, rows=2) == 2
    assert "not prepared" in E.last_error()
    assert L.elb_append_enqueue(append.h, p(out), p(k), p(v), p(q), p(kd), p(kd), p(b.table), p(b.lengths_t), None, 2, 2, b.pages, b.width, None) == 2
    assert "not prepared" in E.last_error()
    assert rotary.prepare() == 0 and append.prepare() == 0
    bad = [(dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(seqs=-1), "sequences"), (dict(seqs=1 << 25), "sequences"), (dict(pages=-1), "pages"), (dict(pages=1 << 31), "pages"),
           (dict(width=-1), "width"), (dict(width=1 << 31), "width"), (dict(rows=3), "starts are wanted"), (dict(out=None), "null"), (dict(q=None), "null"), (dict(k=None), "null"),
           (dict(v=None), "null"), (dict(table=None), "null"), (dict(lengths=None), "null"), (dict(out=p(out) + 1), "misaligned"), (dict(q=p(q) + 1), "misaligned"),
           (dict(k=p(k) + 1), "misaligned"), (dict(v=p(v) + 1), "misaligned"), (dict(table=p(b.table) + 2), "misaligned"), (dict(lengths=p(b.lengths_t) + 1), "misaligned"),
           (dict(starts=p(b.lengths_t) + 2), "misaligned"), (dict(op=dense), "dense"), (dict(op=rotary), ""), (dict(op=append), "")]
    for kw, word in bad:
        assert attend(**kw) == 2, kw
        assert word in E.last_error(), (kw, E.last_error())

    def put(q_out=p(out), kc=p(k), vc=p(v), q=p(q), nk=p(kd), nv=p(kd), table=p(b.table), lengths=p(b.lengths_t), rows=2, seqs=2):
        return L.elb_append_enqueue(append.h, q_out, kc, vc, q, nk, nv, table, lengths, None, rows, seqs, b.pages, b.width, None)
    before = k.clone()
    for kw, word in [(dict(rows=-1), "rows"), (dict(rows=3), "starts are wanted"), (dict(q_out=p(out) + 1), "misaligned"), (dict(kc=p(k) + 1), "misaligned"), (dict(nv=p(kd) + 1), "misaligned")] + \
            [({n: None}, "null") for n in ("q_out", "kc", "vc", "q", "nk", "nv", "table", "lengths")]:
        assert put(**kw) == 2, kw
        assert word in E.last_error(), (kw, E.last_error())
    for args, word in [((None, p(kd), p(q), p(kd), p(at), 2), "null"), ((p(q), p(kd), p(q), p(kd), None, 2), "null"), ((p(q), p(kd), p(q), p(kd), p(at), -2), "rows"),
                       ((p(q) + 1, p(kd), p(q), p(kd), p(at), 2), "misaligned"), ((p(q), p(kd), p(q), p(kd), p(at) + 2, 2), "misaligned")]:
        assert L.elb_rotary_enqueue(rotary.h, *args, None) == 2
        assert word in E.last_error()
    assert attend(rows=0) == 0 and attend(seqs=0, rows=2) == 0 and put(rows=0) == 0
    torch.cuda.synchronize()
    assert bool((out == POISON).all()) and torch.equal(k.nan_to_num(POISON), before.nan_to_num(POISON))
    assert plan.device_status() == append.device_status() == rotary.device_status() == 0
    assert plan.launch_count() == append.launch_count() == rotary.launch_count() == 0
