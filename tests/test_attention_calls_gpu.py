"""Calls of the attention operators that their documentation allows and that are easy to get wrong: plans used right after they are prepared, values that are not
finite in long caches, the largest scores, strides and batches."""
import pytest
import torch

import attentionutil as A
from oputil import E, POISON, close, randn

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
    plan, out, held_t = E.Attention(heads, kv_heads, d, dtype=dt, page_size=page), A.poisoned(seqs, heads, d, dt=dt), A.ints(lengths)

    def call():
        assert plan.enqueue(out, q, k, v, table, held_t, rows=seqs, seqs=seqs) == 0, E.last_error()
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


# ------------------------------------------------------------------------------------------- values that are not finite
def filled(new, lengths, heads, kv_heads, d, page_size, dt=E.bf16, seed=1, causal=True, bad=(), width=None):
    """(call, out, want, bound, rows that no value spoils): a plan over a cache, or dense keys with ``page_size`` 0, whose values have ``bad`` (sequence, key, head, channel, value)."""
    b = A.batch(new, lengths, page_size or 16, seed, width=width)
    q, kv = A.inputs(b, heads, kv_heads, d, dt, seed)
    want, err, _ = A.wanted(b, q, kv, causal, d ** -0.5, dt)
    spoilt = torch.zeros(want.shape, dtype=torch.bool, device="cuda")
    group = heads // kv_heads
    for s, j, h, c, what in bad:
        kv[s][1][j, h, c] = what
        for i in range(b.new[s]):
            if not causal or j <= lengths[s] - b.new[s] + i:
                spoilt[b.starts[s] + i, h * group:(h + 1) * group, c] = True
    if page_size:
        (k, k_view, ld), (v, v_view, _) = A.cache(b, kv_heads, d, dt), A.cache(b, kv_heads, d, dt)
        for s, (ks, vs) in enumerate(kv):
            A.put(b, k_view, s, ks)
            A.put(b, v_view, s, vs)
        rest = (b.table, b.lengths_t, b.starts_t)
    else:
        k = torch.full((b.seqs, max(lengths), kv_heads, d), A.NAN, dtype=q.dtype, device="cuda")
        v, ld, rest = k.clone(), {}, (None, b.lengths_t, b.starts_t)
        for s, (ks, vs) in enumerate(kv):
            k[s, :lengths[s]], v[s, :lengths[s]] = ks, vs
    plan, out = E.Attention(heads, kv_heads, d, dtype=dt, page_size=page_size, causal=causal, **ld), A.poisoned(b.rows, heads, d, dt=dt)

    def call():
        assert plan.enqueue(out, q, k, v, *rest, rows=b.rows, seqs=b.seqs) == 0, E.last_error()
        return plan
    torch.cuda.synchronize()
    return call, out, want, err, spoilt


SHAPES = [([5, 5], [5, 200], 8, 2, 128), ([8], [3001], 4, 4, 64), ([2, 7, 32], [40, 1000, 32], 2, 2, 96), ([16, 16], [16, 90], 2, 1, 64), ([200], [200], 8, 2, 128), ([130, 300], [700, 300], 6, 2, 64),
          ([300], [4100], 4, 1, 128), ([40, 3], [33, 3], 5, 1, 80), ([260], [20000], 2, 2, 64)]


@pytest.mark.parametrize("new,lengths,heads,kv_heads,d", SHAPES, ids=str)
@pytest.mark.parametrize("page_size", [16, 24, 72, 136, 0])
@pytest.mark.parametrize("dt", [E.bf16, E.f16])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(new, lengths, heads, kv_heads, d, page_size, dt):
    """Some thirty values anywhere among the last keys, of which rows see some, all or none: a channel that a row sees one in is not finite, every other is right."""
    g = torch.Generator().manual_seed(7)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=g))                                                         # noqa: E731
    bad = []
    for s, (n, m) in enumerate(zip(new, lengths)):
        places = [m - 1, max(0, m - n), max(0, m - n - 1)] + [m - 1 - draw(min(m, 2 * n)) for _ in range(8)]
        bad += [(s, j, draw(kv_heads), draw(d), [A.NAN, float("inf"), -float("inf")][draw(3)]) for j in places]
    call, out, want, err, spoilt = filled(new, lengths, heads, kv_heads, d, page_size, dt, bad=bad)
    plan = call()
    assert plan.device_status() == 0
    assert not bool(out[spoilt].isfinite().any())
    out[spoilt], want[spoilt] = 0, 0
    close(out, want, err, dt)
    first = out.clone()
    call()
    torch.cuda.synchronize()
    out[spoilt] = 0
    assert torch.equal(out, first)


def milliseconds(call):
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    call()
    torch.cuda.synchronize()
    begin.record()
    call()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end)


@pytest.mark.parametrize("new,length,heads,kv_heads,d", [(8, 100000, 4, 1, 128), (8, 100000, 4, 1, 64), (4096, 4096, 8, 2, 128), (4096, 4096, 4, 2, 64)])
@pytest.mark.parametrize("place", ["seen", "half"])
def test_a_value_that_is_not_finite_costs_little(new, length, heads, kv_heads, d, place):
    """A row worked out again by a warp takes half a microsecond for each of its keys: 50 ms here for one of these rows, and seconds for longer ones."""
    bad = [(0, 5 if place == "seen" else length - new // 2, 0, 3, float("inf"))]
    call, out, want, err, spoilt = filled([new], [length], heads, kv_heads, d, 16, bad=bad)
    clean, _, _, _, _ = filled([new], [length], heads, kv_heads, d, 16)
    took, usual = milliseconds(call), milliseconds(clean)
    assert not bool(out[spoilt].isfinite().any())
    out[spoilt], want[spoilt] = 0, 0
    close(out, want, err, E.bf16)
    assert took <= 3 * usual + 2.0, (took, usual)


# ------------------------------------------------------------------------------------------- strides and batches
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("what", ["page", "row", "dense"])
def test_strides_that_no_tiled_copy_takes(n, what):
    """Rows and pages of which there is one may lie as far apart as the description takes."""
    far, d, dt = 1 << 40, 64, E.bf16
    q, k, v = (randn(m, 1, d, dtype=A.TORCH[dt], seed=m) for m in (n, 50, 51))
    v = v[:50].contiguous()
    out = A.poisoned(n, 1, d, dt=dt)
    rows, table, lengths = 1 if what == "row" else n, A.ints([[0]]), A.ints([50])
    if what == "page":
        plan = E.Attention(1, 1, d, page_size=64, ld_page=far)
        kc, vc = (torch.cat([x, x.new_zeros(14, 1, d)]).permute(1, 0, 2)[None].contiguous() for x in (k, v))
        args = (kc.data_ptr(), vc.data_ptr(), table.data_ptr(), lengths.data_ptr(), None, rows, 1, 1, 1)
    else:
        plan = E.Attention(1, 1, d, **(dict(ld_page=far) if what == "dense" else dict(ld_input=far, ld_output=far)))
        args = (k.data_ptr(), v.data_ptr(), None, None, None, rows, 1, 1, 50)
    torch.cuda.synchronize()
    assert E.lib.elb_attention_enqueue(plan.h, out.data_ptr(), q.data_ptr(), *args, None) == 0, E.last_error()
    assert plan.device_status() == 0
    want, err = A.attention64(q[:rows], k, v, rows, True, d ** -0.5, dt)
    close(out[:rows], want, err, dt)


# ------------------------------------------------------------------------------------------- the largest scores
@pytest.mark.parametrize("n,length", [(1, 700), (3, 500), (1, 40000), (90, 300), (130, 20000)])
@pytest.mark.parametrize("d,scale", [(64, 1.0), (128, 1.0), (64, 0.125), (64, 0.01), (128, 60.0)])
@pytest.mark.parametrize("scores", ["lowest", "lowest but one", "highest", "rising", "both"])
def test_scores_up_to_the_ends_of_fp32(n, length, d, scale, scores):
    """Scores of up to 1.75 * 2^127, whose products with log2 e are rounded to far more than one, or are none of fp32's numbers: the largest share the sum alone."""
    size, dt = 1.75 * 2.0 ** 63, E.bf16
    k0 = torch.full((length,), {"lowest": -size, "lowest but one": -size, "highest": size, "rising": 0.0, "both": -size}[scores], dtype=torch.float64, device="cuda")
    if scores == "lowest but one":
        k0[length // 3] = 0.0
    if scores == "rising":
        k0 = torch.linspace(-1.0, 1.0, length, dtype=torch.float64, device="cuda") * size
    if scores == "both":
        k0[::5] = size
    k0 = k0.to(A.TORCH[dt])
    k = torch.zeros(1, length, 2, d, dtype=A.TORCH[dt], device="cuda")
    k[0, :, :, 5] = k0[:, None]
    q = torch.zeros(n, 4, d, dtype=A.TORCH[dt], device="cuda")
    q[..., 5] = 2.0 ** 64
    v = randn(1, length, 2, d, dtype=A.TORCH[dt], seed=4)
    plan, out = E.Attention(4, 2, d, dtype=dt, causal=False, scale=scale), A.poisoned(n, 4, d, dt=dt)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, rows=n, seqs=1) == 0, E.last_error()
    assert plan.device_status() == 0
    top = k0 == k0.max()
    mean, size = (f(v[0].double()[top]).mean(0).repeat_interleave(2, 0).expand(n, -1, -1) for f in (lambda x: x, torch.abs))
    close(out, mean, (2.0 ** -17 + (4 * int(top.sum()) ** 0.5 + 8) * 2.0 ** -23) * 2 * size, dt)


@pytest.mark.parametrize("n", [1, 3, 90])
@pytest.mark.parametrize("power", [10, 20, 24, 27, 28, 31, 40, 60])
@pytest.mark.parametrize("dt", [E.bf16, E.f16])
def test_large_scores_that_are_near_one_another(n, power, dt):
    """Scores of 2^power and a few of their own last places below it, exact in 32 bits: the definition's weights, whatever the product with log2 e is rounded to."""
    if dt == E.f16 and power > 28:
        return
    length, d = 300, 64
    half = power // 2
    scale = 1.0 if power > 20 else 0.75
    k = torch.zeros(1, length, 1, d, dtype=A.TORCH[dt], device="cuda")
    q = torch.zeros(n, 2, d, dtype=A.TORCH[dt], device="cuda")
    steps = torch.arange(length, device="cuda") % 5                                      # 0, 1, 2, 3, 4 last places (of 2^(power - 22)) below the largest
    last = 2.0 ** max(power - 22, -3)
    q[..., 0], q[..., 1] = 2.0 ** half, -2.0 ** min(half, 10)
    k[..., 0] = 2.0 ** (power - half)
    k[0, :, 0, 1] = (steps * last / 2.0 ** min(half, 10)).to(k.dtype)
    v = randn(1, length, 1, d, dtype=A.TORCH[dt], seed=4)
    plan, out = E.Attention(2, 1, d, dtype=dt, causal=False, scale=scale), A.poisoned(n, 2, d, dt=dt)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, rows=n, seqs=1) == 0, E.last_error()
    assert plan.device_status() == 0
    s = (q[0, 0].double() @ k[0, :, 0].double().T) * scale
    w = torch.softmax(s, -1)
    want = (w @ v[0, :, 0].double()).expand(n, 2, -1)
    size = (w @ v[0, :, 0].double().abs()).expand(n, 2, -1)
    # the terms' rounding and the exponential's; above 2^27 the power of two above scale * log2 e stands in for it: a last place is then 8 or more of its powers of two, and a term
    # of 2^-8 / 2^-11.5 at most the other
    off = 2.0 ** -16 + {E.bf16: 2.0 ** -8, E.f16: 2.0 ** -11}[dt] + (2.0 ** -8 if power >= 27 else 0.0)
    close(out, want, off * 2 * size, dt)


# ------------------------------------------------------------------------------------------- far positions
def test_fast_frequencies_at_the_farthest_positions():
    """Angles of up to 10^13 radians against their definition in rational numbers: the bound of every other position."""
    from fractions import Fraction
    turns = Fraction(15915494309189533576888376337251436203445964574045644874766734405889, 10 ** 68)     # 1 / (2 pi)
    f = torch.tensor([1.0, 1000.0, -777.7, 333.3, 7.5, 5000.0, 0.1, 62.83], dtype=torch.float32)
    pos = A.ints([2 ** 31 - 1, 2 ** 31 - 2, -(2 ** 31), 2 ** 30 + 12345, 10 ** 9 + 7, 10 ** 6 + 3, -1999999999])
    x = randn(len(pos), 2, 16, dtype=torch.float32, seed=1)
    plan, out = E.Rotary(2, 0, 16, dtype=E.f32), torch.empty_like(x)
    assert plan.prepare(f) == 0, E.last_error()
    assert plan.enqueue(out, None, x, None, pos, rows=len(pos)) == 0, E.last_error()
    assert plan.device_status() == 0
    angle = torch.tensor([[float((Fraction(p) * Fraction(w) * turns) % 1) for w in f.tolist()] for p in pos.tolist()], dtype=torch.float64, device="cuda")[:, None] * 2.0 * torch.pi
    a, b = x.double().chunk(2, -1)
    want = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
    off = (a.abs() + b.abs()).repeat(1, 1, 2) * 2.0 ** -20                                                # (as turn64's)
    close(out, want, off, E.f32)


# ------------------------------------------------------------------------------------------- many sequences
def many(new, lengths, heads, kv_heads, d, causal=True, aligned=True):
    """Sequences of up to 16 tokens over one page each, against the definition for those that have new tokens."""
    seqs, rows, dt = len(new), int(new.sum()), E.bf16
    starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    starts[1:] = new.cumsum(0)
    some = new.nonzero()[:, 0]
    pages = len(some) + 1
    table = torch.full((seqs, 1), A.FAR_PAGE, dtype=torch.int32, device="cuda")
    table[some, 0] = torch.randperm(pages, device="cuda")[:len(some)].to(torch.int32)
    k, v = (randn(pages, kv_heads, 16, d, dtype=A.TORCH[dt], seed=i) for i in (1, 2))
    q = randn(rows, heads, d, dtype=A.TORCH[dt], seed=3)
    plan = E.Attention(heads, kv_heads, d, page_size=16, causal=causal, **({} if aligned else dict(ld_input=heads * d + 4)))
    if not aligned:
        wide = torch.empty(rows, heads * d + 4, dtype=q.dtype, device="cuda")
        wide[:, :heads * d] = q.flatten(1)
        q_in = wide[:, :heads * d]
    else:
        q_in = q
    out = A.poisoned(rows, heads, d, dt=dt)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q_in, k, v, table, lengths, starts, rows=rows, seqs=seqs) == 0, E.last_error()
    assert plan.device_status() == 0
    where = torch.repeat_interleave(torch.arange(seqs, device="cuda"), new)
    place = torch.arange(rows, device="cuda") - starts[where]
    group, at = heads // kv_heads, table[where, 0].long()
    s = torch.einsum("rhd,rhmd->rhm", q.double(), k[at].double().repeat_interleave(group, 1)) * d ** -0.5
    seen = lengths[where] - (new[where] - 1 - place if causal else 0)
    s = s.masked_fill(torch.arange(16, device="cuda") >= seen[:, None, None], -float("inf"))
    w = torch.softmax(s, -1).nan_to_num(0.0)
    want, size = (torch.einsum("rhm,rhmd->rhd", w, x.repeat_interleave(group, 1)) for x in (v[at].double(), v[at].double().abs()))
    close(out, want, (2.0 ** -8 + 2.0 ** -16) * 1.1 * size, dt)


@pytest.mark.parametrize("seqs", [33, 64, 1000, 5000])
@pytest.mark.parametrize("heads,kv_heads,d,aligned", [(4, 4, 64, True), (8, 1, 128, True), (3, 1, 64, True), (2, 2, 64, False)])
def test_many_ragged_sequences(seqs, heads, kv_heads, d, aligned):
    g = torch.Generator(device="cuda").manual_seed(seqs)
    new = torch.randint(0, 17, (seqs,), generator=g, device="cuda") * (torch.rand(seqs, generator=g, device="cuda") < 0.6)
    lengths = (new + torch.randint(0, 17, (seqs,), generator=g, device="cuda")).clamp(max=16).to(torch.int32)
    many(new, lengths, heads, kv_heads, d, True, aligned)
    many(new, lengths, heads, kv_heads, d, False, aligned)


@pytest.mark.parametrize("count", [7, 4000])
@pytest.mark.parametrize("aligned", [True, False])
def test_a_few_of_a_million_sequences(count, aligned):
    """A call's CTAs find their sequences by searching: looked at one after the other, 2^20 of them would cost each CTA some milliseconds, and a call of 2^20 CTAs half a
    minute."""
    seqs = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(count)
    new = torch.zeros(seqs, dtype=torch.int64, device="cuda")
    some = torch.randperm(seqs, generator=g, device="cuda")[:count]
    new[some] = torch.randint(1, 4, (count,), generator=g, device="cuda")
    lengths = torch.where(new > 0, new + 9, 0).to(torch.int32)
    many(new, lengths, 2, 1, 64, True, aligned)
    # and into the cache
    rows = int(new.sum())
    starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    starts[1:] = new.cumsum(0)
    table = torch.full((seqs, 1), A.FAR_PAGE, dtype=torch.int32, device="cuda")
    some = new.nonzero()[:, 0]
    table[some, 0] = torch.arange(count, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(count, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, nk, nv = (randn(rows, h, 64, dtype=torch.bfloat16, seed=i) for i, h in enumerate((2, 1, 1)))
    plan, q_out = E.CacheAppend(2, 1, 64, 16, rotary_dim=0), torch.empty_like(q)
    assert plan.prepare() == 0
    torch.cuda.synchronize()
    assert plan.enqueue(q_out, k, v, q, nk, nv, table, lengths, starts, rows=rows, seqs=seqs) == 0, E.last_error()
    assert plan.device_status() == 0
    where = torch.repeat_interleave(torch.arange(seqs, device="cuda"), new)
    at = lengths[where].long() - new[where] + torch.arange(rows, device="cuda") - starts[where]
    page = table[where, 0].long()
    assert torch.equal(q_out, q) and torch.equal(k[page, :, at], nk) and torch.equal(v[page, :, at], nv)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("empty", [0, -7])
def test_empty_slots_of_a_padded_batch(new, empty):
    """A step of answers, captured once, in which some places of the batch hold no sequence: nothing is written for them, attention gives them zeros, and nothing is wrong."""
    seqs, d = 6, 64
    rows, lengths = seqs * new, A.ints([empty if i in (1, 4) else 20 + i for i in range(seqs)])
    table = A.ints([[-1, -1] if i in (1, 4) else [2 * i, 2 * i + 1] for i in range(seqs)])
    k, v = (torch.zeros(2 * seqs, 2, 16, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, nk, nv = (randn(rows, h, d, dtype=torch.bfloat16, seed=h) for h in (4, 2, 3))
    nv = nv[:, :2].contiguous()
    q_out, out = torch.full_like(q, POISON), A.poisoned(rows, 4, d, dt=E.bf16)
    append, attention, s = E.CacheAppend(4, 2, d, 16, rotary_dim=0), E.Attention(4, 2, d, page_size=16), torch.cuda.Stream()
    assert append.prepare() == 0

    def step():
        assert append.enqueue(q_out, k, v, q, nk, nv, table, lengths, rows=rows, seqs=seqs, stream=s.cuda_stream) == 0, E.last_error()
        assert attention.enqueue(out, q_out, k, v, table, lengths, rows=rows, seqs=seqs, stream=s.cuda_stream) == 0, E.last_error()
    torch.cuda.synchronize()
    step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    graph.replay()
    torch.cuda.synchronize()
    assert append.device_status() == attention.device_status() == 0
    for i in range(seqs):
        r = slice(i * new, (i + 1) * new)
        if i in (1, 4):
            assert bool((q_out[r] == POISON).all()) and bool((out[r] == 0).all())
            continue
        at = torch.arange(20 + i - new, 20 + i, device="cuda")
        assert torch.equal(q_out[r], q[r]) and torch.equal(k[2 * i + at // 16, :, at % 16], nk[r]) and torch.equal(v[2 * i + at // 16, :, at % 16], nv[r])
    assert not bool(k[[2, 3, 8, 9]].any()) and not bool(v[[2, 3, 8, 9]].any())


@pytest.mark.parametrize("n", [1, 4, 60])
@pytest.mark.parametrize("aligned", [True, False])
def test_sequences_without_new_tokens_have_no_pages(n, aligned):
    """Their lengths may be anything and their entries of the table no pages: nobody reads them, and nothing is wrong."""
    d, lengths = 64, [70, 200, 90, 33]
    b = A.batch([0, n, 0, 0], [lengths[0], 200 + n, lengths[2], lengths[3]], 16, ragged=True)
    q, kv = A.inputs(b, 4, 2, d, E.bf16)
    (k, k_view, ld), (v, v_view, _) = A.cache(b, 2, d, E.bf16), A.cache(b, 2, d, E.bf16)
    A.put(b, k_view, 1, kv[1][0])
    A.put(b, v_view, 1, kv[1][1])
    want, err, _ = A.wanted(b, q, kv, True, d ** -0.5, E.bf16)
    for s in (0, 2, 3):
        b.table[s] = -1 if s else A.FAR_PAGE
    if not aligned:
        wide = torch.empty(n, 4 * d + 4, dtype=q.dtype, device="cuda")
        wide[:, :4 * d] = q.flatten(1)
        q = wide[:, :4 * d]
    plan = E.Attention(4, 2, d, page_size=16, ld_input=0 if aligned else 4 * d + 4, **ld)
    out = A.poisoned(n, 4, d, dt=E.bf16)
    torch.cuda.synchronize()
    assert plan.enqueue(out, q, k, v, b.table, b.lengths_t, b.starts_t, rows=n, seqs=4) == 0, E.last_error()
    assert plan.device_status() == 0
    close(out, want, err, E.bf16)
