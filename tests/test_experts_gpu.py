"""``Experts`` against its definition in 64 bits, and the four operators together as a user runs them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def U(pkg):
    import oputil
    return oputil


def _want(U, x, ids, share, w_in, w_out, act, gated, dt):
    """Expert by expert; the middle tensor's one rounding is a relative UNIT of each of its values."""
    rows, ic = x.shape
    y = torch.zeros(rows, w_out.shape[1], dtype=torch.float64, device="cuda")
    err = torch.zeros_like(y)
    for e in range(w_in.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        z, dz = U.product64(x[t], w_in[e])
        h, dh = U.activated64(z, dz, act, gated)
        dh = dh + U.UNIT[dt] * (h.abs() + dh) + U.TINY[dt]
        w = w_out[e].double()
        o = h @ w.t()
        do = dh @ w.abs().t() + (4.0 * math.sqrt(w.shape[1]) + 8.0) * 2.0 ** -23 * (h.abs() @ w.abs().t())
        s = share[t, j].double()[:, None]
        y.index_add_(0, t, o * s)
        err.index_add_(0, t, (do + 2.0 ** -21 * o.abs()) * s.abs())
    return y, err


def _run(U, rows, experts, k, ic, mid, dt="bf16", act="silu", gated=True, ids=None, pad=(0, 0), shift=(0, 0), max_rows=None, seed=1, plan=None, x=None):
    E = U.E
    ed = getattr(E, dt)
    td = U.TORCH[ed]
    wide = 2 * mid if gated else mid
    x = U.randn(rows, ic, dtype=td, seed=seed + 5) if x is None else x
    w_in = U.randn(experts, wide, ic, dtype=td, seed=seed, scale=1.5 / math.sqrt(ic))
    w_out = U.randn(experts, ic, mid, dtype=td, seed=seed + 1, scale=1.5 / math.sqrt(mid))
    if ids is None:
        ids = U.randn(rows, experts, dtype=torch.float32, seed=seed + 2).topk(k, dim=1).indices.to(torch.int32)
    share = torch.softmax(U.randn(rows, k, dtype=torch.float32, seed=seed + 3), dim=1)
    xs, _ = U.strided(rows, ic, ic + pad[0], td, shift[0], source=x)
    ys, yb = U.strided(rows, ic, ic + pad[1], td, shift[1])
    op = plan or E.Experts(experts, k, ic, mid, max_rows=max_rows or rows, dtype=ed, activation=U.ACTS[act], gated=gated, ld_input=ic + pad[0],
                           ld_output=ic + pad[1])
    assert op.prepare(w_in, w_out) == 0, E.last_error()
    assert op.enqueue(ys, xs, ids, share, rows=rows) == 0, E.last_error()
    assert op.device_status() == 0
    U.untouched(ys, yb)
    U.close(ys, *_want(U, x, ids, share, w_in, w_out, act, gated, ed), ed, f"{rows} rows")
    return op, ys


@pytest.mark.parametrize("case", [(1, 1, 1, 1, 1), (1, 8, 2, 64, 128), (1, 64, 8, 256, 192), (2, 4, 3, 65, 33), (5, 16, 4, 200, 300), (33, 7, 2, 129, 65), (64, 4, 1, 136, 72),
                                  (100, 100, 6, 128, 40), (257, 8, 2, 320, 256), (300, 3, 3, 72, 1000), (1000, 16, 4, 256, 130), (2100, 4, 2, 192, 257),
                                  (40, 1024, 32, 16, 8)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_sizes(U, case, gated, dt):
    _run(U, *case, dt=dt, gated=gated, act="silu" if gated else "gelu")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_activations(U, act):
    _run(U, 30, 4, 2, 100, 60, act=act)
    _run(U, 30, 4, 2, 100, 60, act=act, gated=False, dt="f16")


@pytest.mark.parametrize("rows", [3, 70, 400])
def test_loads(U, rows):
    """All tokens to one expert, experts without any, slots without an expert, the same expert twice, rows without any."""
    k, experts = 4, 9
    ids = torch.full((rows, k), 5, dtype=torch.int32, device="cuda")
    _run(U, rows, experts, k, 96, 80, ids=ids)
    ids = torch.randint(-2, experts + 2, (rows, k), generator=torch.Generator().manual_seed(rows)).to(torch.int32).cuda()
    ids[0] = -1
    ids[1] = torch.tensor([2147483647, -2147483648, 9, 8], dtype=torch.int32, device="cuda")
    _, y = _run(U, rows, experts, k, 96, 80, ids=ids)
    assert bool((y[0] == 0).all())
    _, y = _run(U, rows, experts, k, 96, 80, ids=torch.full((rows, k), -1, dtype=torch.int32, device="cuda"))
    assert bool((y == 0).all())


@pytest.mark.parametrize("pad,shift", [((8, 8), (8, 8)), ((1, 0), (0, 0)), ((0, 1), (0, 0)), ((0, 0), (1, 1)), ((3, 5), (2, 6))], ids=str)
@pytest.mark.parametrize("ic", [96, 101])
def test_strides_and_alignment(U, ic, pad, shift):
    _run(U, 50, 6, 3, ic, 72, pad=pad, shift=shift)


def test_one_plan_many_row_counts(U):
    E = U.E
    op, _ = _run(U, 300, 8, 2, 128, 96, max_rows=300)
    for rows in (1, 17, 299, 64, 2):
        _run(U, rows, 8, 2, 128, 96, plan=op)
    y = torch.empty(301, 128, dtype=torch.bfloat16, device="cuda")
    n = op.launch_count()
    ids, share = torch.zeros(301, 2, dtype=torch.int32, device="cuda"), torch.zeros(301, 2, device="cuda")
    assert op.enqueue(y, y, ids, share, rows=301) == E.ELB_GENERAL_ERROR and "300" in E.last_error()
    assert op.enqueue(y, y, ids, share, rows=0) == E.ELB_OK
    assert op.enqueue(y, y, ids, None, rows=3) == E.ELB_GENERAL_ERROR
    assert op.launch_count() == n


def test_values_that_are_not_finite_stay_in_their_rows(U):
    E = U.E
    rows, ic, mid = 60, 70, 50
    x = U.randn(rows, ic, dtype=torch.bfloat16, seed=3)
    w_in, w_out = U.randn(4, 2 * mid, ic, dtype=torch.bfloat16, seed=4), U.randn(4, ic, mid, dtype=torch.bfloat16, seed=5)
    ids = torch.randint(0, 4, (rows, 2), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    share = torch.rand(rows, 2, device="cuda")
    op = E.Experts(4, 2, ic, mid, max_rows=rows)
    clean, y = torch.empty_like(x), torch.empty_like(x)
    assert op.prepare(w_in, w_out) == 0 and op.enqueue(clean, x, ids, share, rows=rows) == 0
    x[7, 69], x[20, 0] = float("nan"), float("inf")
    assert op.enqueue(y, x, ids, share, rows=rows) == 0
    torch.cuda.synchronize()
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[[7, 20]] = True
    assert torch.equal(y[~hit], clean[~hit]) and bool(y[7].isnan().all()) and not bool(y[20].isfinite().all())


def test_streams_graphs_and_repeats(U):
    E = U.E
    rows, experts, k, ic, mid = 90, 8, 2, 136, 104
    w_in, w_out = U.randn(experts, 2 * mid, ic, dtype=torch.bfloat16, seed=1, scale=0.1), U.randn(experts, ic, mid, dtype=torch.bfloat16, seed=2, scale=0.1)
    op = E.Experts(experts, k, ic, mid, max_rows=rows)
    assert op.prepare(w_in, w_out) == 0
    data = []
    for s in range(4):
        ids = U.randn(rows, experts, dtype=torch.float32, seed=20 + s).topk(k, dim=1).indices.to(torch.int32)
        data.append((U.randn(rows, ic, dtype=torch.bfloat16, seed=10 + s), ids, torch.softmax(U.randn(rows, k, dtype=torch.float32, seed=30 + s), 1)))
    outs = [torch.empty(rows, ic, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for i in range(16):                     # one workspace, calls on four streams at once
        x, ids, share = data[i % 4]
        assert op.enqueue(outs[i % 4], x, ids, share, rows=rows, stream=streams[i % 4].cuda_stream) == 0, E.last_error()
    torch.cuda.synchronize()
    for o, (x, ids, share) in zip(outs, data):
        U.close(o, *_want(U, x, ids, share, w_in, w_out, "silu", True, E.bf16), E.bf16)
        again = torch.empty_like(o)
        assert op.enqueue(again, x, ids, share, rows=rows) == 0
        torch.cuda.synchronize()
        assert torch.equal(o, again)        # whatever place a slot was given
    x, ids, share = (t.clone() for t in data[0])
    y, g, s = torch.empty_like(outs[0]), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        assert op.enqueue(y, x, ids, share, rows=rows, stream=s.cuda_stream) == 0, E.last_error()
    for n in (2, 3):
        for t, v in zip((x, ids, share), data[n]):
            t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, outs[n])


@pytest.mark.parametrize("rows,channels,dtype", [(1, 256, "bf16"), (3, 512, "f16"), (40, 264, "bf16"), (300, 1024, "bf16"), (700, 520, "f16")])
def test_the_four_together(U, rows, channels, dtype):
    """The example's two feed-forward halves against the same chain in 64 bits.  Each of its seven 16-bit tensors rounds once (a relative
    half unit in the last place at most, in the norm of a vector a third root of that at most), what a rounding becomes on its way
    through a product is about as large as it was, and through the gate at most twice: 16 roundings are allowed."""
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("feed_forward", Path(__file__).resolve().parent.parent / "examples" / "feed_forward.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    E = U.E
    dt = getattr(E, dtype)
    ff = mod.FeedForward(channels, 4 * channels, 32, 4, channels // 2, rows, dt)
    x = U.randn(rows, channels, dtype=U.TORCH[dt], seed=1)
    s0 = U.randn(rows, channels, dtype=torch.float32, seed=2, scale=2.0)
    s = s0.clone()
    torch.cuda.synchronize()
    out = ff(x, s).clone()
    torch.cuda.synchronize()
    assert all(p.device_status() == 0 for p in ff.plans())
    want, want_s = ff.in_64_bits(x, s0, ff.ids[:rows])
    for got, w in ((out, want), (s, want_s)):
        assert float((got.double() - w).norm() / w.norm()) <= 16 * U.UNIT[dt]
    # captured, the pass gives the same bits
    s2, y2 = s0.clone(), torch.empty_like(out)
    g, q = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=q):
        ff(x, s2, stream=q.cuda_stream)
    s2.copy_(s0)
    g.replay()
    torch.cuda.synchronize()
    y2.copy_(ff.out[:rows])
    assert torch.equal(y2, out) and torch.equal(s2, s)


@pytest.mark.parametrize("rows", [513, 700, 3000])
def test_loads_of_counted_calls(U, rows):
    """More than 2048 slots, which a kernel of its own counts, over several of its blocks: all tokens to one expert, ids outside the experts,
    experts that nobody wants, rows without any."""
    k, experts = 4, 9
    ids = torch.full((rows, k), 5, dtype=torch.int32, device="cuda")
    _run(U, rows, experts, k, 96, 80, ids=ids)
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-2, experts + 2, (rows, k), generator=g).to(torch.int32)
    ids[(ids == 3) | (ids == 0)] = 8
    ids[0] = -1
    ids[1] = torch.tensor([2147483647, -2147483648, 9, 8], dtype=torch.int32)
    ids[rows // 2:rows // 2 + 40] = -1
    _, y = _run(U, rows, experts, k, 96, 80, ids=ids.cuda())
    assert bool((y[0] == 0).all()) and bool((y[rows // 2:rows // 2 + 40] == 0).all())
    _, y = _run(U, rows, experts, k, 96, 80, ids=torch.full((rows, k), -1, dtype=torch.int32, device="cuda"))
    assert bool((y == 0).all())
    ids = torch.full((rows, k), -1, dtype=torch.int32, device="cuda")
    ids[rows - 1, k - 1] = 1                       # one slot, the last
    _, y = _run(U, rows, experts, k, 96, 80, ids=ids)
    assert bool((y[:rows - 1] == 0).all())


def test_one_plan_counted_and_not(U):
    """Calls of one plan on both sides of 2048 slots, in any order."""
    op, _ = _run(U, 1500, 8, 2, 128, 96, max_rows=1500)
    for n, rows in enumerate((1024, 1025, 3, 1400, 1500, 64, 1025, 1, 1024, 1499)):
        g = torch.Generator().manual_seed(n)
        _run(U, rows, 8, 2, 128, 96, plan=op, ids=torch.randint(-1, 9, (rows, 2), generator=g).to(torch.int32).cuda())


def test_counted_calls_on_streams_and_in_graphs(U):
    """One workspace and one set of counts: calls on four streams at once, long and short in turn, and a captured one between them."""
    E = U.E
    experts, k, ic, mid, sizes = 8, 3, 136, 104, (900, 50, 1200, 700)
    w_in, w_out = U.randn(experts, 2 * mid, ic, dtype=torch.bfloat16, seed=1, scale=0.1), U.randn(experts, ic, mid, dtype=torch.bfloat16, seed=2, scale=0.1)
    op = E.Experts(experts, k, ic, mid, max_rows=max(sizes))
    assert op.prepare(w_in, w_out) == 0
    data, outs = [], []
    for s, rows in enumerate(sizes):
        ids = U.randn(rows, experts, dtype=torch.float32, seed=20 + s).topk(k, dim=1).indices.to(torch.int32)
        ids[::7, 1] = -1
        data.append((U.randn(rows, ic, dtype=torch.bfloat16, seed=10 + s), ids, torch.softmax(U.randn(rows, k, dtype=torch.float32, seed=30 + s), 1)))
        outs.append(torch.empty(rows, ic, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    for i in range(20):
        x, ids, share = data[i % 4]
        assert op.enqueue(outs[i % 4], x, ids, share, rows=sizes[i % 4], stream=streams[i % 4].cuda_stream) == 0, E.last_error()
    torch.cuda.synchronize()
    for o, (x, ids, share) in zip(outs, data):
        U.close(o, *_want(U, x, ids, share, w_in, w_out, "silu", True, E.bf16), E.bf16)
    y, g, s = torch.empty_like(outs[2]), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    x, ids, share = (t.clone() for t in data[2])
    with torch.cuda.graph(g, stream=s):
        assert op.enqueue(y, x, ids, share, rows=sizes[2], stream=s.cuda_stream) == 0, E.last_error()
    for n in range(3):
        again = torch.empty_like(outs[n])
        assert op.enqueue(again, *data[n], rows=sizes[n]) == 0
        torch.cuda.synchronize()
        assert torch.equal(again, outs[n])
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, outs[2])
    assert op.device_status() == 0
