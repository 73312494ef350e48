"""``Linear`` against its definition in 64 bits: sizes around the tiles, types, activations, strides, alignment, residuals, and
values that are not finite."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def U(pkg):
    import oputil
    return oputil


def _run(U, rows, ic, oc, dt=None, out=None, act="none", gated=False, bias=None, residual=False, scale=1.0, hwio=False, pad=(0, 0, 0),
         offset=(0, 0, 0), in_place=False, seed=1, x=None, w=None, plan=None):
    """One call with poison around the output and NaN between the input's rows; compares and returns (output, plan)."""
    E = U.E
    dt = E.bf16 if dt is None else dt
    out = dt if out is None else out
    wide = 2 * oc if gated else oc
    x = U.randn(rows, ic, dtype=U.TORCH[dt], seed=seed) if x is None else x
    w = U.randn(wide, ic, dtype=U.TORCH[dt], seed=seed + 1, scale=1.5 / math.sqrt(ic)) if w is None else w
    b = None if bias is None else U.randn(wide, dtype=U.TORCH[bias], seed=seed + 2)
    r = U.randn(rows, oc, dtype=U.TORCH[out], seed=seed + 3, scale=2.0) if residual else None
    xs, xbuf = U.strided(rows, ic, ic + pad[0], U.TORCH[dt], offset[0], source=x)
    gap = torch.ones_like(xbuf, dtype=torch.bool)
    torch.as_strided(gap, xs.shape, xs.stride(), xs.storage_offset()).fill_(False)
    xbuf[gap] = float("nan")
    ys, ybuf = U.strided(rows, oc, oc + pad[1], U.TORCH[out], offset[1], source=r if in_place else None)
    rs = None
    if residual and not in_place:
        rs, _ = U.strided(rows, oc, oc + pad[2], U.TORCH[out], offset[2], source=r)
    lin = plan or E.Linear(ic, oc, dtype=dt, out_dtype=out, activation=U.ACTS[act], gated=gated, with_bias=bias is not None,
                           bias_dtype=E.f32 if bias is None else bias, with_residual=residual, scale=scale,
                           weights_format=E.hwio if hwio else E.oihw, ld_input=ic + pad[0], ld_output=oc + pad[1],
                           ld_residual=oc + (pad[1] if in_place else pad[2]))
    assert lin.prepare(w.t().contiguous() if hwio else w, b) == 0, E.last_error()
    rc = lin.enqueue(ys, xs, ys if in_place else rs, rows=rows)
    assert rc == 0, E.last_error()
    assert lin.device_status() == 0
    U.untouched(ys, ybuf)
    want, err = U.linear64(x, w, b, r, act, gated, scale)
    U.close(ys, want, err, out, f"{rows}x{ic}->{oc}")
    return ys, lin


SIZES = [(1, 1, 1), (1, 64, 128), (1, 7, 3), (2, 65, 129), (3, 128, 127), (5, 4096, 256), (8, 1000, 1001), (15, 63, 2), (16, 64, 130),
         (17, 192, 255), (31, 72, 640), (32, 520, 64), (33, 1003, 257), (63, 64, 384), (64, 2048, 128), (65, 80, 511), (96, 4100, 72),
         (127, 264, 256), (128, 256, 512), (129, 257, 513), (200, 640, 2500), (255, 65, 256), (256, 1024, 1024), (257, 72, 1000),
         (300, 33, 16), (511, 2048, 320), (513, 130, 260), (1000, 520, 776), (1025, 64, 4096), (2300, 192, 2049), (4099, 96, 130)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_sizes(U, size, dt):
    _run(U, *size, dt=getattr(U.E, dt))


# every tile width, with and without shared channels, pairs of CTAs with full, ragged and several tiles, and CUDA cores
FORMS = [(5, 4096, 4096, False), (24, 4096, 8192, True), (33, 2048, 4096, False), (64, 4096, 2048, True), (128, 4096, 4096, False), (200, 3000, 2048, True),
         (256, 4096, 4096, False), (512, 2048, 4096, False), (1024, 4096, 2100, True), (1500, 640, 5120, False), (4000, 256, 1280, False), (3000, 1024, 511, True),
         (240, 2048, 18944, False), (20, 4096, 9000, False), (160, 1024, 10000, True), (96, 8192, 1024, False), (1000, 7168, 250, False), (2, 4096, 4096, True),
         (7, 1000, 600, True), (1, 16384, 300, False)]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "x".join(map(str, f)))
def test_every_form(U, form):
    rows, ic, oc, gated = form
    _run(U, rows, ic, oc, act="silu" if gated else "gelu_tanh", gated=gated, bias=U.E.f32, residual=True, scale=0.5)
    _run(U, rows, ic, oc, dt=U.E.f16, gated=gated, seed=5)


@pytest.mark.parametrize("size", [(1, 64, 1), (3, 200, 129), (16, 1003, 64), (40, 256, 192), (130, 320, 333), (300, 512, 1024), (1100, 1000, 515)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_epilogues(U, size, act, gated):
    E = U.E
    k = size[0] % 3
    _run(U, *size, dt=(E.bf16, E.f16, E.bf16)[k], act=act, gated=gated, bias=(E.f32, E.f16, E.bf16)[k], residual=True, scale=(1.0, 0.5, -1.25)[k])


@pytest.mark.parametrize("rows,ic,oc", [(1, 300, 200), (20, 300, 200), (150, 300, 200), (700, 520, 400)])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_fp32_output(U, rows, ic, oc, dt, gated):
    _run(U, rows, ic, oc, dt=getattr(U.E, dt), out=U.E.f32, act="silu" if gated else "none", gated=gated, bias=U.E.f32, residual=True)


@pytest.mark.parametrize("rows", [1, 21, 140, 530])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("pad,offset", [((8, 8, 8), (8, 8, 8)), ((1, 0, 0), (0, 0, 0)), ((0, 1, 0), (0, 0, 0)), ((0, 0, 1), (0, 0, 0)), ((0, 0, 0), (1, 0, 0)),
                                        ((0, 0, 0), (0, 1, 0)), ((0, 0, 0), (0, 0, 1)), ((4, 2, 6), (4, 2, 6)), ((3, 5, 7), (1, 3, 5))], ids=str)
def test_strides_and_alignment(U, rows, gated, pad, offset):
    _run(U, rows, 136, 264, act="silu", gated=gated, residual=True, pad=pad, offset=offset)


@pytest.mark.parametrize("rows", [1, 40, 400])
def test_hwio_weights_and_residual_in_place(U, rows):
    _run(U, rows, 100, 150, hwio=True, gated=True, act="gelu", bias=U.E.f32)
    _run(U, rows, 100, 150, hwio=True, residual=True, in_place=True, pad=(0, 3, 3))


def test_one_plan_many_row_counts_and_no_rows(U):
    E = U.E
    _, lin = _run(U, 7, 200, 300)
    for rows in (1, 600, 33, 2, 129):
        _run(U, rows, 200, 300, plan=lin)
    assert lin.launch_count() > 0
    n = lin.launch_count()
    assert lin.enqueue(torch.empty(1, device="cuda"), torch.empty(1, device="cuda"), rows=0) == E.ELB_OK
    assert lin.launch_count() == n
    # the weights were read once
    assert lin.prepare(torch.zeros(300, 200, dtype=torch.bfloat16, device="cuda")) == 0
    _run(U, 9, 200, 300, plan=lin)


@pytest.mark.parametrize("rows", [5, 90, 600])
def test_values_that_are_not_finite_stay_in_their_rows(U, rows):
    """NaN and infinities in a row of the input reach that row of the output and no other; infinite weights their channel."""
    E = U.E
    ic, oc = 130, 200
    x = U.randn(rows, ic, dtype=torch.bfloat16, seed=5)
    w = U.randn(oc, ic, dtype=torch.bfloat16, seed=6, scale=0.1)
    clean = torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda")
    lin = E.Linear(ic, oc)
    assert lin.prepare(w) == 0 and lin.enqueue(clean, x, rows=rows) == 0
    x[1, 3], x[3, 129], x[rows - 1, 0] = float("nan"), float("inf"), float("-inf")
    y = torch.empty_like(clean)
    assert lin.enqueue(y, x, rows=rows) == 0
    torch.cuda.synchronize()
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[[1, 3, rows - 1]] = True
    assert torch.equal(y[~hit], clean[~hit])
    assert bool(y[1].isnan().all()) and not bool(y[3].isfinite().any()) and not bool(y[rows - 1].isfinite().any())
    assert torch.equal(y[3] > 0, w[:, 129] > 0)


def test_results_do_not_depend_on_the_run(U):
    """The same call gives the same bits (no sum's order depends on timing)."""
    E = U.E
    for rows, ic, oc in ((1, 8192, 512), (24, 4096, 640), (300, 2048, 1000), (2000, 512, 2048)):
        x, w = U.randn(rows, ic, dtype=torch.bfloat16, seed=1), U.randn(oc, ic, dtype=torch.bfloat16, seed=2, scale=0.02)
        lin = E.Linear(ic, oc, out_dtype=E.f32)
        assert lin.prepare(w) == 0
        ys = [torch.empty(rows, oc, device="cuda") for _ in range(4)]
        for y in ys:
            assert lin.enqueue(y, x, rows=rows) == 0
        torch.cuda.synchronize()
        assert all(torch.equal(ys[0], y) for y in ys[1:])


def test_offsets_past_32_bits(U):
    """Rows so far apart that the last ones lie behind 2^32 bytes and 2^31 elements."""
    E = U.E
    rows, ic, oc, ld = 70001, 64, 96, 32000
    x, w = U.randn(rows, ic, dtype=torch.bfloat16, seed=1), U.randn(oc, ic, dtype=torch.bfloat16, seed=2, scale=0.2)
    big = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda")
    y = torch.as_strided(big, (rows, oc), (ld, 1))
    lin = E.Linear(ic, oc, ld_output=ld)
    assert lin.prepare(w) == 0 and lin.enqueue(y, x, rows=rows) == 0, E.last_error()
    want, err = U.linear64(x, w, None, None, "none", False, 1.0)
    U.close(y.clone(), want, err, E.bf16)
    xb = torch.as_strided(big, (rows, ic), (ld, 1), 1024)
    xb.copy_(x)
    y2 = torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda")
    lin2 = E.Linear(ic, oc, ld_input=ld)
    assert lin2.prepare(w) == 0 and lin2.enqueue(y2, xb, rows=rows) == 0, E.last_error()
    torch.cuda.synchronize()
    assert torch.equal(y2, y)


def test_streams_and_graphs(U):
    """Calls on other streams than the tensors' own, ordered by events, and a captured call replayed on new inputs."""
    E = U.E
    for rows, ic in ((3, 512), (40, 333), (600, 333), (600, 512)):
        oc = 320
        w = U.randn(oc, ic, dtype=torch.bfloat16, seed=2, scale=0.05)
        lin = E.Linear(ic, oc)
        assert lin.prepare(w) == 0
        y = torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda")
        inputs = [U.randn(rows, ic, dtype=torch.bfloat16, seed=10 + k) for k in range(4)]
        torch.cuda.synchronize()
        streams, outs = [torch.cuda.Stream() for _ in range(4)], [torch.empty_like(y) for _ in range(4)]
        for k in range(12):           # calls of one plan on four streams at once
            assert lin.enqueue(outs[k % 4], inputs[k % 4], rows=rows, stream=streams[k % 4].cuda_stream) == 0, E.last_error()
        torch.cuda.synchronize()
        for o, x in zip(outs, inputs):
            U.close(o, *U.linear64(x, w, None, None, "none", False, 1.0), E.bf16)
        x = inputs[0].clone()
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=s):
            assert lin.enqueue(y, x, rows=rows, stream=s.cuda_stream) == 0, E.last_error()
        for k in (1, 2):
            x.copy_(inputs[k])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, outs[k])
        assert lin.device_status() == 0


def test_a_captured_call_outlives_a_larger_workspace(U):
    """Inputs that are not aligned go through the plan's workspace; a graph captured with a small one is right after larger calls."""
    E = U.E
    ic, oc = 333, 320
    w = U.randn(oc, ic, dtype=torch.bfloat16, seed=2, scale=0.05)
    lin = E.Linear(ic, oc)
    assert lin.prepare(w) == 0
    x, y = U.randn(300, ic, dtype=torch.bfloat16, seed=1), torch.empty(300, oc, dtype=torch.bfloat16, device="cuda")
    assert lin.enqueue(y, x, rows=300) == 0
    want = y.clone()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        assert lin.enqueue(y, x, rows=300, stream=s.cuda_stream) == 0, E.last_error()
    for rows in (900, 5000, 20000):
        big, out = U.randn(rows, ic, dtype=torch.bfloat16, seed=rows), torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda")
        assert lin.enqueue(out, big, rows=rows) == 0
        torch.cuda.synchronize()
        filler = torch.full((rows, ic), float("nan"), dtype=torch.bfloat16, device="cuda")     # takes memory that was given back
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        U.close(out, *U.linear64(big, w, None, None, "none", False, 1.0), E.bf16)
        del filler


def test_host_weights(U):
    E = U.E
    x, w = U.randn(10, 70, dtype=torch.float16, seed=1), U.randn(90, 70, dtype=torch.float16, seed=2)
    lin = E.Linear(70, 90, dtype=E.f16, with_bias=True)
    b = torch.randn(90)
    assert lin.prepare(w.cpu(), b) == 0, E.last_error()
    y = torch.empty(10, 90, dtype=torch.float16, device="cuda")
    assert lin.enqueue(y, x, rows=10) == 0
    U.close(y, *U.linear64(x, w, b.cuda(), None, "none", False, 1.0), E.f16)


def test_refusals_of_calls(U):
    E = U.E
    lin = E.Linear(64, 64, with_residual=True, with_bias=True)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    assert lin.enqueue(x, x, x, rows=4) == E.ELB_GENERAL_ERROR and "not prepared" in E.last_error()
    w, b = torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, device="cuda")
    assert lin.prepare(w) == E.ELB_GENERAL_ERROR and lin.prepare(None) == E.ELB_GENERAL_ERROR
    for bad in (x, w.float(), w.t(), w[:, :32], w.cpu().float().numpy()):
        with pytest.raises(ValueError):
            lin.prepare(bad, b)
    with pytest.raises(ValueError):
        lin.prepare(w, b.half())
    assert lin.prepare(w, b) == 0
    assert lin.enqueue(x, x, None, rows=4) == E.ELB_GENERAL_ERROR
    assert lin.enqueue(None, x, x, rows=4) == E.ELB_GENERAL_ERROR
    assert lin.enqueue(x, x, x, rows=-1) == E.ELB_GENERAL_ERROR
    assert lin.enqueue(x.data_ptr() + 1, x, x, rows=1) == E.ELB_GENERAL_ERROR
    with pytest.raises(ValueError):
        lin.enqueue(x, x.cpu(), x, rows=4)
    assert lin.launch_count() == 0
    # a plan of another operator
    norm = E.BlockNorm(64)
    assert E.lib.elb_linear_enqueue(norm.h, x.data_ptr(), x.data_ptr(), None, 4, None) == E.ELB_GENERAL_ERROR


@pytest.mark.parametrize("rows,ic", [(1, 64), (3, 64), (24, 4096), (90, 512), (700, 512)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_activations_far_from_zero(U, rows, ic, act, gated):
    """Sums of any size, the type's lowest value among them, on every route: one product with 1, the others with 0.

    The logistic factor 1 / (1 + 2^t): t carries a relative 2^-22 (a constant, three products and sums), so the exponential 126 * 2^-22 * ln 2
    at most before it is flushed to zero, which 2^-15 covers with the other roundings.  Behind t = 126 the factor is 0 for a value of 90 at
    most (silu; the tanh form: 7), an error under 90 * 2^-126 < 2^-119."""
    E = U.E
    v = torch.tensor([-3.3895313892515355e38, -1e30, -1e20, -1e10, -40000.0, -300.0, -126.0, -90.0, -86.5, -64.0, -50.0, -44.0, -20.0, -11.0, -6.0, -4.5, -3.0,
                      -1.0, -0.01, 0.0, 0.5, 3.0, 20.0, 70.0, 1e4, 1e20, 3e38, float("inf"), float("-inf"), float("nan")], device="cuda").to(torch.bfloat16)
    if gated:
        v = v[:-3]                                 # (the up row's product with 0 makes NaN of those)
    rows = max(rows, 1)
    oc = 150
    x = torch.zeros(rows, ic, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2 * oc if gated else oc, ic, dtype=torch.bfloat16, device="cuda")
    w[:oc, 5], w[oc:, 9] = 1.0, 1.0
    x[:, 9] = 1.0
    for out in (E.f32, E.bf16):
        lin = E.Linear(ic, oc, out_dtype=out, activation=U.ACTS[act], gated=gated)
        assert lin.prepare(w) == 0
        for k in range(0, len(v), rows):           # every value in some row
            x[:, 5] = v[(torch.arange(rows, device="cuda") + k) % len(v)]
            y = torch.empty(rows, oc, dtype=U.TORCH[out], device="cuda")
            assert lin.enqueue(y, x, rows=rows) == 0
            torch.cuda.synchronize()
            z = x[:, 5:6].double()
            t = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
            want = (z * torch.sigmoid(t)).expand(rows, oc)
            odd = want.isnan()
            assert bool(y[odd].isnan().all()), "an infinite sum times a factor of zero, and NaN, are NaN as in the formula"
            U.close(y[~odd], want[~odd], 2.0 ** -15 * want[~odd].abs() + 2.0 ** -119, out)


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_channels_that_are_not_finite_stay_alone(U, rows, act, gated):
    """A NaN or an infinity in some channels of a token changes no bit of the others (two of them share a reciprocal)."""
    E = U.E
    ic, oc = 64, 96
    x = U.randn(rows, ic, dtype=torch.bfloat16, seed=1)
    w = U.randn(2 * oc if gated else oc, ic, dtype=torch.bfloat16, seed=2, scale=0.3)
    odd = torch.zeros(oc, dtype=torch.bool, device="cuda")
    odd[[0, 9, 18, 27, 37, 63, 95]] = True
    ys = []
    for value in (None, float("nan"), float("inf"), 3e38):
        wv = w.clone()
        if value is not None:
            wv[:oc][odd] = value
        lin, y = E.Linear(ic, oc, activation=U.ACTS[act], gated=gated), torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda")
        assert lin.prepare(wv) == 0 and lin.enqueue(y, x, rows=rows) == 0
        torch.cuda.synchronize()
        ys.append(y)
        assert torch.equal(y[:, ~odd], ys[0][:, ~odd])
    assert bool(ys[1][:, odd].isnan().all())


def test_per_thread_streams_take_turns_in_the_workspace(U):
    """cudaStreamPerThread is one handle for a stream of each thread: a call in one thread comes behind the other thread's call of the plan."""
    import threading
    E = U.E
    rows, ic, oc, per_thread = 500, 333, 200, 2
    w = U.randn(oc, ic, dtype=torch.bfloat16, seed=2, scale=0.05)
    xs = [U.randn(rows, ic, dtype=torch.bfloat16, seed=k) for k in range(2)]
    ys = [torch.empty(rows, oc, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    lin = E.Linear(ic, oc)
    assert lin.prepare(w) == 0
    first_done, results = torch.cuda.Event(), []
    for x, y in zip(xs, ys):
        assert lin.enqueue(y, x, rows=rows) == 0
        y.zero_()
    torch.cuda.synchronize()

    def call(k):
        stream = torch.cuda.ExternalStream(per_thread)
        with torch.cuda.stream(stream):
            if k == 0:
                torch.cuda._sleep(200_000_000)             # 0.1 s in front of the first thread's call
            results.append(lin.enqueue(ys[k], xs[k], rows=rows, stream=per_thread))
            if k == 0:
                first_done.record(stream)
            else:
                stream.synchronize()
                results.append(first_done.query())

    for k in range(2):
        t = threading.Thread(target=call, args=(k,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert results == [0, 0, True]
    for x, y in zip(xs, ys):
        U.close(y, *U.linear64(x, w, None, None, "none", False, 1.0), E.bf16)


@pytest.mark.parametrize("rows", [1, 20, 300, 700])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_gelu_keeps_its_relative_precision(U, rows, gated):
    """fp32 results of gelu's erf form, of both signs until they vanish: each sum is one product with 1.

    Relative error: the fit of erfc, its evaluation, a reciprocal (2^-23), an exponential (2^-22) and three products, 2^-19 together; the exponential's
    argument z^2 / 2 is 2.5 * 2^-24 off, relatively, which 2^-23 z^2 covers.  Flushed to zero below 2^-126, with |z| under 14."""
    E = U.E
    ic, oc = 64, 1801
    z = torch.linspace(-14.0, 14.0, oc, device="cuda").to(torch.bfloat16)
    x = torch.zeros(rows, ic, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2 * oc if gated else oc, ic, dtype=torch.bfloat16, device="cuda")
    x[:, 5] = x[:, 9] = 1.0
    w[:oc, 5], w[oc:, 9] = z, 1.0
    lin, y = E.Linear(ic, oc, out_dtype=E.f32, activation=E.ACT_GELU, gated=gated), torch.empty(rows, oc, device="cuda")
    assert lin.prepare(w) == 0 and lin.enqueue(y, x, rows=rows) == 0
    torch.cuda.synchronize()
    zd = z.double()
    want = (zd * 0.5 * torch.erfc(-zd / math.sqrt(2.0))).expand(rows, oc)
    U.close(y, want, want.abs() * (2.0 ** -19 + 2.0 ** -23 * zd * zd) + 14 * 2.0 ** -126, E.f32)
