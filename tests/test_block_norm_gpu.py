"""``BlockNorm`` against its definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def U(pkg):
    import oputil
    return oputil


def _normed64(v, dv, kind, w, b, eps):
    """(norm of v, what it may be off in 32 bits): mean and variance are sums of n values, each a few roundings of 2^-24 off
    (a tree of additions: at most log2 n + a few of them in a row, 40 taken); dv is the error of v that comes in."""
    n = v.shape[1]
    if kind == "none":
        return v, dv
    u = 40 * 2.0 ** -24
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    dmean = (u * v.abs().mean(1, keepdim=True) + dv.mean(1, keepdim=True)) if kind == "layer" else 0.0
    c = v - mean
    dc = dv + dmean + 2.0 ** -23 * c.abs()
    var = (c * c).mean(1, keepdim=True)
    dvar = u * var + 2 * (c.abs() * dc).mean(1, keepdim=True) + (dc * dc).mean(1, keepdim=True)
    by = 1.0 / torch.sqrt(var + eps)
    dby = by * (dvar / (var + eps) + 4 * 2.0 ** -24)
    y = c * by * w
    dy = (dc * by + c.abs() * dby + dc * dby) * w.abs() + 2.0 ** -22 * y.abs()
    if b is not None:
        y = y + b
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy


def _run(U, rows, n, dt="bf16", res="same", wt="f32", post="none", pre="rms", gate_rows=0, scale=1.0, offset=0.0, with_residual=True, pad=0,
         shift=0, want_sum=True, in_place=False, seed=1, mean=0.5, eps=1e-5):
    E = U.E
    kinds = {"none": E.NORM_NONE, "rms": E.NORM_RMS, "layer": E.NORM_LAYER}
    ed, er = getattr(E, dt), getattr(E, dt if res == "same" else res)
    ew = getattr(E, wt)
    td, tr, tw = U.TORCH[ed], U.TORCH[er], U.TORCH[ew]
    x, xb = U.strided(rows, n, n + pad, td, shift, source=U.randn(rows, n, dtype=torch.float32, seed=seed, scale=1.5) + mean)
    r = rb = g = None
    if with_residual:
        r, rb = U.strided(rows, n, n + pad, tr, shift, source=U.randn(rows, n, dtype=torch.float32, seed=seed + 1, scale=3.0))
    if gate_rows:
        g, _ = U.strided(-(-rows // gate_rows), n, n + pad, td, shift, source=U.randn(-(-rows // gate_rows), n, dtype=torch.float32, seed=seed + 2))
    ws = [None if k == "none" else (U.randn(n, dtype=torch.float32, seed=seed + 3 + i, scale=0.3) + 1.0 - offset).to(tw) for i, k in enumerate((post, pre))]
    bs = [U.randn(n, dtype=tw, seed=seed + 5 + i, scale=0.3) if k == "layer" else None for i, k in enumerate((post, pre))]
    r64 = r.double().clone() if r is not None else 0.0
    if in_place:
        s, sb = r, rb
    else:
        s, sb = U.strided(rows, n, n + pad, tr, shift) if want_sum else (None, None)
    y, yb = U.strided(rows, n, n + pad, td, shift)
    op = E.BlockNorm(n, dtype=ed, residual_dtype=er, weights_dtype=ew, post=kinds[post], pre=kinds[pre], post_eps=eps, pre_eps=eps, weight_offset=offset,
                     scale=scale, with_residual=with_residual, gate_rows=gate_rows,
                     **{f"ld_{k}": n + pad for k in ("input", "residual", "gate", "sum", "output")})
    assert op.prepare(ws[0], bs[0], ws[1], bs[1]) == 0, E.last_error()
    assert op.enqueue(y if pre != "none" else None, s, x, r, g, rows=rows) == 0, E.last_error()
    torch.cuda.synchronize()
    w64 = [None if w is None else w.double() + offset for w in ws]
    b64 = [None if b is None else b.double() for b in bs]
    v, dv = _normed64(x.double(), torch.zeros(rows, n, dtype=torch.float64, device="cuda"), post, w64[0], b64[0], eps)
    if g is not None:
        gg = g.double().repeat_interleave(gate_rows, 0)[:rows]
        v, dv = v * gg, dv * gg.abs()
    v, dv = v * scale, dv * abs(scale) + 2.0 ** -22 * (v * scale).abs()
    want, err = r64 + v, dv + 2.0 ** -23 * (r64 + v).abs()
    if s is not None:
        U.close(s, want, err, er, "sum")
        U.untouched(s, sb, "sum")
    if pre != "none":
        wy, ey = _normed64(want, err, pre, w64[1], b64[1], eps)
        U.close(y, wy, ey, ed, "output")
        U.untouched(y, yb, "output")
    else:
        assert bool((yb == U.POISON).all())
    return op


SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 31), (4, 32), (6, 33), (4, 256), (7, 264), (5, 512), (3, 520), (4, 1023), (5, 1024), (3, 1025), (2, 1032),
         (130, 1155), (1, 4096), (3, 4095), (2, 4104), (2, 8192), (2, 16384), (2, 16392), (1, 16385), (1, 32768), (1, 32767), (1000, 96), (4001, 8)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("types", [("bf16", "same"), ("bf16", "f32"), ("f16", "same"), ("f16", "f32"), ("f32", "same")], ids="-".join)
def test_sizes_and_types(U, size, types):
    _run(U, *size, dt=types[0], res=types[1], post="rms", pre="layer")


@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("n", [40, 777, 2048, 2500])
def test_kinds(U, post, pre, n):
    _run(U, 11, n, "bf16", "f32", post=post, pre=pre, scale=0.7, gate_rows=4)
    _run(U, 3, n, "f16", post=post, pre=pre, with_residual=False)


@pytest.mark.parametrize("gate_rows", [1, 2, 3, 10, 11, 100])
def test_gates(U, gate_rows):
    _run(U, 11, 300, gate_rows=gate_rows, post="rms")
    _run(U, 11, 1032, gate_rows=gate_rows, pre="none")


@pytest.mark.parametrize("pad,shift", [(8, 8), (8, 0), (0, 1), (1, 0), (4, 4), (3, 5)])
@pytest.mark.parametrize("n", [64, 1000, 1600, 5000])
def test_strides_and_alignment(U, n, pad, shift):
    _run(U, 9, n, "bf16", "f32", post="layer", pre="rms", gate_rows=5, pad=pad, shift=shift)


@pytest.mark.parametrize("rows,n", [(3001, 2048), (2500, 4096), (1300, 4104), (1200, 8192), (1500, 1544)])
@pytest.mark.parametrize("types", [("bf16", "same"), ("f16", "f32"), ("f32", "same")], ids="-".join)
def test_long_calls(U, rows, n, types):
    """Rows that stream through shared memory, more of them than blocks at a time."""
    _run(U, rows, n, *types, post="rms", pre="layer", gate_rows=7, scale=0.5)
    _run(U, rows, n, *types, post="none", pre="rms")
    _run(U, rows, n, *types, post="layer", pre="none", with_residual=False, pad=16)


@pytest.mark.parametrize("rows,n", [(297, 1032), (890, 1544), (2700, 2824), (445, 4096), (447, 4104), (600, 6152), (299, 8192)])
@pytest.mark.parametrize("types", [("bf16", "same"), ("f16", "f32"), ("f32", "same")], ids="-".join)
def test_blocks_that_walk_rows(U, rows, n, types):
    """Row counts around those of resident blocks: some blocks have one row more than others, or one alone."""
    _run(U, rows, n, *types, post="rms", pre="rms", in_place=True)
    _run(U, rows, n, *types, post="layer", pre="layer", gate_rows=rows - 1, pad=8, scale=-2.0, want_sum=False)
    _run(U, rows, n, *types, post="none", pre="layer", with_residual=False)
    _run(U, rows, n, *types, post="layer", pre="none", gate_rows=1)


def test_walked_rows_that_are_not_finite_stay_alone(U):
    E = U.E
    rows, n = 1500, 4096
    x = U.randn(rows, n, dtype=torch.bfloat16, seed=1)
    odd = torch.arange(rows, device="cuda") % 7 == 3
    x[odd, 5] = float("nan")
    op = E.BlockNorm(n, post=E.NORM_RMS, pre=E.NORM_LAYER, with_residual=False)
    y, s = torch.empty_like(x), torch.empty_like(x)
    assert op.prepare() == 0 and op.enqueue(y, s, x, rows=rows) == 0
    torch.cuda.synchronize()
    assert bool(y[odd].isnan().all()) and bool(s[odd].isnan().all()) and bool(y[~odd].isfinite().all()) and bool(s[~odd].isfinite().all())


@pytest.mark.parametrize("n", [9, 37, 250, 511, 1001, 1155, 1537, 2049, 4099, 9001, 16387])
@pytest.mark.parametrize("types", [("bf16", "same"), ("f16", "f32"), ("f32", "same")], ids="-".join)
@pytest.mark.parametrize("rows", [3, 9, 700])
def test_rows_that_start_anywhere(U, n, types, rows):
    """Dense rows of odd lengths: every place of a 16-byte boundary occurs."""
    if rows * n > 4_000_000:
        rows = 17
    _run(U, rows, n, *types, post="layer", pre="rms", gate_rows=2)
    _run(U, rows, n, *types, pre="layer", shift=5, in_place=True)


def test_weights_types_offset_and_no_sum(U):
    _run(U, 5, 200, wt="bf16", post="rms", pre="layer", offset=1.0)
    _run(U, 5, 2000, "f16", wt="f16", post="rms", pre="rms", offset=1.0, want_sum=False)
    _run(U, 5, 333, want_sum=False, with_residual=False)
    _run(U, 5, 4096, in_place=True)
    _run(U, 70, 77, "f16", "f32", in_place=True, post="rms")


def test_default_weights_are_ones(U):
    E = U.E
    x = U.randn(4, 100, dtype=torch.float32, seed=1)
    op, y = E.BlockNorm(100, dtype=E.f32, pre=E.NORM_LAYER, with_residual=False, weight_offset=1.0), torch.empty(4, 100, device="cuda")
    assert op.prepare() == 0 and op.enqueue(y, None, x, rows=4) == 0
    want, err = _normed64(x.double(), torch.zeros_like(x, dtype=torch.float64), "layer", torch.ones(100, dtype=torch.float64, device="cuda"), None, 1e-6)
    U.close(y, want, err, E.f32)


def test_variance_around_a_large_mean(U):
    """Values of 1000 +- 1: a difference of sums would lose the variance, the sum around the mean does not."""
    _run(U, 6, 3000, "f32", post="none", pre="layer", mean=1000.0, with_residual=False, eps=1e-6)
    _run(U, 6, 800, "f32", post="layer", pre="none", mean=1000.0, eps=1e-6)


def test_rows_of_zeros_and_values_that_are_not_finite(U):
    E = U.E
    for n in (48, 1155, 4096):
        x = U.randn(6, n, dtype=torch.bfloat16, seed=1)
        x[0], x[2, 3], x[4, n - 1] = 0.0, float("nan"), float("inf")
        op = E.BlockNorm(n, pre=E.NORM_RMS, with_residual=False)
        y, s = torch.empty_like(x), torch.empty_like(x)
        assert op.prepare() == 0 and op.enqueue(y, s, x, rows=6) == 0
        torch.cuda.synchronize()
        assert bool((y[0] == 0).all()) and bool(y[2].isnan().all()) and bool(y[4, n - 1].isnan()) and bool((y[4, :n - 1] == 0).all())
        assert bool(y[[1, 3, 5]].isfinite().all())


def test_offsets_past_32_bits(U):
    E = U.E
    rows, n, ld = 70001, 64, 32000
    big = torch.zeros(rows * ld, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (rows, n), (ld, 1), 0)
    y = torch.as_strided(big, (rows, n), (ld, 1), 128)
    x.copy_(U.randn(rows, n, dtype=torch.bfloat16, seed=3))
    op = E.BlockNorm(n, with_residual=False, ld_input=ld, ld_output=ld)
    assert op.prepare() == 0 and op.enqueue(y, None, x, rows=rows) == 0
    want, err = _normed64(x.double(), torch.zeros(rows, n, dtype=torch.float64, device="cuda"), "rms", torch.ones(n, dtype=torch.float64, device="cuda"), None, 1e-6)
    U.close(y.clone(), want, err, E.bf16)


def test_refusals_of_calls(U):
    E = U.E
    op = E.BlockNorm(64, gate_rows=2)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    assert op.enqueue(x, x, x, x, x, rows=4) == E.ELB_GENERAL_ERROR and "not prepared" in E.last_error()
    assert op.prepare() == 0
    assert op.enqueue(None, x, x, x, x, rows=4) == E.ELB_GENERAL_ERROR
    assert op.enqueue(x, x, x, None, x, rows=4) == E.ELB_GENERAL_ERROR
    assert op.enqueue(x, x, x, x, None, rows=4) == E.ELB_GENERAL_ERROR
    assert op.enqueue(x, x, x.data_ptr() + 1, x, x, rows=1) == E.ELB_GENERAL_ERROR
    assert op.enqueue(x, x, x, x, x, rows=0) == E.ELB_OK and op.launch_count() == 0


@pytest.mark.parametrize("rows,n", [(297, 2064), (445, 4096), (900, 4088), (447, 4104), (600, 6144), (299, 8192), (1000, 8184)])
@pytest.mark.parametrize("types", [("bf16", "same"), ("f16", "f32"), ("f32", "same")], ids="-".join)
def test_walked_rows_without_a_gate(U, rows, n, types):
    """Rows of 257 vectors and more without a gate: a scale, no sum, rows further apart, one output in the residual's place."""
    _run(U, rows, n, *types, post="rms", pre="layer", scale=-2.0, want_sum=False)
    _run(U, rows, n, *types, post="layer", pre="rms", scale=0.3, pad=8)
    _run(U, rows, n, *types, post="rms", pre="rms", scale=-0.5, in_place=True, pad=24)
    _run(U, rows, n, *types, post="layer", pre="layer", with_residual=False, want_sum=False)
    _run(U, rows, n, *types, post="layer", pre="none", scale=-2.0)
    _run(U, rows, n, *types, post="rms", pre="none")
