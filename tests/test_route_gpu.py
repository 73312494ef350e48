"""``Route`` against its definition: whole rows of choices, ties, groups, masks, and weights in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def U(pkg):
    import oputil
    return oputil


def _reference(z, k, sigmoid, bias, groups, top_groups, group_best, renormalise, scale):
    """z: [rows, experts] in 64 bits.  Returns ids, weights and, for each row, the smallest gap between choices
    (and groups) that decided; equal choices are decided by the index."""
    z = np.where(np.isnan(z), -np.inf, z)
    rows, n = z.shape
    top = z.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        if sigmoid:
            score = 1.0 / (1.0 + np.exp(-z))
            whole = None
        else:
            d = np.where(z == top, 0.0, z - top)
            score = np.where(np.isneginf(z), 0.0, np.exp(d))
            whole = score.sum(1, keepdims=True)
            score = np.where(whole > 0, score / np.where(whole > 0, whole, 1.0), 0.0)
    choice = score + bias if bias is not None else score.copy()
    choice[np.isnan(choice)] = -np.inf
    gap = np.full(rows, np.inf)
    if groups > 1:
        by = choice.reshape(rows, groups, -1)
        best = -np.sort(-by, axis=2)[:, :, :group_best].sum(2)
        order = np.argsort(-best, axis=1, kind="stable")
        s = np.take_along_axis(best, order, 1)
        if top_groups < groups:
            with np.errstate(all="ignore"):
                d = s[:, top_groups - 1] - s[:, top_groups]
            gap = np.minimum(gap, np.where(d > 0, d, np.inf))
        shut = np.ones((rows, groups), bool)
        np.put_along_axis(shut, order[:, :top_groups], False, 1)
        by[shut] = -np.inf
        choice = by.reshape(rows, n)
    order = np.argsort(-choice, axis=1, kind="stable")
    s = np.take_along_axis(choice, order, 1)[:, :k + 1]
    with np.errstate(all="ignore"):
        d = s[:, :-1] - s[:, 1:]
    gap = np.minimum(gap, np.where(d > 0, d, np.inf).min(1, initial=np.inf))
    ids = order[:, :k]
    w = np.take_along_axis(score, ids, 1)
    if renormalise:
        t = w.sum(1, keepdims=True)
        w = np.where(t > 0, w / np.where(t > 0, t, 1.0), 0.0)
    return ids, w * scale, gap


def _run(U, z, k, dt="f32", sigmoid=False, bias=None, groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0, pad=0, sure_rows=1.0):
    E = U.E
    rows, n = z.shape
    td = U.TORCH[getattr(E, dt)]
    zs, _ = U.strided(rows, n, n + pad, td, pad, source=z)
    op = E.Route(n, k, dtype=getattr(E, dt), score=E.SCORE_SIGMOID if sigmoid else E.SCORE_SOFTMAX, with_bias=bias is not None, groups=groups,
                 top_groups=top_groups, group_best=group_best, renormalise=renormalise, scale=scale, ld_logits=n + pad)
    assert op.prepare(bias) == 0, E.last_error()
    ids = torch.full((rows + 1, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((rows + 1, k), U.POISON, device="cuda")
    assert op.enqueue(ids, w, zs, rows=rows) == 0, E.last_error()
    torch.cuda.synchronize()
    assert bool((ids[rows] == -7).all()) and bool((w[rows] == U.POISON).all())
    want_ids, want_w, gap = _reference(zs.double().cpu().numpy(), k, sigmoid, None if bias is None else bias.double().cpu().numpy(), groups,
                                       top_groups, group_best, renormalise, scale)
    got = ids[:rows].cpu().numpy()
    # choices in 32 bits are a few 2^-24 off: rows whose decisions are nearer than that say nothing
    sure = gap > 2.0 ** -21
    assert sure.mean() >= sure_rows, sure.mean()
    assert np.array_equal(got[sure], want_ids[sure])
    # softmax: exp, a sum of n, a division, the renormalisation's sum and division, the scale: under 64 roundings
    g = w[:rows].double().cpu().numpy()
    assert np.all(np.abs(g - want_w)[sure] <= (64 * 2.0 ** -24 * np.abs(want_w) + 1e-37)[sure])
    return got, w[:rows]


def _spread(U, rows, n, seed):
    """Logits whose neighbours in order lie apart: a random permutation of distinct steps for each row."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.rand(rows, n, generator=g, device="cuda").argsort(dim=1).float()
    return (order - n / 2) * (6.0 / n) + 0.3


@pytest.mark.parametrize("n,k", [(1, 1), (2, 2), (3, 1), (8, 2), (31, 4), (32, 32), (33, 8), (60, 4), (64, 8), (65, 3), (128, 1), (160, 6), (256, 8), (300, 32),
                                 (512, 8), (1000, 10), (1024, 32)])
@pytest.mark.parametrize("rows", [1, 2, 7, 130])
@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
def test_sizes(U, n, k, rows, sigmoid):
    _run(U, _spread(U, rows, n, n + rows), k, sigmoid=sigmoid, scale=2.5)


@pytest.mark.parametrize("n,groups,top,best", [(64, 8, 3, 2), (256, 8, 4, 2), (256, 8, 4, 1), (160, 8, 3, 1), (96, 32, 10, 2), (60, 4, 2, 2), (32, 32, 12, 2), (1024, 16, 1, 2)])
@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True], ids=["", "bias"])
def test_groups(U, n, groups, top, best, sigmoid, with_bias):
    # the bias is a multiple of 1/64 from a few values, so that choices stay apart as the scores are
    z = _spread(U, 50, n, n + top)
    bias = None
    if with_bias:
        bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(n)).float().cuda() / 64
    k = min(8, n // groups * top)
    _run(U, z, k, sigmoid=sigmoid, bias=bias, groups=groups, top_groups=top, group_best=best, renormalise=n != 160, sure_rows=0.8)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [40, 256])
def test_ties_go_to_the_lowest_index(U, dt, n):
    E = U.E
    g = torch.Generator(device="cuda").manual_seed(n)
    z = torch.randint(-2, 3, (60, n), generator=g, device="cuda").float()
    for sigmoid in (False, True):
        _run(U, z, 8, dt, sigmoid=sigmoid)
        _run(U, z, 8, dt, sigmoid=sigmoid, renormalise=False, pad=3)
    _run(U, z * 0, 5, dt)
    _run(U, z, 4, dt, sigmoid=True, groups=8, top_groups=3, group_best=2)
    zero = torch.zeros(3, n, device="cuda")
    zero[:, ::2] = -0.0
    got, _ = _run(U, zero, 6, dt)
    assert got[0].tolist() == [0, 1, 2, 3, 4, 5]


def test_masked_experts_and_rows(U):
    """-inf, NaN, the type's lowest value, +inf and rows where nothing is left."""
    inf, low = float("inf"), torch.finfo(torch.float32).min
    z = _spread(U, 8, 48, 1)
    z[0, :40] = -inf
    z[1, 5:] = low
    z[2] = -inf
    z[3] = low
    z[4, 7] = float("nan")
    z[5] = float("nan")
    z[6, 9] = inf
    z[7, 9], z[7, 11] = inf, inf
    for sigmoid in (False, True):
        got, w = _run(U, z, 6, sigmoid=sigmoid)
        assert bool(w.isfinite().all())
        for row in got:
            assert len(set(row.tolist())) == 6
    got, w = _run(U, z, 6, renormalise=False)
    assert got[2].tolist() == [0, 1, 2, 3, 4, 5] and bool((w[2] == 0).all()) and bool((w[5] == 0).all())
    assert w[6, 0] == 1.0 and w[7].tolist()[:2] == [0.5, 0.5]
    # a bias that shuts experts
    bias = torch.zeros(48, device="cuda")
    bias[10:40] = -inf
    bias[3] = float("nan")
    got, _ = _run(U, _spread(U, 20, 48, 2), 8, sigmoid=True, bias=bias)
    assert not np.isin(got, list(range(10, 40)) + [3]).any()


def test_choice_and_weights_in_32_bits_as_written(U):
    """The scores are the formulas' own 32-bit operations: the same choices as torch's, bit for bit, also where they are near."""
    E = U.E
    z = U.randn(20000, 256, dtype=torch.float32, seed=9, scale=1.5)
    b = U.randn(256, dtype=torch.float32, seed=10, scale=0.1)
    choice = 1.0 / (1.0 + torch.exp(-z)) + b
    op, ids = E.Route(256, 8, score=E.SCORE_SIGMOID, with_bias=True), torch.empty(20000, 8, dtype=torch.int32, device="cuda")
    assert op.prepare(b) == 0 and op.enqueue(ids, None, z, rows=20000) == 0
    assert torch.equal(ids.long(), choice.sort(dim=1, descending=True, stable=True).indices[:, :8])
    op2 = E.Route(256, 8)
    assert op2.prepare() == 0 and op2.enqueue(ids, None, z, rows=20000) == 0
    choice = torch.exp(z - z.max(1, keepdim=True).values)
    assert torch.equal(ids.long(), choice.sort(dim=1, descending=True, stable=True).indices[:, :8])


def test_refusals_of_calls(U):
    E = U.E
    op = E.Route(16, 2, with_bias=True)
    z, ids = torch.zeros(4, 16, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    assert op.enqueue(ids, None, z, rows=4) == E.ELB_GENERAL_ERROR
    assert op.prepare(None) == E.ELB_GENERAL_ERROR
    assert op.prepare(torch.zeros(16)) == 0
    assert op.enqueue(None, None, z, rows=4) == E.ELB_GENERAL_ERROR
    assert op.enqueue(ids, None, None, rows=4) == E.ELB_GENERAL_ERROR
    assert op.enqueue(ids, None, z, rows=-3) == E.ELB_GENERAL_ERROR
    assert op.enqueue(ids, None, z, rows=0) == E.ELB_OK and op.launch_count() == 0


@pytest.mark.parametrize("n,groups,top", [(64, 8, 2), (256, 8, 4), (60, 4, 2), (96, 32, 6), (40, 5, 3)])
@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
@pytest.mark.parametrize("shut", [float("-inf"), float("nan")], ids=["-inf", "nan"])
def test_only_experts_of_open_groups(U, n, groups, top, sigmoid, shut):
    """A bias that leaves each group one expert that counts: the others of the open groups come next, by their index, and no expert of a
    closed group does, however low its index."""
    E = U.E
    size, rows = n // groups, 40
    z = _spread(U, rows, n, n)
    bias = torch.full((n,), shut, device="cuda")
    bias[size - 1::size] = 0.0
    k = min(8, size * top)
    op = E.Route(n, k, score=E.SCORE_SIGMOID if sigmoid else E.SCORE_SOFTMAX, with_bias=True, groups=groups, top_groups=top, renormalise=False)
    ids, w = torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda")
    assert op.prepare(bias) == 0 and op.enqueue(ids, w, z, rows=rows) == 0
    torch.cuda.synchronize()
    zd = z.double()
    score = torch.sigmoid(zd) if sigmoid else torch.softmax(zd, 1)
    for t in range(rows):
        best = score[t, size - 1::size].sort(descending=True).indices[:top].tolist()
        want = [g * size + size - 1 for g in best]
        want += sorted(g * size + i for g in best for i in range(size - 1))
        assert ids[t].tolist() == want[:k]
    got = score.gather(1, ids.long())
    assert bool(((w.double() - got).abs() <= 64 * 2.0 ** -24 * got).all())
