"""What ``enqueue`` of the transformer operators takes, without a GPU: the library is a stand-in that notes its calls, tensors say that they are on one."""
import pytest
import torch


class _Library:
    """create gives a null handle (which the library itself destroys without harm); enqueue notes the addresses."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_enqueue"):
                self.calls.append(args)
            return 0
        return call


class Tensor:
    """A CPU tensor that says it is a GPU's."""
    is_cuda = True

    def __init__(self, t, device=0):
        self.t, self.device = t, device

    def get_device(self):
        return self.device

    def __getattr__(self, name):
        return getattr(self.t, name)


BF, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def new(*shape, dtype=BF):
    return Tensor(torch.empty(*shape, dtype=dtype))


@pytest.fixture()
def E(pkg, monkeypatch):
    monkeypatch.setattr(pkg, "lib", _Library())
    return pkg


def _plans(E):
    """name -> (plan, good tensors of a call of 6 rows)"""
    return {
        "linear": (E.Linear(64, 96, out_dtype=E.f32, with_residual=True), dict(output=new(6, 96, dtype=F32), input=new(6, 64), residual=new(6, 96, dtype=F32))),
        "norm": (E.BlockNorm(64, residual_dtype=E.f32, gate_rows=4), dict(output=new(6, 64), sum=new(6, 64, dtype=F32), input=new(6, 64),
                                                                         residual=new(6, 64, dtype=F32), gate=new(2, 64))),
        "route": (E.Route(16, 2), dict(ids=new(6, 2, dtype=I32), weights=new(6, 2, dtype=F32), logits=new(6, 16, dtype=F32))),
        "experts": (E.Experts(8, 2, 64, 32, 100), dict(output=new(6, 64), input=new(6, 64), ids=new(6, 2, dtype=I32), weights=new(6, 2, dtype=F32))),
    }


ARGUMENTS = [(k, a) for k, names in (("linear", ("output", "input", "residual")), ("norm", ("output", "sum", "input", "residual", "gate")),
                                     ("route", ("ids", "weights", "logits")), ("experts", ("output", "input", "ids", "weights"))) for a in names]


@pytest.mark.parametrize("kind,argument", ARGUMENTS)
def test_tensors_that_do_not_hold_the_rows_are_refused(E, kind, argument):
    plan, good = _plans(E)[kind]
    assert plan.enqueue(**good, rows=6) == 0 and len(E.lib.calls) == 1
    assert [a for a in E.lib.calls[0][1:] if isinstance(a, int) and a > 64] == [t.data_ptr() for t in good.values()]
    t = good[argument].t
    n, other = t.shape[1], F16 if t.dtype != F16 else BF
    bad = [t.to(other), t.to(torch.int64), t[:-1], t[:-1].clone(), t[0], torch.empty(n, t.shape[0], dtype=t.dtype).t(), torch.empty(2 * t.shape[0], n, dtype=t.dtype)[::2],
           torch.empty(t.shape[0], 2 * n, dtype=t.dtype)[:, ::2], torch.empty(t.shape[0], n + 8, dtype=t.dtype)[:, :n], t[:, :-1], torch.empty(1, n, dtype=t.dtype).expand(t.shape[0], n),
           torch.empty(0, n, dtype=t.dtype), torch.empty((), dtype=t.dtype)]
    for b in bad:
        with pytest.raises(ValueError, match=argument):
            plan.enqueue(**{**good, argument: Tensor(b)}, rows=6)
    for elsewhere in (t, Tensor(t, device=1)):
        with pytest.raises(ValueError, match="device 0"):
            plan.enqueue(**{**good, argument: elsewhere}, rows=6)
    assert len(E.lib.calls) == 1
    # what holds them in another shape, more of them, an address, and calls without rows, which use none
    for fine in (torch.empty(2, t.shape[0] // 2, n, dtype=t.dtype), torch.empty(t.numel() + 5, dtype=t.dtype), torch.empty(t.shape[0] + 3, n, dtype=t.dtype)):
        assert plan.enqueue(**{**good, argument: Tensor(fine)}, rows=6) == 0
    assert plan.enqueue(**{**good, argument: 4096}, rows=6) == 0
    assert plan.enqueue(**{**good, argument: new(1, dtype=torch.int64)}, rows=0) == 0
    assert len(E.lib.calls) == 6


def test_rows_that_lie_apart(E):
    plan = E.Linear(64, 96, ld_input=80, ld_output=100, with_residual=True, ld_residual=96)
    wide, out, res = torch.empty(6, 80, dtype=BF), torch.empty(6, 100, dtype=BF), new(6, 96)

    def call(x, y, rows=6):
        return plan.enqueue(Tensor(y), Tensor(x), res, rows=rows)

    flat = torch.empty(5 * 80 + 64, dtype=BF)
    for x in (wide, wide[:, :64], flat, torch.as_strided(flat, (6, 64), (80, 1)), torch.empty(2, 3, 80, dtype=BF)[:, :, 8:72], torch.empty(6, 1, 80, dtype=BF)):
        assert call(x, out) == 0 and call(x, out[:, 2:98]) == 0
    assert call(torch.empty(1, 64, dtype=BF), torch.empty(1, 96, dtype=BF), rows=1) == 0
    for x in (torch.empty(6, 64, dtype=BF), torch.empty(6, 96, dtype=BF), wide[:, :63], wide[:5], flat[1:], torch.empty(3, 2, 96, dtype=BF)[:, :, :64],
              torch.empty(12, 80, dtype=BF)[::2], torch.empty(2, 4, 80, dtype=BF)[:, :3]):
        with pytest.raises(ValueError, match="input"):
            call(x, out)
    with pytest.raises(ValueError, match="output"):
        call(wide, torch.empty(6, 96, dtype=BF))


def test_tensors_that_a_plan_does_not_use_are_not_looked_at(E):
    assert E.Linear(64, 96).enqueue(new(6, 96), new(6, 64), new(1, dtype=F32), rows=6) == 0
    assert E.BlockNorm(64, pre=E.NORM_NONE, with_residual=False).enqueue(new(1), new(6, 64), new(6, 64), new(1), new(1), rows=6) == 0
    with pytest.raises(ValueError):
        E.Linear(64, 96).enqueue(new(6, 96), new(6, 64), torch.empty(6, 96), rows=6)
