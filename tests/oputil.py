"""Helpers of the operator tests: the operators' definitions in 64 bits, with error bounds that follow from the formulas."""
from __future__ import annotations

import importlib
import math

import torch

E = importlib.import_module("deep-learning-math-kernel-research_b200")

TORCH = {E.bf16: torch.bfloat16, E.f16: torch.float16, E.f32: torch.float32}
UNIT = {E.bf16: 2.0 ** -8, E.f16: 2.0 ** -11, E.f32: 2.0 ** -24}        # half a unit in the last place, relative
TINY = {E.bf16: 2.0 ** -133, E.f16: 2.0 ** -25, E.f32: 2.0 ** -149}     # and absolute, among the subnormals
ACTS = {"none": E.ACT_NONE, "relu": E.ACT_RELU, "gelu": E.ACT_GELU, "gelu_tanh": E.ACT_GELU_TANH, "silu": E.ACT_SILU}
SLOPE = 1.13                                                           # no activation here is steeper (the tanh form of gelu: 1.129)
POISON = 7.25


def act64(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    if act == "gelu_tanh":
        return v * 0.5 * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def act_error(v):
    """What the activation itself may be off in 32 bits: a few roundings and an exponential of up to |2u|, whose argument's
    rounding it multiplies.  erf's form loses the relative precision of large negative values, not the absolute."""
    return 2.0 ** -20 * (1.0 + v.abs())


def product64(x, w):
    """x w^T in 64 bits and what a sum of as many products in 32 bits may be off: each of the additions rounds (or cuts off) to
    2^-23 of a partial sum, which is at most sum |x w|; the errors of n of them grow as their root (factor 4: the tail)."""
    z = x.double() @ w.double().t()
    return z, (4.0 * math.sqrt(x.shape[1]) + 8.0) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()) + 1e-37


def activated64(z, dz, act, gated):
    if not gated:
        return act64(z, act), SLOPE * dz + act_error(z)
    n = z.shape[-1] // 2
    g, u, dg, du = z[..., :n], z[..., n:], dz[..., :n], dz[..., n:]
    a, da = act64(g, act), SLOPE * dg + act_error(g)
    return a * u, da * u.abs() + a.abs() * du + da * du + 2.0 ** -23 * (a * u).abs()


def linear64(x, w, b, r, act, gated, scale):
    z, dz = product64(x, w)
    if b is not None:
        z = z + b.double()
        dz = dz + 2.0 ** -23 * z.abs()
    y, dy = activated64(z, dz, act, gated)
    y, dy = scale * y, abs(scale) * dy + 2.0 ** -23 * (scale * y).abs()
    if r is not None:
        y = y + r.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy


def close(got, want, err, dt, what=""):
    """Each value within its bound: the computation's error, then one rounding to the result's type."""
    got = got.double()
    bound = 1.01 * err + UNIT[dt] * (want.abs() + err) + TINY[dt]
    off = (got - want).abs()
    # a value that rounds past the type's largest is infinite
    top = torch.finfo(TORCH[dt]).max
    fine = (off <= bound) | ((want.abs() + bound >= top) & got.isinf())
    bad = ~fine
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} (bound {bound.expand_as(got)[bad][0]})")


def strided(rows, n, ld, dtype, offset=0, fill=None, source=None):
    """(view [rows, n] of rows ld apart, the whole buffer): `offset` elements in front, poison around."""
    buf = torch.full((offset + max(rows, 1) * ld + 64,), POISON, dtype=dtype, device="cuda")
    view = torch.as_strided(buf, (rows, n), (ld, 1), offset)
    if source is not None:
        view.copy_(source)
    elif fill is not None:
        view.fill_(fill)
    return view, buf


def untouched(view, buf, what=""):
    """Nothing around the view's elements was written."""
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, view.shape, view.stride(), view.storage_offset()).fill_(False)
    assert bool((buf[mask] == POISON).all()), f"{what}: written outside the tensor"


def randn(*shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)
