"""Helpers of the attention operators' tests: batches over caches of pages and dense tensors, the definitions in 64 bits with error bounds that follow from
the formulas."""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

from oputil import E, POISON, TINY, TORCH, UNIT, randn

NAN = float("nan")
FAR_PAGE = 1 << 30                # in entries of a table that nobody may read


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def batch(new, lengths, page_size, seed=0, spare=3, width=None, behind=0, ragged=None):
    """Sequences of ``lengths`` tokens, the last ``new`` of each among them, over pages in no order; ``behind`` rows follow the last sequence."""
    rng = random.Random(seed)
    held = [-(-n // page_size) for n in lengths]
    width = max(held + [1]) if width is None else width
    pages = sum(held) + spare
    order = rng.sample(range(pages), pages)
    table, used = torch.full((len(new), width), FAR_PAGE, dtype=torch.int32), []
    for s, n in enumerate(held):
        table[s, :n] = torch.tensor(order[len(used):len(used) + n], dtype=torch.int32)
        used += order[len(used):len(used) + n]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    ragged = len(set(new)) > 1 or behind > 0 if ragged is None else ragged
    return SimpleNamespace(new=new, lengths=lengths, page_size=page_size, pages=pages, width=width, table=table.cuda(), lengths_t=ints(lengths), starts=starts,
                           starts_t=ints(starts) if ragged else None, rows=starts[-1] + behind, seqs=len(new))


def cache(b, kv_heads, head_dim, dtype, order="heads", ld_extra=0, fill=NAN):
    """A cache filled with ``fill``, its strides as the plan wants them, and a view [pages, kv_heads, page_size, head_dim] of it."""
    d = head_dim + ld_extra
    if order == "heads":
        t = torch.full((b.pages, kv_heads, b.page_size, d), fill, dtype=TORCH[dtype], device="cuda")[..., :head_dim]
        return t, t, dict(ld_page=kv_heads * b.page_size * d, ld_head=b.page_size * d, ld_token=d)
    t = torch.full((b.pages, b.page_size, kv_heads, d), fill, dtype=TORCH[dtype], device="cuda")[..., :head_dim]
    return t, t.permute(0, 2, 1, 3), dict(ld_page=kv_heads * b.page_size * d, ld_head=d, ld_token=kv_heads * d)


def put(b, view, s, x):
    """x: [length, kv_heads, head_dim] of sequence s, into its pages"""
    for p in range(-(-x.shape[0] // b.page_size)):
        part = x[p * b.page_size:(p + 1) * b.page_size]
        view[int(b.table[s, p]), :, :part.shape[0]] = part.permute(1, 0, 2)


def attention64(q, k, v, n, causal, scale, dt):
    """One sequence: q [n, heads, d], k and v [length, kv_heads, d].  (out, its bound before the last rounding) in 64 bits.

    A score is a sum of d products in 32 bits: (4 sqrt(d) + 8) 2^-23 of the sum of their sizes (see product64), scaled with one rounding, and its distance
    from the running maximum is rounded to 2^-23 of the two; a term's exponential is right to 2^-17 and rounded to dt.  The sums over the keys add
    (4 sqrt(length) + 8) 2^-23 of the sum of the terms' sizes.  A term that falls among f16's subnormals is off by TINY, beside a largest of one or more."""
    group, length = q.shape[1] // k.shape[1], k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    if length == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = torch.einsum("nhd,mhd->hnm", q, k) * scale
    size = torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * abs(scale)
    seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(length - n)
    s = s.masked_fill(~seen, -math.inf)
    top = s.max(-1, keepdim=True).values
    none = (top == -math.inf)
    w = torch.where(seen, torch.exp(s - top.masked_fill(none, 0.0)), torch.zeros_like(s))
    whole = w.sum(-1, keepdim=True)
    w = torch.where(none, torch.zeros_like(w), w / whole.masked_fill(none, 1.0))
    ds = (4.0 * math.sqrt(q.shape[2]) + 8.0) * 2.0 ** -23 * size + 2.0 ** -21 * (s.masked_fill(~seen, 0.0).abs() + top.masked_fill(none, 0.0).abs())
    # the running maximum, too, comes from scores that are off
    rel = 1.1 * (ds + 2.0 ** -17) + (4.0 * math.sqrt(length) + 8.0) * 2.0 ** -23
    out = torch.einsum("hnm,mhd->nhd", w, v)
    err = torch.einsum("hnm,mhd->nhd", w * (rel + UNIT[dt]), v.abs()) + (w * rel).sum(-1).t()[..., None] * out.abs()
    err = err + TINY[dt] * torch.einsum("nm,mhd->nhd", seen.double(), v.abs())
    return out, err


def inputs(b, heads, kv_heads, head_dim, dt, seed=1, scale=1.0):
    """q [rows, heads, d] and each sequence's keys and values"""
    q = randn(b.rows, heads, head_dim, dtype=TORCH[dt], seed=seed, scale=1.5 * scale)
    kv = [(randn(n, kv_heads, head_dim, dtype=TORCH[dt], seed=seed + 10 + 2 * s, scale=scale), randn(n, kv_heads, head_dim, dtype=TORCH[dt], seed=seed + 11 + 2 * s))
          for s, n in enumerate(b.lengths)]
    return q, kv


def wanted(b, q, kv, causal, scale, dt):
    """(out, bound, rows that a sequence has) of the whole batch"""
    out, err = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for s, (k, v) in enumerate(kv):
        r = slice(b.starts[s], b.starts[s] + b.new[s])
        out[r], err[r] = attention64(q[r], k, v, b.new[s], causal, scale, dt)
    return out, err, b.starts[-1]


def poisoned(*shape, dt):
    return torch.full(shape, POISON, dtype=TORCH[dt], device="cuda")


def turn64(x, positions, r, layout, steps, magnitude, inverse=False):
    """Rotary positions of x [rows, heads, d] in 64 bits and what 32 bits may be off: the argument of sine and cosine is a 32-bit fraction of half a turn (2^-25
    of a half turn, 2^-23 in radians), they are right to 2^-22, the products and the sum round three times."""
    y = x.double().clone()
    near = layout == E.ROTARY_NEIGHBOURS
    a, b = (x[..., 0:r:2].double(), x[..., 1:r:2].double()) if near else (x[..., :r // 2].double(), x[..., r // 2:r].double())
    angle = positions.double()[:, None, None] * steps.double().cuda() * (-1.0 if inverse else 1.0)
    u, w = magnitude * (a * angle.cos() - b * angle.sin()), magnitude * (b * angle.cos() + a * angle.sin())
    err = torch.zeros_like(y)
    off = abs(magnitude) * (a.abs() + b.abs()) * 2.0 ** -20
    if near:
        y[..., 0:r:2], y[..., 1:r:2], err[..., 0:r:2], err[..., 1:r:2] = u, w, off, off
    else:
        y[..., :r // 2], y[..., r // 2:r], err[..., :r // 2], err[..., r // 2:r] = u, w, off, off
    return y, err


def steps64(r, base=10000.0, scaling=None, factor=1.0, slow=1.0, fast=4.0, original=8192):
    f = torch.tensor([base ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64)
    if scaling == E.SCALE_LINEAR:
        f = f / factor
    if scaling == E.SCALE_BY_PARTS:
        s = ((original * f / (2.0 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = s * f + (1.0 - s) * f / factor
    return f
