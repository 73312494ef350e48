"""Performance cases of the attention operators: the attention half of a transformer block over a paged cache of keys and values or over dense
tensors, through the public entry points of the package (``Rotary``, ``CacheAppend``, ``Attention``).

A case is a dict of plain values.  ``op`` names the operator:

  rotary     queries and keys turned by their positions: pairs (i, i + r/2) or (2i, 2i + 1) of the first r channels of a head
  append     queries turned, keys turned and written to their places in the cache's pages, values written there
  attention  out[t] = sum_j softmax_j(scale * q[t] k[j]) v[j] over the keys that token t sees, in pages of a cache or in dense tensors

Sequences have between ``least`` and ``keys`` tokens, the new ones included, spread evenly; each brings ``new`` new tokens, or between one and ``new`` where
``ragged``.  With ``own`` false ``run`` computes the operators in elementary torch operations in 32 bits (angles in 64), rounded once at the end.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BASE, FACTOR, SLOW, FAST, ORIGINAL, MAGNITUDE = 500000.0, 8.0, 1.0, 4.0, 8192, 1.1


def _rotary(rows, heads, kv_heads, dim, rotary=0, layout="halves", scaling="none", dtype="bf16", far=4096):
    """``rotary``: channels of a head that are turned, 0 for all; ``far``: the largest position."""
    return dict(op="rotary", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary or dim, layout=layout, scaling=scaling, dtype=dtype, far=far)


def _append(seqs, new, least, keys, heads, kv_heads, dim, page, rotary=0, layout="halves", scaling="none", dtype="bf16", ragged=False):
    return dict(op="append", seqs=seqs, new=new, least=max(least, new), keys=max(keys, new), heads=heads, kv_heads=kv_heads, dim=dim, page=page, rotary=rotary or dim,
                layout=layout, scaling=scaling, dtype=dtype, ragged=ragged)


def _attention(seqs, new, least, keys, heads, kv_heads, dim, page, causal=True, dtype="bf16", ragged=False):
    """``page``: tokens of a page of the cache, 0 for dense tensors.  A causal case's new tokens are the last of their sequence."""
    return dict(op="attention", seqs=seqs, new=new, least=max(least, new if causal else 1), keys=max(keys, new if causal else 1), heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, causal=causal, dtype=dtype, ragged=ragged)


def listed():
    return [
        # the turn in front of an attention without a cache, for four tokens far into their texts: latency
        dict(_rotary(4, 32, 8, 128, far=100000), name="rotary_tokens"),
        # an encoder's prompt of odd length, heads turned in part, neighbouring pairs, positions stretched
        dict(_rotary(3001, 16, 16, 80, 32, "neighbours", "linear", "f16", far=3000), name="rotary_prompt_partial"),
        # a step of 64 answers: one token each
        dict(_append(64, 1, 100, 4000, 32, 8, 128, 16), name="append_tokens"),
        # prompts of uneven length that start 12 answers, a long-context scaling
        dict(_append(12, 2500, 2500, 2500, 32, 8, 128, 64, 0, "halves", "by_parts", ragged=True), name="append_prompts"),
        # one answer, one token
        dict(_attention(1, 1, 3900, 3900, 32, 8, 128, 16), name="token_one"),
        # a full batch of answers of very uneven length
        dict(_attention(64, 1, 500, 16000, 32, 8, 128, 64), name="token_batch"),
        # a batch whose heads do not share keys, half as wide
        dict(_attention(24, 1, 1, 3001, 12, 12, 64, 32, dtype="f16"), name="token_batch_unshared"),
        # four proposed tokens behind the last one are looked at together, five heads to a key head
        dict(_attention(8, 5, 1000, 7000, 40, 8, 128, 16), name="token_proposals"),
        # a long prompt: the largest
        dict(_attention(1, 8192, 8192, 8192, 32, 8, 128, 64), name="prompt_long"),
        # pieces of prompts of uneven length behind what is in the cache already
        dict(_attention(6, 700, 700, 5000, 32, 4, 128, 32, ragged=True), name="prompt_pieces"),
        # a decoder's tokens over a padded batch of encoder states of other lengths
        dict(_attention(8, 448, 300, 1500, 20, 20, 64, 0, causal=False, dtype="f16"), name="cross_prompt"),
        # one token each over encoder states
        dict(_attention(16, 1, 1500, 1500, 20, 20, 64, 0, causal=False, dtype="f16"), name="cross_tokens"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 12, 16])
    return kv * rng.choice([1, 1, 4, 4, 5, 7, 8] if kv <= 8 else [1, 2]), kv


def _draw_once(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "attention"])
    heads, kv = _heads(rng)
    dim, dtype = rng.choice([64, 64, 80, 96, 128, 128, 128]), rng.choice(["bf16", "bf16", "f16"])
    page, turn = rng.choice([16, 16, 32, 64, 128]), (rng.choice([0, 0, 32]), rng.choice(["halves", "neighbours"]), rng.choice(["none", "linear", "by_parts"]))
    if op == "rotary":
        return _rotary(_log(rng, 1, 16000), heads, kv, dim, *turn, dtype=rng.choice([dtype, "f32"]), far=_log(rng, 100, 200000))
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 30000 // seqs))
        return _append(seqs, new, new + rng.randint(0, 50), new + _log(rng, 50, 2000), heads, kv, dim, page, *turn, dtype=dtype, ragged=new > 1 and rng.random() < 0.5)
    kind = rng.choice(["token", "token", "prompt", "cross"])
    if kind == "token":
        return _attention(_log(rng, 1, 96), rng.choice([1, 1, 1, 2, 4]), 1, _log(rng, 10, 20000), heads, kv, dim, page, dtype=dtype)
    if kind == "prompt":
        seqs, new = _log(rng, 1, 12), _log(rng, 16, 8192)
        keys = new + (0 if rng.random() < 0.5 else _log(rng, 10, 4000))
        return _attention(seqs, new, keys * 3 // 4, keys, heads, kv, dim, page, dtype=dtype, ragged=rng.random() < 0.5)
    keys = _log(rng, 20, 3000)
    return _attention(_log(rng, 1, 32), _log(rng, 1, 1500), keys // 3 + 1, keys, heads, kv, dim, 0, causal=False, dtype=dtype)


def _scores(c):
    return c["seqs"] * c["heads"] * c["new"] * c["keys"] if c["op"] == "attention" else 0


def draw(rng):
    top = listed()
    most_bytes, most_flops, most_scores = max(work(c)["bytes"] for c in top), max(work(c)["flops"] for c in top), max(_scores(c) for c in top)
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and _scores(c) <= most_scores:
            return c


# ------------------------------------------------------------------------------------------- sizes and inputs
def _spread(n, lo, hi, turn):
    """n numbers from lo to hi, evenly spread, in an order without a trend; the last is hi."""
    return [hi if i == n - 1 else lo + int((hi - lo + 1) * ((i * 0.6180339887 + turn) % 1.0)) for i in range(n)]


def _lengths(c):
    """(tokens of each sequence, new tokens of each)"""
    new = _spread(c["seqs"], 1, c["new"], 0.3) if c["ragged"] else [c["new"]] * c["seqs"]
    return _spread(c["seqs"], c["least"], c["keys"], 0.1), new


def _make(c, seed):
    """The tensors of a case, from its sizes and the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    dt = DTYPES[c["dtype"]]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")                     # noqa: E731

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "rotary":
        far = torch.randint(0, c["far"] + 1, (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        return dict(q=normal(c["rows"], h, d), k=normal(c["rows"], kv, d), positions=far)
    lengths, new = _lengths(c)
    rows = sum(new)
    first = [sum(new[:i]) for i in range(len(new) + 1)]
    t = dict(rows=rows, lengths=ints(lengths), starts=ints(first) if c["ragged"] else None)
    # what the plain form wants to know of each row: its sequence, its place among the new tokens
    t["seq"] = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), ints(new).long())
    t["place"] = torch.arange(rows, device="cuda") - ints(first).long()[t["seq"]]
    t["new"] = ints(new).long()
    t["q"] = normal(rows, h, d, scale=1.5)
    if c["op"] == "attention" and c["page"] == 0:
        t["k"], t["v"] = normal(c["seqs"], c["keys"], kv, d), normal(c["seqs"], c["keys"], kv, d)
        t["table"] = None
        return t
    page = c["page"]
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + 3                                    # a pool in which pages lie in no order, a few of them nobody's
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], max(held)), -1, dtype=torch.int32, device="cuda")
    mask = torch.arange(max(held), device="cuda")[None, :] < ints(held)[:, None]
    table[mask] = order[:sum(held)]
    t["table"] = table
    t["k"], t["v"] = normal(pages, kv, page, d), normal(pages, kv, page, d)
    if c["op"] == "append":
        t["new_k"], t["new_v"] = normal(rows, kv, d), normal(rows, kv, d)
    return t


def _plan(c, t):
    """The plan that a user's program makes once for a layer, and the tensors that it writes."""
    E = importlib.import_module("deep-learning-math-kernel-research_b200")
    dtype = {"bf16": E.bf16, "f16": E.f16, "f32": E.f32}[c["dtype"]]
    if c["op"] == "attention":
        return E.Attention(c["heads"], c["kv_heads"], c["dim"], dtype=dtype, page_size=c["page"], causal=c["causal"]), dict(out=torch.empty_like(t["q"]))
    turn = dict(rotary_dim=c["rotary"], layout=E.ROTARY_NEIGHBOURS if c["layout"] == "neighbours" else E.ROTARY_HALVES, base=BASE,
                scaling={"none": E.SCALE_NONE, "linear": E.SCALE_LINEAR, "by_parts": E.SCALE_BY_PARTS}[c["scaling"]], factor=FACTOR, slow=SLOW, fast=FAST,
                original=ORIGINAL, magnitude=MAGNITUDE if c["scaling"] == "by_parts" else 1.0)
    if c["op"] == "rotary":
        plan = E.Rotary(c["heads"], c["kv_heads"], c["dim"], dtype=dtype, **turn)
        _ok(plan.prepare())
        return plan, dict(q=torch.empty_like(t["q"]), k=torch.empty_like(t["k"]))
    plan = E.CacheAppend(c["heads"], c["kv_heads"], c["dim"], page_size=c["page"], dtype=dtype, **turn)
    _ok(plan.prepare())
    return plan, dict(q=torch.empty_like(t["q"]), k=t["k"], v=t["v"])


def prepare(case, seed):
    t = _make(case, seed)
    plan, out = _plan(case, t) if own else (None, None)
    return dict(case=case, t=t, plan=plan, out=out)


def _ok(rc):
    if rc != 0:
        raise RuntimeError("rc=%d" % rc)


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    c, t = state["case"], state["t"]
    if not own:
        return PLAIN[c["op"]](c, t)
    plan, out = state["plan"], state["out"]
    if c["op"] == "rotary":
        _ok(plan.enqueue(out["q"], out["k"], t["q"], t["k"], t["positions"], rows=c["rows"]))
    elif c["op"] == "append":
        _ok(plan.enqueue(out["q"], out["k"], out["v"], t["q"], t["new_k"], t["new_v"], t["table"], t["lengths"], t["starts"], rows=t["rows"], seqs=c["seqs"]))
    else:
        _ok(plan.enqueue(out["out"], t["q"], t["k"], t["v"], t["table"], t["lengths"], t["starts"], rows=t["rows"], seqs=c["seqs"]))
    return out


# ------------------------------------------------------------------------------------------- plain forms
def _plain_turn(c, x, positions):
    """x: [rows, heads, dim] in 32 bits"""
    r = c["rotary"]
    step = BASE ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if c["scaling"] == "linear":
        step = step / FACTOR
    elif c["scaling"] == "by_parts":
        turns = ORIGINAL * step / (2.0 * math.pi)
        kept = ((turns - SLOW) / (FAST - SLOW)).clamp(0.0, 1.0)
        step = step * kept + step / FACTOR * (1.0 - kept)
    angle = positions.double()[:, None, None] * step
    size = MAGNITUDE if c["scaling"] == "by_parts" else 1.0
    cos, sin = (torch.cos(angle) * size).float(), (torch.sin(angle) * size).float()
    near = c["layout"] == "neighbours"
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if near else (x[..., :r // 2], x[..., r // 2:r])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), dim=-1).flatten(-2) if near else torch.cat((u, w), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _plain_rotary(c, t):
    return dict(q=_plain_turn(c, t["q"].float(), t["positions"]).to(t["q"].dtype), k=_plain_turn(c, t["k"].float(), t["positions"]).to(t["k"].dtype))


def _plain_append(c, t):
    at = t["lengths"].long()[t["seq"]] - t["new"][t["seq"]] + t["place"]
    page, offset = t["table"][t["seq"], at // c["page"]].long(), at % c["page"]
    t["k"][page, :, offset] = _plain_turn(c, t["new_k"].float(), at).to(t["k"].dtype)
    t["v"][page, :, offset] = t["new_v"]
    return dict(q=_plain_turn(c, t["q"].float(), at).to(t["q"].dtype), k=t["k"], v=t["v"])


def _plain_attention(c, t):
    kv, d, group = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    if t["table"] is None:
        k, v = t["k"].float().permute(0, 2, 1, 3), t["v"].float().permute(0, 2, 1, 3)          # [seqs, kv heads, keys, dim]
    else:
        table = t["table"].clamp(min=0).long()
        k = t["k"][table].float().permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, -1, d)
        v = t["v"][table].float().permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, -1, d)
    q = torch.zeros(c["seqs"], c["new"], kv, group, d, device="cuda")
    q[t["seq"], t["place"]] = t["q"].float().reshape(-1, kv, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, -1, d) * (1.0 / math.sqrt(d))           # rows: new token, head of the group
    s = (q @ k.transpose(2, 3)).reshape(c["seqs"], kv, c["new"], group, -1)
    seen = t["lengths"].long()[:, None].expand(-1, c["new"])
    if c["causal"]:
        seen = seen - t["new"][:, None] + 1 + torch.arange(c["new"], device="cuda")
    s = s.masked_fill(torch.arange(s.shape[-1], device="cuda") >= seen[:, None, :, None, None], -math.inf)
    s = torch.exp(s - s.max(dim=-1, keepdim=True).values)
    whole = s.sum(dim=-1)
    o = (s.reshape(c["seqs"], kv, -1, s.shape[-1]) @ v).reshape(c["seqs"], kv, c["new"], group, d) / whole[..., None]
    return dict(out=o.permute(0, 2, 1, 3, 4)[t["seq"], t["place"]].reshape(-1, c["heads"], d).to(t["q"].dtype))


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    e, h, kv, d = BYTES[c["dtype"]], c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "rotary":
        return {"bytes": c["rows"] * (2 * e * (h + kv) * d + 4), "flops": 3.0 * c["rows"] * (h + kv) * c["rotary"]}
    lengths, new = _lengths(c)
    rows = sum(new)
    if c["op"] == "append":
        return {"bytes": 2 * e * rows * (h + 2 * kv) * d + 4 * sum(-(-n // c["page"]) + 1 for n in new), "flops": 3.0 * rows * (h + kv) * c["rotary"]}
    seen = sum(n * m - (n * (n - 1) // 2 if c["causal"] else 0) for m, n in zip(lengths, new))      # pairs of a token and a key that it sees
    table = 4 * sum(-(-m // c["page"]) for m in lengths) if c["page"] else 0
    return {"bytes": 2 * e * (rows * h * d + sum(lengths) * kv * d) + table + 4 * c["seqs"], "flops": 4.0 * seen * h * d}


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_turn(c, x, positions):
    r, near, y = c["rotary"], c["layout"] == "neighbours", x.double().clone()
    for i in range(r // 2):
        w = math.exp(-2.0 * i / r * math.log(BASE))
        if c["scaling"] == "linear":
            w /= FACTOR
        if c["scaling"] == "by_parts":
            share = min(1.0, max(0.0, (ORIGINAL * w / (2.0 * math.pi) - SLOW) / (FAST - SLOW)))
            w = share * w + (1.0 - share) * w / FACTOR
        turn = torch.polar(torch.full_like(positions, MAGNITUDE if c["scaling"] == "by_parts" else 1.0, dtype=torch.float64), positions.double() * w)[:, None]
        m, n = (2 * i, 2 * i + 1) if near else (i, i + r // 2)
        z = torch.complex(x[:, :, m].double(), x[:, :, n].double()) * turn
        y[:, :, m], y[:, :, n] = z.real, z.imag
    return y


def exact(case, seed):
    c, t = case, _make(case, seed)
    if c["op"] == "rotary":
        return dict(q=_exact_turn(c, t["q"], t["positions"]), k=_exact_turn(c, t["k"], t["positions"]))
    lengths, new = _lengths(c)
    if c["op"] == "append":
        at = torch.cat([torch.arange(m - n, m, device="cuda") for m, n in zip(lengths, new)])
        turned, k, v = _exact_turn(c, t["new_k"], at), t["k"].double(), t["v"].double()
        row = 0
        for s, n in enumerate(new):
            places = at[row:row + n]
            pages = t["table"][s].long()[torch.div(places, c["page"], rounding_mode="floor")]
            k[pages, :, places.remainder(c["page"])] = turned[row:row + n]
            v[pages, :, places.remainder(c["page"])] = t["new_v"][row:row + n].double()
            row += n
        return dict(q=_exact_turn(c, t["q"], at), k=k, v=v)
    group, row, out = c["heads"] // c["kv_heads"], 0, torch.zeros_like(t["q"], dtype=torch.float64)
    for s, (m, n) in enumerate(zip(lengths, new)):
        for j in range(c["kv_heads"]):
            if t["table"] is None:
                k, v = t["k"][s, :m, j].double(), t["v"][s, :m, j].double()
            else:
                pages = t["table"][s, :-(-m // c["page"])].long()
                k, v = t["k"][pages, j].flatten(0, 1)[:m].double(), t["v"][pages, j].flatten(0, 1)[:m].double()
            q = t["q"][row:row + n, j * group:(j + 1) * group].double()
            z = torch.einsum("nhd,md->hnm", q, k) / math.sqrt(c["dim"])
            if c["causal"]:
                z.masked_fill_(torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1), -math.inf)
            out[row:row + n, j * group:(j + 1) * group] = torch.einsum("hnm,md->nhd", torch.softmax(z, dim=-1), v)
        row += n
    return dict(out=out)
