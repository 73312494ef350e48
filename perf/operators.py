"""Performance cases of the transformer operators: the feed-forward half of a block, dense or routed to experts, through the
public entry points of the package (``Linear``, ``BlockNorm``, ``Route``, ``Experts``).

A case is a dict of plain values.  ``op`` names the operator:

  linear    y = r + scale * act(x w^T + b), or act(gate) * up where ``gated``; 16-bit operands
  norm      s = r + scale * gate * post(x);  y = pre(s); both are returned
  route     scores of the logits, a bias for balance, groups, the top_k experts of a row and their weights
  experts   y[t] = sum_j weight[t][j] * w_out[e] act(w_in[e] x[t]), e = id[t][j]

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits, rounded once at the end.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _linear(rows, ic, oc, dtype="bf16", act="none", gated=False, bias=False, residual=False, scale=1.0):
    return dict(op="linear", rows=rows, ic=ic, oc=oc, dtype=dtype, act=act, gated=gated, bias=bias, residual=residual, scale=scale)


def _norm(rows, channels, dtype="bf16", residual="bf16", post="none", pre="rms", gate_rows=0, scale=1.0):
    """``residual``: the type of the residual stream; ``gate_rows``: consecutive rows that share a row of the gate, 0 for none."""
    return dict(op="norm", rows=rows, channels=channels, dtype=dtype, residual=residual, post=post, pre=pre, gate_rows=gate_rows, scale=scale)


def _route(rows, experts, top_k, dtype="f32", score="softmax", bias=False, groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0):
    return dict(op="route", rows=rows, experts=experts, top_k=top_k, dtype=dtype, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_best=group_best, renormalise=renormalise, scale=scale)


def _experts(rows, experts, top_k, ic, mid, dtype="bf16", act="silu", gated=True):
    return dict(op="experts", rows=rows, experts=experts, top_k=top_k, ic=ic, mid=mid, dtype=dtype, act=act, gated=gated)


def listed():
    return [
        # the projection behind a block while one sequence is answered token by token: the weights are read once, latency counts
        dict(_linear(1, 4096, 4096, residual=True), name="linear_token"),
        # the gated first product of a feed-forward layer for a batch of sequences, one token each
        dict(_linear(24, 4096, 8192, "f16", "silu", gated=True), name="linear_batch_gated"),
        # an encoder layer of odd sizes: rows of 2006 and 4042 bytes, which no 16-byte access fits
        dict(_linear(333, 1003, 2021, "f16", "gelu", bias=True, residual=True), name="linear_ragged"),
        # the gated first product over a long prompt: the largest
        dict(_linear(8192, 4096, 8192, "bf16", "silu", gated=True), name="linear_prompt_gated"),
        # the norm between two blocks for one token
        dict(_norm(1, 4096), name="norm_token"),
        # norms on both sides of a block over a long prompt, the residual stream kept in 32 bits
        dict(_norm(16384, 4096, "bf16", "f32", post="rms", pre="rms", scale=0.5), name="norm_both_prompt"),
        # layer norm with a gate for each sequence of a batch, odd width
        dict(_norm(2500, 1155, "f16", "f16", post="layer", pre="layer", gate_rows=500), name="norm_gated_ragged"),
        # a few tokens to two of 64 experts
        dict(_route(5, 64, 2), name="route_tokens"),
        # a long prompt to eight of 256 experts in four of eight groups, with a bias for balance
        dict(_route(16384, 256, 8, score="sigmoid", bias=True, groups=8, top_groups=4, group_best=2, scale=2.5), name="route_groups_prompt"),
        # one token through its eight experts: their weights are read once
        dict(_experts(1, 64, 8, 2048, 1024), name="experts_token"),
        # a batch through experts of odd sizes without a gate
        dict(_experts(200, 16, 2, 1000, 721, "f16", "gelu", gated=False), name="experts_batch_ragged"),
        # a long prompt through eight of 64 experts
        dict(_experts(4096, 64, 8, 2048, 1024), name="experts_prompt"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _rows(rng, hi):
    return max(1, min(hi, int(_log(rng, 1, hi + 1))))


def _width(rng, lo, hi):
    """Three in four as networks have them (a power of two, or five or seven quarters of one), the others odd."""
    v = _log(rng, lo, hi)
    if rng.random() < 0.25:
        return int(v) | 1
    p = 2 ** int(math.log2(v))
    return min(hi, rng.choice([p, p, p * 5 // 4, p * 7 // 4]))


def _draw_once(rng):
    op = rng.choice(["linear", "linear", "norm", "route", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "linear":
        return _linear(_rows(rng, 8192), _width(rng, 64, 8192), _width(rng, 64, 16384), dtype,
                       rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), rng.random() < 0.4, rng.random() < 0.5,
                       rng.random() < 0.5, rng.choice([1.0, 1.0, 0.5]))
    if op == "norm":
        rows = _rows(rng, 16384)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return _norm(rows, _width(rng, 64, 8192), dtype, rng.choice([dtype, "f32"]), rng.choice(["none", "rms", "layer"]),
                     rng.choice(["rms", "rms", "layer"]), rng.choice([0, 0, 1, rows, (rows + 3) // 4]), rng.choice([1.0, 1.0, 0.5]))
    if op == "route":
        experts = rng.choice([4, 8, 16, 20, 60, 64, 128, 160, 256, 384])
        k = rng.randint(1, min(8, experts))
        if rng.random() < 0.5:
            return _route(_rows(rng, 16384), experts, k, rng.choice(["f32", "f32", "bf16"]), renormalise=rng.random() < 0.5)
        groups = rng.choice([1, 4]) if experts >= 16 else 1
        return _route(_rows(rng, 16384), experts, k, "f32", "sigmoid", True, groups, max(1, groups // 2) if experts // 2 >= 8 else groups, 2, scale=2.5)
    experts = rng.choice([4, 8, 16, 32, 64, 100, 128])
    return _experts(_rows(rng, 4096), experts, rng.randint(1, min(8, experts)), _width(rng, 256, 2048), _width(rng, 128, 2048),
                    dtype, rng.choice(["silu", "gelu", "relu"]), rng.random() < 0.75)


def draw(rng):
    top = [work(c) for c in listed()]
    most_bytes, most_flops = max(w["bytes"] for w in top), max(w["flops"] for w in top)
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return c


# ------------------------------------------------------------------------------------------- inputs
def _make(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    c, dt = case, DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if c["op"] == "linear":
        wide = c["oc"] * (2 if c["gated"] else 1)
        return dict(x=normal(c["rows"], c["ic"]), w=normal(wide, c["ic"], scale=1.5 / math.sqrt(c["ic"])),
                    b=normal(wide, scale=0.5, dtype=torch.float32) if c["bias"] else None,
                    r=normal(c["rows"], c["oc"], scale=2.0) if c["residual"] else None)
    if c["op"] == "norm":
        n = c["channels"]
        gates = -(-c["rows"] // c["gate_rows"]) if c["gate_rows"] else 0

        def weights(kind):
            w = (1.0 + normal(n, scale=0.2, dtype=torch.float32)) if kind != "none" else None
            return w, normal(n, scale=0.2, dtype=torch.float32) if kind == "layer" else None

        (pw, pb), (qw, qb) = weights(c["post"]), weights(c["pre"])
        return dict(x=normal(c["rows"], n, scale=1.5) + 0.25, r=normal(c["rows"], n, scale=3.0, dtype=DTYPES[c["residual"]]),
                    g=normal(gates, n) if gates else None, post_w=pw, post_b=pb, pre_w=qw, pre_b=qb)
    if c["op"] == "route":
        return dict(logits=normal(c["rows"], c["experts"], scale=1.5), b=normal(c["experts"], scale=0.1, dtype=torch.float32) if c["bias"] else None)
    # as a router leaves them: some experts are asked for several times as often as others
    liking = normal(c["experts"], scale=0.7, dtype=torch.float32)
    best, ids = torch.topk(normal(c["rows"], c["experts"], dtype=torch.float32) + liking, c["top_k"])
    wide = c["mid"] * (2 if c["gated"] else 1)
    return dict(x=normal(c["rows"], c["ic"]), ids=ids.to(torch.int32), weights=torch.softmax(best, dim=1),
                w_in=normal(c["experts"], wide, c["ic"], scale=1.5 / math.sqrt(c["ic"])),
                w_out=normal(c["experts"], c["ic"], c["mid"], scale=1.5 / math.sqrt(c["mid"])))


def _plan(c, t):
    """The plan that a user's program makes once for a layer, and the tensors that it writes."""
    E = importlib.import_module("deep-learning-math-kernel-research_b200")
    kinds = {"bf16": E.bf16, "f16": E.f16, "f32": E.f32}
    acts = {"none": E.ACT_NONE, "relu": E.ACT_RELU, "gelu": E.ACT_GELU, "gelu_tanh": E.ACT_GELU_TANH, "silu": E.ACT_SILU}
    norms = {"none": E.NORM_NONE, "rms": E.NORM_RMS, "layer": E.NORM_LAYER}
    dt, rows = DTYPES[c["dtype"]], c["rows"]
    if c["op"] == "linear":
        plan = E.Linear(c["ic"], c["oc"], dtype=kinds[c["dtype"]], activation=acts[c["act"]], gated=c["gated"], with_bias=c["bias"],
                        with_residual=c["residual"], scale=c["scale"])
        _ok(plan.prepare(t["w"], t["b"]))
        return plan, dict(y=torch.empty(rows, c["oc"], dtype=dt, device="cuda"))
    if c["op"] == "norm":
        plan = E.BlockNorm(c["channels"], dtype=kinds[c["dtype"]], residual_dtype=kinds[c["residual"]], post=norms[c["post"]],
                           pre=norms[c["pre"]], gate_rows=c["gate_rows"], scale=c["scale"])
        _ok(plan.prepare(t["post_w"], t["post_b"], t["pre_w"], t["pre_b"]))
        return plan, dict(y=torch.empty_like(t["x"]), s=torch.empty_like(t["r"]))
    if c["op"] == "route":
        plan = E.Route(c["experts"], c["top_k"], dtype=kinds[c["dtype"]], score=E.SCORE_SIGMOID if c["score"] == "sigmoid" else E.SCORE_SOFTMAX,
                       with_bias=c["bias"], groups=c["groups"], top_groups=c["top_groups"], group_best=c["group_best"],
                       renormalise=c["renormalise"], scale=c["scale"])
        _ok(plan.prepare(t["b"]))
        return plan, dict(ids=torch.empty(rows, c["top_k"], dtype=torch.int32, device="cuda"),
                          weights=torch.empty(rows, c["top_k"], device="cuda"))
    plan = E.Experts(c["experts"], c["top_k"], c["ic"], c["mid"], max_rows=rows, dtype=kinds[c["dtype"]], activation=acts[c["act"]], gated=c["gated"])
    _ok(plan.prepare(t["w_in"], t["w_out"]))
    return plan, dict(y=torch.empty(rows, c["ic"], dtype=dt, device="cuda"))


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
    if c["op"] == "linear":
        _ok(plan.enqueue(out["y"], t["x"], t["r"], rows=c["rows"]))
    elif c["op"] == "norm":
        _ok(plan.enqueue(out["y"], out["s"], t["x"], t["r"], t["g"], rows=c["rows"]))
    elif c["op"] == "route":
        _ok(plan.enqueue(out["ids"], out["weights"], t["logits"], rows=c["rows"]))
    else:
        _ok(plan.enqueue(out["y"], t["x"], t["ids"], t["weights"], rows=c["rows"]))
    return out


# ------------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _activated(z, act, gated):
    if not gated:
        return _act(z, act)
    half = z.shape[-1] // 2
    return _act(z[..., :half], act) * z[..., half:]


def _plain_linear(c, t):
    z = t["x"].float() @ t["w"].float().t()
    if t["b"] is not None:
        z = z + t["b"]
    z = _activated(z, c["act"], c["gated"])
    if c["scale"] != 1.0:
        z = z * c["scale"]
    if t["r"] is not None:
        z = z + t["r"].float()
    return dict(y=z.to(t["x"].dtype))


def _plain_normed(v, kind, w, b):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * w
    return v + b if b is not None else v


def _plain_norm(c, t):
    v = _plain_normed(t["x"].float(), c["post"], t["post_w"], t["post_b"])
    if t["g"] is not None:
        v = v * t["g"].float()[torch.arange(c["rows"], device="cuda") // c["gate_rows"]]
    s = t["r"].float() + c["scale"] * v
    y = _plain_normed(s, c["pre"], t["pre_w"], t["pre_b"])
    return dict(y=y.to(t["x"].dtype), s=s.to(t["r"].dtype))


def _plain_route(c, t):
    z = t["logits"].float()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-z))
        whole = None
    else:
        score = torch.exp(z - z.max(dim=1, keepdim=True).values)   # the order of the softmax is that of its numerators
        whole = score.sum(dim=1, keepdim=True)
    choice = score + t["b"] if t["b"] is not None else score
    if c["groups"] > 1:
        by = choice.reshape(c["rows"], c["groups"], -1)
        best = by.sort(dim=2, descending=True, stable=True).values[:, :, :c["group_best"]].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(open_[:, :, None], by, torch.full_like(by, -math.inf)).reshape(c["rows"], -1)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = score.gather(1, ids)
    if c["renormalise"]:
        w = w / w.sum(dim=1, keepdim=True)
    elif whole is not None:
        w = w / whole
    return dict(ids=ids.to(torch.int32), weights=w * c["scale"])


def _plain_experts(c, t):
    rows, k = c["rows"], c["top_k"]
    ids = t["ids"].long().reshape(-1)
    x, share = t["x"].float(), t["weights"].reshape(-1, 1)
    if rows * k <= c["experts"]:                             # few slots: a product with each slot's own weights
        h = (t["w_in"][ids].float() @ x.repeat_interleave(k, dim=0)[:, :, None])[:, :, 0]
        h = _activated(h, c["act"], c["gated"])
        o = (t["w_out"][ids].float() @ h[:, :, None])[:, :, 0]
        return dict(y=(o * share).reshape(rows, k, -1).sum(dim=1).to(t["x"].dtype))
    order = ids.argsort(stable=True)                         # the slots of an expert side by side, in a bucket for each
    count = torch.zeros(c["experts"], dtype=torch.long, device="cuda").index_add_(0, ids, torch.ones_like(ids))
    at, by = torch.arange(rows * k, device="cuda") - (count.cumsum(0) - count)[ids[order]], ids[order]
    bucket = torch.zeros(c["experts"], int(count.max()), c["ic"], device="cuda")
    bucket[by, at] = x[order // k]
    h = _activated(bucket @ t["w_in"].float().transpose(1, 2), c["act"], c["gated"])
    o = h @ t["w_out"].float().transpose(1, 2)
    slots = torch.empty(rows * k, c["ic"], device="cuda")
    slots[order] = o[by, at]
    return dict(y=(slots * share).reshape(rows, k, -1).sum(dim=1).to(t["x"].dtype))


PLAIN = {"linear": _plain_linear, "norm": _plain_norm, "route": _plain_route, "experts": _plain_experts}


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "linear":
        wide, e = c["oc"] * (2 if c["gated"] else 1), BYTES[c["dtype"]]
        return {"bytes": e * (wide * c["ic"] + c["rows"] * (c["ic"] + c["oc"] * (2 if c["residual"] else 1))) + (4 * wide if c["bias"] else 0),
                "flops": 2.0 * c["rows"] * c["ic"] * wide}
    if c["op"] == "norm":
        n, e, f = c["rows"] * c["channels"], BYTES[c["dtype"]], BYTES[c["residual"]]
        gates = -(-c["rows"] // c["gate_rows"]) * c["channels"] if c["gate_rows"] else 0
        return {"bytes": n * (2 * e + 2 * f) + gates * e + 8 * c["channels"], "flops": 12.0 * n}
    if c["op"] == "route":
        n = c["rows"] * c["experts"]
        return {"bytes": n * BYTES[c["dtype"]] + 8 * c["rows"] * c["top_k"], "flops": 8.0 * n}
    wide, e, slots = c["mid"] * (2 if c["gated"] else 1), BYTES[c["dtype"]], c["rows"] * c["top_k"]
    hit = c["experts"] * (1.0 - (1.0 - c["top_k"] / c["experts"]) ** c["rows"])
    return {"bytes": e * (hit * c["ic"] * (wide + c["mid"]) + 2 * c["rows"] * c["ic"]) + 8 * slots,
            "flops": 2.0 * slots * c["ic"] * (wide + c["mid"])}


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_f(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def _exact_norm(v, kind, w, b):
    if kind == "none":
        return v
    centre = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    power = ((v - centre) ** 2).mean(1, keepdim=True)
    return (v - centre) * torch.rsqrt(power + 1e-6) * w.double() + (b.double() if b is not None else 0.0)


def exact(case, seed):
    c, t = case, _make(case, seed)
    if c["op"] == "linear":
        w, b = t["w"].chunk(2) if c["gated"] else (t["w"],), None
        if t["b"] is not None:
            b = t["b"].chunk(2) if c["gated"] else (t["b"],)
        parts = [t["x"].double() @ p.double().T + (b[i].double() if b else 0.0) for i, p in enumerate(w)]
        y = _exact_f(parts[0], c["act"]) * (parts[1] if c["gated"] else 1.0) * c["scale"]
        return dict(y=y + (t["r"].double() if t["r"] is not None else 0.0))
    if c["op"] == "norm":
        v = _exact_norm(t["x"].double(), c["post"], t["post_w"], t["post_b"]) * c["scale"]
        if t["g"] is not None:
            v = v * t["g"].double().repeat_interleave(c["gate_rows"], dim=0)[:c["rows"]]
        s = t["r"].double() + v
        return dict(y=_exact_norm(s, c["pre"], t["pre_w"], t["pre_b"]), s=s)
    if c["op"] == "route":
        z = t["logits"].double()
        score = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.softmax(z, dim=1)
        choice = score + t["b"].double() if t["b"] is not None else score.clone()
        if c["groups"] > 1:
            by = choice.unflatten(1, (c["groups"], -1))
            best = by.topk(c["group_best"], dim=2).values.sum(2)
            shut = best < best.topk(c["top_groups"], dim=1).values[:, -1:]
            choice = by.masked_fill(shut[:, :, None], -math.inf).flatten(1)
        w = score.gather(1, choice.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]])
        return dict(ids=None, weights=w * c["scale"] / (w.sum(1, keepdim=True) if c["renormalise"] else 1.0))
    y = torch.zeros(c["rows"], c["ic"], dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        token, place = torch.nonzero(t["ids"] == e, as_tuple=True)
        h = t["x"][token].double() @ t["w_in"][e].double().T
        h = _exact_f(h[:, :c["mid"]], c["act"]) * h[:, c["mid"]:] if c["gated"] else _exact_f(h, c["act"])
        y.index_add_(0, token, (h @ t["w_out"][e].double().T) * t["weights"][token, place].double()[:, None])
    return dict(y=y)
