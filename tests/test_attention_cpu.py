"""The attention operators without a GPU: descriptions and calls are refused before a device is looked for, tensors that do not fit are refused in Python."""
import ctypes as C

import pytest
import torch

from test_op_tensors_cpu import Tensor, _Library, new
from test_ops_cpu import _refused

BF, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def test_struct_layouts(pkg):
    assert C.sizeof(pkg.ElbRotaryDesc) == 15 * 4 + 4 + 4 * 8
    assert C.sizeof(pkg.ElbAppendDesc) == 15 * 4 + 4 + 4 * 8 + 8 + 4 * 8
    assert C.sizeof(pkg.ElbAttentionDesc) == 8 * 4 + 5 * 8


INF, NAN = float("inf"), float("nan")
BAD_ROTARY = [(dict(heads=-1), 2, "heads"), (dict(heads=0, kv_heads=0), 2, "heads"), (dict(kv_heads=5000), 2, "heads"), (dict(head_dim=0), 2, "channels"), (dict(head_dim=2048), 2, "channels"),
              (dict(rotary_dim=33), 2, "turn"), (dict(rotary_dim=66), 2, "turn"), (dict(rotary_dim=-2), 2, "turn"), (dict(dtype=3), 1, "fp32"), (dict(layout=2), 2, "layout"),
              (dict(scaling=3), 2, "scaling"), (dict(base=0.0), 2, "base"), (dict(base=NAN), 2, "base"), (dict(magnitude=INF), 2, "magnitude"), (dict(scaling=1, factor=0.0), 2, "factor"),
              (dict(scaling=2, factor=INF), 2, "factor"), (dict(scaling=2, factor=2.0, slow=4.0, fast=4.0), 2, "slow"), (dict(scaling=2, factor=2.0, original=0), 2, "original"),
              (dict(ld_q=255), 2, "apart"), (dict(ld_k=-1), 2, "apart"), (dict(ld_q_out=1), 2, "apart")]


@pytest.mark.parametrize("kw,code,word", BAD_ROTARY + [(dict(rotary_dim=0), 2, "turn"), (dict(ld_k_out=127), 2, "apart")], ids=str)
def test_rotary_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.Rotary(**{**dict(heads=4, kv_heads=2, head_dim=64), **kw}), code, word)


@pytest.mark.parametrize("kw,code,word", BAD_ROTARY + [(dict(kv_heads=0), 2, "cache"), (dict(page_size=0), 2, "pages"), (dict(page_size=1 << 21), 2, "pages"), (dict(ld_v=100), 2, "apart"),
                                                       (dict(ld_token=63), 2, "overlap"), (dict(ld_head=1000), 2, "overlap"), (dict(ld_page=2000), 2, "overlap"), (dict(ld_head=-64), 2, "strides"),
                                                       (dict(ld_head=64, ld_token=127), 2, "overlap"), (dict(ld_page=1 << 41), 2, "strides")], ids=str)
def test_append_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.CacheAppend(**{**dict(heads=4, kv_heads=2, head_dim=64, page_size=16), **kw}), code, word)


@pytest.mark.parametrize("kw,code,word", [(dict(heads=0), 2, "heads"), (dict(kv_heads=0), 2, "heads"), (dict(heads=5), 2, "multiple"), (dict(heads=8192), 2, "4096"), (dict(head_dim=0), 2, "channels"),
                                          (dict(head_dim=257), 1, "256"), (dict(dtype=1), 1, "bf16"), (dict(dtype=3), 1, "bf16"), (dict(page_size=-1), 2, "pages"), (dict(scale=INF), 2, "scale"),
                                          (dict(ld_input=255), 2, "apart"), (dict(ld_output=-4), 2, "apart"), (dict(ld_head=63), 2, "overlap"), (dict(page_size=0, ld_head=63), 2, "apart"),
                                          (dict(page_size=0, ld_token=63), 2, "apart"), (dict(page_size=0, ld_page=-1), 2, "apart")], ids=str)
def test_attention_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.Attention(**{**dict(heads=4, kv_heads=2, head_dim=64, page_size=16), **kw}), code, word)


def test_no_cpu_fallback_and_null_plans(pkg):
    lib = pkg.lib
    for create in (lib.elb_rotary_create, lib.elb_append_create, lib.elb_attention_create):
        assert create(None, None) == pkg.ELB_GENERAL_ERROR
    assert lib.elb_rotary_prepare(None, None) == lib.elb_append_prepare(None, None) == pkg.ELB_GENERAL_ERROR
    assert lib.elb_attention_enqueue(*[None] * 8, 1, 1, 1, 1, None) == pkg.ELB_GENERAL_ERROR
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for make in (lambda: pkg.Rotary(4, 2, 64), lambda: pkg.CacheAppend(4, 2, 64, 16), lambda: pkg.Attention(4, 2, 64)):
        _refused(pkg, make, 2, "CUDA")


# ------------------------------------------------------------------------------------------- what enqueue takes
@pytest.fixture()
def E(pkg, monkeypatch):
    monkeypatch.setattr(pkg, "lib", _Library())
    return pkg


def _ints(*shape):
    return new(*shape, dtype=I32)


def _plans(E):
    """name -> (plan, good tensors of a call of 6 rows and 2 sequences, its numbers)"""
    pages = lambda: new(9, 2, 16, 64)                  # noqa: E731
    return {
        "rotary": (E.Rotary(4, 2, 64), dict(q_out=new(6, 4, 64), k_out=new(6, 2, 64), q=new(6, 4, 64), k=new(6, 128), positions=_ints(6)), dict(rows=6)),
        "append": (E.CacheAppend(4, 2, 64, 16), dict(q_out=new(6, 4, 64), k_cache=pages(), v_cache=pages(), q=new(6, 4, 64), k=new(6, 2, 64), v=new(6, 2, 64), table=_ints(2, 5),
                                                     lengths=_ints(2), starts=_ints(3)), dict(rows=6, seqs=2)),
        "attention": (E.Attention(4, 2, 64, page_size=16), dict(output=new(6, 4, 64), input=new(6, 4, 64), k=pages(), v=pages(), table=_ints(2, 5), lengths=_ints(2), starts=_ints(3)),
                      dict(rows=6, seqs=2)),
        "dense": (E.Attention(4, 2, 64), dict(output=new(6, 4, 64), input=new(6, 4, 64), k=new(2, 10, 2, 64), v=new(2, 10, 2, 64), lengths=_ints(2), starts=_ints(3)), dict(rows=6, seqs=2)),
    }


@pytest.mark.parametrize("kind", ["rotary", "append", "attention", "dense"])
def test_tensors_that_do_not_fit_are_refused(E, kind):
    plan, good, numbers = _plans(E)[kind]
    assert plan.enqueue(**good, **numbers) == 0 and len(E.lib.calls) == 1
    sent = [a for a in E.lib.calls[0][1:] if isinstance(a, int) and a > 64]
    assert sent == [t.data_ptr() for t in good.values()]
    for name, x in good.items():
        t = x.t
        wide = torch.empty(t.shape[0], 2 * t.shape[-1] if len(t.shape) > 1 else 2, dtype=t.dtype)
        bad = [t.to(torch.int64), t.to(F16 if t.dtype != F16 else BF), wide[:, ::2] if len(t.shape) > 1 else wide[:, 0], torch.empty((), dtype=t.dtype)]
        if name not in ("k_cache", "v_cache") and not (kind == "attention" and name in ("k", "v")):
            bad += [t[:-1], t[:-1].clone()]                        # (fewer pages are another pool)
        if len(t.shape) == 4:
            bad += [t[:, :, :-1], t[..., :-1], t.flatten(0, 1), torch.empty(*t.shape[:3], t.shape[3] + 8, dtype=t.dtype)[..., :t.shape[3]]]
        for b in bad:
            with pytest.raises(ValueError, match=name):
                plan.enqueue(**{**good, name: Tensor(b)}, **numbers)
        for elsewhere in (t, Tensor(t, device=1)):
            with pytest.raises(ValueError, match="device 0"):
                plan.enqueue(**{**good, name: elsewhere}, **numbers)
    assert len(E.lib.calls) == 1


def test_addresses_want_their_sizes(E):
    plan, good, numbers = _plans(E)["attention"]
    with pytest.raises(ValueError, match="pages"):
        plan.enqueue(**{**good, "k": 4096, "v": 4096}, **numbers)
    with pytest.raises(ValueError, match="width"):
        plan.enqueue(**{**good, "table": 4096}, **numbers)
    assert plan.enqueue(**{**good, "k": 4096, "v": 8192, "table": 4096}, **numbers, pages=9, width=5) == 0
    assert E.lib.calls[-1][-5:] == (6, 2, 9, 5, None)
    with pytest.raises(ValueError, match="10 pages"):
        plan.enqueue(**good, **numbers, pages=10)
    with pytest.raises(ValueError, match="table"):
        plan.enqueue(**good, **numbers, width=4)
    with pytest.raises(ValueError, match="v_cache"):              # a pool of values with fewer pages than that of keys
        a, g, n = _plans(E)["append"]
        a.enqueue(**{**g, "v_cache": new(8, 2, 16, 64)}, **n)
    plan, good, numbers = _plans(E)["dense"]
    with pytest.raises(ValueError, match="width"):
        plan.enqueue(**{**good, "k": 4096}, **numbers)
    with pytest.raises(ValueError, match="table"):
        plan.enqueue(**good, table=_ints(2, 5), **numbers)
    assert plan.enqueue(**good, **numbers) == 0 and E.lib.calls[-1][-5:] == (6, 2, 0, 10, None)


def test_orders_and_strides_of_keys(E):
    """Tokens in front of heads, heads in front of tokens, channels further apart; sizes of one have no stride."""
    tokens = E.Attention(4, 2, 64, page_size=16, ld_head=64, ld_token=128, ld_page=2048)
    base = _plans(E)["attention"][1]
    good = {**base, "k": new(9, 16, 2, 64), "v": new(9, 16, 2, 64)}
    assert tokens.enqueue(**good, rows=6, seqs=2) == 0
    assert tokens.enqueue(**{**good, "k": Tensor(torch.empty(9, 16, 2, 64, dtype=BF).permute(0, 2, 1, 3))}, rows=6, seqs=2) == 0
    with pytest.raises(ValueError, match="k:"):
        tokens.enqueue(**base, rows=6, seqs=2)
    fused = E.Attention(4, 2, 64, ld_token=256)                  # keys and values of one projection, side by side
    both = torch.empty(2, 10, 4, 64, dtype=BF)
    dense = {**_plans(E)["dense"][1], "k": Tensor(both[:, :, :2]), "v": Tensor(both[:, :, 2:])}
    assert fused.enqueue(**dense, rows=6, seqs=2) == 0
    with pytest.raises(ValueError, match="k:"):
        _plans(E)["dense"][0].enqueue(**dense, rows=6, seqs=2)
    one = E.Attention(4, 1, 64)
    assert one.enqueue(new(6, 4, 64), new(6, 4, 64), new(1, 10, 1, 64), new(1, 10, 1, 64), rows=6, seqs=1) == 0
