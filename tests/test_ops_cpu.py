"""The transformer operators without a GPU: descriptions are refused before a device is looked for, and nothing computes."""
import ctypes as C

import pytest


def _refused(pkg, make, code, word):
    with pytest.raises(RuntimeError) as err:
        make()
    assert f"rc={code}" in str(err.value) and word in str(err.value)


def test_struct_layouts(pkg):
    assert C.sizeof(pkg.ElbLinearDesc) == 12 * 4 + 3 * 8
    assert C.sizeof(pkg.ElbNormDesc) == 13 * 4 + 4 + 5 * 8
    assert C.sizeof(pkg.ElbRouteDesc) == 11 * 4 + 4 + 8
    assert C.sizeof(pkg.ElbExpertsDesc) == 8 * 4 + 3 * 8


BAD_LINEAR = [(dict(ic=0), 2, "channels"), (dict(oc=-1), 2, "channels"), (dict(ic=1 << 21), 2, "channels"), (dict(dtype=1), 1, "bf16"), (dict(dtype=3), 1, "bf16"),
              (dict(out_dtype=2), 1, "fp32"), (dict(bias_dtype=2), 1, "bias"), (dict(weights_format=7), 1, "hwio"), (dict(activation=5), 2, "activation"),
              (dict(scale=float("inf")), 2, "scale"), (dict(ld_input=63), 2, "apart"), (dict(ld_output=-1), 2, "apart"), (dict(ld_residual=127), 2, "apart")]


@pytest.mark.parametrize("kw,code,word", BAD_LINEAR, ids=str)
def test_linear_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.Linear(**{**dict(ic=64, oc=128), **kw}), code, word)


BAD_NORM = [(dict(channels=0), 2, "channels"), (dict(channels=32769), 1, "32768"), (dict(dtype=3), 1, "fp32"), (dict(residual_dtype=2), 1, "residual"), (dict(weights_dtype=2), 1, "weights"),
            (dict(post=3), 2, "kind"), (dict(pre=-1), 2, "kind"), (dict(pre_eps=-1.0), 2, "eps"), (dict(post_eps=float("nan")), 2, "eps"), (dict(scale=float("nan")), 2, "scale"),
            (dict(gate_rows=-1), 2, "gate_rows"), (dict(ld_gate=3), 2, "apart")]


@pytest.mark.parametrize("kw,code,word", BAD_NORM, ids=str)
def test_norm_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.BlockNorm(**{**dict(channels=64), **kw}), code, word)


BAD_ROUTE = [(dict(experts=0), 2, "experts"), (dict(top_k=0), 2, "experts"), (dict(top_k=65), 2, "experts"), (dict(experts=1025), 1, "1024"), (dict(top_k=33), 1, "32"), (dict(dtype=3), 1, "logits"),
             (dict(score=2), 2, "score"), (dict(groups=5), 2, "groups"), (dict(groups=8, top_groups=9), 2, "groups"), (dict(groups=64, top_groups=8), 1, "groups"),
             (dict(groups=8, top_groups=2, group_best=3), 1, "best"), (dict(groups=8, top_groups=1, top_k=9), 2, "groups"), (dict(scale=float("inf")), 2, "scale"), (dict(ld_logits=5), 2, "apart")]


@pytest.mark.parametrize("kw,code,word", BAD_ROUTE, ids=str)
def test_route_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.Route(**{**dict(experts=64, top_k=4), **kw}), code, word)


BAD_EXPERTS = [(dict(experts=0), 2, "experts"), (dict(experts=2000), 1, "1024"), (dict(top_k=33), 1, "32"), (dict(ic=0), 2, "channels"), (dict(mid=0), 2, "channels"), (dict(dtype=1), 1, "bf16"),
               (dict(activation=-1), 2, "activation"), (dict(max_rows=0), 2, "max_rows"), (dict(max_rows=1 << 31), 2, "max_rows"), (dict(max_rows=1 << 62, top_k=4), 2, "max_rows"), (dict(ld_input=1), 2, "apart")]


@pytest.mark.parametrize("kw,code,word", BAD_EXPERTS, ids=str)
def test_experts_refusals(pkg, kw, code, word):
    _refused(pkg, lambda: pkg.Experts(**{**dict(experts=8, top_k=2, ic=64, mid=64, max_rows=16), **kw}), code, word)


def test_no_cpu_fallback(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for make in (lambda: pkg.Linear(64, 64), lambda: pkg.BlockNorm(64), lambda: pkg.Route(8, 2), lambda: pkg.Experts(8, 2, 64, 64, 4)):
        _refused(pkg, make, 2, "CUDA")


def test_null_plans(pkg):
    assert pkg.lib.elb_linear_enqueue(None, None, None, None, 1, None) == pkg.ELB_GENERAL_ERROR
    assert pkg.lib.elb_norm_prepare(None, None, None, None, None) == pkg.ELB_GENERAL_ERROR
    assert pkg.lib.elb_op_device_status(None) == -1 and pkg.lib.elb_op_launch_count(None) == 0
    pkg.lib.elb_op_destroy(None)
    for create in (pkg.lib.elb_linear_create, pkg.lib.elb_norm_create, pkg.lib.elb_route_create, pkg.lib.elb_experts_create):
        assert create(None, None) == pkg.ELB_GENERAL_ERROR
