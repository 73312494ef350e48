"""The attention operators together, as a program uses them (examples/encoder_decoder.py): an encoder layer, prompts, then answers token by token from the cache."""
import importlib.util
from pathlib import Path

import pytest

from oputil import E, UNIT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("encoder_decoder", Path(__file__).resolve().parent.parent / "examples" / "encoder_decoder.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [E.bf16, E.f16])
@pytest.mark.parametrize("seqs,heads,kv_heads,dim,steps,graph", [(1, 4, 4, 64, 3, False), (6, 8, 2, 64, 20, True), (5, 6, 2, 80, 9, False), (33, 4, 1, 128, 4, True)])
def test_layers(example, dtype, seqs, heads, kv_heads, dim, steps, graph):
    rel, _, layers = example.run(seqs, heads, kv_heads, dim, steps, dtype, graph)
    # A result has gone through some twelve tensors of 16 bits one after the other, each off by at most a unit and by far less of it on the average; sums of
    # hundreds of such terms do not add up their errors.  A wrong place, page, position or length moves results by their own size.
    assert max(rel) <= 12 * UNIT[dtype], rel
    assert all(p.launch_count() > 0 for p in layers.plans())
