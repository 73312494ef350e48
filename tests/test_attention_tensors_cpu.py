"""Tensors of the attention operators' calls that have to be taken, whatever their number of rows, without a GPU."""
import pytest
import torch

from test_op_tensors_cpu import Tensor, _Library, new

BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture()
def E(pkg, monkeypatch):
    monkeypatch.setattr(pkg, "lib", _Library())
    return pkg


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("heads", [1, 4])
def test_heads_in_rows_that_lie_apart(E, rows, heads):
    """q, k and v as [rows, heads, channels] in the rows of one product: one row of them is a dense tensor too."""
    wide, n = (heads + 2) * 64, heads * 64
    h = torch.empty(rows, wide, dtype=BF)
    q, k, v = (Tensor(t.unflatten(1, (-1, 64))) for t in (h[:, :n], h[:, n:n + 64], h[:, n + 64:]))
    ints = lambda *shape: new(*shape, dtype=I32)                                                                         # noqa: E731
    turn = E.Rotary(heads, 1, 64, ld_q=wide, ld_k=wide, ld_q_out=wide, ld_k_out=wide)
    assert turn.enqueue(q, k, q, k, ints(rows), rows=rows) == 0
    append, pages = E.CacheAppend(heads, 1, 64, 16, ld_q=wide, ld_k=wide, ld_v=wide), new(9, 1, 16, 64)
    assert append.enqueue(new(rows, heads, 64), pages, pages, q, k, v, ints(rows, 5), ints(rows), rows=rows, seqs=rows) == 0
    attention = E.Attention(heads, 1, 64, page_size=16, ld_input=wide, ld_output=wide)
    assert attention.enqueue(q, q, pages, pages, ints(rows, 5), ints(rows), rows=rows, seqs=rows) == 0
    assert len(E.lib.calls) == 3
    short = Tensor(torch.empty(rows, heads, 56, dtype=BF))
    for bad in (short, Tensor(q.t.to(torch.float16))):
        with pytest.raises(ValueError, match="input"):
            attention.enqueue(q, bad, pages, pages, ints(rows, 5), ints(rows), rows=rows, seqs=rows)
    if rows > 1:                                             # rows elsewhere than the plan says
        with pytest.raises(ValueError, match="input"):
            attention.enqueue(q, new(rows, heads, 64), pages, pages, ints(rows, 5), ints(rows), rows=rows, seqs=rows)
    with pytest.raises(ValueError, match="output"):
        attention.enqueue(q, q, pages, pages, ints(rows + 1, 5), ints(rows + 1), rows=rows + 1, seqs=rows + 1)
