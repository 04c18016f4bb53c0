"""fa_cache_append at the ends of what its arguments may hold."""
import pytest
import torch

from test_cache_gpu import Case, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


@pytest.mark.parametrize("kind", ["16", "u4"])
def test_numbers_of_new_tokens_of_any_size(op, dev, kind):
    """num_new below zero stores nothing, above T everything, at the ends of 32 bits too."""
    new = [-2 ** 31, 2 ** 31 - 1, -1, 0, 6]
    c = Case(dev, "f16", 5, 5, 4, 2, 64, 40, seed=4)
    got = _run(op, c, kind, None, [40] * 5, new)
    clamped = [min(max(x, 0), 5) for x in new]
    c.g.manual_seed(7)
    q, caches, before = _run(op, c, kind, None, [40] * 5, new)
    c.g.manual_seed(7)
    want_q, want, _ = _run(op, c, kind, None, [40] * 5, clamped)
    assert torch.equal(q, want_q) and torch.equal(got[0], want_q)
    for x, y in zip(caches, want):
        assert x is None and y is None or torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    assert torch.equal(caches[0][0].view(torch.uint8), before[0][0].view(torch.uint8)) and not q[0].any()
