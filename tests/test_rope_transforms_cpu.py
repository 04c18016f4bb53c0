"""The eager short cut of ``rope`` under torch's transforms, with a stand-in for the kernel: the same linear map in plain torch."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture()
def op(fa, monkeypatch):
    import __graft_entry__ as ge
    op = ge.load_module("torch_op")

    def turn(x, inv_freq, positions, interleaved, amplitude, inverse):
        p = torch.arange(x.shape[2]) if positions is None else positions
        a = (p.double()[..., None] * inv_freq * (-1 if inverse else 1))
        a = a[:, None] if a.dim() == 3 else a
        c, s, h = amplitude * a.cos(), amplitude * a.sin(), inv_freq.numel()
        u, v = x[..., :h].double(), x[..., h:2 * h].double()
        return torch.cat((u * c - v * s, v * c + u * s, x[..., 2 * h:].double()), -1).to(x.dtype)

    def stand_in(q, k, inv_freq, positions, interleaved, amplitude, inverse):
        with torch.no_grad():                          # a kernel leaves no trace, and knows data alone
            q, k = (torch.from_numpy(x.detach().numpy().copy()) for x in (q, k))
            return tuple(torch.from_numpy(turn(x, inv_freq, positions, interleaved, amplitude, inverse).numpy()) for x in (q, k))

    monkeypatch.setattr(op, "_run_rope", stand_in)
    return op


def _inputs(op):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn((2, 3, 8, 64), generator=g), torch.randn((2, 1, 8, 64), generator=g)
    return q, k, op.rope_frequencies(32)[0], torch.arange(8) * 3


def test_traced_by_jit(op):
    q, k, f, pos = _inputs(op)
    traced = torch.jit.trace(lambda a, b: op.rope(a, b, f, pos), (q, k), check_trace=False)
    assert "fa_b200::rope" in str(traced.graph)
    for x, y in zip(traced(q + 1, k - 1), op.rope(q + 1, k - 1, f, pos)):
        assert torch.equal(x, y)
