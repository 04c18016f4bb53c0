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


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode(op, grad):
    """The map is linear: the tangent of R(x) along u is R(u), for q and k each by itself, with or without a gradient to come."""
    q, k, f, pos = _inputs(op)
    u, w = torch.randn_like(q), torch.randn_like(k)
    want_u, want_w = op.rope(u, w, f, pos, False, 1.25, True)
    with fwd.dual_level():
        for tq, tk in ((u, w), (u, None), (None, w)):
            a, b = (x.clone().requires_grad_(grad) for x in (q, k))
            a = a if tq is None else fwd.make_dual(a, tq)
            b = b if tk is None else fwd.make_dual(b, tk)
            for y, t, want in zip(op.rope(a, b, f, pos, False, 1.25, True), (tq, tk), (want_u, want_w)):
                got = fwd.unpack_dual(y).tangent
                if t is None:
                    assert got is None or not got.any()
                else:
                    assert torch.equal(got, want)
        plain = op.rope(q, k, f, pos)                  # no tangents at all
        assert fwd.unpack_dual(plain[0]).tangent is None or not fwd.unpack_dual(plain[0]).tangent.any()


def test_functional_jvp_and_gradients(op):
    q, k, f, pos = _inputs(op)
    u, w = torch.randn_like(q), torch.randn_like(k)
    out, tangents = torch.func.jvp(lambda a, b: op.rope(a, b, f, pos), (q, k), (u, w))
    for x, y in zip((*out, *tangents), (*op.rope(q, k, f, pos), *op.rope(u, w, f, pos))):
        assert torch.equal(x, y)
    a = q.clone().requires_grad_()
    op.rope(a, k, f, pos)[0].square().sum().backward()
    # the derivative of sum R(x)^2 in direction u, from the gradient and from the tangent: 32-bit sums of 3000 products
    y, t = op.rope(q, k, f, pos)[0], op.rope(u, k, f, pos)[0]
    assert abs(float((a.grad * u).sum() - 2 * (y * t).sum())) < 1e-3 * float((y * t).abs().sum())


def test_forward_mode_is_refused_by_the_registered_operator(op):
    """Below the dispatcher a tangent cannot be seen for certain: an error instead of a result without its tangent."""
    q, k, f, pos = _inputs(op)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.ops.fa_b200.rope(fwd.make_dual(q, q), k, f, pos)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda a: torch.ops.fa_b200.rope(a, k, f, pos)[0], (q,), (q,))
    torch.ops.fa_b200.rope(q, k, f, pos)
