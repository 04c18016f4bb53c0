"""Rotary positions (fa_rope, torch.ops.fa_b200.rope) against the formula in 64 bits; bounds in cache_reference.py."""
import numpy as np
import pytest
import torch

from cache_reference import angles, close16, rotate

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def _x(dev, dtype, seed, *shape):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev).to(DT[dtype])


def _check(got, x, pos, f, inter, amp=1.0, inverse=False):
    """x [B,H,S,D] torch, pos [S] or [B,S]."""
    ang = angles(pos, f)
    ang = ang[None, None] if ang.ndim == 2 else ang[:, None]
    want, size = rotate(x.double().cpu().numpy(), ang, inter, amp, inverse)
    close16(got, want, size, x.dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (64, 16), (64, 48), (128, 128), (128, 64), (128, 16), (128, 112)])
@pytest.mark.parametrize("b,hq,hkv,s", [(1, 1, 1, 1), (2, 6, 2, 77)])
def test_rope(op, dev, dtype, inter, d, rot, b, hq, hkv, s):
    q, k = _x(dev, dtype, 1, b, hq, s, d), _x(dev, dtype, 2, b, hkv, s, d)
    f, _ = op.rope_frequencies(rot)
    qo, ko = op.rope(q, k, f, None, inter)
    for x, y in ((q, qo), (k, ko)):
        _check(y, x, np.arange(s), f, inter)
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,hq,hkv,s", [(5, 3, 2, 1001), (2, 13, 1, 3000), (300, 5, 0, 15)])
def test_rope_many_tokens_of_small_heads(op, dev, inter, b, hq, hkv, s):
    """d_head 64 with enough tokens for the larger blocks, which the last ones do not fill."""
    q, k = _x(dev, "f16", 5, b, hq, s, 64), _x(dev, "f16", 6, b, hkv, s, 64)
    f, _ = op.rope_frequencies(64)
    qo, ko = op.rope(q, k, f, None, inter)
    _check(qo, q, np.arange(s), f, inter)
    if hkv:
        _check(ko, k, np.arange(s), f, inter)


@pytest.mark.parametrize("b,hq,hkv,s", [(1, 40, 8, 3), (3, 5, 1, 9), (1, 71, 0, 130), (2, 32, 8, 1000), (5, 3, 3, 8)])
def test_rope_sizes(op, dev, b, hq, hkv, s):
    q, k = _x(dev, "bf16", 3, b, hq, s, 128), _x(dev, "bf16", 4, b, hkv, s, 128)
    f, _ = op.rope_frequencies(128)
    qo, ko = op.rope(q, k, f)
    _check(qo, q, np.arange(s), f, False)
    assert ko.shape == k.shape
    if hkv:
        _check(ko, k, np.arange(s), f, False)


@pytest.mark.parametrize("inter", [False, True])
def test_positions_near_far_and_negative(op, dev, inter):
    b, h, d = 2, 3, 64
    pos = np.array([[0, 1, -1, 7, -12345, 131071, 1000003, 2 ** 31 - 1, -2 ** 31, 5],
                    [9, 8, 7, 6, 5, 4, 3, 2, 1, 2 ** 30 + 1]])
    q = _x(dev, "f16", 5, b, h, pos.shape[1], d)
    f, _ = op.rope_frequencies(d, 5e5)
    # 64-bit products of the largest positions are off by 2^31 * 2^-53 rad: nothing at these bounds
    for p in (pos, pos[1]):
        for t in (torch.int32, torch.int64):
            qo, ko = op.rope(q, q, f, torch.tensor(p, device=dev, dtype=t), inter)
            _check(qo, q, p, f, inter)
            assert torch.equal(qo, ko)


def test_position_offset_in_place_and_amplitude(fa, op, dev):
    b, h, s, d = 2, 4, 33, 128
    x = _x(dev, "f16", 6, b, h, s, d)
    f, amp = op.rope_frequencies(d, scaling="parts", factor=8.0, original_length=512, slow=1, fast=32)
    assert amp > 1.1
    y = x.clone()
    fa.rope(y, None, y, None, b, h, 0, s, d, f, d, amplitude=amp, dtype="f16", position_offset=100001,
            stream=torch.cuda.current_stream())
    _check(y, x, np.arange(s) + 100001, f, False, amp)


def test_strided_inputs_and_outputs(fa, op, dev):
    """[B, S, H, D] parts of one projection, as views; and strided outputs through the binding, with a guard around."""
    b, s, hq, hkv, d = 2, 19, 4, 2, 64
    qkv = _x(dev, "bf16", 7, b, s, hq + 2 * hkv, d)
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hkv].transpose(1, 2)
    f, _ = op.rope_frequencies(d)
    qo, ko = op.rope(q, k, f)
    assert qo.is_contiguous() and ko.is_contiguous()
    _check(qo, q, np.arange(s), f, False)
    _check(ko, k, np.arange(s), f, False)
    pool = torch.full((b, s, hq + 1, d + 8), 7.0, device=dev, dtype=q.dtype)
    st = pool.stride()
    fa.rope(q, None, pool, None, b, hq, 0, s, d, f, d, dtype="bf16", q_strides=(q.stride(0), q.stride(1), q.stride(2)),
            q_out_strides=(st[0], st[2], st[1]), stream=torch.cuda.current_stream())
    assert torch.equal(pool[:, :, :hq, :d].transpose(1, 2), qo)
    pool[:, :, :hq, :d] = 7.0
    assert (pool == 7.0).all()
    odd = _x(dev, "bf16", 8, b, hq, s, d + 1)[..., 1:]          # misaligned rows are copied by the operator
    _check(op.rope(odd, odd, f)[0], odd, np.arange(s), f, False)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("inter,rot", [(False, 64), (True, 32)])
def test_gradient(op, dev, dtype, inter, rot):
    b, hq, hkv, s, d = 2, 4, 2, 37, 64
    q, k = _x(dev, dtype, 9, b, hq, s, d).requires_grad_(), _x(dev, dtype, 10, b, hkv, s, d).requires_grad_()
    gq, gk = _x(dev, dtype, 11, b, hq, s, d), _x(dev, dtype, 12, b, hkv, s, d)
    f, amp = op.rope_frequencies(rot, scaling="parts", factor=4.0, original_length=64, slow=1, fast=32)
    pos = torch.randint(0, 10 ** 6, (b, s), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    qo, ko = op.rope(q, k, f, pos, inter, amp)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    p = pos.cpu().numpy()
    _check(dq, gq, p, f, inter, amp, inverse=True)
    _check(dk, gk, p, f, inter, amp, inverse=True)
    # differences: the map is linear, so <g, R(u) - R(0)> = <R'g, u> for any u.  Each 16-bit element of R u and R'g is
    # off by at most eps / 2 of it (and far less before that): the sums differ by at most the sum of those.
    eps = torch.finfo(q.dtype).eps
    a, c = (qo.detach().double() * gq.double()), (q.detach().double() * dq.double())
    assert abs(float(a.sum() - c.sum())) <= eps * float(a.abs().sum() + c.abs().sum())
    # one output alone, and an expanded gradient
    only_k, = torch.autograd.grad(ko, k, gk, retain_graph=True)
    assert torch.equal(only_k, dk)
    ones, = torch.autograd.grad(qo.sum(), q)
    _check(ones, torch.ones_like(gq), p, f, inter, amp, inverse=True)


@pytest.mark.parametrize("which", ["positions", "inv_freq"])
@pytest.mark.parametrize("registered", [False, True])
def test_overwritten_before_the_backward_pass(op, dev, which, registered):
    q = torch.randn((1, 2, 8, 64), device=dev).half().requires_grad_()
    k = torch.randn((1, 1, 8, 64), device=dev).half()
    f, pos = op.rope_frequencies(64)[0], torch.arange(8, device=dev, dtype=torch.int32)
    qo, _ = (torch.ops.fa_b200.rope if registered else op.rope)(q, k, f, pos)
    (pos if which == "positions" else f).mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        qo.float().sum().backward()


def test_nan_and_inf_stay_in_their_pair(op, dev):
    s, d, rot = 4, 64, 32
    x = _x(dev, "f16", 13, 1, 1, s, d)
    x[0, 0, 1, 3], x[0, 0, 2, 50] = float("nan"), float("inf")
    f, _ = op.rope_frequencies(rot)
    y, _ = op.rope(x, x, f)
    bad = ~torch.isfinite(y[0, 0])
    assert bad.nonzero().tolist() == [[1, 3], [1, 3 + rot // 2], [2, 50]]


def test_refused_by_the_operator(op, dev):
    q = _x(dev, "f16", 14, 1, 2, 8, 64)
    f, _ = op.rope_frequencies(64)
    for args, err in (((q.float(), q.float(), f), TypeError), ((q, q.bfloat16(), f), TypeError), ((q, q[:, :, :4], f), ValueError),
                      ((q, q, f.to(dev)), TypeError), ((q, q, f.float()), TypeError),
                      ((q, q, f, torch.zeros(7, device=dev, dtype=torch.int32)), ValueError),
                      ((q, q, f, torch.zeros(8, device=dev)), ValueError), ((q, q, f, torch.zeros(8, dtype=torch.int32)), ValueError)):
        with pytest.raises(err):
            op.rope(*args)


def test_captured_and_replayed_with_training_step(op, dev):
    """Forward and backward in one graph, replayed on new contents: the same bits as direct calls."""
    b, h, s, d = 1, 2, 50, 64
    q = _x(dev, "f16", 15, b, h, s, d)
    g = _x(dev, "f16", 16, b, h, s, d)
    f, _ = op.rope_frequencies(d)

    def step():
        x = q.detach().requires_grad_()
        y, z = op.rope(x, x, f)
        return y, z, torch.autograd.grad((y, z), x, (g, g))[0]

    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    q.copy_(_x(dev, "f16", 17, b, h, s, d))
    graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(outs, step()):
        assert torch.equal(a, c)


def test_registered_operator_is_the_same_with_its_gradient(op, dev):
    """torch.ops.fa_b200.rope (what compiled code reaches) and the eager call: the same bits, forward and backward."""
    q, k = _x(dev, "bf16", 18, 2, 4, 21, 64).requires_grad_(), _x(dev, "bf16", 19, 2, 1, 21, 64).requires_grad_()
    g, h = _x(dev, "bf16", 20, 2, 4, 21, 64), _x(dev, "bf16", 21, 2, 1, 21, 64)
    f, _ = op.rope_frequencies(64)
    pos = torch.arange(21, device=dev) * 1000
    results = []
    for fn in (op.rope, torch.ops.fa_b200.rope):
        a, b = fn(q, k, f, pos, True, 1.25)
        results.append((a, b, *torch.autograd.grad((a, b), (q, k), (g, h))))
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_side_stream(op, dev):
    """Work on another stream than the tensors' own, ordered by the caller."""
    x = _x(dev, "f16", 22, 1, 8, 300, 128)
    f, _ = op.rope_frequencies(128)
    want = op.rope(x, x, f)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = op.rope(x, x, f)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
def test_every_operation_is_rounded_by_itself(op, dev, dtype, inter):
    """Products and their sum rounded to 32 bits one by one, then once to 16: the same bits as separate 32-bit operations,
    which a cache in 4 bits depends on.  (One multiply-add instead gives 1e-4 of fp16 results another value.)"""
    s, d = 2000, 128
    x = _x(dev, dtype, 23, 1, 8, s, d)
    f, _ = op.rope_frequencies(d)
    y, _ = op.rope(x, x, f, None, inter)
    ang = torch.arange(s, device=dev).double()[:, None] * f.to(dev)
    c, sn = ang.cos().float(), ang.sin().float()
    v = x.float()
    a, b = (v[..., 0::2], v[..., 1::2]) if inter else (v[..., :d // 2], v[..., d // 2:])
    want = torch.stack((a * c - b * sn, b * c + a * sn), -1 if inter else -2).flatten(-2).to(x.dtype)
    # cos and sin come from angles in 64 bits by two ways: a value next to a border of 32 bits may round either way (2^-29
    # relative a rounding of 2^-24, a few of 10^6), and then a 16-bit one in 2^13 or less of these
    assert int((y != want).sum()) <= 2
