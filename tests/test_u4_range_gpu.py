"""4-bit caches of other origin whose values leave fp16's range at either end: offset + scale * code up to +-65504 and past it."""
import pytest
import torch

from cache_reference import u4_unpack

pytestmark = pytest.mark.gpu
EDGE = 65504.0


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def _cache(dev, b, rows, hkv, d, seed):
    """Ordinary rows (values of order 1), and rows that reach past +-65504 in some codes, by scales of either sign."""
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = torch.randint(0, 256, (b, rows, hkv, d // 2), generator=g, device=dev, dtype=torch.uint8)
    params = torch.empty((b, rows, hkv, d // 64, 2), device=dev, dtype=torch.float16)
    params[..., 0], params[..., 1] = 0.2, -1.5
    edge = torch.tensor([[8736.0, -65504.0], [-8736.0, 65504.0], [60000.0, 0.0], [-60000.0, 0.0], [65504.0, 65504.0], [-65504.0, -65504.0]],
                        device=dev, dtype=torch.float16)
    params[:, ::5] = edge[torch.randint(0, 6, params[:, ::5].shape[:-1], generator=g, device=dev)]
    codes[:, ::5, :, :3], codes[:, ::5, :, 3:5] = 0xFF, 0
    return codes, params


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_read(op, dev, dtype, d):
    (kc, kp), (vc, vp) = _cache(dev, 2, 61, 3, d, 1), _cache(dev, 2, 61, 3, d, 2)
    for got, c, p in zip(op.cache_read_u4(kc, kp, vc, vp, 2, 61, dtype), (kc, vc), (kp, vp)):
        want = u4_unpack(c, p)                                  # a sum of at most 24 bits: exact in 32, then one rounding
        assert torch.equal(got, (want.clamp(-EDGE, EDGE) if dtype == torch.float16 else want).to(dtype))
        assert torch.isfinite(got).all() and bool((want < -EDGE).any()) and bool((want > EDGE).any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_of_many_rows(op, dev, dtype, which):
    """The copy in fp16 holds +-65504 in the place of values past them, and nothing becomes infinite.  K: queries so small that
    scores stay of order 1.  Bounds: scores are off by d = sum |q k| scale (2^-11 + 2^-20), P by exp(+-2d) and 2^-11, V^ by 2^-11 (half steps of
    fp16)."""
    b, t, hq, hkv, n, d = 1, 40, 8, 2, 640, 64
    kc, kp = _cache(dev, b, n, hkv, d, 3)
    vc, vp = _cache(dev, b, n, hkv, d, 4)
    for c, p, x in ((kc, kp, "k"), (vc, vp, "v")):
        if x != which:
            p[..., 0], p[..., 1] = 0.2, -1.5
    g = torch.Generator(device=dev).manual_seed(5)
    q = (torch.randn((b, t, hq, d), generator=g, device=dev) * (1e-5 if which == "k" else 1.0)).to(dtype)
    o, lse = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.125)
    k, v = (u4_unpack(c, p)[0].clamp(-EDGE, EDGE) for c, p in ((kc, kp), (vc, vp)))
    x = q[0].double().view(t, hkv, hq // hkv, d)
    s = torch.einsum("thgd,nhd->thgn", x, k) * 0.125
    see = torch.arange(n, device=dev)[None] <= (n - t + torch.arange(t, device=dev))[:, None]
    s = s.masked_fill(~see[:, None, None, :], float("-inf"))
    p = torch.softmax(s, -1)
    want = torch.einsum("thgn,nhd->thgd", p, v)
    off = 0.125 * torch.einsum("thgd,hd->thg", x.abs(), k.abs().amax(0)).max() * (2.0 ** -11 + 2.0 ** -20)
    tol = torch.einsum("thgn,nhd->thgd", p, v.abs()) * (2.0 ** -10 + 2.0 ** -18 + torch.expm1(2 * off)) + want.abs() * torch.finfo(dtype).eps / 2 + n * 2.0 ** -25 * v.abs().max() + 2.0 ** -25
    assert ((o[0].double().view_as(want) - want).abs() <= tol).all()
    assert ((lse[0].double().view(t, hkv, -1) - torch.logsumexp(s, -1)).abs() <= off + 2.0 ** -18).all()
