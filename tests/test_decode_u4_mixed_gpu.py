"""Attention over a 4-bit cache where the query rows of one KV head differ: in magnitude, in being numbers at all."""
import pytest
import torch

from cache_reference import u4_unpack
from test_decode_u4_gpu import Cache, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def check_rows(q, cache, o, lse, scale, rows):
    """The query rows that `rows` [B, T, Hq] names, each against 64 bits within a bound of its own.  Many rows go through a copy of
    the cache in fp16, which rounds V^ and P (2^-12 each) and K^ (2^-12 of its elements); fewer rows round P times V's
    scale (2^-12 of at most 2 |V^| + |V^|).  A score is off by at most d = scale * sum |q k| (2^-12 + 2^-20), the second for the
    32-bit sums, so P by exp(+-2d); then O's own rounding."""
    want, want_l, _, _ = reference(q, cache, scale)
    b, t, hq, d = q.shape
    hkv = cache.tensors[0].shape[2]
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        k, v = u4_unpack(kc, kp), u4_unpack(vc, vp)
        x = q[i].double().abs().view(t, hkv, hq // hkv, d)
        dev = scale * torch.einsum("thgd,hd->thg", x, k.abs().amax(0)).reshape(t, hq) * (2.0 ** -12 + 2.0 ** -20)
        top = v.abs().amax(0).repeat_interleave(hq // hkv, 0)[None]
        tol = top * (3 * 2.0 ** -12 + 2.0 ** -18 + torch.expm1(2 * dev)[..., None]) + want[i].abs() * (torch.finfo(q.dtype).eps / 2 + 2.0 ** -12) + 2.0 ** -24
        m = rows[i]
        assert bool(m.any())
        assert ((o[i].double() - want[i]).abs() <= tol)[m].all()
        assert ((lse[i].double() - want_l[i]).abs() <= dev + 2.0 ** -18)[m].all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,skv,page", [
    (1, 5, 8, 2, 1024, 0),              # few rows a KV head
    (1, 24, 8, 2, 1024, 0),             # the smallest number that goes by the copy
    (2, 40, 6, 2, 1030, 16),
    (2, 130, 5, 1, 700, 0),             # several query tiles
])
def test_rows_of_any_size_side_by_side(op, dev, dtype, d, b, t, hq, hkv, skv, page):
    """Rows of order 1, 1e-3 and 1e12 (fp16: 6e4), and rows that hold a NaN or an infinity, within each KV head, by head and
    by token: what the numbers of one row are is nothing to another.  (The rows of 1e12 themselves are not looked at: their scores
    are of order 1e13, where a 32-bit maximum times scale is off by half a step, 2^19, and exp of that is anything.)"""
    q, cache = make(dev, dtype, b, t, hq, hkv, skv, d, [skv] * b, page, seed=t)
    huge = 1e12 if dtype == "bf16" else 6e4
    kind = torch.randint(0, 5, (b, t, hq), device=dev, generator=torch.Generator(device=dev).manual_seed(d + t))
    kind[:, -1, 0], kind[:, 0, -1] = 0, 1
    q = torch.where((kind == 1)[..., None], q * 1e-3, q)
    q = torch.where((kind == 2)[..., None], (q.sign() * huge).to(q.dtype), q)
    q[..., 7] = torch.where(kind == 3, torch.full_like(q[..., 7], float("nan")), q[..., 7])
    q[..., 3] = torch.where(kind == 4, torch.full_like(q[..., 3], float("-inf")), q[..., 3])
    o, lse = run(op, q, cache, d ** -0.5)
    check_rows(torch.where((kind < 2)[..., None], q, torch.ones_like(q)), cache, o, lse, d ** -0.5, kind < 2)


@pytest.mark.parametrize("t", [4, 40])
def test_padding_of_a_batch_holds_anything(op, dev, t):
    """The tokens before a left-padded sequence's first see no key; whatever their q holds, they give zeros and reach nothing."""
    lens = [700, t - 3, 1]
    b, hq, hkv, d = 3, 8, 2, 128
    q, cache = make(dev, "bf16", b, t, hq, hkv, 700, d, lens, seed=3)
    clean, clean_l = run(op, q, cache, 0.0884)
    dirty = q.clone()
    for i, n in enumerate(lens):
        pad = max(t - n, 0)
        for j, x in enumerate((float("nan"), float("inf"), 3e38, -1e30)):
            dirty[i, :pad, j::4] = x
    o, lse = run(op, dirty, cache, 0.0884)
    assert torch.equal(o, clean) and torch.equal(lse, clean_l)
    for i, n in enumerate(lens):
        pad = max(t - n, 0)
        assert not o[i, :pad].any() and torch.isinf(lse[i, :pad]).all()


@pytest.mark.parametrize("d,t,skv", [(64, 5, 1024), (64, 40, 1024), (128, 40, 1024), (128, 64, 9000), (64, 48, 20000)])
def test_results_far_below_fp16(op, dev, d, t, skv):
    """V of 1e-6 and bf16: O is rounded once, to bf16, also where few keys are split over many CTAs and merged.  All of V^ is
    positive, so O = sum p V^ carries the relative errors of its terms: V^ is a multiple of 2^-24 and exact in fp16, P is off by 2^-12
    (below 2^-14 by 2^-25, on a sum of P of 1 and more), and by the scores' error d as in check_rows; then half a step of bf16."""
    b, hq, hkv = 1, 8, 2
    g = torch.Generator(device=dev).manual_seed(d + t)
    q = torch.randn((b, t, hq, d), generator=g, device=dev).bfloat16()
    k = torch.randn((b, skv, hkv, d), generator=g, device=dev).bfloat16()
    v = (1e-6 + 1e-6 * torch.rand((b, skv, hkv, d), generator=g, device=dev)).bfloat16()
    cache = Cache(dev, k, v, [skv])
    o, lse = run(op, q, cache, 0.05)
    want, _, _, _ = reference(q, cache, 0.05)
    kk = u4_unpack(*cache.packed[0][0])
    dev_s = 0.05 * float(torch.einsum("thgd,hd->thg", q[0].double().abs().view(t, hkv, hq // hkv, d), kk.abs().amax(0)).max()) * (2.0 ** -12 + 2.0 ** -20)
    terms = 2.0 ** -12 + skv * 2.0 ** -25 + 2.0 ** -18 + float(torch.expm1(torch.tensor(2 * dev_s)))
    rel = ((o.double() - want).abs() / want).max()
    assert rel <= (1 + terms) * (1 + 2.0 ** -8) - 1, float(rel)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.125, 1e-9, 1e-30])
@pytest.mark.parametrize("t", [5, 40])
def test_queries_of_zeros(op, dev, dtype, scale, t):
    """Every score is 0 whatever the scale: O is the mean of the V^ that a token sees, LSE the logarithm of their number.  Rows of
    zeros, of numbers so small that their power of two times the scale leaves 32 bits, and of ordinary ones."""
    q, cache = make(dev, dtype, 2, t, 8, 2, 600, 64, [600, 514], seed=t)
    q[:, :, 0::4] = 0
    q[:, :, 1::4] = 1e-38 if dtype == "bf16" else 6e-8
    o, lse = run(op, q, cache, scale)
    check_rows(q, cache, o, lse, scale, torch.ones(q.shape[:3], dtype=torch.bool, device=dev))
