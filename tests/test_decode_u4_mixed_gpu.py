"""Attention over a 4-bit cache where the query rows of one KV head differ: in magnitude, in being numbers at all."""
import pytest
import torch

from cache_reference import u4_unpack
from test_decode_u4_gpu import Cache, check, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def check_rows(q, cache, o, lse, scale, rows):
    """The query rows that `rows` [B, T, Hq] names, each against 64 bits within a bound of its own.  A rounding to fp16
    is off by half a step, finfo.eps / 2 = 2^-11.  Many rows go through a copy of the cache in fp16, which rounds V^ and P (2^-11
    each) and K^ (2^-11 of its elements), fp16 queries P alone; fewer rows round P times V's scale (2^-11 of at most 2 |V^| + |V^|).
    A score is off by at most d = scale * sum |q k| (2^-11 + 2^-20), the second for the 32-bit sums, so P by exp(+-2d); then O's
    own rounding."""
    want, want_l, _, _ = reference(q, cache, scale)
    b, t, hq, d = q.shape
    hkv = cache.tensors[0].shape[2]
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        k, v = u4_unpack(kc, kp), u4_unpack(vc, vp)
        x = q[i].double().abs().view(t, hkv, hq // hkv, d)
        dev = scale * torch.einsum("thgd,hd->thg", x, k.abs().amax(0)).reshape(t, hq) * (2.0 ** -11 + 2.0 ** -20)
        top = v.abs().amax(0).repeat_interleave(hq // hkv, 0)[None]
        tol = top * (3 * 2.0 ** -11 + 2.0 ** -18 + torch.expm1(2 * dev)[..., None]) + want[i].abs() * (torch.finfo(q.dtype).eps / 2 + 2.0 ** -11) + 2.0 ** -24
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
    (2, 1, 128, 1, 700, 0),             # one token of a group that fills a query tile
    (2, 2, 300, 3, 5000, 16),           # a group of 100, split over the keys
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
    positive, so O = sum p V^ carries the relative errors of its terms: V^ is a multiple of 2^-24 and exact in fp16, P is off by 2^-11
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
    dev_s = 0.05 * float(torch.einsum("thgd,hd->thg", q[0].double().abs().view(t, hkv, hq // hkv, d), kk.abs().amax(0)).max()) * (2.0 ** -11 + 2.0 ** -20)
    terms = 2.0 ** -11 + skv * 2.0 ** -25 + 2.0 ** -18 + float(torch.expm1(torch.tensor(2 * dev_s)))
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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [1, 3])
@pytest.mark.parametrize("small", [-6, -11, -15])
def test_a_v_row_of_no_weight_and_a_huge_scale(op, dev, d, t, small):
    """One key of V^ up to 65504 whose weight is about 2^-60, between keys of values 2^small.  P times V's scale is rounded to fp16 in
    units of 2^E with 2^E at most a 16th of the largest scale, so below 2^-14 by 2^-25 of such a unit: times a code of up to 8,
    at most 2^-26 of the largest scale for each key, on a sum of P of at least sum exp(s - max s).  That beside
    half a step, 2^-11, of the terms."""
    b, hq, hkv, n = 2, 4, 1, 200
    g = torch.Generator(device=dev).manual_seed(t)
    base = torch.randn((d,), generator=g, device=dev).sign()
    q = (base + 0.3 * torch.randn((b, t, hq, d), generator=g, device=dev)).half()
    k = torch.randn((b, n, hkv, d), generator=g, device=dev) * 0.7
    v = torch.rand((b, n, hkv, d), generator=g, device=dev) * 2.0 ** small * 7.5
    k[:, 70] = -base * 0.5 * (128 / d)
    v[:, 70, :, ::2], v[:, 70, :, 1::2] = 65504.0, -65504.0
    cache = Cache(dev, k.half(), v.half(), [n] * b)
    scale = 0.65
    o, lse = run(op, q, cache, scale)
    want, want_l, amount, worst = reference(q, cache, scale)
    off = 16 * 2.0 ** -23 * 79 * worst + 2.0 ** -22
    steps = (n // 16 + 16) * 2.0 ** -23
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        s = torch.einsum("thd,nd->thn", q[i].double(), u4_unpack(kc, kp)[:, 0]) * scale
        see = torch.arange(n, device=dev)[None] <= (n - t + torch.arange(t, device=dev))[:, None]
        s = s.masked_fill(~see[:, None], float("-inf"))
        assert (s[..., 70] - torch.logsumexp(s, -1) < -30).all()
        l = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1)
        tol = amount[i] * (2.0 ** -11 + 2 * off + steps) + want[i].abs() * 2.0 ** -11 + 2.0 ** -25 + (n * 2.0 ** -26 * float(vp[..., 0].max()) / l)[..., None]
        assert ((o[i].double() - want[i]).abs() <= tol).all()


@pytest.mark.parametrize("d,hq", [(64, 8), (128, 24), (64, 80)])
def test_a_huge_v_row_costs_its_own_tile_alone(op, dev, d, hq):
    """Keys 64 .. 127 have weights below 2^-60 and one of them V^ up to 65504; the thousands after it, of values 2^-13, keep every digit
    within `check`'s bound, which has no absolute term (but O's own half step, 2^-25)."""
    b, hkv, n = 32, 8, 4000
    g = torch.Generator(device=dev).manual_seed(d)
    base = torch.randn((d,), generator=g, device=dev).sign()
    q = (base + 0.3 * torch.randn((b, 1, hq, d), generator=g, device=dev)).half()
    k = torch.randn((b, n, hkv, d), generator=g, device=dev) * 0.7
    v = torch.rand((b, n, hkv, d), generator=g, device=dev) * 2.0 ** -13 * 7.5
    k[:, 64:128] = -base * 0.5 * (128 / d)
    v[:, 70, :, ::2], v[:, 70, :, 1::2] = 65504.0, -65504.0
    cache = Cache(dev, k.half(), v.half(), [n] * b)
    o, lse = run(op, q, cache, 0.65)
    check(q, cache, o, lse, 0.65, n)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("t", [3, 40])
def test_rows_that_are_not_numbers(op, dev, dtype, t):
    """A NaN in a query, or in a key that a token sees: NaN with few rows; O = 0 and LSE = -inf with many, as fa_decode_gqa has it.
    Tokens and heads that do not meet it keep every bit."""
    q, cache = make(dev, dtype, 2, t, 8, 2, 640, 64, seed=2)
    clean, clean_l = run(op, q, cache, 0.125, lens=False)
    q[1, 1, 2, 5] = float("nan")
    kp = cache.tensors[1]
    kp[0, 639, 1] = float("nan")                               # the last token's own key, KV head 1
    o, lse = run(op, q, cache, 0.125, lens=False)
    hit = torch.zeros(q.shape[:3], dtype=torch.bool, device=dev)
    hit[1, 1, 2] = True
    hit[0, t - 1, 4:] = True
    assert torch.equal(o[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_l[~hit])
    if t == 3:
        assert o[hit].isnan().all() and lse[hit].isnan().all()
    else:
        assert not o[hit].any() and (lse[hit] == float("-inf")).all()


@pytest.mark.parametrize("t", [1, 6])
def test_an_infinite_scale_stays_in_its_64_elements(op, dev, t):
    """A pair of V (of another origin) whose scale is infinite: its 64 elements are lost, the row's other ones are not."""
    b, hq, hkv, n, d = 32, 8, 4, 1500, 128
    q, cache = make(dev, "f16", b, t, hq, hkv, n, d, seed=t)
    clean, clean_l = run(op, q, cache, 0.0884, lens=False)
    check(q, cache, clean, clean_l, 0.0884, n)
    for i in range(b):
        cache.tensors[3][i, 70 + 20 * i, :, i % 2, 0] = float("inf")
    o, lse = run(op, q, cache, 0.0884, lens=False)
    assert torch.equal(lse, clean_l)
    _, _, amount, _ = reference(q, cache, 0.0884)
    for i in range(b):
        other = slice(64, 128) if i % 2 == 0 else slice(0, 64)
        # both are P times V's scale rounded and O rounded (2^-11 each); and the tile of the infinity, 64 keys, counts in units for a scale of
        # 65504, 2^-26 of that a key at most, on a sum of P of sum exp(s - max s)
        k = u4_unpack(*cache.packed[0][i])
        s = torch.einsum("thgd,nhd->thgn", q[i].double().view(t, hkv, hq // hkv, d), k) * 0.0884
        l = torch.exp(clean_l[i].double().view(t, hkv, -1) - s.amax(-1)).view(t, hq, 1)
        tol = 2 * (amount[i] * 2.0 ** -11 + clean[i].double().abs() * 2.0 ** -11) + 64 * 2.0 ** -26 * 65504 / l + 2.0 ** -24
        assert ((o[i].double() - clean[i].double()).abs() <= tol)[..., other].all()
        assert not torch.isfinite(o[i, :, :, 64 * (i % 2)]).all()
