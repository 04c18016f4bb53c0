"""Attention over a 4-bit cache (fa_decode_gqa_u4) against 64-bit attention over the values that the cache stands for.

Bounds.  The codes are exact on the tensor core and every sum is held in 32 bits; what is rounded to fewer is P times
V's scale, to fp16 (half a step: 2^-12 of the term), and O.  The terms' roundings add up to at most 2^-12 * sum_k p_k |s_k (c_k - 8)|
<= 2^-12 * A with A = sum_k p_k (|V^_k| + |z_k + 8 s_k|); `ab` below computes A exactly.  32-bit parts: a score is a sum of 2 * 128 products of
up to 79 |q| (the tensor core sees 64 + code) with ~2^-23 lost at each of its 8 to 16 steps, so off by at most
d = 16 * 2^-23 * 79 * scale * s_max * sum |q|, and
p by the factor d and ex2's 2^-22; the running sums of tiles lose at most 2^-23 a step (one for 16 keys of a warp)."""
import numpy as np
import pytest
import torch

from cache_reference import u4_pack, u4_unpack

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


class Cache:
    """A 4-bit cache of K and V rows [B, Skv, Hkv, D]; what no sequence reaches holds NaN params and arbitrary codes."""

    def __init__(self, dev, k, v, lens, page=0, head_major=True, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed + 99)
        b, skv, hkv, d = k.shape
        self.lens, self.table, self.k, self.v = lens, None, [], []
        n_pages = -(-skv // page) if page else 1
        rows, blocks = page or skv, b * n_pages + (2 if page else 0)
        if page:
            self.table = torch.randperm(blocks, generator=g, device=dev)[:b * n_pages].to(torch.int32).view(b, n_pages)
        self.tensors = []
        for x in (k, v):
            shape = (blocks, hkv, rows) if head_major else (blocks, rows, hkv)
            codes = torch.randint(0, 256, (*shape, d // 2), generator=g, device=dev, dtype=torch.uint8)
            params = torch.full((*shape, d // 64, 2), float("nan"), device=dev, dtype=torch.float16)
            if head_major:
                codes, params = codes.transpose(1, 2), params.transpose(1, 2)
            for i in range(b):
                n = min(max(lens[i], 0), skv)
                c, p = u4_pack(x[i, :n])
                for r0 in range(0, n, rows):
                    m = min(rows, n - r0)
                    blk = int(self.table[i, r0 // rows]) if page else i
                    codes[blk, :m], params[blk, :m] = c[r0:r0 + m], p[r0:r0 + m]
            self.tensors += [codes, params]
        if page:                                                 # entries past a sequence's end are never looked at
            for i in range(b):
                self.table[i, -(-min(max(lens[i], 0), skv) // page):] = 2 ** 31 - 1
        self.packed = [[u4_pack(x[i, :min(max(lens[i], 0), skv)]) for i in range(b)] for x in (k, v)]


def reference(q, cache, scale):
    """O, LSE in 64 bits, the bound's A, and the largest sum |q| * s_max."""
    b, t, hq, d = q.shape
    hkv = cache.tensors[0].shape[2]
    group = hq // hkv
    o, lse, amount = (torch.zeros((b, t, hq, d), dtype=torch.float64, device=q.device) for _ in range(3))
    lse = torch.full((b, t, hq), float("-inf"), dtype=torch.float64, device=q.device)
    worst = 0.0
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        n = kc.shape[0]
        if n == 0:
            continue
        k, v = u4_unpack(kc, kp), u4_unpack(vc, vp)
        mid = (vp[..., 1].double() + 8 * vp[..., 0].double()).abs().repeat_interleave(64, -1)
        x = q[i].double().view(t, hkv, group, d)
        s = torch.einsum("thgd,nhd->thgn", x, k) * scale
        see = torch.arange(n, device=q.device)[None] <= (n - t + torch.arange(t, device=q.device))[:, None]
        s = s.masked_fill(~see[:, None, None, :], float("-inf"))
        l = torch.logsumexp(s, -1)
        p = torch.exp(s - torch.where(torch.isfinite(l), l, torch.zeros_like(l))[..., None])
        o[i] = torch.einsum("thgn,nhd->thgd", p, v).reshape(t, hq, d)
        amount[i] = torch.einsum("thgn,nhd->thgd", p, v.abs() + mid).reshape(t, hq, d)
        lse[i] = l.reshape(t, hq)
        worst = max(worst, float(x.abs().sum(-1).max() * kp[..., 0].double().max()) * scale)
    return o, lse, amount, worst


def check(q, cache, o, lse, scale, keys):
    want, want_l, amount, worst = reference(q, cache, scale)
    d = 16 * 2.0 ** -23 * 79 * worst + 2.0 ** -22
    steps = (keys // 16 + 16) * 2.0 ** -23
    tol = amount * (2.0 ** -12 + 2 * d + steps) + want.abs() * torch.finfo(q.dtype).eps / 2 + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    err = (o.double() - want).abs()
    assert not (~(err <= tol)).any(), (float(err.max()), float((err / tol.clamp_min(1e-30)).max()))
    assert torch.equal(torch.isinf(lse), torch.isinf(want_l))
    fin = torch.isfinite(want_l)
    # one rounding of the result on top
    assert ((lse.double() - want_l)[fin].abs() <= 2 * d + steps + 2.0 ** -23 * want_l[fin].abs()).all()


def make(dev, dtype, b, t, hq, hkv, skv, d, lens=None, page=0, head_major=True, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn((b, t, hq, d), generator=g, device=dev).to(DT[dtype])
    rows = -(-skv // page) * page if page else skv           # what the pages hold: lengths are clamped to that
    k, v = (torch.randn((b, rows, hkv, d), generator=g, device=dev).to(DT[dtype]) for _ in range(2))
    return q, Cache(dev, k, v, lens or [skv] * b, page, head_major, seed)


def run(op, q, cache, scale, lens=True):
    kc, kp, vc, vp = cache.tensors
    return op.decode_gqa_u4(q, kc, kp, vc, vp, scale, torch.tensor(cache.lens, device=q.device, dtype=torch.int32) if lens else None,
                            cache.table)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,skv,page,hm", [
    (1, 1, 1, 1, 1, 0, True),               # one key
    (2, 1, 8, 2, 33, 0, False),             # a key past a tile
    (1, 1, 8, 1, 1000, 16, True),
    (3, 1, 3, 3, 257, 0, True),             # no groups
    (2, 1, 12, 4, 1537, 64, False),
    (1, 1, 16, 1, 500, 0, True),            # 16 rows
    (1, 1, 71, 1, 300, 16, False),          # 71 rows: three blocks, the last ragged
    (2, 3, 6, 2, 100, 0, True),             # 9 rows of three tokens
    (1, 7, 10, 2, 200, 32, True),           # 35 rows
    (1, 64, 4, 2, 64, 0, False),            # a prompt from nothing
    (2, 100, 4, 4, 333, 16, True),
    (1, 1, 256, 1, 64, 0, True),            # a group of 256
])
def test_against_64_bits(op, dev, dtype, d, b, t, hq, hkv, skv, page, hm):
    q, cache = make(dev, dtype, b, t, hq, hkv, skv, d, None, page, hm, seed=skv)
    scale = d ** -0.5
    o, lse = run(op, q, cache, scale, lens=page != 0)       # without lengths the last page would count whole
    check(q, cache, o, lse, scale, skv)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("t", [1, 2, 5])
@pytest.mark.parametrize("page", [0, 16, 256])
def test_lengths(op, dev, dtype, t, page):
    """Lengths of every kind, among them 0, fewer keys than tokens, tile and page borders, out of range."""
    lens = [700, 0, 1, 16, 31, 32, 33, 5, 64, 511, -3, 9999, 256, 257, 2]
    q, cache = make(dev, dtype, len(lens), t, 8, 2, 700, 128, lens, page, seed=t)
    o, lse = run(op, q, cache, 0.0884)
    check(q, cache, o, lse, 0.0884, 700)
    assert not o[1].any() and torch.isinf(lse[1]).all()


@pytest.mark.parametrize("b", [255, 256, 257, 600])
def test_many_short_sequences(op, dev, b):
    """More sequences than threads look their lengths up at once; a warp does several."""
    lens = np.random.RandomState(b).randint(0, 70, b).tolist()
    q, cache = make(dev, "bf16", b, 1, 2, 1, 70, 64, lens, seed=b)
    o, lse = run(op, q, cache, 0.125)
    check(q, cache, o, lse, 0.125, 70)


@pytest.mark.parametrize("lens", [[40000], [20000, 3, 19000], [1] * 3 + [30000] + [2] * 3])
def test_long_sequences_over_many_ctas(op, dev, lens):
    q, cache = make(dev, "f16", len(lens), 1, 8, 2, max(lens), 128, lens, seed=1)
    o, lse = run(op, q, cache, 0.0884)
    check(q, cache, o, lse, 0.0884, max(lens))
    # the same bits on every run
    o2, lse2 = run(op, q, cache, 0.0884)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_few_keys_of_a_large_capacity(op, dev):
    """The plan is made for the capacity, the sequences are short: most CTAs have nothing."""
    lens = [3, 300, 0, 95]
    q, cache = make(dev, "f16", 4, 1, 8, 2, 8192, 128, lens, seed=2)
    o, lse = run(op, q, cache, 0.0884)
    check(q, cache, o, lse, 0.0884, 300)


def test_large_scores_and_uneven_scales(op, dev):
    """Scores up to hundreds with late maxima, V rows whose scales differ by 2^20, and constant rows (scale 0)."""
    b, hq, hkv, skv, d = 1, 8, 1, 900, 128
    g = torch.Generator(device=dev).manual_seed(3)
    q = (torch.randn((b, 1, hq, d), generator=g, device=dev) * 8).half()
    k = torch.randn((b, skv, hkv, d), generator=g, device=dev)
    k *= torch.linspace(0.01, 3.0, skv, device=dev)[None, :, None, None]
    v = torch.randn((b, skv, hkv, d), generator=g, device=dev)
    v *= torch.exp2(torch.randint(-14, 7, (b, skv, hkv, 1), generator=g, device=dev).float())
    v[:, ::7] = 0.5
    v[:, :40] = 0.0
    k, v = k.half(), v.half()
    cache = Cache(dev, k, v, [skv])
    for scale in (0.0884, 0.002, 1.0):
        o, lse = run(op, q, cache, scale)
        check(q, cache, o, lse, scale, skv)


@pytest.mark.parametrize("t", [1, 3])
def test_scales_of_either_sign(op, dev, t):
    """The same values written from the other end: offset + 15 scale as offset, -scale, 15 - code."""
    b, hq, hkv, skv, d = 2, 8, 2, 700, 128
    q, cache = make(dev, "f16", b, t, hq, hkv, skv, d, seed=14)
    for x in (0, 1):
        for i in range(b):
            codes, params = cache.packed[x][i]
            turn = torch.rand(params.shape[:2], device=dev) < 0.5 if t == 3 else torch.ones(params.shape[:2], device=dev, dtype=torch.bool)
            z, s = params[..., 1].float(), params[..., 0].float()
            new = torch.stack([-s, z + 15 * s], -1).half()
            params.copy_(torch.where(turn[..., None, None], new, params))
            codes.copy_(torch.where(turn[..., None], 255 - codes, codes))          # both codes of a byte
            cache.tensors[2 * x][i, :skv], cache.tensors[2 * x + 1][i, :skv] = codes, params
    o, lse = run(op, q, cache, 0.0884)
    want, want_l, amount, worst = reference(q, cache, 0.0884)
    largest = max(float(p[..., 0].abs().max()) for p in (cache.packed[0][0][1], cache.packed[0][1][1]))
    d0 = 16 * 2.0 ** -23 * 79 * float(q.double().abs().sum(-1).max()) * largest * 0.0884 + 2.0 ** -22     # as in check(), of |scale|
    steps = (skv // 16 + 16) * 2.0 ** -23
    tol = amount * (2.0 ** -12 + 2 * d0 + steps) + want.abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((o.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_l).abs() <= 2 * d0 + steps + 2.0 ** -23 * want_l.abs()).all()


def test_nan_in_a_key_reaches_its_head_alone(op, dev):
    q, cache = make(dev, "f16", 2, 1, 4, 2, 100, 64, seed=4)
    kc, kp, vc, vp = cache.tensors
    kp[1, 50, 1] = float("nan")
    o, lse = run(op, q, cache, 0.125)
    assert o[1, 0, 2:].isnan().all() and lse[1, 0, 2:].isnan().all()
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[1, 0, :2]).all()


def test_rows_of_pages_that_do_not_exist_count_as_zero(op, dev):
    """As in the other paged attention: K^ = V^ = 0 there."""
    q, cache = make(dev, "f16", 1, 1, 4, 2, 96, 64, page=32, seed=5)
    cache.table[0, 1] = -1
    o, lse = run(op, q, cache, 0.125)
    for x in (0, 1):
        c, p = cache.packed[x][0]
        c[32:64], p[32:64] = 0, 0
    check(q, cache, o, lse, 0.125, 96)


def test_outputs_alone_are_written_and_lse_is_optional(fa, op, dev):
    b, hq, hkv, skv, d = 2, 8, 2, 400, 128
    q, cache = make(dev, "bf16", b, 1, hq, hkv, skv, d, seed=6)
    want, _ = run(op, q, cache, 0.1)
    kc, kp, vc, vp = cache.tensors
    need = fa.decode_gqa_u4_workspace_bytes(b, hq, hkv, 1, skv, d)
    guard = torch.full((need + 512,), 77, device=dev, dtype=torch.uint8)
    o = torch.full((b * hq * d + 64,), 5.0, device=dev, dtype=torch.bfloat16)
    kw = dict(dtype="bf16", kv_strides=(kc.stride(0), kc.stride(2), kc.stride(1)),
              param_strides=(kp.stride(0) // 2, kp.stride(2) // 2, kp.stride(1) // 2), stream=torch.cuda.current_stream())
    args = (q, kc, kp, vc, vp, o, None, b, hq, hkv, skv, d, 0.1)
    assert fa.decode_gqa_u4_raw(*args, workspace=guard, workspace_bytes=need - 1, **kw) == fa.FA_ERR_WORKSPACE
    assert fa.decode_gqa_u4_raw(*args, workspace=None, workspace_bytes=need, **kw) == fa.FA_ERR_WORKSPACE
    fa.decode_gqa_u4(*args, workspace=guard, workspace_bytes=need, **kw)
    torch.cuda.synchronize()
    assert (guard[need:] == 77).all() and (o[b * hq * d:] == 5.0).all()
    assert torch.equal(o[:b * hq * d].view_as(want), want)


def test_long_cache_past_32_bit_offsets(op, dev):
    """Rows 2^31 bytes and more from the start of the cache: a token-major pool of 2.3 GB of which two sequences use pages
    at both ends."""
    hkv, d, page = 64, 128, 256
    n_pages = (2 ** 31 + 2 ** 28) // (page * hkv * d // 2)
    g = torch.Generator(device=dev).manual_seed(7)
    codes = torch.empty((n_pages, page, hkv, d // 2), device=dev, dtype=torch.uint8)
    params = torch.empty((n_pages, page, hkv, 2, 2), device=dev, dtype=torch.float16)
    table = torch.tensor([[n_pages - 1, 0], [1, n_pages - 2]], device=dev, dtype=torch.int32)
    k = torch.randn((2, 2 * page, hkv, d), generator=g, device=dev).half()
    lens = [2 * page, page + 40]
    small = Cache(dev, k, k, lens, page, head_major=False)
    for i in range(2):
        c, p = small.packed[0][i]
        for r0 in range(0, lens[i], page):
            n = min(page, lens[i] - r0)
            codes[int(table[i, r0 // page]), :n], params[int(table[i, r0 // page]), :n] = c[r0:r0 + n], p[r0:r0 + n]
    q = torch.randn((2, 1, hkv, d), generator=g, device=dev).half()
    o, lse = op.decode_gqa_u4(q, codes, params, codes, params, 0.0884, torch.tensor(lens, device=dev, dtype=torch.int32), table)
    check(q, small, o, lse, 0.0884, 512)
    kk, vv = op.cache_read_u4(codes, params, codes, params, 2, 512, torch.float16, None, torch.tensor(lens, device=dev), table)
    want = u4_unpack(*small.packed[0][0]).half()
    assert torch.equal(kk[0], want) and torch.equal(vv, kk)
    codes2, params2 = codes[:, :, :, :], params
    x = torch.randn((2, 3, hkv, d), generator=g, device=dev).half()
    op.cache_append(x, x, x, codes2, codes2, params2, params2, None, torch.tensor(lens, device=dev), table)
    kk, _ = op.cache_read_u4(codes, params, codes, params, 2, 3, torch.float16, torch.tensor([509, 293], device=dev), torch.tensor(lens, device=dev), table)
    assert torch.equal(kk, u4_unpack(*u4_pack(x)).half())


def test_together_prompt_then_tokens(op, dev):
    """As a server uses them: a left-padded batch of prompts in one chunk, then token by token, rotation, append and
    attention each step; against 64-bit attention over what the cache holds, and against the prefill of the read-back rows."""
    b, hq, hkv, d, page, cap = 3, 8, 2, 128, 16, 96
    g = torch.Generator(device=dev).manual_seed(8)
    f, amp = op.rope_frequencies(d, 5e5, "parts", 4.0, 64, 1, 32)
    n = cap // page
    table = torch.randperm(b * n + 2, generator=g, device=dev)[:b * n].to(torch.int32).view(b, n)
    (kc, kp), (vc, vp) = op.u4_cache(b * n + 2, page, hkv, d, dev), op.u4_cache(b * n + 2, page, hkv, d, dev)
    lens = torch.tensor([40, 33, 7], device=dev, dtype=torch.int32)
    new, t = lens.clone(), 40
    for step in range(4):
        x = torch.randn((b, t, hq + 2 * hkv, d), generator=g, device=dev).half()
        q = op.cache_append(x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:], kc, vc, kp, vp, f, lens, table, False, amp, new)
        o, lse = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, table)
        class View:
            tensors = [kc, kp, vc, vp]
            packed = [[], []]
        for i in range(b):
            m = int(lens[i])
            for out, (c, p) in zip(View.packed, ((kc, kp), (vc, vp))):
                blk = table[i].long()
                out.append((c[blk].flatten(0, 1)[:m], p[blk].flatten(0, 1)[:m]))
        check(q, View, o, lse, 0.0884, cap)
        if step == 0:
            k, v = op.cache_read_u4(kc, kp, vc, vp, b, t, torch.float16, None, lens, table)
            i = 0                                              # the sequence without padding: its prompt is a plain prefill
            rep = lambda y: y[i:i + 1].transpose(1, 2).repeat_interleave(hq // hkv, 1).contiguous()
            want, _ = op.prefill(q[i:i + 1].transpose(1, 2).contiguous(), rep(k), rep(v), 0.0884, True)
            # K^, V^, P and O rounded to fp16 there: a few steps of values of order 1
            assert (want.transpose(1, 2).float() - o[i:i + 1].float()).abs().max() < 8 * 2.0 ** -11 * float(want.abs().max())
        t = 1 if step < 2 else 3
        new = torch.full_like(lens, t)
        lens += t


def test_two_streams_with_a_workspace_each_and_a_replayed_graph(fa, op, dev):
    q, cache = make(dev, "f16", 4, 1, 8, 2, 3000, 128, [3000, 10, 777, 1500], page=16, seed=9)
    lens = torch.tensor(cache.lens, device=dev, dtype=torch.int32)
    want = run(op, q, cache, 0.0884)
    torch.cuda.synchronize()
    kc, kp, vc, vp = cache.tensors
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table))
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    side = streams[0]
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
    torch.cuda.synchronize()
    q.copy_(q.flip(0))
    lens.copy_(torch.tensor([9, 8, 700, 1], device=dev))
    graph.replay()
    torch.cuda.synchronize()
    want = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refused_by_the_operator(op, dev):
    q, cache = make(dev, "f16", 2, 1, 4, 2, 64, 64, seed=10)
    kc, kp, vc, vp = cache.tensors
    for args, err in (((q.float(), kc, kp, vc, vp, 0.1), TypeError), ((q, kc, kp, vc[:, :32], vp, 0.1), ValueError),
                      ((q, kc, kp.float(), vc, vp, 0.1), ValueError), ((q[:1], kc, kp, vc, vp, 0.1), ValueError),
                      ((q[0], kc, kp, vc, vp, 0.1), ValueError), ((q[:, :0], kc, kp, vc, vp, 0.1), ValueError), ((q, kc.float(), kp, vc.float(), vp, 0.1), TypeError),
                      ((q, kc, kp, vc, vp, 0.1, torch.zeros(3, device=dev, dtype=torch.int32)), ValueError)):
        with pytest.raises(err):
            op.decode_gqa_u4(*args)


def check_many(q, cache, o, lse, scale):
    """Many query rows go through a copy of the cache in fp16: beside O's rounding, V^ (2^-12 of it), P (2^-12) and K^
    (2^-12 of its elements) are rounded.  Scores are off by at most d = scale * 2^-12 * sum |q k| (and 32-bit parts, taken as
    2^-20 of the same sum), so P by the factors exp(+-2d), and O by at most sum p |V^| (2^-12 + 2^-12 + exp(2d) - 1 ...)."""
    want, want_l, _, _ = reference(q, cache, scale)
    b, t, hq, d = q.shape
    hkv = cache.tensors[0].shape[2]
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        if kc.shape[0] == 0:
            assert not o[i].any() and torch.isinf(lse[i]).all()
            continue
        k, v = u4_unpack(kc, kp), u4_unpack(vc, vp)
        x = q[i].double().abs().view(t, hkv, hq // hkv, d)
        dev = scale * float(torch.einsum("thgd,hd->thg", x, k.abs().amax(0)).max()) * (2.0 ** -12 + 2.0 ** -20)
        top = v.abs().amax(0).repeat_interleave(hq // hkv, 0)[None]             # sum p |V^| <= max |V^|
        tol = top * (2.0 ** -11 + 2.0 ** -18 + np.expm1(2 * dev)) + want[i].abs() * (torch.finfo(q.dtype).eps / 2 + 2.0 ** -12) + 2.0 ** -24
        assert ((o[i].double() - want[i]).abs() <= tol).all()
        fin = torch.isfinite(want_l[i])
        assert torch.equal(torch.isfinite(lse[i]), fin)
        assert ((lse[i].double() - want_l[i])[fin].abs() <= dev + 2.0 ** -18).all()
        # and on average the roundings are as small as theirs are: sqrt of the sum of their squares, 4 of 2^-12 / sqrt(3), doubled
        rel = float((o[i].double() - want[i]).norm() / want[i].norm())
        assert rel < 2 * (2 * 2.0 ** -12 + torch.finfo(q.dtype).eps / 2), rel


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,skv,page,lens", [
    (1, 96, 1, 1, 512, 0, None),                       # the smallest that counts as many rows
    (2, 33, 8, 2, 1100, 16, [1100, 700]),
    (3, 100, 6, 3, 1500, 0, [1500, 40, 0]),            # fewer keys than tokens, and none
    (2, 300, 5, 1, 1027, 64, [1027, 1026]),
])
def test_many_tokens(op, dev, dtype, d, b, t, hq, hkv, skv, page, lens):
    q, cache = make(dev, dtype, b, t, hq, hkv, skv, d, lens, page, seed=t)
    o, lse = run(op, q, cache, d ** -0.5, lens=lens is not None or page != 0)
    check_many(q, cache, o, lse, d ** -0.5)


def test_many_tokens_of_any_magnitude(op, dev):
    """bf16 queries far outside fp16's range, another for each sequence and KV head."""
    b, t, hq, hkv, skv, d = 2, 40, 8, 2, 1024, 64
    q, cache = make(dev, "bf16", b, t, hq, hkv, skv, d, seed=11)
    size = torch.tensor([[1e-9, 1e9], [3e5, 1.0]], device=dev).repeat_interleave(hq // hkv, 1)[:, None, :, None]
    for i in range(2):
        for h in range(2):                             # one magnitude at a time decides the scale
            s = float(size[i, 0, h * 4, 0])
            qs = (q.float() * size).bfloat16()
            o, lse = run(op, qs, cache, 0.125 / s)
            small = qs[i:i + 1, :, h * 4:h * 4 + 4]
            class View:
                tensors = [cache.tensors[0][:, :, h:h + 1]]
                packed = [[(c[:, h:h + 1], p[:, h:h + 1])] for c, p in (cache.packed[0][i], cache.packed[1][i])]
            check_many(small, View, o[i:i + 1, :, h * 4:h * 4 + 4], lse[i:i + 1, :, h * 4:h * 4 + 4], 0.125 / s)


def test_many_tokens_copy_in_parts(op, dev):
    """More sequences than one copy holds (256 MB of K and V): the same bits as sequence by sequence with the same splits."""
    b, t, hq, hkv, skv, d = 3, 16, 32, 8, 24000, 128
    lens = [24000, 17, 20001]
    q, cache = make(dev, "f16", b, t, hq, hkv, skv, d, lens, seed=12)
    o, lse = run(op, q, cache, 0.0884)
    kc, kp, vc, vp = cache.tensors
    for i in range(b):
        oi, li = op.decode_gqa_u4(q[i:i + 1], kc[i:i + 1], kp[i:i + 1], vc[i:i + 1], vp[i:i + 1], 0.0884,
                                  torch.tensor(lens[i:i + 1], device=dev, dtype=torch.int32))
        assert torch.equal(torch.isinf(li), torch.isinf(lse[i:i + 1]))
        fin = torch.isfinite(li)
        assert (li - lse[i:i + 1])[fin].abs().max() < 1e-4 and (oi.float() - o[i:i + 1].float()).abs().max() < 4 * 2.0 ** -11


def test_many_tokens_captured_and_replayed(op, dev):
    q, cache = make(dev, "bf16", 2, 40, 8, 2, 1100, 128, [1100, 900], page=16, seed=13)
    lens = torch.tensor(cache.lens, device=dev, dtype=torch.int32)
    kc, kp, vc, vp = cache.tensors
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
    torch.cuda.synchronize()
    q.copy_(q.flip(0) * 100)
    lens.copy_(torch.tensor([500, 60], device=dev))
    graph.replay()
    torch.cuda.synchronize()
    want = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_tokens_whatever_the_workspace_holds(fa, op, dev, dtype):
    """Rows past a sequence's end are not copied: what lies there, here NaN, reaches nothing."""
    b, t, hq, hkv, skv, d = 3, 50, 8, 2, 1100, 128
    lens = [1100, 513, 7]
    q, cache = make(dev, dtype, b, t, hq, hkv, skv, d, lens, seed=15)
    want, want_l = run(op, q, cache, 0.0884)
    check_many(q, cache, want, want_l, 0.0884)
    kc, kp, vc, vp = cache.tensors
    need = fa.decode_gqa_u4_workspace_bytes(b, hq, hkv, t, skv, d)
    o, lse = torch.full_like(want, float("nan")), torch.full_like(want_l, float("nan"))
    fa.decode_gqa_u4(q, kc, kp, vc, vp, o, lse, b, hq, hkv, skv, d, 0.0884, dtype=dtype, num_q_tokens=t,
                     kv_strides=(kc.stride(0), kc.stride(2), kc.stride(1)),
                     param_strides=(kp.stride(0) // 2, kp.stride(2) // 2, kp.stride(1) // 2),
                     seq_lens=torch.tensor(lens, device=dev, dtype=torch.int32),
                     workspace=torch.full((need,), 255, device=dev, dtype=torch.uint8), workspace_bytes=need,
                     stream=torch.cuda.current_stream())
    assert torch.equal(o, want) and torch.equal(lse, want_l)
