"""Filling KV caches (fa_cache_append) and reading the 4-bit one back (fa_cache_read_u4), against plain forms.

A 16-bit cache is held to the formula in 64 bits (bounds in cache_reference.py); e4m3 and 4-bit caches hold exactly what their
format makes of the rows that the 16-bit cache gets, so they are compared bit for bit."""
import numpy as np
import pytest
import torch

from cache_reference import angles, close16, rotate, u4_pack, u4_unpack

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


class Case:
    """Tokens and caches of one kind, every byte of the caches known beforehand."""

    def __init__(self, dev, dtype="f16", b=2, t=3, hq=4, hkv=2, d=128, skv=64, page=0, head_major=False, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.__dict__.update(dev=dev, dtype=dtype, b=b, t=t, hq=hq, hkv=hkv, d=d, skv=skv, page=page)
        x = torch.randn((b, t, hq + 2 * hkv, d), generator=g, device=dev).to(DT[dtype])
        self.q, self.k, self.v = x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]
        self.n_pages = -(-skv // page) if page else 1
        self.rows = page or skv
        self.blocks = b * self.n_pages + (3 if page else 0)      # some pages belong to nobody
        self.table = torch.randperm(self.blocks, generator=g, device=dev)[:b * self.n_pages].to(torch.int32).view(b, self.n_pages) if page else None
        self.head_major, self.g = head_major, g

    def cache(self, kind):
        shape = (self.blocks, self.hkv, self.rows) if self.head_major else (self.blocks, self.rows, self.hkv)
        view = (lambda x: x.transpose(1, 2)) if self.head_major else (lambda x: x)
        if kind == "u4":
            codes = torch.randint(0, 256, (*shape, self.d // 2), generator=self.g, device=self.dev, dtype=torch.uint8)
            params = torch.randn((*shape, self.d // 64, 2), generator=self.g, device=self.dev).half()
            return view(codes), view(params)
        if kind == "e4m3":
            return view(torch.randint(0, 126, (*shape, self.d), generator=self.g, device=self.dev, dtype=torch.uint8).view(torch.float8_e4m3fn)), None
        return view(torch.randn((*shape, self.d), generator=self.g, device=self.dev).to(DT[self.dtype])), None

    def places(self, lens, num_new=None):
        """(b, t, block, row within, row of the sequence) of every stored token."""
        out = []
        for b in range(self.b):
            n = min(max(lens[b], 0), self.skv)
            for t in range(self.t):
                r = n - self.t + t
                if r < 0 or (num_new is not None and t < self.t - num_new[b]):
                    continue
                if self.page:
                    out.append((b, t, int(self.table[b, r // self.page]), r % self.page, r))
                else:
                    out.append((b, t, b, r, r))
        return out


def _i32(x, dev):
    return None if x is None else torch.tensor(x, device=dev, dtype=torch.int32)


def _bytes(x):
    return x.contiguous().view(torch.uint8)


def _run(op, c, kind, f, lens=None, num_new=None, inter=False, amp=1.0, positions=None, scales=None):
    (kc, kp), (vc, vp) = c.cache(kind), c.cache(kind)
    before = [None if x is None else x.clone() for x in (kc, vc, kp, vp)]
    kw = {} if scales is None else dict(zip(("q_scale", "k_scale", "v_scale"), scales))
    q = op.cache_append(c.q, c.k, c.v, kc, vc, kp, vp, f, _i32(lens, c.dev), c.table, inter, amp, _i32(num_new, c.dev),
                        positions, **kw)
    return q, (kc, vc, kp, vp), before


def _check16(c, q, caches, before, f, lens, num_new=None, inter=False, amp=1.0, positions=None):
    where = c.places(lens, num_new)
    live = {(b, t) for b, t, *_ in where}
    kc, vc = caches[0].clone(), caches[1].clone()
    for b, t, blk, row, r in where:
        p = r if positions is None else int(positions[b, t])
        ang = angles(np.array(p), f) if f is not None else np.zeros((0,))
        for got, x in ((q[b, t], c.q[b, t]), (kc[blk, row], c.k[b, t])):
            want, size = rotate(x.double().cpu().numpy(), ang[None], inter, amp)
            close16(got, want, size, x.dtype)
        assert torch.equal(vc[blk, row], c.v[b, t])
        kc[blk, row], vc[blk, row] = before[0][blk, row], before[1][blk, row]
    assert torch.equal(_bytes(kc), _bytes(before[0])) and torch.equal(_bytes(vc), _bytes(before[1]))   # nothing else was touched
    for b in range(c.b):
        for t in range(c.t):
            if (b, t) not in live:
                assert not _bytes(q[b, t]).any()


SHAPES = [
    # dtype, b, t, hq, hkv, d, skv, page, head_major, lens, num_new
    ("f16", 1, 1, 1, 1, 64, 1, 0, False, None, None),
    ("bf16", 3, 1, 8, 2, 128, 100, 16, False, [100, 1, 17], None),
    ("f16", 2, 5, 6, 3, 64, 40, 16, True, [40, 3], None),                 # fewer rows than tokens
    ("bf16", 4, 7, 5, 1, 128, 33, 0, True, [33, 0, -4, 99], [7, 3, 2, 0]),    # no rows; lengths out of range; padding
    ("f16", 2, 40, 4, 4, 128, 64, 32, False, [64, 41], [0, 40]),
    ("bf16", 1, 300, 3, 1, 64, 300, 0, False, None, [123]),
    ("f16", 2, 3, 300, 300, 128, 5, 0, False, [5, 2], None),              # many KV heads
    ("bf16", 3, 801, 3, 1, 64, 900, 0, True, [900, 850, 3], None),        # the largest blocks, across sequences
    ("f16", 2, 1201, 4, 2, 128, 1300, 16, False, [1300, 1250], [1201, 700]),
]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_append_16bit(op, dev, shape, inter):
    dtype, b, t, hq, hkv, d, skv, page, hm, lens, new = shape
    c = Case(dev, dtype, b, t, hq, hkv, d, skv, page, hm, seed=b * 100 + t)
    f, _ = op.rope_frequencies(d)
    q, caches, before = _run(op, c, "16", f, lens, new, inter)
    _check16(c, q, caches, before, f, lens or [skv] * b, new, inter)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("kind", ["e4m3", "u4"])
@pytest.mark.parametrize("shape", SHAPES)
def test_append_quantised(op, dev, shape, kind, inter):
    dtype, b, t, hq, hkv, d, skv, page, hm, lens, new = shape
    if kind == "e4m3" and d != 128:
        pytest.skip("e4m3 caches are d_head 128")
    c = Case(dev, dtype, b, t, hq, hkv, d, skv, page, hm, seed=b * 100 + t)
    f, _ = op.rope_frequencies(d, 5e5)
    q16, (k16, v16, *_), _ = _run(op, c, "16", f, lens, new, inter)
    scales = None
    if kind == "e4m3":
        # one head's values leave the range on purpose
        scales = [torch.linspace(0.001, 0.02, b * hkv, device=dev) for _ in range(3)]
    q, caches, before = _run(op, c, kind, f, lens, new, inter, scales=scales)
    got = [None if x is None else x.clone() for x in caches]
    where = c.places(lens or [skv] * b, new)
    for bb, tt, blk, row, _ in where:
        for i, x16 in ((0, k16), (1, v16)):
            x = x16[blk, row]
            if kind == "u4":
                codes, params = u4_pack(x)
                assert torch.equal(got[i][blk, row], codes)
                assert torch.equal(got[2 + i][blk, row], params)
                got[2 + i][blk, row] = before[2 + i][blk, row]
            else:
                inv = (1.0 / scales[1 + i]).view(b, hkv)[bb]
                want = (x.float() * inv[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                assert torch.equal(_bytes(got[i][blk, row]), _bytes(want))
            got[i][blk, row] = before[i][blk, row]
        if kind == "e4m3":
            inv = (1.0 / scales[0]).view(b, hkv)[bb].repeat_interleave(hq // hkv)
            want = (q16[bb, tt].float() * inv[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            assert torch.equal(_bytes(q[bb, tt]), _bytes(want))
    for g, o in zip(got, before):
        assert g is None or torch.equal(_bytes(g), _bytes(o))
    if kind == "u4":
        assert torch.equal(q, q16)


def test_append_without_rotation_without_q_and_with_positions(fa, op, dev):
    c = Case(dev, "f16", 2, 4, 4, 2, 64, 32, 16, seed=3)
    q, caches, before = _run(op, c, "16", None, [9, 32])
    _check16(c, q, caches, before, None, [9, 32])
    assert torch.equal(q, c.q)
    f, amp = op.rope_frequencies(32, scaling="parts", factor=2.0, original_length=64, slow=1, fast=8)
    pos = torch.tensor([[5, 5, 1000003, 0], [1, 2, 3, 2 ** 31 - 1]], device=dev)
    q, caches, before = _run(op, c, "16", f, [9, 32], amp=amp, positions=pos)
    _check16(c, q, caches, before, f, [9, 32], amp=amp, positions=pos)
    kc, vc = c.cache("16")[0], c.cache("16")[0]
    st = kc.stride()
    fa.cache_append(c.k.contiguous(), c.v.contiguous(), kc, vc, 2, 4, 2, 32, 64, dtype="f16", cache_dtype="f16",
                    kv_strides=(st[0], st[2], st[1]), block_table=c.table, block_table_stride=2, page_size=16,
                    num_pages=c.blocks, seq_lens=_i32([9, 32], dev), inv_freq=f, rotary_dim=32, amplitude=amp, positions=pos.int(),
                    stream=torch.cuda.current_stream())
    for _, _, blk, row, _ in c.places([9, 32]):
        assert torch.equal(kc[blk, row], caches[0][blk, row]) and torch.equal(vc[blk, row], caches[1][blk, row])


@pytest.mark.parametrize("kind", ["16", "u4"])
def test_rows_of_pages_that_do_not_exist_are_dropped(op, dev, kind):
    """The page numbers -1, one past the pool and the largest int: their rows are left out, the others stored, and reading
    them gives zero."""
    c = Case(dev, "f16", 1, 64, 2, 1, 64, 64, 16, seed=4)
    good = c.table.clone()
    c.table[0, 1], c.table[0, 2], c.table[0, 3] = -1, c.blocks, 2 ** 31 - 1
    q, caches, before = _run(op, c, kind, None)
    page = int(good[0, 0])
    for got, old in zip(caches, before):
        if got is not None:
            a, o = got.clone(), old.clone()
            a[page], o[page] = 0, 0
            assert torch.equal(_bytes(a), _bytes(o))
    assert torch.equal(q, c.q)
    if kind == "u4":
        k, v = op.cache_read_u4(caches[0], caches[2], caches[1], caches[3], 1, 64, torch.float16, None, None, c.table)
        codes, params = u4_pack(c.k[0, :16])
        assert torch.equal(k[0, :16], u4_unpack(codes, params).half())
        assert not k[0, 16:].any() and not v[0, 16:].any()


def test_u4_values_at_the_edges(op, dev):
    """Constant groups, subnormal ranges, the largest values, infinities and NaN."""
    d, big = 64, 65504.0
    rows = torch.zeros((10, d), device=dev)
    rows[0] = 3.25                                       # no range: scale 0
    rows[1, 7] = 2.0 ** -24                              # a range below the smallest scale
    rows[2] = torch.linspace(0, 2.0 ** -20, d)
    rows[3] = torch.linspace(-big, big, d)
    rows[4], rows[4, 0] = 1.0, float("inf")
    rows[5], rows[5, 1] = 1.0, float("-inf")
    rows[6, 9] = float("nan")
    rows[7] = -0.0
    rows[8] = torch.linspace(1000, 1001, d)
    rows[9, ::2] = -1.0
    for dtype in (torch.float16, torch.bfloat16):
        k = rows.to(dtype).view(1, 10, 1, d)
        if dtype == torch.bfloat16:
            k = k.clone()
            k[0, 4, 0, 3] = 3e38                         # past fp16
        codes, params = op.u4_cache(1, 10, 1, d, dev)
        vcodes, vparams = op.u4_cache(1, 10, 1, d, dev)
        op.cache_append(k, k, k, codes, vcodes, params, vparams, None)
        want_c, want_p = u4_pack(k[0])
        nan = want_p.isnan()
        assert torch.equal(params[0].isnan(), nan) and nan[6].all() and not nan[:6].any()
        assert torch.equal(torch.nan_to_num(params[0].float()), torch.nan_to_num(want_p.float()))
        keep = [i for i in range(10) if i != 6]
        assert torch.equal(codes[0][keep], want_c[keep])
        assert torch.equal(vcodes, codes)
        out, _ = op.cache_read_u4(codes, params, vcodes, vparams, 1, 10, dtype)
        assert out[0, 6].isnan().all() and torch.isfinite(out[0, keep].float()).all()
        x, y = k[0, keep].double().clamp(-big, big), out[0, keep].double()
        # half a step of the levels, the levels' own rounding (scale: 15 codes of 2^-11, or 2^-25 where subnormal), the
        # offset's where it is subnormal, and the 16-bit result's rounding
        s = params[0, keep][..., 0].double()
        tol = s * (0.5 + 15 * 2.0 ** -11) + 16 * 2.0 ** -25 + y.abs() * torch.finfo(dtype).eps / 2
        assert ((x - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("b,hkv,d,skv,page,hm,n,lens,first", [
    (1, 1, 64, 1, 0, False, 1, None, None),
    (2, 3, 128, 200, 16, True, 200, [200, 37], None),
    (3, 2, 64, 333, 0, True, 70, [333, 60, 0], [263, -3, 0]),
    (2, 8, 128, 1024, 256, False, 513, [1000, 2000], [511, 400]),
    (1, 2, 128, 90, 0, False, 300, None, [2 ** 31 - 5]),
])
def test_read(op, dev, dtype, b, hkv, d, skv, page, hm, n, lens, first):
    c = Case(dev, dtype, b, 1, hkv, hkv, d, skv, page, hm, seed=n)
    (kc, kp), (vc, vp) = c.cache("u4"), c.cache("u4")
    k, v = op.cache_read_u4(kc, kp, vc, vp, b, n, DT[dtype], _i32(first, dev), _i32(lens, dev), c.table)
    for got, codes, params in ((k, kc, kp), (v, vc, vp)):
        want = torch.zeros_like(got)
        x = u4_unpack(codes, params).float().to(DT[dtype])         # exact sums of 32 bits at most, rounded once more
        for bb in range(b):
            length = min(lens[bb], skv) if lens else skv
            f = first[bb] if first else 0
            for i in range(n):
                r = f + i
                if 0 <= r < length:
                    blk, row = (int(c.table[bb, r // page]), r % page) if page else (bb, r)
                    want[bb, i] = x[blk, row]
        assert torch.equal(got, want)


def test_refused_by_the_operators(op, dev):
    c = Case(dev, "f16", 2, 3, 4, 2, 128, 64, seed=5)
    f, _ = op.rope_frequencies(128)
    k16, _ = c.cache("16")
    (kc, kp), (vc, vp) = c.cache("u4"), c.cache("u4")
    bad = [
        (dict(k_cache=k16.bfloat16(), v_cache=k16.bfloat16()), TypeError),
        (dict(v_cache=k16[:, :32]), ValueError),
        (dict(k_cache=k16[..., ::2], v_cache=k16[..., ::2]), ValueError),
        (dict(k_cache=k16[:1], v_cache=k16[:1]), ValueError),
        (dict(k_cache=kc, v_cache=vc), TypeError),
        (dict(k_cache=kc, v_cache=vc, k_params=kp), TypeError),
        (dict(k_cache=kc, v_cache=vc, k_params=kp, v_params=vp[:, :32]), ValueError),
        (dict(k_cache=kc, v_cache=vc, k_params=kp.float(), v_params=vp.float()), ValueError),
        (dict(q=c.q.bfloat16()), TypeError), (dict(k=c.k[:, :2]), ValueError), (dict(seq_lens=torch.zeros(3, device=dev, dtype=torch.int32)), ValueError),
        (dict(positions=torch.zeros(2, device=dev, dtype=torch.int32)), ValueError), (dict(inv_freq=f.to(dev)), TypeError),
        (dict(k_cache=k16.to(torch.float8_e4m3fn), v_cache=k16.to(torch.float8_e4m3fn)), ValueError),
        (dict(block_table=torch.zeros((1, 2), device=dev, dtype=torch.int32)), ValueError),
    ]
    for change, err in bad:
        args = dict(q=c.q, k=c.k, v=c.v, k_cache=k16.clone(), v_cache=k16.clone(), k_params=None, v_params=None, inv_freq=f)
        args.update(change)
        with pytest.raises(err):
            op.cache_append(**args)
    with pytest.raises(TypeError):
        op.cache_read_u4(kc, kp, vc, vp, 2, 3, torch.float32)


def test_append_then_attention(fa, op, dev):
    """A prompt by fa_rope and fa_prefill at once, and the same prompt in chunks through a paged cache and
    decode_gqa: the same attention.  f16: both round q and k alike (the same kernels' arithmetic), P and O each
    within a few steps: 4 * 2^-11 of values of order 1."""
    b, s, hq, hkv, d, page = 2, 90, 4, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn((b, s, hq + 2 * hkv, d), generator=g, device=dev).half()
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]
    f, _ = op.rope_frequencies(d)
    qr, kr = op.rope(q.transpose(1, 2), k.transpose(1, 2), f)
    want, _ = op.prefill(qr, kr.repeat_interleave(2, 1), v.transpose(1, 2).repeat_interleave(2, 1).contiguous(), 0.125, True)
    table = torch.randperm(12, generator=g, device=dev).to(torch.int32).view(2, 6)
    kc, vc = (torch.full((12, page, hkv, d), float("nan"), device=dev, dtype=torch.float16) for _ in range(2))
    done = 0
    for t in (40, 1, 1, 48):
        done += t
        lens = torch.full((b,), done, device=dev, dtype=torch.int32)
        qc = op.cache_append(q[:, done - t:done], k[:, done - t:done], v[:, done - t:done], kc, vc, None, None, f, lens, table)
        assert torch.equal(qc, qr[:, :, done - t:done].transpose(1, 2))
        o, _ = op.decode_gqa(qc, kc, vc, 0.125, lens, table)
        assert (o.transpose(1, 2).float() - want[:, :, done - t:done].float()).abs().max() < 4 * 2.0 ** -11 * float(want.abs().max())
    assert done == s


def test_captured_and_replayed(op, dev):
    c = Case(dev, "bf16", 3, 2, 4, 2, 128, 50, 16, True, seed=7)
    f, _ = op.rope_frequencies(128)
    (kc, kp), (vc, vp) = c.cache("u4"), c.cache("u4")
    lens = torch.tensor([50, 9, 2], device=dev, dtype=torch.int32)

    def step():
        q = op.cache_append(c.q, c.k, c.v, kc, vc, kp, vp, f, lens, c.table)
        return (q, *op.cache_read_u4(kc, kp, vc, vp, 3, 50, torch.bfloat16, None, lens, c.table))

    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    lens.copy_(torch.tensor([30, 41, 1], device=dev))
    c.q.copy_(c.q.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    for a, x in zip(outs, step()):
        assert torch.equal(a, x)
