"""The operators around attention as a server strings them together, in the types and layouts that one test alone does not have."""
import numpy as np
import pytest
import torch

from cache_reference import u4_unpack
from test_cache_gpu import Case, _i32
from test_decode_u4_gpu import DT, Cache, check, check_many, make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def _held(table, lens, kc, kp, vc, vp):
    """What a paged cache holds, as the checks want it."""
    class View:
        tensors = [kc, kp, vc, vp]
        packed = [[], []]
    for i, n in enumerate(lens.tolist()):
        blk = table[i].long()
        for out, (c, p) in zip(View.packed, ((kc, kp), (vc, vp))):
            out.append((c[blk].flatten(0, 1)[:n], p[blk].flatten(0, 1)[:n]))
    return View


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,hq,hkv,cap,prompts", [
    (128, 8, 2, 96, [40, 33, 7]),           # few rows or a short cache
    (64, 6, 2, 640, [130, 600, 1]),         # a chunk of many rows, by the copy; its padding too
])
def test_prompt_then_tokens(op, dev, dtype, d, hq, hkv, cap, prompts):
    """A left-padded batch of prompts in one chunk, one token twice, then three at a time: rotation, append, attention."""
    b, page = len(prompts), 16
    g = torch.Generator(device=dev).manual_seed(d)
    f, amp = op.rope_frequencies(d, 5e5, "smooth", 8.0, 64, 1, 4)
    n = cap // page
    table = torch.randperm(b * n + 2, generator=g, device=dev)[:b * n].to(torch.int32).view(b, n)
    (kc, kp), (vc, vp) = op.u4_cache(b * n + 2, page, hkv, d, dev), op.u4_cache(b * n + 2, page, hkv, d, dev)
    lens = torch.tensor(prompts, device=dev, dtype=torch.int32)
    new, t = lens.clone(), max(prompts)
    for step in range(4):
        x = torch.randn((b, t, hq + 2 * hkv, d), generator=g, device=dev).to(DT[dtype])
        for i in range(b):                                     # what a padded token holds is nobody's business
            x[i, :max(t - int(new[i]), 0)] = float("nan")
        q = op.cache_append(x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:], kc, vc, kp, vp, f, lens, table, True, amp, new)
        o, lse = op.decode_gqa_u4(q, kc, kp, vc, vp, d ** -0.5, lens, table)
        many = t * hq // hkv >= 96 and cap >= 512
        (check_many if many else check)(q, _held(table, lens, kc, kp, vc, vp), o, lse, d ** -0.5, *(() if many else (cap,)))
        t = 1 if step < 2 else 3
        new = torch.full_like(lens, t)
        lens += t


@pytest.mark.parametrize("t", [1, 4, 40])
@pytest.mark.parametrize("page", [0, 16])
def test_e4m3_append_then_attention(fa, op, dev, t, page):
    """q, K and V as e4m3 codes from cache_append, then fa_decode_gqa on them, against 64 bits over what codes and scales stand for.
    There P is rounded to fp16 (2^-11 of each term), O to bf16; scores are sums of exact products in 32 bits (2^-20 of sum |q k|)."""
    lens = [200, 77]
    c = Case(dev, "bf16", 2, t, 8, 2, 128, 200, page, seed=t)
    f, _ = op.rope_frequencies(128)
    scales = [torch.linspace(a, 2 * a, 4, device=dev) for a in (0.012, 0.01, 0.009)]
    kv = [x.clone().view(torch.uint8) for x in (c.cache("e4m3")[0], c.cache("e4m3")[0])]
    kc, vc = (((x.float() / 126 - 0.5) * 400).to(torch.float8_e4m3fn) for x in kv)         # older rows: of order 1 under the scales
    q = op.cache_append(c.q, c.k, c.v, kc, vc, None, None, f, _i32(lens, dev), c.table, q_scale=scales[0], k_scale=scales[1], v_scale=scales[2])
    o, lse = torch.empty((2, t, 8, 128), device=dev, dtype=torch.bfloat16), torch.empty((2, t, 8), device=dev)
    kw = dict(block_table=c.table, block_table_stride=c.n_pages, page_size=page, num_pages=c.blocks, kv_page_stride=kc.stride(0)) if page else {}
    need = fa.decode_workspace_bytes(2, t * 8, 128, fa.decode_gqa_default_splits(2, 2, 200))
    fa.decode_gqa(q, kc, vc, o, lse, 2, 8, 2, 200, 128, 0.0884, dtype="e4m3", num_q_tokens=t, kv_strides=(kc.stride(0), kc.stride(2), kc.stride(1)),
                  seq_lens=_i32(lens, dev), q_scale=scales[0], k_scale=scales[1], v_scale=scales[2],
                  workspace=torch.empty(need, device=dev, dtype=torch.uint8), workspace_bytes=need, stream=torch.cuda.current_stream(), **kw)
    for i, n in enumerate(lens):
        k, v = ((x[c.table[i].long()].flatten(0, 1) if page else x[i])[:n].double() for x in (kc, vc))
        sq, sk, sv = (s.double().view(2, 2)[i] for s in scales)
        k, v = k * sk[:, None], v * sv[:, None]
        x = q[i].double().view(t, 2, 4, 128) * sq[None, :, None, None]
        s = torch.einsum("thgd,nhd->thgn", x, k) * 0.0884
        see = torch.arange(n, device=dev)[None] <= (n - t + torch.arange(t, device=dev))[:, None]
        s = s.masked_fill(~see[:, None, None, :], float("-inf"))
        p = torch.softmax(s, -1)
        want, size = torch.einsum("thgn,nhd->thgd", p, v), torch.einsum("thgn,nhd->thgd", p, v.abs())
        off = 0.0884 * float(torch.einsum("thgd,hd->thg", x.abs(), k.abs().amax(0)).max()) * 2.0 ** -20
        tol = size * (2.0 ** -11 + np.expm1(2 * off) + 2.0 ** -18) + n * 2.0 ** -25 * v.abs().max() + want.abs() * 2.0 ** -8
        assert ((o[i].double().view_as(want) - want).abs() <= tol).all()
        assert ((lse[i].double().view(t, 2, 4) - torch.logsumexp(s, -1)).abs() <= off + 2.0 ** -18).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page", [0, 64])
def test_many_tokens_copy_in_parts(op, dev, dtype, page):
    """More sequences than one copy of 256 MB holds, 128 rows a KV head, each of a size of its own: offsets of every part, against 64
    bits."""
    b, t, hq, hkv, skv, d = 4, 32, 32, 8, 24000, 128
    lens = [24000, 17, 20001, 23999]
    q, cache = make(dev, dtype, b, t, hq, hkv, skv, d, lens, page, seed=12)
    q = (q.float() * torch.exp2(torch.randint(-6, 1, (b, t, hq, 1), device=dev, generator=torch.Generator(device=dev).manual_seed(1)).float())).to(q.dtype)
    o, lse = run(op, q, cache, 0.0884)
    check_many(q, cache, o, lse, 0.0884)


def test_registered_operators_keep_their_contracts(op, dev):
    """Schemas (what is written, what aliases), shapes without data, and tracing, as torch checks them."""
    check_op = torch.library.opcheck
    g = torch.Generator(device=dev).manual_seed(2)
    f, _ = op.rope_frequencies(64)
    q, k = (torch.randn((2, h, 9, 64), generator=g, device=dev).half() for h in (4, 2))
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    check_op(torch.ops.fa_b200.rope, (q, k, f), test_utils=tests)
    check_op(torch.ops.fa_b200.rope, (q.clone().requires_grad_(), k, f, torch.arange(9, device=dev), True, 1.5), test_utils=tests + ("test_aot_dispatch_static",))
    (kc, kp), (vc, vp) = op.u4_cache(2, 32, 2, 64, dev), op.u4_cache(2, 32, 2, 64, dev)
    x, y = q.transpose(1, 2), k.transpose(1, 2)
    lens = torch.tensor([9, 20], device=dev, dtype=torch.int32)
    check_op(torch.ops.fa_b200.cache_append, (x, y, y, kc, vc, kp, vp, f, lens), test_utils=tests)
    check_op(torch.ops.fa_b200.cache_append, (x, y, y, torch.zeros((2, 32, 2, 64), device=dev).half(), torch.zeros((2, 32, 2, 64), device=dev).half(), None, None, None),
             test_utils=tests)
    op.cache_append(x, y, y, kc, vc, kp, vp, f, lens)
    check_op(torch.ops.fa_b200.cache_read_u4, (kc, kp, vc, vp, 2, 5, torch.bfloat16, lens), test_utils=tests)
    check_op(torch.ops.fa_b200.decode_gqa_u4, (x, kc, kp, vc, vp, 0.125, lens), test_utils=tests)
