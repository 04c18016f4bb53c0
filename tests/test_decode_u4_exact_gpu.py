"""fp16 attention of many rows over a 4-bit cache counts K^ and V^ with the digits that the few-row kernel gives them.

K^ and V^ go in as fp16 values and remainders (22 bits), so what is rounded to fewer bits than 32 is P and O, to fp16 each.
A rounding to fp16 is off by 2^-10 / sqrt(12) of its binade's lower end on average, which over values spread evenly by their logarithm is
sqrt(0.541 / 12) * 2^-10 = 2.07e-4 of the value; the terms of O are of either sign and rounded independently of one another, so P's
roundings are 2.07e-4 of O's norm as O's own are: together 2.93e-4.  (With K^ and V^ rounded as well, 4.1e-4.)"""
import numpy as np
import pytest
import torch

from cache_reference import u4_unpack
from test_decode_u4_gpu import Cache, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def check_f16(q, cache, o, lse, scale):
    """Below the border (96 rows a KV head, 128 with d_head 128) it is P times V's scale that is rounded, half a step of
    p |s (c - 8)| <= p (|V^| + |z + 8 s|), `amount` of the reference.  From there on P's rounding, half a step (2^-11) of a term
    and at least 2^-25 of V^ on a sum of P of 1 or more; 22 bits of V^; scores off by scale * sum |q k| (2^-22 + 2^-20), the second
    for 32-bit sums; O's half step.  Element by element, and the norm of it all."""
    want, want_l, amount, _ = reference(q, cache, scale)
    b, t, hq, d = q.shape
    hkv = cache.tensors[0].shape[2]
    few = t * hq // hkv < (128 if d == 128 else 96)
    for i in range(b):
        (kc, kp), (vc, vp) = cache.packed[0][i], cache.packed[1][i]
        n = kc.shape[0]
        if n == 0:
            assert not o[i].any() and torch.isinf(lse[i]).all()
            continue
        k, v = u4_unpack(kc, kp), u4_unpack(vc, vp)
        x = q[i].double().view(t, hkv, hq // hkv, d)
        off = scale * float(torch.einsum("thgd,hd->thg", x.abs(), k.abs().amax(0)).max()) * (2.0 ** -22 + 2.0 ** -20)
        see = torch.arange(n, device=q.device)[None] <= (n - t + torch.arange(t, device=q.device))[:, None]
        s = (torch.einsum("thgd,nhd->thgn", x, k) * scale).masked_fill(~see[:, None, None, :], float("-inf"))
        p = torch.softmax(s, -1).nan_to_num()
        size = amount[i] if few else torch.einsum("thgn,nhd->thgd", p, v.abs()).reshape(t, hq, d)
        tol = size * (2.0 ** -11 + 2.0 ** -18 + np.expm1(2 * off)) + n * 2.0 ** -25 * float(v.abs().max()) + want[i].abs() * 2.0 ** -11 + 2.0 ** -25
        assert ((o[i].double() - want[i]).abs() <= tol).all()
        fin = torch.isfinite(want_l[i])
        assert torch.equal(torch.isfinite(lse[i]), fin) and ((lse[i].double() - want_l[i])[fin].abs() <= off + 2.0 ** -18).all()
        rel = float((o[i].double() - want[i]).norm() / want[i].norm())
        assert rel < 1.15 * 2.93e-4, rel


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,skv,page,lens", [
    (1, 96, 1, 1, 512, 0, None),                       # the smallest that counts as many rows (d_head 64)
    (1, 128, 1, 1, 512, 0, None),                      # (d_head 128)
    (2, 33, 8, 2, 1100, 16, [1100, 700]),
    (3, 100, 6, 3, 1500, 0, [1500, 140, 0]),
    (2, 300, 5, 1, 1027, 64, [1027, 1026]),            # several query tiles, a ragged one
    (1, 512, 8, 8, 513, 0, None),                      # a prompt from next to nothing, one key past a tile
    (8, 64, 16, 2, 4000, 0, None),                     # several tiles a CTA, several items
    (1, 32, 4, 1, 30000, 16, [29999]),                 # split over the keys, and merged
    (4, 127, 2, 2, 2000, 0, [2000, 1999, 127, 1]),     # a row below the border of d_head 128
    (2, 1, 128, 1, 700, 0, [700, 3]),                  # one token of a group that fills a query tile
    (2, 2, 300, 3, 5000, 16, [4999, 2500]),            # a group of 100, split over the keys
])
def test_many_rows(op, dev, d, b, t, hq, hkv, skv, page, lens):
    q, cache = make(dev, "f16", b, t, hq, hkv, skv, d, lens, page, seed=t)
    o, lse = run(op, q, cache, d ** -0.5, lens=lens is not None or page != 0)
    check_f16(q, cache, o, lse, d ** -0.5)
    again = run(op, q, cache, d ** -0.5, lens=lens is not None or page != 0)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


def test_more_sequences_than_one_copy_holds(op, dev):
    b, t, hq, hkv, skv, d = 4, 32, 32, 8, 12000, 128           # 128 rows a KV head; 98 MB a sequence, values and remainders
    q, cache = make(dev, "f16", b, t, hq, hkv, skv, d, [12000, 17, 11001, 11999], 64, seed=12)
    o, lse = run(op, q, cache, 0.0884)
    check_f16(q, cache, o, lse, 0.0884)


@pytest.mark.parametrize("lens", [None, [900, 513]])
def test_whatever_the_workspace_holds(fa, op, dev, lens):
    """Rows past a sequence's end are copied in neither half: NaN there reaches nothing."""
    b, t, hq, hkv, skv, d = 2, 50, 8, 2, 900, 128
    q, cache = make(dev, "f16", b, t, hq, hkv, skv, d, lens, seed=15)
    kc, kp, vc, vp = cache.tensors
    need = fa.decode_gqa_u4_workspace_bytes(b, hq, hkv, t, skv, d)
    guard = torch.full((need + 256,), 255, device=dev, dtype=torch.uint8)
    o, lse = torch.full_like(q, float("nan")), torch.full((b, t, hq), float("nan"), device=dev)
    fa.decode_gqa_u4(q, kc, kp, vc, vp, o, lse, b, hq, hkv, skv, d, 0.0884, dtype="f16", num_q_tokens=t,
                     kv_strides=(kc.stride(0), kc.stride(2), kc.stride(1)),
                     param_strides=(kp.stride(0) // 2, kp.stride(2) // 2, kp.stride(1) // 2),
                     seq_lens=None if lens is None else torch.tensor(lens, device=dev, dtype=torch.int32),
                     workspace=guard, workspace_bytes=need, stream=torch.cuda.current_stream())
    check_f16(q, cache, o, lse, 0.0884)
    assert (guard[need:] == 255).all()


def test_small_values(op, dev):
    """V^ and K^ of order 2^-8: the remainder, in steps of 2^-24, still gives 16 times the digits, and the norm is as above."""
    b, t, hq, hkv, n, d = 1, 64, 8, 2, 700, 128
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn((b, t, hq, d), generator=g, device=dev).half()
    k, v = (torch.randn((b, n, hkv, d), generator=g, device=dev) * 2.0 ** -8 for _ in range(2))
    cache = Cache(dev, k.half(), v.half(), [n])
    o, lse = run(op, q, cache, 0.0884 * 2 ** 8)
    check_f16(q, cache, o, lse, 0.0884 * 2 ** 8)


def test_captured_and_replayed(op, dev):
    """The copy of both halves in a graph: new queries and lengths at replay, the same bits as a direct call."""
    q, cache = make(dev, "f16", 2, 40, 8, 2, 1100, 128, [1100, 900], page=16, seed=13)
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
    q.copy_(q.flip(0))
    lens.copy_(torch.tensor([500, 60], device=dev))
    graph.replay()
    torch.cuda.synchronize()
    want = op.decode_gqa_u4(q, kc, kp, vc, vp, 0.0884, lens, cache.table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
