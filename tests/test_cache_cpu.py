"""Rotary positions and KV caches without a GPU: refusals on the host, the frequencies, where rows lie, the PyTorch
operators' shapes."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cache_rows(tmp_path):
    exe = tmp_path / "cache_row_host"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "flash-attention-ptx-cuda_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpu", "cache_row_host.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr


def _freqs(n=64):
    return (ctypes.c_double * n)(*[1e4 ** (-i / n) for i in range(n)])


def _rope(fa, **kw):
    base = dict(q=16, k=16, q_out=16, k_out=16, batch_size=1, num_q_heads=4, num_kv_heads=2, seq_len=8, d_head=64,
                inv_freq=_freqs(), rotary_dim=64)
    base.update(kw)
    names = ("q", "k", "q_out", "k_out", "batch_size", "num_q_heads", "num_kv_heads", "seq_len", "d_head", "inv_freq", "rotary_dim")
    return fa.rope_raw(*[base.pop(n) for n in names], **base)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), "INVALID_ARGUMENT"), (dict(q_out=None), "INVALID_ARGUMENT"), (dict(k=None), "INVALID_ARGUMENT"),
    (dict(k=None, k_out=None), "INVALID_ARGUMENT"), (dict(num_kv_heads=0), "INVALID_ARGUMENT"),
    (dict(batch_size=0), "INVALID_ARGUMENT"), (dict(seq_len=0), "INVALID_ARGUMENT"), (dict(num_q_heads=0), "INVALID_ARGUMENT"),
    (dict(inv_freq=None), "INVALID_ARGUMENT"), (dict(rotary_dim=0), "INVALID_ARGUMENT"), (dict(rotary_dim=-16), "INVALID_ARGUMENT"),
    (dict(rotary_dim=24), "UNSUPPORTED"), (dict(rotary_dim=80), "UNSUPPORTED"), (dict(d_head=96), "UNSUPPORTED"),
    (dict(dtype=2), "UNSUPPORTED"), (dict(amplitude=float("nan")), "INVALID_ARGUMENT"),
    (dict(inv_freq=(ctypes.c_double * 32)(*[float("inf")] * 32)), "INVALID_ARGUMENT"),
    (dict(position_offset=2 ** 31 - 8 + 1), "INVALID_ARGUMENT"), (dict(positions=16, positions_stride=-1), "INVALID_ARGUMENT"),
    (dict(q=24), "MISALIGNED"), (dict(q_strides=(4096, 512, 68)), "MISALIGNED"), (dict(k_out_strides=(0, -64, 64)), "INVALID_ARGUMENT"),
    (dict(q_strides=(4096, 64, 256)), "INVALID_ARGUMENT"), (dict(k_out_strides=(4096, 64, 128)), "INVALID_ARGUMENT"),   # in place, elsewhere
    (dict(num_q_heads=2 ** 30, num_kv_heads=2 ** 30), "INVALID_ARGUMENT"), (dict(seq_len=2 ** 31 - 1), "INVALID_ARGUMENT"),
])
def test_rope_refusals(fa, change, code):
    assert _rope(fa, **change) == getattr(fa, "FA_ERR_" + code)


def _append(fa, **kw):
    base = dict(k=16, v=16, k_cache=16, v_cache=16, batch_size=2, num_tokens=3, num_kv_heads=2, seq_len_kv=64, d_head=128,
                q=16, q_out=16, num_q_heads=4, kv_strides=(64 * 256, 128, 256), inv_freq=_freqs(), rotary_dim=128)
    base.update(kw)
    names = ("k", "v", "k_cache", "v_cache", "batch_size", "num_tokens", "num_kv_heads", "seq_len_kv", "d_head")
    return fa.cache_append_raw(*[base.pop(n) for n in names], **base)


def test_append_types_by_name_and_number(fa):
    """Past the types, the next check is the alignment."""
    for dtype, cache in (("f16", None), ("f16", "f16"), (0, "f16"), (1, "bf16"), (1, None), ("bf16", "bf16"), ("bf16", 0)):
        assert _append(fa, dtype=dtype, cache_dtype=cache, k_cache=8) == fa.FA_ERR_MISALIGNED
    for dtype, cache in (("f16", "bf16"), (0, "bf16"), (1, "f16")):
        assert _append(fa, dtype=dtype, cache_dtype=cache, k_cache=8) == fa.FA_ERR_UNSUPPORTED


U4 = dict(cache_dtype="u4", kv_strides=(64 * 128, 64 * 64, 64), param_strides=(256, 128, 2), k_params=16, v_params=16)
E4M3 = dict(cache_dtype="e4m3", q_scale=16, k_scale=16, v_scale=16)
PAGED = dict(block_table=16, block_table_stride=4, page_size=16, num_pages=9)


@pytest.mark.parametrize("change,code", [
    (dict(k=None), "INVALID_ARGUMENT"), (dict(v_cache=None), "INVALID_ARGUMENT"), (dict(q=None), "INVALID_ARGUMENT"),
    (dict(q_out=None), "INVALID_ARGUMENT"), (dict(num_q_heads=3), "INVALID_ARGUMENT"), (dict(num_q_heads=0), "INVALID_ARGUMENT"),
    (dict(num_tokens=0), "INVALID_ARGUMENT"), (dict(num_tokens=65), "INVALID_ARGUMENT"), (dict(seq_len_kv=0), "INVALID_ARGUMENT"),
    (dict(d_head=80), "UNSUPPORTED"), (dict(dtype="e4m3"), "UNSUPPORTED"), (dict(cache_dtype=5), "UNSUPPORTED"),
    (dict(cache_dtype="bf16"), "UNSUPPORTED"), (dict(rotary_dim=40), "UNSUPPORTED"), (dict(rotary_dim=-1), "INVALID_ARGUMENT"),
    (dict(kv_strides=(64 * 256, 128, 120)), "INVALID_ARGUMENT"), (dict(kv_strides=(0, 128, 256)), "INVALID_ARGUMENT"),
    (dict(kv_strides=(64 * 256, 132, 256)), "MISALIGNED"), (dict(token_strides=(512, 260, 256)), "MISALIGNED"),
    (dict(token_strides=(512, 128, 256)), "INVALID_ARGUMENT"), (dict(k_cache=8), "MISALIGNED"),
    (dict(E4M3, k_scale=None), "INVALID_ARGUMENT"), (dict(E4M3, q_scale=None), "INVALID_ARGUMENT"),
    (dict(E4M3, d_head=64, rotary_dim=64), "UNSUPPORTED"), (dict(E4M3, num_kv_heads=1025, num_q_heads=1025), "UNSUPPORTED"), (dict(E4M3, kv_strides=(64 * 256, 136, 256)), "MISALIGNED"),
    (dict(E4M3), "INVALID_ARGUMENT"), (dict(token_strides=(1024, 0, 0)), "INVALID_ARGUMENT"),       # q_out is q, of other places
    (dict(num_kv_heads=2 ** 30, num_q_heads=2 ** 30), "INVALID_ARGUMENT"), (dict(batch_size=2 ** 30, num_tokens=64), "INVALID_ARGUMENT"),
    (dict(U4, k_params=None), "INVALID_ARGUMENT"), (dict(U4, param_strides=(0, 0, 0)), "INVALID_ARGUMENT"),
    (dict(U4, param_strides=(256, 129, 2)), "MISALIGNED"), (dict(U4, kv_strides=(64 * 128, 64 * 64, 56)), "INVALID_ARGUMENT"),
    (dict(U4, kv_strides=(64 * 128, 64 * 64, 72)), "MISALIGNED"),
    (dict(PAGED, page_size=24), "INVALID_ARGUMENT"), (dict(PAGED, page_size=8), "INVALID_ARGUMENT"),
    (dict(PAGED, num_pages=0), "INVALID_ARGUMENT"), (dict(PAGED, block_table_stride=3), "INVALID_ARGUMENT"),
])
def test_append_refusals(fa, change, code):
    assert _append(fa, **change) == getattr(fa, "FA_ERR_" + code)


@pytest.mark.parametrize("change,code", [
    (dict(k_out=None), "INVALID_ARGUMENT"), (dict(k_params=None), "INVALID_ARGUMENT"), (dict(num_rows=0), "INVALID_ARGUMENT"),
    (dict(num_rows=2 ** 31 - 1), "INVALID_ARGUMENT"), (dict(d_head=32), "UNSUPPORTED"), (dict(dtype="e4m3"), "UNSUPPORTED"),
    (dict(v_out=24), "MISALIGNED"), (dict(param_strides=(256, 128, 1)), "INVALID_ARGUMENT"), (dict(PAGED, page_size=48), "INVALID_ARGUMENT"),
])
def test_read_refusals(fa, change, code):
    base = dict(k_cache=16, k_params=16, v_cache=16, v_params=16, k_out=16, v_out=16, batch_size=2, num_kv_heads=2,
                seq_len_kv=64, d_head=128, num_rows=5, kv_strides=U4["kv_strides"], param_strides=U4["param_strides"])
    base.update(change)
    names = ("k_cache", "k_params", "v_cache", "v_params", "k_out", "v_out", "batch_size", "num_kv_heads", "seq_len_kv",
             "d_head", "num_rows")
    assert fa.cache_read_u4_raw(*[base.pop(n) for n in names], **base) == getattr(fa, "FA_ERR_" + code)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), "INVALID_ARGUMENT"), (dict(v_params=None), "INVALID_ARGUMENT"), (dict(o=None), "INVALID_ARGUMENT"),
    (dict(num_q_heads=3), "INVALID_ARGUMENT"), (dict(batch_size=0), "INVALID_ARGUMENT"), (dict(seq_len_kv=0), "INVALID_ARGUMENT"),
    (dict(seq_len_kv=2 ** 31 - 1), "INVALID_ARGUMENT"), (dict(scale=0.0), "INVALID_ARGUMENT"),
    (dict(scale=float("inf")), "INVALID_ARGUMENT"), (dict(num_q_tokens=-1), "INVALID_ARGUMENT"),
    (dict(num_q_tokens=65), "INVALID_ARGUMENT"), (dict(d_head=96), "UNSUPPORTED"), (dict(dtype="e4m3"), "UNSUPPORTED"),
    (dict(kv_strides=(64 * 128, 64 * 64 + 8, 64)), "MISALIGNED"), (dict(param_strides=(257, 128, 2)), "MISALIGNED"),
    (dict(param_strides=(256, 0, 2)), "INVALID_ARGUMENT"), (dict(PAGED, page_size=100), "INVALID_ARGUMENT"),
    (dict(q=24), "MISALIGNED"), (dict(lse=18), "MISALIGNED"),
])
def test_attention_refusals(fa, change, code):
    base = dict(q=16, k_cache=16, k_params=16, v_cache=16, v_params=16, o=16, lse=16, batch_size=2, num_q_heads=4,
                num_kv_heads=2, seq_len_kv=64, d_head=128, scale=0.1, kv_strides=U4["kv_strides"],
                param_strides=U4["param_strides"])
    base.update(change)
    names = ("q", "k_cache", "k_params", "v_cache", "v_params", "o", "lse", "batch_size", "num_q_heads", "num_kv_heads",
             "seq_len_kv", "d_head", "scale")
    assert fa.decode_gqa_u4_raw(*[base.pop(n) for n in names], **base) == getattr(fa, "FA_ERR_" + code)


def test_attention_workspace(fa):
    size = fa.decode_gqa_u4_workspace_bytes
    assert size(0, 4, 2, 1, 64, 128) == size(1, 3, 2, 1, 64, 128) == size(1, 4, 2, 1, 64, 96) == 0
    assert 0 < size(1, 4, 2, 1, 64, 128) <= size(8, 4, 2, 1, 4096, 128) == size(8, 4, 2, 0, 4096, 128)
    assert size(2, 128, 1, 0, 4096, 128) == size(2, 128, 1, 1, 4096, 128) > 0     # no number of tokens: one, of many rows here
    assert size(64, 32, 8, 1, 4096, 128) > 148 * 10 * 8 * 130 * 4 - 1      # parts of the line: 10 records an SM


@pytest.mark.parametrize("name", ["RopeArgs", "CacheAppendArgs", "CacheReadArgs", "DecodeGqaU4Args"])
def test_packed_arguments_have_the_structures_layout(fa, name):
    cls, values, at = getattr(fa, name), [], [0]

    def fill(obj):
        for field, t in obj._fields_:
            if issubclass(t, ctypes.Structure):
                fill(getattr(obj, field))
            else:
                at[0] += 1
                v = at[0] + 0.5 if t in (ctypes.c_float, ctypes.c_double) else at[0]
                setattr(obj, field, v)
                values.append(v)
    obj = cls()
    fill(obj)
    assert fa._packer(cls)(*values) == bytes(obj)


def test_null_arguments(fa):
    lib = fa.lib()
    for name in ("fa_rope", "fa_cache_append", "fa_cache_read_u4", "fa_decode_gqa_u4"):
        assert getattr(lib, name)(None) == fa.FA_ERR_INVALID_ARGUMENT
    assert lib.fa_rope_inv_freq(None, 64, None, None) == fa.FA_ERR_INVALID_ARGUMENT


def _np_inv_freq(dim, base, scaling, factor, length, slow, fast):
    i = np.arange(dim // 2, dtype=np.float64)
    if scaling == "base":
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2 * i / dim)
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        place = [dim * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
        lo, hi = max(math.floor(place[0]), 0), min(math.ceil(place[1]), dim - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f * (1 - ramp) + f / factor * ramp
    if scaling == "smooth":
        mix = np.clip((length * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        return f * mix + f / factor * (1 - mix)
    return f


@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("base", [1e4, 5e5])
@pytest.mark.parametrize("scaling,args", [("plain", (1, 0, 0, 0)), ("linear", (4, 0, 0, 0)), ("base", (8, 0, 0, 0)),
                                          ("parts", (16, 4096, 1, 32)), ("smooth", (8, 8192, 1, 4)), ("parts", (1, 64, 1, 2))])
def test_frequencies(fa, dim, base, scaling, args):
    factor, length, slow, fast = args
    got, amp = fa.rope_inv_freq(dim, base, scaling, factor, length, slow, fast)
    want = _np_inv_freq(dim, base, scaling, factor, length, slow, fast)
    # a power, a product and a sum in doubles: a few roundings of 2^-53, the power's exponent up to ln(base) of them
    np.testing.assert_allclose(np.array(got), want, rtol=64 * 2.0 ** -53)
    assert amp == np.float32(0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0)


@pytest.mark.parametrize("dim,kw", [(24, {}), (0, {}), (256, {}), (64, dict(base=1.0)), (64, dict(scaling="linear", factor=0.5)),
                                    (64, dict(scaling="parts", factor=2)), (64, dict(scaling="smooth", factor=2, original_length=8, slow=2, fast=1))])
def test_frequency_refusals(fa, dim, kw):
    with pytest.raises(fa.FaError):
        fa.rope_inv_freq(dim, **kw)


def test_operators_registered_and_fake_shapes(fa):
    import __graft_entry__ as ge
    op = ge.load_module("torch_op")
    from torch._subclasses.fake_tensor import FakeTensorMode
    f, amp = op.rope_frequencies(64)
    assert f.shape == (32,) and f.dtype == torch.float64 and amp == 1.0
    with FakeTensorMode(allow_non_fake_inputs=True):
        q, k = torch.empty((2, 6, 40, 64), dtype=torch.float16), torch.empty((2, 3, 40, 64), dtype=torch.float16)
        a, b = torch.ops.fa_b200.rope(q, k, f)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == torch.float16
        q, k = torch.empty((2, 5, 6, 128), dtype=torch.bfloat16), torch.empty((2, 5, 3, 128), dtype=torch.bfloat16)
        codes, params = torch.empty((2, 64, 3, 64), dtype=torch.uint8), torch.empty((2, 64, 3, 2, 2), dtype=torch.float16)
        assert torch.ops.fa_b200.cache_append(q, k, k, codes, codes, params, params, f).shape == q.shape
        e = torch.empty((2, 64, 3, 128), dtype=torch.float8_e4m3fn)
        assert torch.ops.fa_b200.cache_append(q, k, k, e, e, None, None, f).dtype == torch.float8_e4m3fn
        o, lse = torch.ops.fa_b200.decode_gqa_u4(q, codes, params, codes, params, 0.1)
        assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (2, 5, 6) and lse.dtype == torch.float32
        kk, vv = torch.ops.fa_b200.cache_read_u4(codes, params, codes, params, 2, 7, torch.float16)
        assert kk.shape == vv.shape == (2, 7, 3, 128) and kk.dtype == torch.float16


def test_cpu_tensors_are_rejected(fa):
    import __graft_entry__ as ge
    op = ge.load_module("torch_op")
    f, _ = op.rope_frequencies(64)
    q = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError):
        op.rope(q, q, f)
    codes, params = op.u4_cache(1, 32, 2, 64, device="cpu")
    assert codes.shape == (1, 32, 2, 32) and params.shape == (1, 32, 2, 1, 2)
    with pytest.raises(RuntimeError):
        op.cache_append(q.transpose(1, 2), q.transpose(1, 2), q.transpose(1, 2), codes, codes, params, params, f)
    with pytest.raises(RuntimeError):
        op.cache_read_u4(codes, params, codes, params, 1, 4, torch.float16)
