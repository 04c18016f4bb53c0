"""PyTorch custom operators over the C ABI: ``torch.ops.fa_b200.prefill`` / ``decode`` /
``decode_gqa`` / ``prefill_backward`` / ``rope`` / ``cache_append`` / ``cache_read_u4`` /
``decode_gqa_u4``.

``prefill`` is differentiable with respect to q, k and v (``fa_backward``); the gradient of its LSE
output is not supported.  ``rope`` is differentiable with respect to q and k.  The others are forward
only.  Tensors use the layout of
``torch.nn.functional.scaled_dot_product_attention``: ``[B, H, S, D]``,
contiguous, fp16 or bf16, on a CUDA device; the kernels see them as the
reference's ``[B*H, S, D]`` (include/flash_attention.h:46-61).  The operators
launch on the current CUDA stream of the tensors' device and allocate their
outputs (and the decode workspace) with torch.

``sdpa()`` is a convenience with the keyword names of
``scaled_dot_product_attention`` for the cases this library covers.

There is no fallback: on a machine without the library or without a B200-class
GPU the operators raise.
"""
from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import is_in_torch_dispatch_mode

import fa_b200 as _fa
from fa_b200 import FaError

_DTYPES = {torch.float16: "f16", torch.bfloat16: "bf16"}
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_HERE = contextlib.nullcontext()


def _check(q, k, v):
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("fa_b200: q, k, v must share dtype float16 or bfloat16")
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("fa_b200: tensors must be on a CUDA device (there is no CPU path)")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("fa_b200: expected [B, H, S, D] tensors")


@torch.library.custom_op("fa_b200::prefill", mutates_args=())
def prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
            causal: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Self-attention forward.  Returns (O [B,H,S,D] in the input dtype, LSE [B,H,S] fp32, natural log)."""
    _check(q, k, v)
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("fa_b200::prefill: q, k, v must have the same shape")
    b, h, s, d = q.shape
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q)
    lse = torch.empty((b, h, s), device=q.device, dtype=torch.float32)
    with torch.cuda.device(q.device):
        _fa.prefill(q, k, v, o, lse, b, h, s, d, float(scale), bool(causal), dtype=_DTYPES[q.dtype],
                    stream=torch.cuda.current_stream(q.device))
    return o, lse


@prefill.register_fake
def _(q, k, v, scale, causal):
    b, h, s, _ = q.shape
    return torch.empty_like(q), q.new_empty((b, h, s), dtype=torch.float32)


@torch.library.custom_op("fa_b200::prefill_backward", mutates_args=())
def prefill_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                     d_o: torch.Tensor, scale: float, causal: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dQ, dK, dV) of ``prefill`` for the upstream gradient ``d_o`` of O."""
    _check(q, k, v)
    b, h, s, d = q.shape
    q, k, v, o, d_o, lse = (t.contiguous() for t in (q, k, v, o, d_o.to(q.dtype), lse))
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    with torch.cuda.device(q.device):
        wsb = _fa.backward_workspace_bytes(b, h, s)
        ws = torch.empty(wsb, device=q.device, dtype=torch.uint8)
        _fa.backward(q, k, v, o, d_o, lse, dq, dk, dv, b, h, s, d, float(scale), bool(causal),
                     dtype=_DTYPES[q.dtype], workspace=ws, workspace_bytes=wsb,
                     stream=torch.cuda.current_stream(q.device))
    return dq, dk, dv


@prefill_backward.register_fake
def _(q, k, v, o, lse, d_o, scale, causal):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def _prefill_setup_context(ctx, inputs, output):
    q, k, v, scale, causal = inputs
    o, lse = output
    ctx.save_for_backward(q, k, v, o, lse)
    ctx.scale, ctx.causal = scale, causal


def _prefill_backward(ctx, d_o, d_lse):
    q, k, v, o, lse = ctx.saved_tensors
    dq, dk, dv = prefill_backward(q, k, v, o, lse, d_o, ctx.scale, ctx.causal)
    return dq, dk, dv, None, None


torch.library.register_autograd("fa_b200::prefill", _prefill_backward, setup_context=_prefill_setup_context)


@torch.library.custom_op("fa_b200::decode", mutates_args=())
def decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
           num_splits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """One query row per head against a KV cache: q [B,H,1,D], k/v [B,H,Skv,D].

    Returns (O [B,H,1,D], LSE [B,H,1]).  ``num_splits`` 0 picks the library default."""
    _check(q, k, v)
    b, h, one, d = q.shape
    if one != 1 or k.shape[:2] != (b, h) or k.shape[3] != d or v.shape != k.shape:
        raise ValueError("fa_b200::decode: expected q [B,H,1,D] and k, v [B,H,Skv,D]")
    skv = k.shape[2]
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q)
    lse = torch.empty((b, h, 1), device=q.device, dtype=torch.float32)
    with torch.cuda.device(q.device):
        splits = num_splits if num_splits > 0 else _fa.decode_default_splits(b, h, skv)
        ws_bytes = _fa.decode_workspace_bytes(b, h, d, splits)
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8)
        _fa.decode(q, k, v, o, lse, None, b, h, skv, d, float(scale), dtype=_DTYPES[q.dtype],
                   num_splits=splits, workspace=ws, workspace_bytes=ws_bytes,
                   stream=torch.cuda.current_stream(q.device))
    return o, lse


@decode.register_fake
def _(q, k, v, scale, num_splits):
    b, h, _, _ = q.shape
    return torch.empty_like(q), q.new_empty((b, h, 1), dtype=torch.float32)


@torch.library.custom_op("fa_b200::decode_gqa", mutates_args=())
def decode_gqa(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scale: float,
               seq_lens: torch.Tensor | None = None,
               block_table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Grouped-query attention of new tokens over a KV cache (``fa_decode_gqa``).

    q ``[B, T, Hq, D]`` (the T tokens are the last T cache entries of each sequence; token t sees keys
    up to its own position).  Cache, not paged: ``[B, Skv, Hkv, D]``; paged (``block_table`` int32
    ``[B, max_pages]``): page pools ``[P, page_size, Hkv, D]``.  ``seq_lens`` int32 ``[B]`` optional.
    Returns (O ``[B, T, Hq, D]``, LSE ``[B, T, Hq]``)."""
    if q.dtype not in _DTYPES or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise TypeError("fa_b200::decode_gqa: q and the cache must share dtype float16 or bfloat16")
    if not (q.is_cuda and k_cache.is_cuda and v_cache.is_cuda):
        raise RuntimeError("fa_b200: tensors must be on a CUDA device (there is no CPU path)")
    if q.dim() != 4 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("fa_b200::decode_gqa: expected q [B,T,Hq,D] and 4-D caches of equal shape")
    b, t, hq, d = q.shape
    q, k_cache, v_cache = q.contiguous(), k_cache.contiguous(), v_cache.contiguous()
    hkv = k_cache.shape[2]
    kw = {}
    if block_table is None:
        if k_cache.shape[0] != b:
            raise ValueError("fa_b200::decode_gqa: cache batch differs from q")
        skv = k_cache.shape[1]
        kw["kv_strides"] = (skv * hkv * d, d, hkv * d)
    else:
        n_pages, page = k_cache.shape[0], k_cache.shape[1]
        block_table = block_table.to(torch.int32).contiguous()
        skv = block_table.shape[1] * page
        kw.update(kv_strides=(0, d, hkv * d), block_table=block_table, block_table_stride=block_table.shape[1],
                  page_size=page, num_pages=n_pages, kv_page_stride=page * hkv * d)
    if seq_lens is not None:
        kw["seq_lens"] = seq_lens.to(torch.int32).contiguous()
    o = torch.empty_like(q)
    lse = torch.empty((b, t, hq), device=q.device, dtype=torch.float32)
    with torch.cuda.device(q.device):
        group = hq // hkv
        n_qt = -(-t // max(1, min(t, 128 // group)))
        splits = _fa.decode_gqa_default_splits(b * n_qt, hkv, skv)
        ws_bytes = _fa.decode_workspace_bytes(b, t * hq, d, splits)
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8)
        _fa.decode_gqa(q, k_cache, v_cache, o, lse, b, hq, hkv, skv, d, float(scale), dtype=_DTYPES[q.dtype],
                       num_splits=splits, num_q_tokens=t, workspace=ws, workspace_bytes=ws_bytes,
                       stream=torch.cuda.current_stream(q.device), **kw)
    return o, lse


@decode_gqa.register_fake
def _(q, k_cache, v_cache, scale, seq_lens=None, block_table=None):
    b, t, hq, _ = q.shape
    return torch.empty_like(q), q.new_empty((b, t, hq), dtype=torch.float32)


def _rows(t: torch.Tensor, what: str, elem_per_16: int = 8, copy: bool = False) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """A 4-D tensor with the strides of its first three dimensions, as the library wants them: contiguous last dimension,
    16-byte multiples.  Another one is copied if ``copy``, else refused."""
    if t.is_contiguous() and t.shape[3] % elem_per_16 == 0 and t.data_ptr() % 16 == 0:
        _, n1, n2, n3 = t.shape
        return t, (n1 * n2 * n3, n2 * n3, n3)

    def strides(x):
        return tuple(x.shape[3] if n == 1 else s for n, s in zip(x.shape[:3], x.stride()[:3]))

    st = strides(t)
    if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % elem_per_16 == 0 for s in st) and (any(st) or not copy):
        return t, st
    if not copy:
        raise ValueError(f"fa_b200: {what} needs a contiguous last dimension and strides of multiples of 16 bytes")
    t = t.clone(memory_format=torch.contiguous_format)
    return t, strides(t)


def _inv_freq(f: torch.Tensor) -> torch.Tensor:
    if f.is_cuda or f.dim() != 1 or f.dtype != torch.float64:
        raise TypeError("fa_b200: inv_freq is a 1-D float64 tensor in CPU memory (rope_frequencies makes one)")
    return f.contiguous()


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
                     original_length: float = 0.0, slow: float = 0.0, fast: float = 0.0) -> tuple[torch.Tensor, float]:
    """(inv_freq, amplitude) for ``rope`` and ``cache_append``: radians per position of each pair (``fa_rope_inv_freq``)."""
    out, amp = _fa.rope_inv_freq(rotary_dim, base, scaling, factor, original_length, slow, fast)
    return torch.tensor(list(out), dtype=torch.float64), amp


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on(device: torch.device):
    """torch.cuda.device(device), at no cost where it is the current one."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _run_rope(q, k, inv_freq, positions, interleaved, amplitude, inverse):
    dtype, device, q_shape, k_shape = q.dtype, q.device, q.shape, k.shape
    if dtype not in _DTYPES or k.dtype != dtype:
        raise TypeError("fa_b200: q and k must share dtype float16 or bfloat16")
    if not (q.is_cuda and k.is_cuda):
        raise RuntimeError("fa_b200: tensors must be on a CUDA device (there is no CPU path)")
    if len(q_shape) != 4 or len(k_shape) != 4 or q_shape[0] != k_shape[0] or q_shape[2:] != k_shape[2:] or k.device != device:
        raise ValueError("fa_b200::rope: expected q [B,Hq,S,D] and k [B,Hkv,S,D] on one device")
    b, hq, s, d = q_shape
    hkv = k_shape[1]
    inv_freq = _inv_freq(inv_freq)
    (q, qs), (k, ks) = _rows(q, "q", copy=True), _rows(k, "k", copy=True)
    q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q_shape)      # the first costs half
    k_out = torch.empty_like(k) if k.is_contiguous() else k.new_empty(k_shape)
    pos_stride = 0
    if positions is not None:
        if positions.is_floating_point() or tuple(positions.shape) not in ((s,), (b, s)) or positions.device != device:
            raise ValueError("fa_b200::rope: positions are integers [S] or [B, S] on q's device")
        positions = positions.to(torch.int32).contiguous()
        pos_stride = s if positions.dim() == 2 else 0
    with _on(device):
        _fa.rope(q, k if hkv else None, q_out, k_out if hkv else None, b, hq, hkv, s, d, inv_freq.data_ptr(), 2 * inv_freq.numel(),
                 interleaved, amplitude, _DTYPES[dtype], positions, pos_stride, 0, inverse, qs, ks, stream=_stream(device))
    return q_out, k_out


@torch.library.custom_op("fa_b200::rope", mutates_args=())
def _rope_op(q: torch.Tensor, k: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor | None = None,
             interleaved: bool = False, amplitude: float = 1.0, inverse: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    if forward_ad._current_level >= 0:                         # a tangent need not be visible down here, and would be lost
        raise NotImplementedError("fa_b200::rope: the registered operator has no forward-mode derivative; call rope() of this module")
    return _run_rope(q, k, inv_freq, positions, interleaved, amplitude, inverse)


@_rope_op.register_fake
def _(q, k, inv_freq, positions=None, interleaved=False, amplitude=1.0, inverse=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rope_setup_context(ctx, inputs, output):
    _, _, inv_freq, positions, interleaved, amplitude, inverse = inputs
    ctx.save_for_backward(inv_freq, positions)                 # so that autograd sees if one is overwritten in between
    ctx.how = interleaved, amplitude, not inverse


def _rope_backward(ctx, d_q, d_k):
    """The map is linear: its gradient is the transposed one, the rotation back (with the same amplitude)."""
    d_q, d_k = rope(d_q, d_k, *ctx.saved_tensors, *ctx.how)
    return d_q, d_k, None, None, None, None, None


torch.library.register_autograd("fa_b200::rope", _rope_backward, setup_context=_rope_setup_context)


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, interleaved, amplitude, inverse):
        _rope_setup_context(ctx, (q, k, inv_freq, positions, interleaved, amplitude, inverse), None)
        return _run_rope(q, k, inv_freq, positions, interleaved, amplitude, inverse)

    @staticmethod
    def backward(ctx, d_q, d_k):
        return _rope_backward(ctx, d_q, d_k)


class _RopeForwardMode(torch.autograd.Function):
    """_Rope in the form that forward-mode differentiation takes, at two to three times its host time a call."""

    @staticmethod
    def forward(q, k, inv_freq, positions, interleaved, amplitude, inverse):
        return _run_rope(q, k, inv_freq, positions, interleaved, amplitude, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _rope_setup_context(ctx, inputs, output)
        ctx.save_for_forward(inputs[2], inputs[3])
        ctx.zeros = inputs[0].new_zeros, inputs[0].shape, inputs[1].shape

    @staticmethod
    def backward(ctx, d_q, d_k):
        return _rope_backward(ctx, d_q, d_k)

    @staticmethod
    def jvp(ctx, d_q, d_k, *_):
        """The map is linear: its tangents are those of its inputs, turned."""
        zeros, q_shape, k_shape = ctx.zeros
        d_q, d_k = zeros(q_shape) if d_q is None else d_q, zeros(k_shape) if d_k is None else d_k
        interleaved, amplitude, back = ctx.how
        return rope(d_q, d_k, *ctx.saved_tensors, interleaved, amplitude, not back)


def rope(q: torch.Tensor, k: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor | None = None,
         interleaved: bool = False, amplitude: float = 1.0, inverse: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions (``fa_rope``) of q ``[B, Hq, S, D]`` and k ``[B, Hkv, S, D]`` (any strides; Hkv may be 0).

    ``inv_freq`` float64 ``[rotary_dim / 2]`` in CPU memory; ``positions`` integer ``[S]`` or ``[B, S]`` on the device
    (taken as int32), default 0 .. S-1; ``inverse`` turns back.  Returns the rotated (q, k), contiguous.

    ``torch.ops.fa_b200.rope`` is the same; plain tensors in eager mode go to the kernel without the dispatcher, whose
    20 us a call (50 with a gradient) a short prompt would feel; and forward-mode tangents are known here alone."""
    if forward_ad._current_level >= 0 and not torch.compiler.is_compiling():
        return _RopeForwardMode.apply(q, k, inv_freq, positions, interleaved, amplitude, inverse)
    if (type(q) in _PLAIN and type(k) in _PLAIN and not torch.compiler.is_compiling() and not is_in_torch_dispatch_mode()
            and not torch._C._is_tracing() and not torch._C._are_functorch_transforms_active()):
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
            return _Rope.apply(q, k, inv_freq, positions, interleaved, amplitude, inverse)
        return _run_rope(q, k, inv_freq, positions, interleaved, amplitude, inverse)
    return torch.ops.fa_b200.rope(q, k, inv_freq, positions, interleaved, amplitude, inverse)


def u4_cache(blocks: int, rows: int, num_kv_heads: int, d_head: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An empty (zero) 4-bit cache for K or V: codes uint8 ``[blocks, rows, Hkv, D/2]`` and params fp16
    ``[blocks, rows, Hkv, D/64, 2]`` (scale, offset).  A block is a page or a whole sequence.  The rows of a head lie
    together (both are views of ``[blocks, Hkv, rows, ...]``), which is how attention reads them."""
    codes = torch.zeros((blocks, num_kv_heads, rows, d_head // 2), device=device, dtype=torch.uint8)
    params = torch.zeros((blocks, num_kv_heads, rows, d_head // 64, 2), device=device, dtype=torch.float16)
    return codes.transpose(1, 2), params.transpose(1, 2)


def _param_strides(p: torch.Tensor, codes: torch.Tensor, d: int) -> tuple[int, int, int]:
    """(block, head, row) strides of the params of a 4-bit cache, in pairs."""
    g = d // 64
    if p.device != codes.device:
        raise ValueError("fa_b200: codes and params of a 4-bit cache are on one device")
    if p.dtype != torch.float16 or tuple(p.shape) != (*codes.shape[:3], g, 2):
        raise ValueError("fa_b200: params of a 4-bit cache are float16 [blocks, rows, Hkv, D/64, 2]")
    st = [2 * g if n == 1 else s for n, s in zip(p.shape[:3], p.stride()[:3])]
    if p.stride(4) != 1 or (g > 1 and p.stride(3) != 2) or any(s % (2 * g) for s in st) or p.data_ptr() % 16:
        raise ValueError("fa_b200: the pairs of a 4-bit cache's row must be contiguous and aligned")
    return st[0] // 2, st[2] // 2, st[1] // 2


def _cache_kw(k, v, d, batch, seq_lens, block_table, k_params=None, v_params=None) -> tuple[int, dict]:
    """(seq_len_kv, keyword arguments) that describe a cache ``[blocks, rows, Hkv, ...]`` to the library."""
    u4 = k_params is not None or v_params is not None
    if k.dim() != 4 or v.shape != k.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("fa_b200: expected 4-D caches of equal shape")
    if u4 and (k_params is None or v_params is None or k.dtype != torch.uint8):
        raise TypeError("fa_b200: a 4-bit cache is uint8 codes with the params of both K and V")
    if k.shape[3] != (d // 2 if u4 else d):
        raise ValueError("fa_b200: the cache's rows do not have q's head dimension")
    per_16 = 16 // k.element_size()
    (_, ks), (_, vs) = _rows(k, "k_cache", per_16), _rows(v, "v_cache", per_16)
    if ks != vs:
        raise ValueError("fa_b200: k_cache and v_cache must have the same strides")
    kw = dict(kv_strides=(ks[0], ks[2], ks[1]))
    if u4:
        kw["param_strides"] = _param_strides(k_params, k, d)
        if _param_strides(v_params, v, d) != kw["param_strides"]:
            raise ValueError("fa_b200: k_params and v_params must have the same strides")
    rows = k.shape[1]
    if block_table is None:
        if k.shape[0] != batch:
            raise ValueError("fa_b200: cache batch differs from the tokens'")
    else:
        if block_table.dim() != 2 or block_table.shape[0] != batch:
            raise ValueError("fa_b200: block_table is [B, max_pages]")
        block_table = block_table.to(device=k.device, dtype=torch.int32).contiguous()
        kw.update(block_table=block_table, block_table_stride=block_table.shape[1], page_size=rows, num_pages=k.shape[0])
        rows *= block_table.shape[1]
    if seq_lens is not None:
        kw["seq_lens"] = _per_sequence(seq_lens, batch, k.device, "seq_lens")
    return rows, kw


def _per_sequence(t, batch, device, what):
    if t.is_floating_point() or tuple(t.shape) != (batch,):
        raise ValueError(f"fa_b200: {what} is integers [B]")
    return t.to(device=device, dtype=torch.int32).contiguous()


@torch.library.custom_op("fa_b200::cache_append", mutates_args=("k_cache", "v_cache", "k_params", "v_params"))
def cache_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 k_params: torch.Tensor | None, v_params: torch.Tensor | None, inv_freq: torch.Tensor | None,
                 seq_lens: torch.Tensor | None = None, block_table: torch.Tensor | None = None,
                 interleaved: bool = False, amplitude: float = 1.0,
                 num_new: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 q_scale: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """The newest T tokens into a KV cache, with the rotation of q and k on the way (``fa_cache_append``).

    q ``[B, T, Hq, D]``, k, v ``[B, T, Hkv, D]`` (heads of a token contiguous); caches ``[B, Skv, Hkv, D]`` or page pools
    ``[P, page_size, Hkv, D]`` with ``block_table`` int32 ``[B, max_pages]``, of any strides, in q's dtype, as e4m3 codes
    (``torch.float8_e4m3fn`` with float32 ``{q,k,v}_scale [B * Hkv]``) or in 4 bits (``u4_cache``: uint8 codes with
    params; the others have None there).  ``inv_freq`` None: no rotation.  ``seq_lens [B]`` counts the new tokens in.  Returns the rotated q (e4m3 codes for an e4m3 cache)."""
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("fa_b200::cache_append: q, k, v must share dtype float16 or bfloat16")
    if not all(t.is_cuda and t.device == q.device for t in (q, k, v, k_cache, v_cache)):
        raise RuntimeError("fa_b200: tensors must be on one CUDA device (there is no CPU path)")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or (*q.shape[:2], q.shape[3]) != (*k.shape[:2], k.shape[3]):
        raise ValueError("fa_b200::cache_append: expected q [B,T,Hq,D] and k, v [B,T,Hkv,D]")
    b, t, hq, d = q.shape
    hkv = k.shape[2]
    if k_cache.shape[2] != hkv:
        raise ValueError("fa_b200::cache_append: the cache has another number of KV heads")
    e4m3 = k_cache.dtype == torch.float8_e4m3fn
    if k_params is None and not e4m3 and k_cache.dtype != q.dtype:
        raise TypeError("fa_b200::cache_append: a 16-bit cache has q's dtype")
    skv, kw = _cache_kw(k_cache, v_cache, d, b, seq_lens, block_table, k_params, v_params)
    tokens, strides = [], []
    for x in (q, k, v):                                        # heads side by side, one stride from token to token
        st = x.stride(1) if t > 1 else x.stride(0) if b > 1 else x.shape[2] * d
        ok = x.stride(3) == 1 and (x.shape[2] == 1 or x.stride(2) == d) and (b == 1 or t == 1 or x.stride(0) == t * st)
        if not ok or st % 8 or st < x.shape[2] * d or x.data_ptr() % 16:
            x, st = x.clone(memory_format=torch.contiguous_format), x.shape[2] * d
        tokens.append(x)
        strides.append(st)
    if e4m3:
        for n, sc in (("q_scale", q_scale), ("k_scale", k_scale), ("v_scale", v_scale)):
            if sc is None or sc.numel() != b * hkv or sc.dtype != torch.float32 or sc.device != q.device:
                raise ValueError(f"fa_b200::cache_append: an e4m3 cache needs {n}, float32 [B * Hkv]")
            kw[n] = sc.contiguous()
    if num_new is not None:
        kw["num_new"] = _per_sequence(num_new, b, q.device, "num_new")
    if positions is not None:
        if positions.is_floating_point() or tuple(positions.shape) != (b, t):
            raise ValueError("fa_b200::cache_append: positions are integers [B, T]")
        kw["positions"] = positions.to(device=q.device, dtype=torch.int32).contiguous()
    if inv_freq is not None:
        inv_freq = _inv_freq(inv_freq)
        kw.update(inv_freq=inv_freq.data_ptr(), rotary_dim=2 * inv_freq.numel(), interleaved=interleaved, amplitude=float(amplitude))
    q_out = torch.empty((b, t, hq, d), device=q.device, dtype=k_cache.dtype if e4m3 else q.dtype)
    with _on(q.device):
        _fa.cache_append(tokens[1], tokens[2], k_cache, v_cache, b, t, hkv, skv, d, dtype=_DTYPES[q.dtype],
                         cache_dtype="u4" if k_params is not None else "e4m3" if e4m3 else _DTYPES[q.dtype], q=tokens[0],
                         q_out=q_out, num_q_heads=hq, token_strides=tuple(strides), k_params=k_params, v_params=v_params,
                         stream=_stream(q.device), **kw)
    return q_out


@cache_append.register_fake
def _(q, k, v, k_cache, v_cache, k_params, v_params, inv_freq, seq_lens=None, block_table=None, interleaved=False,
      amplitude=1.0, num_new=None, positions=None, q_scale=None, k_scale=None, v_scale=None):
    return q.new_empty(q.shape, dtype=k_cache.dtype if k_cache.dtype == torch.float8_e4m3fn else q.dtype)


@torch.library.custom_op("fa_b200::cache_read_u4", mutates_args=())
def cache_read_u4(k_cache: torch.Tensor, k_params: torch.Tensor, v_cache: torch.Tensor, v_params: torch.Tensor,
                  batch: int, num_rows: int, dtype: torch.dtype, first_rows: torch.Tensor | None = None,
                  seq_lens: torch.Tensor | None = None,
                  block_table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``first_rows[b]`` (default 0) and on of a 4-bit cache (as for ``cache_append``) as K, V
    ``[B, num_rows, Hkv, D]`` in ``dtype``; zero where a sequence has no such row."""
    if dtype not in _DTYPES:
        raise TypeError("fa_b200::cache_read_u4: dtype is float16 or bfloat16")
    if not all(t.is_cuda and t.device == k_cache.device for t in (k_cache, k_params, v_cache, v_params)):
        raise RuntimeError("fa_b200: tensors must be on one CUDA device (there is no CPU path)")
    d, hkv = 2 * k_cache.shape[-1], k_cache.shape[2]
    skv, kw = _cache_kw(k_cache, v_cache, d, batch, seq_lens, block_table, k_params, v_params)
    if first_rows is not None:
        kw["first_rows"] = _per_sequence(first_rows, batch, k_cache.device, "first_rows")
    k, v = (torch.empty((batch, num_rows, hkv, d), device=k_cache.device, dtype=dtype) for _ in range(2))
    with _on(k_cache.device):
        _fa.cache_read_u4(k_cache, k_params, v_cache, v_params, k, v, batch, hkv, skv, d, num_rows, dtype=_DTYPES[dtype],
                          stream=_stream(k_cache.device), **kw)
    return k, v


@cache_read_u4.register_fake
def _(k_cache, k_params, v_cache, v_params, batch, num_rows, dtype, first_rows=None, seq_lens=None, block_table=None):
    shape = (batch, num_rows, k_cache.shape[2], 2 * k_cache.shape[3])
    return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)


@torch.library.custom_op("fa_b200::decode_gqa_u4", mutates_args=())
def decode_gqa_u4(q: torch.Tensor, k_cache: torch.Tensor, k_params: torch.Tensor, v_cache: torch.Tensor,
                  v_params: torch.Tensor, scale: float, seq_lens: torch.Tensor | None = None,
                  block_table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``decode_gqa`` over a 4-bit cache (``fa_decode_gqa_u4``): codes uint8 ``[B, Skv, Hkv, D/2]`` or page pools
    ``[P, page_size, Hkv, D/2]``, params fp16 ``[..., D/64, 2]``, of any strides (``u4_cache``).

    q ``[B, T, Hq, D]``; returns (O ``[B, T, Hq, D]``, LSE ``[B, T, Hq]``)."""
    if q.dtype not in _DTYPES:
        raise TypeError("fa_b200::decode_gqa_u4: q is float16 or bfloat16")
    if not all(t.is_cuda and t.device == q.device for t in (q, k_cache, k_params, v_cache, v_params)):
        raise RuntimeError("fa_b200: tensors must be on one CUDA device (there is no CPU path)")
    if q.dim() != 4:
        raise ValueError("fa_b200::decode_gqa_u4: expected q [B,T,Hq,D]")
    b, t, hq, d = q.shape
    if t == 0:                                                 # to the library 0 is the default, one token
        raise ValueError("fa_b200::decode_gqa_u4: q has no tokens")
    skv, kw = _cache_kw(k_cache, v_cache, d, b, seq_lens, block_table, k_params, v_params)
    hkv = k_cache.shape[2]
    q, _ = _rows(q.contiguous(), "q", copy=True)
    o = torch.empty_like(q)
    lse = torch.empty((b, t, hq), device=q.device, dtype=torch.float32)
    with _on(q.device):
        ws_bytes = _fa.decode_gqa_u4_workspace_bytes(b, hq, hkv, t, skv, d)
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8)
        _fa.decode_gqa_u4(q, k_cache, k_params, v_cache, v_params, o, lse, b, hq, hkv, skv, d, float(scale),
                          dtype=_DTYPES[q.dtype], num_q_tokens=t, workspace=ws, workspace_bytes=ws_bytes,
                          stream=_stream(q.device), **kw)
    return o, lse


@decode_gqa_u4.register_fake
def _(q, k_cache, k_params, v_cache, v_params, scale, seq_lens=None, block_table=None):
    b, t, hq, _ = q.shape
    return q.new_empty(q.shape), q.new_empty((b, t, hq), dtype=torch.float32)


def sdpa(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attn_mask=None,
         dropout_p: float = 0.0, is_causal: bool = False, scale: float | None = None) -> torch.Tensor:
    """``scaled_dot_product_attention`` for the cases the library covers (no mask, no dropout).

    Self-attention (equal sequence lengths) runs the prefill kernel; a single query row against a
    longer cache runs split-KV decode.  Anything else raises: there is no fallback."""
    if attn_mask is not None or dropout_p != 0.0:
        raise NotImplementedError("fa_b200.sdpa: attn_mask and dropout are not supported")
    d = query.shape[-1]
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(d)
    if query.shape[-2] == key.shape[-2]:
        return prefill(query, key, value, sc, bool(is_causal))[0]
    if query.shape[-2] == 1 and not is_causal:
        return decode(query, key, value, sc, 0)[0]
    raise NotImplementedError("fa_b200.sdpa: only self-attention and single-row decode are covered")


__all__ = ["prefill", "prefill_backward", "decode", "decode_gqa", "rope", "rope_frequencies", "cache_append",
           "cache_read_u4", "decode_gqa_u4", "u4_cache", "sdpa", "FaError"]
