"""Plain 64-bit forms of the rotary positions and the 4-bit cache, shared by the GPU tests.

Rounding bounds.  A result of fa_rope: cos and sin are rounded to 32 bits (2^-24 relative each), two products and a sum
likewise, so the 32-bit value is off by at most 4 * 2^-24 * amplitude * (|x1| + |x2|) (two roundings reach each product, one the
sum, with slack for the amplitude's own product); then one rounding to 16 bits, half a step: eps / 2 relative, and
half the smallest subnormal step of fp16, 2^-25."""
import numpy as np
import torch


def angles(positions, inv_freq):
    """[..., R/2] in 64 bits; positions an integer array."""
    return np.asarray(positions, dtype=np.float64)[..., None] * np.asarray(inv_freq, dtype=np.float64)


def rotate(x, ang, interleaved, amplitude=1.0, inverse=False):
    """x [..., D] float64, ang broadcastable to [..., R/2].  Returns (y, bound of |x1| + |x2| per element)."""
    x = np.asarray(x, dtype=np.float64)
    r = 2 * ang.shape[-1]
    c, s = amplitude * np.cos(ang), amplitude * np.sin(ang) * (-1 if inverse else 1)
    i1, i2 = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
    y, size = x.copy(), np.zeros_like(x)
    a, b = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = a * c - b * s, b * c + a * s
    size[..., i1] = size[..., i2] = amplitude * (np.abs(a) + np.abs(b))
    return y, size


def close16(got, want, size, dtype):
    """Every element within the bound above."""
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    half_step = torch.finfo(dtype).eps / 2
    err32 = 4 * 2.0 ** -24 * size
    tol = err32 + half_step * (np.abs(want) + err32) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want)[bad].max()))


def u4_pack(x):
    """Codes and params of 16-bit rows [..., D] (torch, any device), every operation in fp32 as the format says."""
    g = x.float().clamp(-65504, 65504).unflatten(-1, (-1, 64))
    z = g.amin(-1).half()
    s = ((g.amax(-1) - z.float()) * (1.0 / 15.0)).half()
    inv = torch.where(s.float() > 0, 1.0 / s.float(), torch.zeros_like(s.float()))
    c = ((g - z.float()[..., None]) * inv[..., None]).round().clamp(0, 15)
    c = torch.where(c.isnan(), torch.zeros_like(c), c).to(torch.uint8).flatten(-2)
    return c[..., ::2] | (c[..., 1::2] << 4), torch.stack((s, z), -1)


def u4_unpack(codes, params):
    """Values in 64 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 64)).double()
    return (params[..., 1:].double() + params[..., :1].double() * c).flatten(-2)
