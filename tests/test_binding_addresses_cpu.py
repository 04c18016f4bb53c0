"""What the ctypes binding of the operators around attention takes for an address: device pointers as numbers or tensors, and
host doubles that are there, for the frequencies."""
import ctypes

import pytest
import torch


def _rope(fa, **kw):
    base = dict(q=16, k=None, q_out=24, k_out=None, batch_size=1, num_q_heads=4, num_kv_heads=0, seq_len=8, d_head=64,
                inv_freq=torch.ones(32, dtype=torch.float64), rotary_dim=64)
    base.update(kw)
    return fa.rope_raw(*[base[n] for n in ("q", "k", "q_out", "k_out", "batch_size", "num_q_heads", "num_kv_heads", "seq_len", "d_head",
                                           "inv_freq", "rotary_dim")])


@pytest.mark.parametrize("name", ["q", "q_out"])
@pytest.mark.parametrize("value", [ctypes.c_void_p(32), (ctypes.c_byte * 64)(), "32"])
def test_device_pointers_are_numbers_or_tensors(fa, name, value):
    """A ctypes object's own address lies on the host, where a kernel must not be sent."""
    with pytest.raises((TypeError, AttributeError)):
        _rope(fa, **{name: value})
    with pytest.raises((TypeError, AttributeError)):
        fa.cache_append_raw(value, 16, 16, 16, 1, 1, 1, 64, 64)
    with pytest.raises((TypeError, AttributeError)):
        fa.cache_read_u4_raw(16, value, 16, 16, 16, 16, 1, 1, 64, 64, 1)
    with pytest.raises((TypeError, AttributeError)):
        fa.decode_gqa_u4_raw(16, 16, 16, 16, 16, 16, value, 1, 1, 1, 64, 64, 0.1)


@pytest.mark.parametrize("value", [
    torch.ones(31, dtype=torch.float64), torch.ones(64, dtype=torch.float32), torch.ones(64, dtype=torch.int64),
    torch.ones(64, dtype=torch.float64)[::2], torch.ones(32, dtype=torch.float64, device="meta"), (ctypes.c_double * 31)(),
    (ctypes.c_float * 64)(), ctypes.c_double(1.0), [1.0] * 32,
])
def test_frequencies_that_are_not_there(fa, value):
    """Too few, of another type, with gaps, or not in host memory: they would be read past their end."""
    with pytest.raises((TypeError, ValueError)):
        _rope(fa, inv_freq=value)
    with pytest.raises((TypeError, ValueError)):
        fa.cache_append_raw(16, 16, 16, 16, 1, 1, 1, 64, 64, inv_freq=value, rotary_dim=64)


@pytest.mark.parametrize("value", [torch.ones(32, dtype=torch.float64), torch.ones(40, dtype=torch.float64), (ctypes.c_double * 32)(*[1.0] * 32)])
def test_frequencies_that_are(fa, value):
    """Past the frequencies, the next check is the alignment of q_out; an address is taken as it is."""
    address = value.data_ptr() if isinstance(value, torch.Tensor) else ctypes.addressof(value)
    assert _rope(fa, inv_freq=value) == _rope(fa, inv_freq=address) == fa.FA_ERR_MISALIGNED
    assert fa.cache_append_raw(16, 16, 24, 16, 1, 1, 1, 64, 64, inv_freq=value, rotary_dim=64, kv_strides=(4096, 64, 64)) == fa.FA_ERR_MISALIGNED
