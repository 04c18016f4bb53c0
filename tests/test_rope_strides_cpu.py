"""Strides of fa_rope's results: rows that would fall together are refused, on the host."""
import ctypes

import pytest


def _rope(fa, **kw):
    base = dict(q=16, k=16, q_out=32, k_out=24, batch_size=2, num_q_heads=4, num_kv_heads=2, seq_len=8, d_head=64,
                inv_freq=(ctypes.c_double * 32)(*[1.0] * 32), rotary_dim=64)
    base.update(kw)
    names = ("q", "k", "q_out", "k_out", "batch_size", "num_q_heads", "num_kv_heads", "seq_len", "d_head", "inv_freq", "rotary_dim")
    return fa.rope_raw(*[base.pop(n) for n in names], **base)


@pytest.mark.parametrize("change", [
    dict(q_out_strides=(0, 512, 64)), dict(q_out_strides=(2048, 0, 64)), dict(q_out_strides=(2048, 512, 0)),
    dict(k_out_strides=(0, 512, 64)), dict(k_out_strides=(1024, 0, 64)), dict(k_out_strides=(1024, 512, 0)),
    dict(q=32, q_strides=(0, 512, 64), q_out_strides=(0, 512, 64)),            # in place: turned once for each sequence
])
def test_rows_that_fall_together(fa, change):
    assert _rope(fa, **change) == fa.FA_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change", [
    dict(), dict(q_strides=(0, 512, 64)), dict(k_strides=(0, 0, 64)),           # inputs may be expanded
    dict(batch_size=1, q_out_strides=(0, 512, 64)), dict(num_q_heads=1, q_out_strides=(512, 0, 64)),
    dict(seq_len=1, q_out_strides=(256, 64, 0), k_out_strides=(128, 64, 0)),
])
def test_strides_that_are_taken(fa, change):
    """Past the strides, the next check is the alignment of k_out."""
    assert _rope(fa, **change) == fa.FA_ERR_MISALIGNED
