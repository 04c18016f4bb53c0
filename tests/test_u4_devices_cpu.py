"""A 4-bit cache whose parts lie on different devices is refused before anything is launched (meta tensors stand in for the GPU's)."""
import pytest
import torch


@pytest.fixture(scope="module")
def op(fa):
    import __graft_entry__ as ge
    return ge.load_module("torch_op")


def test_params_on_another_device(op):
    (kc, kp), (vc, vp) = op.u4_cache(2, 32, 2, 64, device="meta"), op.u4_cache(2, 32, 2, 64, device="meta")
    rows, kw = op._cache_kw(kc, vc, 64, 2, None, None, kp, vp)
    assert rows == 32 and kw["param_strides"] == (64, 32, 1)
    for k_params, v_params in ((torch.empty_like(kp, device="cpu"), vp), (kp, torch.empty_like(vp, device="cpu"))):
        with pytest.raises(ValueError, match="device"):
            op._cache_kw(kc, vc, 64, 2, None, None, k_params, v_params)


@pytest.mark.gpu
def test_params_on_the_host(op, dev):
    """Every operator that takes them; refused on the host, so nothing is written."""
    (kc, kp), (vc, vp) = op.u4_cache(1, 32, 2, 64, device=dev), op.u4_cache(1, 32, 2, 64, device=dev)
    x = torch.ones((1, 1, 2, 64), device=dev, dtype=torch.float16)
    for k_params, v_params in ((kp.cpu(), vp), (kp, vp.cpu())):
        for call in (lambda: op.cache_append(x, x, x, kc, vc, k_params, v_params, None),
                     lambda: op.cache_read_u4(kc, k_params, vc, v_params, 1, 4, torch.float16),
                     lambda: op.decode_gqa_u4(x, kc, k_params, vc, v_params, 0.1)):
            with pytest.raises((ValueError, RuntimeError), match="device"):
                call()
    assert not kc.any() and not vc.any()
