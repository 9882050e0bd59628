"""CPU tier: sizes behind what the C ABI's integers hold are refused by name, never cut to their low bits."""
import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    from sm3det_amd import expert_ops, mx4
    made = []
    monkeypatch.setattr(expert_ops, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(mx4, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(mx4, '_call', lambda *a, **k: made.append(a))
    return made


def _wide(rows, k, dtype):
    """a matrix of no memory"""
    return torch.empty(1, dtype=dtype).as_strided((rows, k), (0, 1), 0) if k == 1 else torch.empty(rows, k, dtype=dtype, device='meta')


@pytest.mark.parametrize('k', ((1 << 31) - 127, 1 << 31, (1 << 32) + 8))
def test_rows_longer_than_32_bits(calls, k):
    from sm3det_amd import mx4
    from sm3det_amd._lib import SM3Error
    with pytest.raises(SM3Error):
        mx4.quantize(_wide(1, k, torch.bfloat16))
    kp = mx4.padded(k)
    with pytest.raises(SM3Error):
        mx4.Mx4Tensor(*(torch.empty(1, kp // d, dtype=torch.uint8, device='meta') for d in (2, 32)), k)
    assert not calls


def test_the_longest_rows_are_taken(calls):
    from sm3det_amd import mx4
    k = (1 << 31) - 128
    assert mx4.quantize(_wide(2, k, torch.float16)).shape == (2, k) and calls.pop()[6:8] == (k, k)


def test_the_abi_refuses_them():
    import ctypes

    from sm3det_amd import _lib
    L, a = _lib.lib(), ctypes.c_void_p(1 << 20)
    k = (1 << 31) - 127
    assert L.sm3_mx4_quantize(a, 0, 1, k, k, a, a, None) == -4 and L.sm3_mx4_dequantize(a, a, 1, k, a, 0, None) == -4


@pytest.mark.parametrize('n,k', ((1 << 31, 8), (8, 1 << 31), (1 << 32, 8)))
def test_products_of_such_sizes(calls, n, k, monkeypatch):
    from sm3det_amd import expert_ops
    from sm3det_amd._lib import SM3Error
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: None)
    off = torch.zeros(2, dtype=torch.int32, device='meta')
    with pytest.raises(SM3Error):
        expert_ops.expert_linear(_wide(3, k, torch.float16), torch.empty(1, n, k, dtype=torch.float16, device='meta'), off)
