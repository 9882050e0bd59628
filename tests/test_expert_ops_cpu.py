"""CPU tier of the grouped 16-bit and 4-bit products: what the entry points refuse, and the C ABI's own checks (nothing here
reaches a launch)."""
import ctypes

import numpy as np
import pytest
import torch

from tests.expert_common import E2M1, quantize_ref, spans


@pytest.fixture(scope='module')
def L():
    from sm3det_amd import _lib
    return _lib.lib()


def test_cpu_tensors_are_refused():
    from sm3det_amd import expert_ops, mx4
    from sm3det_amd._lib import SM3Error
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 3, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(SM3Error):
        expert_ops.expert_linear(x, w, off)
    with pytest.raises(SM3Error):
        mx4.quantize(x)
    q = mx4.Mx4Tensor(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), 8)
    for call in (lambda: q.dequantize(), lambda: mx4.linear(x, q), lambda: mx4.linear(q, q)):
        with pytest.raises(SM3Error):
            call()


def test_packed_tensors_are_checked():
    from sm3det_amd import mx4
    from sm3det_amd._lib import SM3Error
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    assert mx4.Mx4Tensor(u(2, 3, 128), u(2, 3, 8), 200).shape == (2, 3, 200)
    assert [mx4.padded(k) for k in (1, 128, 129, 600)] == [128, 128, 256, 640]
    for codes, scales, k in ((u(3, 64), u(3, 4), 129), (u(3, 64), u(3, 3), 100), (u(3, 64), u(2, 4), 100), (u(64), u(4), 100),
                             (u(3, 64).int(), u(3, 4), 100), (u(3, 64), u(3, 4), 0)):
        with pytest.raises(SM3Error):
            mx4.Mx4Tensor(codes, scales, k)


def test_unaligned_packed_storage_is_copied():
    from sm3det_amd import mx4
    flat = torch.zeros(3 * 64 + 1, dtype=torch.uint8)
    q = mx4.Mx4Tensor(flat[1:].view(3, 64), torch.zeros(13, dtype=torch.uint8)[1:].view(3, 4), 8)
    assert q.codes.data_ptr() % 16 == 0 and q.scales.data_ptr() % 4 == 0


def _desc(**kw):
    from sm3det_amd._lib_backbone import ExpertDesc
    d = ExpertDesc()
    base = dict(mode=0, type=2, out_type=2, bias_type=0, act=0, num_groups=1, red=64, cols=64, rows_out=0, rows=4, ldp=64, ldq=64,
                p=1 << 20, q=1 << 20, out=1 << 20, p_scales=1 << 20, q_scales=1 << 20)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


BAD = [dict(mode=3), dict(mode=-1), dict(num_groups=0), dict(num_groups=2), dict(rows=-1), dict(red=0), dict(cols=0), dict(act=2),
       dict(bias_type=3), dict(out_type=5), dict(p=None), dict(q=None), dict(out=None), dict(bias_grad=1 << 20)]


@pytest.mark.parametrize('kw', BAD, ids=str)
def test_the_abi_refuses_bad_descriptors(L, kw):
    for fn in ('sm3_expert_gemm_h16', 'sm3_mx4_gemm'):
        d = _desc(**kw)
        assert getattr(L, fn)(ctypes.byref(d), None, 0, None) == -1, fn
        assert getattr(L, fn + '_workspace_bytes')(ctypes.byref(d)) == 0


def test_the_abi_refuses_types_strides_and_small_workspaces(L):
    f = L.sm3_expert_gemm_h16
    for kw in (dict(type=0), dict(out_type=1), dict(ldp=60), dict(ldq=56), dict(act=1), dict(mode=2, rows_out=0),
               dict(mode=2, rows_out=8, bias=1 << 20), dict(mode=2, rows_out=8, act=1)):
        assert f(ctypes.byref(_desc(**kw)), None, 0, None) == -1, kw
    assert f(ctypes.byref(_desc(red=1 << 23, ldp=1 << 23, ldq=1 << 23)), None, 0, None) == -4
    assert L.sm3_mx4_gemm(ctypes.byref(_desc(mode=1)), None, 0, None) == -1
    for kw in (dict(q_scales=None), dict(q=(1 << 20) + 8), dict(p=(1 << 20) + 8), dict(p_scales=(1 << 20) + 2),
               dict(p_scales=None, type=3), dict(p_scales=None, ldp=63)):
        assert L.sm3_mx4_gemm(ctypes.byref(_desc(**kw)), None, 0, None) == -1, kw
    # operands that have to be copied need room: unaligned or odd 16-bit rows, floating rows of a 4-bit product
    for fn, kw in (('sm3_expert_gemm_h16', dict(p=(1 << 20) + 2)), ('sm3_expert_gemm_h16', dict(red=63)),
                   ('sm3_expert_gemm_h16', dict(ldp=68)), ('sm3_mx4_gemm', dict(p_scales=None, rows=400))):
        d = _desc(**kw)
        assert getattr(L, fn + '_workspace_bytes')(ctypes.byref(d)) > 0, kw
        assert getattr(L, fn)(ctypes.byref(d), None, 0, None) == -2, kw
    assert L.sm3_mx4_gemm(ctypes.byref(_desc(red=1 << 23)), None, 0, None) == -4
    d = _desc(mode=2, rows_out=64, rows=100000, bias_grad=1 << 20)
    need = L.sm3_expert_gemm_h16_workspace_bytes(ctypes.byref(d))
    assert need > 0 and f(ctypes.byref(d), 1 << 20, need - 1, None) == -2 and f(ctypes.byref(d), None, need, None) == -2
    assert f(ctypes.byref(_desc(rows=0)), None, 0, None) == 0 and L.sm3_mx4_gemm(ctypes.byref(_desc(rows=0)), None, 0, None) == 0
    assert L.sm3_expert_gemm_h16(None, None, 0, None) == -1
    P = ctypes.c_void_p(1 << 20)
    assert L.sm3_mx4_quantize(P, 3, 1, 8, 8, P, P, None) == -1 and L.sm3_mx4_quantize(P, 0, 1, 8, 4, P, P, None) == -1
    assert L.sm3_mx4_quantize(None, 0, 1, 8, 8, P, P, None) == -1 and L.sm3_mx4_quantize(P, 0, 0, 8, 8, P, P, None) == 0
    assert L.sm3_mx4_dequantize(P, P, 1, 0, P, 0, None) == -1 and L.sm3_mx4_dequantize(P, P, 0, 8, P, 0, None) == 0


def test_the_references_of_these_tests():
    """the 4-bit reference on values worked out by hand; row ranges of odd offsets"""
    x = np.zeros((2, 32))
    x[0, :8] = [5, 2.5, 3.5, 0.25, 0.75, 1.25, 1.75, 7.9]
    x[1, :3] = [1.0, -0.1, np.inf]
    codes, scales, val = quantize_ref(x)
    assert val[0, :8].tolist() == [4, 2, 4, 0, 1, 1, 2, 6] and scales[0, 0] == 127 and scales[1, 0] == 255
    assert np.isnan(val[1]).all() and codes.shape == (2, 64) and scales.shape == (2, 4)
    _, s, v = quantize_ref(np.array([[1.0, -0.1, 0.13, 3e-3] + [0.0] * 4]))
    assert s[0, 0] == 125 and v[0, :4].tolist() == [1.0, -0.125, 0.125, 0.0]  # grid 0.125 at the bottom, 1.0 = 4 * 2^-2
    assert set(np.abs(quantize_ref(np.linspace(-7, 7, 320).reshape(10, 32))[2].ravel()) / 1.0) <= set(
        (E2M1[:, None] * np.exp2(np.arange(-6.0, 3.0))).ravel())
    assert spans([-5, 40, 30, 1000, 60], 100) == [(0, 40), (40, 40), (40, 100), (100, 100)]
