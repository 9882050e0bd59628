"""Microscaled 4-bit (MXFP4) inference: quantisation, products, products grouped by expert.

A row is cut into blocks of 32 elements; a block keeps one power of two (a byte, exponent + 127) and 32 four-bit elements
(e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) -- 4.25 bits per element.  The block's exponent is floor(log2 max|x|) - 2, elements
are rounded to nearest (ties to the even code) and saturate at 6; a block holding an infinity or a NaN becomes NaN.

    wq = mx4.quantize(w)                       # once: (N, K) or (E, N, K) weights
    y  = mx4.linear(x, wq, b, act='gelu')      # x (M, K) float32 / float16 / bfloat16, quantised on the way in
    y  = mx4.expert_linear(x, wq, offsets, b)  # rows grouped by expert

The products run on the 4-bit matrix instruction with the blocks' scales as its operands and accumulate in fp32; nothing is
dequantised.  Inference only: a call that autograd would have to differentiate is refused.  ``quantize_experts`` puts the
experts of a backbone's MoE blocks (mmrotate/models/backbones/convnext_moe.py:226-248) on these products in evaluation.
"""
import torch

from . import _lib_backbone as LB
from ._lib import SM3Error, require_gpu
from .expert_ops import DTYPES, check_offsets, launch, rows_of

ACTS = {None: 0, 'gelu': 1}


def padded(k):
    """elements a packed row of k elements holds (zeros behind k)"""
    return (k + 127) // 128 * 128


class Mx4Tensor:
    """Packed rows: ``codes`` (..., Kp / 2) uint8 (element 2 i in the low nibble of byte i), ``scales`` (..., Kp / 32) uint8,
    Kp = ``padded(k)``; the elements behind k are zero codes with scale bytes below 255."""

    def __init__(self, codes, scales, k):
        k = int(k)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.device != scales.device:
            raise SM3Error('Mx4Tensor: codes and scales must be uint8 tensors on one device')
        if k < 1 or codes.dim() < 2 or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] * 2 != padded(k) or \
                scales.shape[-1] * 32 != padded(k):
            raise SM3Error(f'Mx4Tensor: rows of {k} elements need codes (..., {padded(max(k, 1)) // 2}) and scales '
                           f'(..., {padded(max(k, 1)) // 32}), got {tuple(codes.shape)} and {tuple(scales.shape)}')
        codes, scales = codes.contiguous(), scales.contiguous()
        # the kernels read 16-byte granules of codes and 4-byte words of scales
        self.codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        self.scales = scales if scales.data_ptr() % 4 == 0 else scales.clone()
        self.k = k

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.k))

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return f'Mx4Tensor(shape={tuple(self.shape)}, device={self.device})'

    def dequantize(self, dtype=torch.float32):
        """the values the rows stand for, rounded to `dtype` (exact in float32 and bfloat16)"""
        if dtype not in DTYPES:
            raise SM3Error(f'dequantize: float32, float16 or bfloat16, not {dtype}')
        require_gpu(self.codes)
        y = torch.empty(self.shape, dtype=dtype, device=self.device)
        rows = self.scales.numel() // self.scales.shape[-1]
        with torch.cuda.device(self.device):
            LB.call('mx4_dequantize', self.codes, self.scales, rows, self.k, y, DTYPES[dtype],
                    nbytes=y.numel() * (y.element_size() + 0.53))
        return y


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise SM3Error(f'{what} is for inference: an input requires a gradient (use torch.no_grad())')


def quantize(x):
    """(..., K) float32 / float16 / bfloat16 -> Mx4Tensor; rows along the last dimension"""
    require_gpu(x)
    _no_grad('mx4.quantize', x)
    if x.dtype not in DTYPES or x.dim() < 2 or x.shape[-1] < 1:
        raise SM3Error(f'mx4.quantize: (..., K) float32, float16 or bfloat16 rows expected, got {tuple(x.shape)} of {x.dtype}')
    K = x.shape[-1]
    if not (x.dim() == 2 and x.shape[0] > 1 and x.stride(1) == 1 and x.stride(0) >= K):
        x = x.contiguous()
    ld = x.stride(0) if x.dim() == 2 and x.shape[0] > 1 else K
    kp = padded(K)
    codes = torch.empty(*x.shape[:-1], kp // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(*x.shape[:-1], kp // 32, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        LB.call('mx4_quantize', x, DTYPES[x.dtype], x.numel() // K, K, ld, codes, scales,
                nbytes=x.numel() * (x.element_size() + 0.53))
    return Mx4Tensor(codes, scales, K)


def _product(what, x, w, offsets, b, act, out_dtype):
    if not isinstance(w, Mx4Tensor):
        raise SM3Error(f'{what}: w must be an Mx4Tensor (mx4.quantize)')
    if act not in ACTS:
        raise SM3Error(f"{what}: act must be None or 'gelu', not {act!r}")
    packed = isinstance(x, Mx4Tensor)
    require_gpu(w.codes, x.codes if packed else x, offsets, b)
    if len(x.shape) != 2 or x.shape[1] != w.k:
        raise SM3Error(f'{what}: x {tuple(x.shape)} does not match w {tuple(w.shape)}')
    if out_dtype is None:
        out_dtype = torch.float32 if packed else x.dtype
    if out_dtype not in DTYPES:
        raise SM3Error(f'{what}: float32, float16 or bfloat16 results, not {out_dtype}')
    groups, N = (1, w.shape[0]) if offsets is None else w.shape[:2]
    if N < 1 or groups < 1:
        raise SM3Error(f'{what}: w {tuple(w.shape)} has no rows')
    if x.device != w.device or (b is not None and b.device != w.device):
        raise SM3Error(f'{what}: x, w and b must be on one device')
    if b is not None:
        if b.shape != w.shape[:-1] or b.dtype not in DTYPES:
            raise SM3Error(f'{what}: b must be {tuple(w.shape[:-1])} of a floating type, got {tuple(b.shape)} of {b.dtype}')
        b = b.contiguous()
    _no_grad(what, None if packed else x, b)
    M = x.shape[0]
    y = torch.empty(M, N, dtype=out_dtype, device=w.device)
    if M == 0:
        return y
    if packed:
        launch('mx4_gemm', w.device, LB.NT, 0, y, x.codes, w.codes, M, w.k, N, groups=groups, offsets=offsets, bias=b, act=ACTS[act],
               p_scales=x.scales, q_scales=w.scales)
    else:
        x, ldx = rows_of(x)
        launch('mx4_gemm', w.device, LB.NT, DTYPES[x.dtype], y, x, w.codes, M, w.k, N, ldp=ldx, groups=groups, offsets=offsets,
               bias=b, act=ACTS[act], q_scales=w.scales)
    return y


def linear(x, w, b=None, act=None, out_dtype=None):
    """act(Q(x) . w^T + b): x (M, K) of a floating type (quantised in the call) or an Mx4Tensor, w an Mx4Tensor (N, K), b (N)
    or None, act None or 'gelu' (erf).  The result has x's type, or out_dtype (float32 where x is packed)."""
    if isinstance(w, Mx4Tensor) and len(w.shape) != 2:
        raise SM3Error(f'mx4.linear: w must be (N, K), got {tuple(w.shape)}')
    return _product('mx4.linear', x, w, None, b, act, out_dtype)


def expert_linear(x, w, offsets, b=None, act=None, out_dtype=None):
    """`linear` with one weight per expert: w an Mx4Tensor (E, N, K), b (E, N) or None, rows [offsets[g], offsets[g + 1]) of x
    belong to expert g (offsets (E + 1) int32 on the device, never read by the host); rows of no expert give zeros."""
    if isinstance(w, Mx4Tensor):
        if len(w.shape) != 3:
            raise SM3Error(f'mx4.expert_linear: w must be (E, N, K), got {tuple(w.shape)}')
        require_gpu(w.codes, offsets)
        offsets = check_offsets(offsets, w.shape[0], w.device, 'mx4.expert_linear')
    return _product('mx4.expert_linear', x, w, offsets, b, act, out_dtype)
