"""Products grouped by expert in 16 bits: one linear layer per expert over expert-major rows, with its gradients.

    y[r] = x[r] . w[g]^T + b[g]          for rows r in [offsets[g], offsets[g + 1])

This is the expert loop of ``MoE_layer.forward`` (mmrotate/models/backbones/convnext_moe.py:243-245) for one ``nn.Linear`` of
the experts, for bf16 / fp16 training -- next to ``backbone_ops.linear`` (fp32, one group) and the fused fp32 / fp16-operand MoE
block of ``backbone_ops.moe_block``.  ``offsets`` are what ``sm3_moe_plan`` leaves on the device (prefix of the experts' slot
counts): the host never reads them, so calls are free of synchronisation and can be captured into a HIP graph.

* types: x, w both bfloat16 or both float16, fp32 accumulation, results rounded once; b of x's type or float32.
* any sizes (rows of a length that is no multiple of 8, or not 16-byte aligned, are copied into padded rows first).
* rows of no expert (before ``offsets[0]``, behind ``offsets[-1]``): y and dx are zero there and they enter no gradient.
  Offsets outside [0, rows] are clamped, decreasing ones made monotone.
* an expert without rows gets zero gradients (never an uninitialised one).
* gradients do not depend on the order in which workgroups run: split reductions are added in a fixed order, no atomics.
"""
import ctypes

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib_backbone as LB
from ._lib import SM3Error, check, lib, require_gpu, stream_ptr, workspace

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def check_offsets(offsets, num_groups, device, name):
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.device != device:
        raise SM3Error(f'{name}: offsets must be a 1-D int32 tensor on {device} (got {offsets.dtype}, '
                       f'{tuple(offsets.shape)} on {offsets.device})')
    if offsets.numel() != num_groups + 1:
        raise SM3Error(f'{name}: {num_groups} experts need {num_groups + 1} offsets, got {offsets.numel()}')
    return offsets.contiguous()


def run_desc(fn, desc, device, flops, nbytes, what):
    """enqueue one grouped product (sm3_<fn>) on the current stream of `device`, its workspace from torch's allocator"""
    L = lib()
    with torch.cuda.device(device):
        need = getattr(L, f'sm3_{fn}_workspace_bytes')(ctypes.byref(desc))
        ws = workspace(need, device) if need else None
        with LB._Prof(what, flops, nbytes):
            check(getattr(L, 'sm3_' + fn)(ctypes.byref(desc), None if ws is None else ws.data_ptr(), need, stream_ptr()),
                  what)


def readable_rows(t):
    """`t` (..., K) as rows the kernels can read: unit stride along K, 16-byte aligned rows, zeros up to the next multiple of
    8 -> (tensor, elements between rows).  A 2-D tensor may keep a row stride; everything else is made contiguous."""
    K = t.shape[-1]
    ld = t.stride(0) if t.dim() == 2 and t.shape[0] > 1 else K
    if t.stride(-1) != 1 and K > 1 or (t.dim() == 2 and ld < K) or (t.dim() != 2 and not t.is_contiguous()):
        t, ld = t.contiguous(), K
    if K % 8 == 0 and ld % 8 == 0 and ld <= 1 << 22 and t.data_ptr() % 16 == 0:
        return t, ld
    kp = (K + 7) // 8 * 8
    rows = t.numel() // K
    out = torch.empty(*t.shape[:-1], kp, dtype=t.dtype, device=t.device)
    with torch.cuda.device(t.device):
        LB.call('pad_rows_h16', t, rows, K, ld, out, kp, nbytes=2.0 * rows * (K + kp))
    return out, kp


def _desc(mode, p, ldp, q, ldq, out, offsets, groups, rows, red, cols, rows_out=0, bias=None, bias_grad=None):
    d = LB.ExpertDesc()
    d.mode, d.type, d.out_type = mode, DTYPES[p.dtype], DTYPES[out.dtype]
    b = bias if bias is not None else bias_grad
    d.bias_type = DTYPES[b.dtype] if b is not None else 0
    d.num_groups, d.red, d.cols, d.rows_out = groups, red, cols, rows_out
    d.rows, d.ldp, d.ldq = rows, ldp, ldq
    d.p, d.q, d.out, d.offsets = LB._p(p), LB._p(q), LB._p(out), LB._p(offsets)
    d.bias, d.bias_grad = LB._p(bias), LB._p(bias_grad)
    return d


class _ExpertLinear(Function):
    @staticmethod
    def forward(ctx, x, w, offsets, b):
        S, K = x.shape
        E, N, _ = w.shape
        y = torch.empty(S, N, dtype=x.dtype, device=x.device)
        xr, ldx = readable_rows(x)
        wr, ldw = readable_rows(w)
        if S:
            run_desc('expert_gemm_h16', _desc(LB.NT, xr, ldx, wr, ldw, y, offsets, E, S, K, N, bias=b), x.device,
                     2.0 * S * N * K, 2.0 * (S * (N + K) + E * N * K), 'expert_linear')
        ctx.save_for_backward(xr, wr, offsets)
        ctx.meta = (S, K, E, N, ldx, ldw, None if b is None else b.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, wr, offsets = ctx.saved_tensors
        S, K, E, N, ldx, ldw, b_dtype = ctx.meta
        dev = xr.device
        dyr, lddy = readable_rows(dy)
        flops, nbytes = 2.0 * S * N * K, 2.0 * (S * (N + K) + E * N * K)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(S, K, dtype=xr.dtype, device=dev)
            if S:
                run_desc('expert_gemm_h16', _desc(LB.NN, dyr, lddy, wr, ldw, dx, offsets, E, S, N, K), dev, flops, nbytes,
                         'expert_linear_dgrad')
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[3]:
            # the bias gradient is a by-product of the weight gradient's pass over dy
            dw = torch.empty(E, N, K, dtype=xr.dtype, device=dev)
            if b_dtype is not None and ctx.needs_input_grad[3]:
                db = torch.empty(E, N, dtype=b_dtype, device=dev)
            run_desc('expert_gemm_h16', _desc(LB.TN, dyr, lddy, xr, ldx, dw, offsets, E, S, 1, K, rows_out=N, bias_grad=db),
                     dev, flops, nbytes, 'expert_linear_wgrad')
            if not ctx.needs_input_grad[1]:
                dw = None
        return dx, dw, None, db


def expert_linear(x, w, offsets, b=None):
    """y (S, N) of x (S, K), one weight (N, K) per expert in w (E, N, K), bias b (E, N) or None; rows grouped by `offsets`
    (E + 1, int32, on the device).  Differentiable in x, w and b."""
    require_gpu(x, w, offsets, b)
    if x.dtype not in (torch.float16, torch.bfloat16) or w.dtype != x.dtype:
        raise SM3Error(f'expert_linear: x and w must both be float16 or both bfloat16 (got {x.dtype}, {w.dtype})')
    if x.dim() != 2 or w.dim() != 3 or w.shape[2] != x.shape[1] or min(w.shape) < 1:
        raise SM3Error(f'expert_linear: x (S, K) and w (E, N, K) with E, N, K >= 1 expected, got {tuple(x.shape)} and '
                       f'{tuple(w.shape)}')
    if w.device != x.device or (b is not None and b.device != x.device):
        raise SM3Error('expert_linear: x, w and b must be on one device')
    if b is not None:
        if b.shape != w.shape[:2] or b.dtype not in (x.dtype, torch.float32):
            raise SM3Error(f'expert_linear: b must be {tuple(w.shape[:2])} of {x.dtype} or float32, got {tuple(b.shape)} of '
                           f'{b.dtype}')
        b = b.contiguous()
    return _ExpertLinear.apply(x, w, check_offsets(offsets, w.shape[0], x.device, 'expert_linear'), b)
