"""Products grouped by expert in 16 bits: one linear layer per expert over expert-major rows, with its gradients.

    y[r] = x[r] . w[g]^T + b[g]          for rows r in [offsets[g], offsets[g + 1])

This is the expert loop of ``MoE_layer.forward`` (mmrotate/models/backbones/convnext_moe.py:243-245) for one ``nn.Linear`` of
the experts, for bf16 / fp16 training -- next to ``backbone_ops.linear`` (fp32, one group) and the fused fp32 / fp16-operand MoE
block of ``backbone_ops.moe_block``.  ``offsets`` are what ``sm3_moe_plan`` leaves on the device (prefix of the experts' slot
counts): the host never reads them, so calls are free of synchronisation and can be captured into a HIP graph.

* types: x, w both bfloat16 or both float16, fp32 accumulation, results rounded once; b of x's type or float32.
* any sizes and row strides, rows and reductions of up to 2^22 elements (rows of a length that is no multiple of 8, or not 16-byte
  aligned, are copied into padded rows of the workspace first).
* rows of no expert (before ``offsets[0]``, behind ``offsets[-1]``): y and dx are zero there and they enter no gradient.
  Offsets outside [0, rows] are clamped, decreasing ones made monotone.
* an expert without rows gets zero gradients (never an uninitialised one).
* first derivatives only, backward mode only: differentiating a gradient raises, and so does an input with a forward-mode tangent.
* gradients do not depend on the order in which workgroups run: split reductions are added in a fixed order, no atomics.
"""
import torch
from torch.autograd import Function, forward_ad

from . import _lib_backbone as LB
from ._lib import SM3Error, check, lib, require_gpu

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def has_tangent(*tensors):
    """whether forward-mode differentiation (which no_grad() does not end) would have to follow one of the tensors; asked where
    `forward_ad._current_level` says that it is on"""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def check_offsets(offsets, num_groups, device, name):
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.device != device:
        raise SM3Error(f'{name}: offsets must be a 1-D int32 tensor on {device} (got {offsets.dtype}, '
                       f'{tuple(offsets.shape)} on {offsets.device})')
    if offsets.numel() != num_groups + 1:
        raise SM3Error(f'{name}: {num_groups} experts need {num_groups + 1} offsets, got {offsets.numel()}')
    return offsets.contiguous()


_NEED = {}  # (entry point, sizes and types of a call) -> bytes of workspace: a query per new size, not per call


def launch(fn, device, mode, dtype, out, p, q, rows, red, cols, *, rows_out=0, ldp=0, ldq=0, groups=1, offsets=None, bias=None,
           bias_grad=None, act=0, p_scales=None, q_scales=None, aligned=0):
    """enqueue one grouped product (sm3_<fn>) on torch's current stream of `device`, workspace from torch's allocator.
    `aligned`: what decides, beside the sizes, whether operands are copied (the operands' addresses modulo 16)."""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return launch(fn, device, mode, dtype, out, p, q, rows, red, cols, rows_out=rows_out, ldp=ldp, ldq=ldq, groups=groups,
                          offsets=offsets, bias=bias, bias_grad=bias_grad, act=act, p_scales=p_scales, q_scales=q_scales,
                          aligned=aligned)
    L = lib()
    b = bias if bias is not None else bias_grad
    out_type = DTYPES[out.dtype]
    try:
        desc = LB.EXPERT_DESC.pack(
            mode, dtype, out_type, 0 if b is None else DTYPES[b.dtype], act, groups, red, cols, rows_out, 0, rows, ldp, ldq,
            p.data_ptr(), q.data_ptr(), 0 if p_scales is None else p_scales.data_ptr(), 0 if q_scales is None else q_scales.data_ptr(),
            0 if offsets is None else offsets.data_ptr(), 0 if bias is None else bias.data_ptr(),
            0 if bias_grad is None else bias_grad.data_ptr(), out.data_ptr())
    except LB.struct.error:
        raise SM3Error(f'{fn}: sizes are counted in 31 bits: reduction {red}, columns {cols}, rows of the result {rows_out}, '
                       f'experts {groups}') from None
    key = (fn, mode, dtype, out_type, groups, red, cols, rows_out, rows, ldp, ldq, offsets is None, bias_grad is None,
           p_scales is None, aligned)
    need = _NEED.get(key)
    if need is None:
        if len(_NEED) > 4096:
            _NEED.clear()
        need = _NEED[key] = getattr(L, f'sm3_{fn}_workspace_bytes')(desc)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    args = (desc, None if ws is None else ws.data_ptr(), need, torch._C._cuda_getCurrentRawStream(device.index))
    if LB.PROFILE is None:
        code = getattr(L, 'sm3_' + fn)(*args)
    else:
        n = rows_out if mode == LB.TN else cols
        with LB._Prof(f'{fn}_{("nt", "nn", "tn")[mode]}', 2.0 * rows * n * (cols if mode == LB.TN else red)):
            code = getattr(L, 'sm3_' + fn)(*args)
    if code:
        check(code, fn)


def rows_of(t):
    """a 2-D tensor as rows with unit stride along them -> (tensor, elements between rows); copied only where it has none"""
    n, k = t.shape
    s0, s1 = t.stride()
    if n <= 1:
        return (t, k) if s1 == 1 or k == 1 else (t.contiguous(), k)
    if (s1 == 1 or k == 1) and s0 >= k:
        return t, s0
    return t.contiguous(), k


def _forward(x, ldx, w, offsets, b):
    S, K = x.shape
    E, N, _ = w.shape
    y = torch.empty(S, N, dtype=x.dtype, device=x.device)
    if S:
        launch('expert_gemm_h16', x.device, LB.NT, DTYPES[x.dtype], y, x, w, S, K, N, ldp=ldx, ldq=K, groups=E, offsets=offsets,
               bias=b, aligned=(x.data_ptr() | w.data_ptr()) & 15 and (x.data_ptr() & 15, w.data_ptr() & 15))
    return y


def _gradients(dy, x, w, offsets, ldx, b_dtype, need):
    """(dx, dw, db), those that `need` (of x, w, b) asks for"""
    S, K = x.shape
    E, N, _ = w.shape
    dev, dt = x.device, DTYPES[x.dtype]
    dy, lddy = rows_of(dy)
    dx = dw = db = None
    if need[0]:
        dx = torch.empty(S, K, dtype=x.dtype, device=dev)
        if S:
            launch('expert_gemm_h16', dev, LB.NN, dt, dx, dy, w, S, N, K, ldp=lddy, ldq=K, groups=E, offsets=offsets,
                   aligned=(dy.data_ptr() | w.data_ptr()) & 15 and (dy.data_ptr() & 15, w.data_ptr() & 15))
    if need[1] or need[2]:
        # the bias gradient is a by-product of the weight gradient's pass over dy
        dw = torch.empty(E, N, K, dtype=x.dtype, device=dev)
        if need[2]:
            db = torch.empty(E, N, dtype=b_dtype, device=dev)
        launch('expert_gemm_h16', dev, LB.TN, dt, dw, dy, x, S, 1, K, rows_out=N, ldp=lddy, ldq=ldx, groups=E, offsets=offsets,
               bias_grad=db, aligned=(dy.data_ptr() | x.data_ptr()) & 15 and (dy.data_ptr() & 15, x.data_ptr() & 15))
        if not need[1]:
            dw = None
    return dx, dw, db


class _Gradients(Function):
    """The gradients where a graph of them is being recorded (create_graph=True): tied to what they were computed from, so that
    differentiating them raises.  (once_differentiable ties them to dy alone: with a dy that needs no gradient, the part of a loss
    that depends on dx through w, or on dw through x, would vanish.)"""

    @staticmethod
    def forward(ctx, dy, x, w, *rest):
        return _gradients(dy, x, w, *rest)

    @staticmethod
    def backward(ctx, *grads):
        raise SM3Error('expert_linear: second derivatives are not implemented')


class _ExpertLinear(Function):
    @staticmethod
    def forward(ctx, x, ldx, w, offsets, b):
        ctx.save_for_backward(x, w, offsets)
        ctx.ldx, ctx.b_dtype = ldx, None if b is None else b.dtype
        return _forward(x, ldx, w, offsets, b)

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        f = _Gradients.apply if torch.is_grad_enabled() else _gradients
        dx, dw, db = f(dy, x, w, offsets, ctx.ldx, ctx.b_dtype, (need[0], need[2], need[4]))
        return dx, None, dw, None, db


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
    if forward_ad._current_level >= 0 and has_tangent(x, w, b):
        raise SM3Error('expert_linear: an input carries a forward-mode tangent; only backward-mode derivatives are implemented')
    offsets = check_offsets(offsets, w.shape[0], x.device, 'expert_linear')
    # (copies are made here, where autograd sees them: what it saves are then the caller's tensors or lead to them)
    (x, ldx), w = rows_of(x), w.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (b is not None and b.requires_grad)):
        return _ExpertLinear.apply(x, ldx, w, offsets, b)
    return _forward(x, ldx, w, offsets, b)
