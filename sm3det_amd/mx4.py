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
from torch.autograd import forward_ad

from . import _lib_backbone as LB
from ._lib import SM3Error, check, lib, require_gpu
from .expert_ops import DTYPES, check_offsets, has_tangent, launch, rows_of

ACTS = {None: 0, 'gelu': 1}
MAX_K = 0x7fffff80  # elements of a row: padded, they are counted in 31 bits


def padded(k):
    """elements a packed row of k elements holds (zeros behind k)"""
    return (k + 127) // 128 * 128


class Mx4Tensor:
    """Packed rows: ``codes`` (..., Kp / 2) uint8 (element 2 i in the low nibble of byte i), ``scales`` (..., Kp / 32) uint8,
    Kp = ``padded(k)``; the elements behind k are zero codes with scale bytes below 255."""

    def __init__(self, codes, scales, k):
        k = int(k)
        cs, ss = codes.shape, scales.shape
        kp = padded(k) if k > 0 else 0
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.device != scales.device:
            raise SM3Error('Mx4Tensor: codes and scales must be uint8 tensors on one device')
        if k > MAX_K:
            raise SM3Error(f'Mx4Tensor: rows of at most {MAX_K} elements, got {k}')
        if kp == 0 or len(cs) < 2 or cs[:-1] != ss[:-1] or cs[-1] * 2 != kp or ss[-1] * 32 != kp:
            raise SM3Error(f'Mx4Tensor: rows of {k} elements need codes (..., {kp // 2}) and scales (..., {kp // 32}), got '
                           f'{tuple(cs)} and {tuple(ss)}')
        codes, scales = codes.contiguous(), scales.contiguous()
        # the kernels read 16-byte granules of codes and 4-byte words of scales
        self.codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        self.scales = scales if scales.data_ptr() % 4 == 0 else scales.clone()
        self.k = k

    @classmethod
    def _of(cls, codes, scales, k):  # storage this module allocated itself
        q = cls.__new__(cls)
        q.codes, q.scales, q.k = codes, scales, k
        return q

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
        y = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        rows = y.numel() // self.k
        if rows:
            _call('mx4_dequantize', self.codes.device, y.numel() * (y.element_size() + 0.53), self.codes.data_ptr(),
                  self.scales.data_ptr(), rows, self.k, y.data_ptr(), DTYPES[dtype])
        return y


def _call(name, device, nbytes, *args):
    """sm3_<name>(*args, current stream of `device`)"""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _call(name, device, nbytes, *args)
    fn = getattr(lib(), 'sm3_' + name)
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if LB.PROFILE is None:
        code = fn(*args, stream)
    else:
        with LB._Prof(name, 0.0, nbytes):
            code = fn(*args, stream)
    if code:
        check(code, name)


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise SM3Error(f'{what} is for inference: an input requires a gradient (use torch.no_grad())')
    if forward_ad._current_level >= 0 and has_tangent(*tensors):
        raise SM3Error(f'{what} is for inference: an input carries a forward-mode tangent')


def quantize(x):
    """(..., K) float32 / float16 / bfloat16 -> Mx4Tensor; rows along the last dimension"""
    require_gpu(x)
    _no_grad('mx4.quantize', x)
    if x.dtype not in DTYPES or x.dim() < 2 or x.shape[-1] < 1:
        raise SM3Error(f'mx4.quantize: (..., K) float32, float16 or bfloat16 rows expected, got {tuple(x.shape)} of {x.dtype}')
    K = x.shape[-1]
    if K > MAX_K:
        raise SM3Error(f'mx4.quantize: rows of at most {MAX_K} elements, got {K}')
    x, ld = rows_of(x) if x.dim() == 2 else (x.contiguous(), K)
    kp = (K + 127) // 128 * 128
    codes = torch.empty(*x.shape[:-1], kp // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(*x.shape[:-1], kp // 32, dtype=torch.uint8, device=x.device)
    n = x.numel()
    if n:
        _call('mx4_quantize', x.device, n * (x.element_size() + 0.53), x.data_ptr(), DTYPES[x.dtype], n // K, K, ld, codes.data_ptr(),
              scales.data_ptr())
    return Mx4Tensor._of(codes, scales, K)


def _product(what, x, w, offsets, b, act, out_dtype):
    if not isinstance(w, Mx4Tensor):
        raise SM3Error(f'{what}: w must be an Mx4Tensor (mx4.quantize)')
    if act not in ACTS:
        raise SM3Error(f"{what}: act must be None or 'gelu', not {act!r}")
    packed = isinstance(x, Mx4Tensor)
    codes, device = w.codes, w.codes.device
    lead, k = codes.shape[:-1], w.k
    if len(lead) != (1 if offsets is None else 2):
        raise SM3Error(f"{what}: w must be {'(N, K)' if offsets is None else '(E, N, K)'}, got {tuple(w.shape)}")
    require_gpu(codes, x.codes if packed else x, b)
    if packed:
        if x.codes.dim() != 2 or x.k != k:
            raise SM3Error(f'{what}: x {tuple(x.shape)} does not match w {tuple(w.shape)}')
    elif x.dim() != 2 or x.shape[1] != k or x.dtype not in DTYPES:
        raise SM3Error(f'{what}: x (M, {k}) of float32, float16 or bfloat16 expected, got {tuple(x.shape)} of {x.dtype}')
    if out_dtype is None:
        out_dtype = torch.float32 if packed else x.dtype
    elif out_dtype not in DTYPES:
        raise SM3Error(f'{what}: float32, float16 or bfloat16 results, not {out_dtype}')
    groups, N = lead if offsets is not None else (1, lead[0])
    if N < 1 or groups < 1:
        raise SM3Error(f'{what}: w {tuple(w.shape)} has no rows')
    if x.device != device or (b is not None and b.device != device):
        raise SM3Error(f'{what}: x, w and b must be on one device')
    if b is not None:
        if b.shape != lead or b.dtype not in DTYPES:
            raise SM3Error(f'{what}: b must be {tuple(lead)} of a floating type, got {tuple(b.shape)} of {b.dtype}')
        b = b.contiguous()
    _no_grad(what, None if packed else x, b)
    if offsets is not None:
        offsets = check_offsets(offsets, groups, device, what)
    M = x.codes.shape[0] if packed else x.shape[0]
    y = torch.empty(M, N, dtype=out_dtype, device=device)
    if M == 0:
        return y
    if packed:
        launch('mx4_gemm', device, LB.NT, 0, y, x.codes, codes, M, k, N, groups=groups, offsets=offsets, bias=b, act=ACTS[act],
               p_scales=x.scales, q_scales=w.scales)
    else:
        x, ldx = rows_of(x)
        launch('mx4_gemm', device, LB.NT, DTYPES[x.dtype], y, x, codes, M, k, N, ldp=ldx, groups=groups, offsets=offsets, bias=b,
               act=ACTS[act], q_scales=w.scales)
    return y


def linear(x, w, b=None, act=None, out_dtype=None):
    """act(Q(x) . w^T + b): x (M, K) of a floating type (quantised in the call) or an Mx4Tensor, w an Mx4Tensor (N, K), b (N)
    or None, act None or 'gelu' (erf).  The result has x's type, or out_dtype (float32 where x is packed)."""
    return _product('mx4.linear', x, w, None, b, act, out_dtype)


def expert_linear(x, w, offsets, b=None, act=None, out_dtype=None):
    """`linear` with one weight per expert: w an Mx4Tensor (E, N, K), b (E, N) or None, rows [offsets[g], offsets[g + 1]) of x
    belong to expert g (offsets (E + 1) int32 on the device, never read by the host); rows of no expert give zeros."""
    if offsets is None:
        raise SM3Error('mx4.expert_linear: offsets (E + 1) are missing')
    return _product('mx4.expert_linear', x, w, offsets, b, act, out_dtype)


def expert_ffn(x, w1, b1, w2, b2, offsets):
    """Linear -> GELU -> Linear of each row's expert (FFN.forward, convnext_moe.py:397-405) on 4-bit operands: x (S, C),
    w1 (E, 4C, C) and w2 (E, C, 4C) packed, -> (S, C) float32.  The hidden rows live as bfloat16 between the two products (their
    8 bits go through a second rounding to e2m1's 2; bfloat16 keeps fp32's range)."""
    h = expert_linear(x, w1, offsets, b1, act='gelu', out_dtype=torch.bfloat16)
    return expert_linear(h, w2, offsets, b2, out_dtype=torch.float32)


class PackedExperts:
    """The experts of one MoE layer as the 4-bit products read them -- packed weights, a copy of the biases -- and the state of the
    four parameters they were made from, so that they are never used for other values."""

    def __init__(self, layer):
        self.w1, self.w2 = quantize(layer.w1.detach()), quantize(layer.w2.detach())
        self.b1, self.b2 = layer.b1.detach().clone(), layer.b2.detach().clone()
        self.stamp(layer)

    def stamp(self, layer):
        """these are `layer`'s parameters as they are now, packed (or copied) on the current stream"""
        self.stream = torch._C._cuda_getCurrentRawStream(self.b1.device.index) if self.b1.is_cuda else None
        # (an optimizer that writes by address does not move the version: it counts its steps, MultiTensorAdamW._writer)
        self.states = []
        for name in ('w1', 'b1', 'w2', 'b2'):
            p = layer._parameters[name]
            writers = getattr(p, '_sm3_writers', ())
            self.states.append((name, p, p.data_ptr(), None if p.is_inference() else p._version, writers, [w.steps for w in writers]))
        # False: writes may come that the host does not see -- an optimizer step inside a captured graph (capturing it counts as a
        # step, so this is as old as the rest), parameters that keep no version
        self.followable = not any(version is None or any(w.captured for w in writers) for *_, version, writers, _ in self.states)

    def made_from(self, layer):
        """whether nothing the host sees has changed the parameters since"""
        now = layer._parameters
        for name, p, address, version, writers, steps in self.states:
            if now.get(name) is not p or p.data_ptr() != address or (version is not None and p._version != version):
                return False
            if getattr(p, '_sm3_writers', ()) != writers or (writers and [w.steps for w in writers] != steps):
                return False
        return True

    def read_here(self):
        """the current stream is about to read them: dropped before it has, they stay allocated until then"""
        device = self.b1.device
        if torch._C._cuda_getCurrentRawStream(device.index) != self.stream:
            stream = torch.cuda.current_stream(device)
            for t in (self.w1.codes, self.w1.scales, self.b1, self.w2.codes, self.w2.scales, self.b2):
                t.record_stream(stream)

    def ffn(self, xslot, offsets):
        return expert_ffn(xslot, self.w1, self.b1, self.w2, self.b2, offsets)

    def __getstate__(self):  # (a copy of the layer has parameters of its own: MoE_layer.__setstate__ stamps)
        return {k: v for k, v in self.__dict__.items() if k not in ('states', 'followable', 'stream')}


def quantize_experts(module):
    """Pack the experts of every MoE layer inside `module` (a backbone or a detector in evaluation mode): its forward under
    ``torch.no_grad()`` then runs them on the 4-bit products -- router, combine, dense blocks and everything else as before.
    -> layers packed.

    The packed weights (and the biases next to them) are a snapshot.  ``train()``, ``load_state_dict()`` and moving the module drop
    them; after any other change of w1, b1, w2 or b2 -- a torch operation in place, a step of ``MultiTensorAdamW``, a broadcast, other
    parameters in their place -- the layer runs its full-precision experts until it is packed again.  Where a captured
    optimizer step writes the parameters, whose replays nobody announces, every forward packs them anew.  Not seen: values
    written past autograd's version counter (``p.data.copy_()``, a foreign kernel); call this again after those.
    A graph captured from such a forward replays the snapshot, which the layer keeps allocated for it: capture again after a change."""
    from .convnext_moe import MoE_layer
    layers = [m for m in module.modules() if isinstance(m, MoE_layer)]
    for m in layers:
        if m.training:
            raise SM3Error('mx4.quantize_experts: call module.eval() first (4-bit experts are for inference)')
    for m, packed in [(m, PackedExperts(m)) for m in layers]:
        m._mx4 = packed
    return len(layers)


def restore_experts(module):
    """undo `quantize_experts`"""
    from .convnext_moe import MoE_layer
    for m in module.modules():
        if isinstance(m, MoE_layer):
            m._mx4 = None
