"""64-bit references and error bounds shared by the tests of the grouped 16-bit and 4-bit products."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def bound(ref, mag, terms, dtype):
    """|computed - ref| of a sum of `terms` products accumulated in fp32 and rounded once to `dtype`; mag = sum of |products|.
    Every fp32 addition, product and alignment inside the matrix unit is off by at most one step, 2^-23 of a partial sum of at
    most mag; the final rounding by half a step of the result (or of the type's smallest number)."""
    acc = (terms + 2) * 2.0 ** -23 * mag
    return acc + HALF_STEP[dtype] * (ref.abs() + acc) + 0.5 * SMALLEST[dtype]


def assert_within(got, ref, tol, what=''):
    off = (got.double() - ref).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert not torch.isnan(got).any(), f'{what}: NaN'
    assert worst <= 0, f'{what}: off by {off.max().item():.3g}, {worst:.3g} over the bound'


def spans(offsets, rows):
    """the experts' row ranges as the operators define them: clamped to [0, rows], made monotone"""
    o = np.maximum.accumulate(np.clip(np.asarray(offsets, dtype=np.int64), 0, rows))
    return list(zip(o[:-1].tolist(), o[1:].tolist()))


def ragged(seed, rows, experts, head=0, tail=0, empty=0.2):
    r = np.random.RandomState(seed)
    w = r.rand(experts) ** 2 * (r.rand(experts) >= empty)
    if not w.any():
        w[r.randint(experts)] = 1.0
    cuts = np.rint(np.cumsum(w) / w.sum() * (rows - head - tail)).astype(int) + head
    return [head] + cuts.tolist()


E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def quantize_ref(x):
    """numpy reference of the 4-bit form, in 64 bits: (codes (R, Kp/2), scales (R, Kp/32), values (R, K) float64)"""
    x = np.asarray(x, dtype=np.float64)
    R, K = x.shape
    kp = (K + 127) // 128 * 128
    v = np.zeros((R, kp // 32, 32))
    v.reshape(R, kp)[:, :K] = x
    m = np.abs(v).max(-1)
    fine = np.isfinite(v).all(-1)
    with np.errstate(divide='ignore', invalid='ignore'):
        e = np.where(fine & (m > 0), np.frexp(np.where(fine, m, 1.0))[1] - 1, -1000)  # floor(log2 m)
    byte = np.where(fine, np.clip(e - 2 + 127, 0, None), 255).astype(np.int64)
    u = np.where(fine[..., None], v, 0.0) / np.exp2(byte - 127.0)[..., None]
    a = np.minimum(np.abs(u), 6.0)
    dist = np.abs(a[..., None] - E2M1)  # (the quotients are exact: ties are seen as ties)
    near = dist == dist.min(-1, keepdims=True)
    code = np.where(near & (np.arange(8) % 2 == 0), np.arange(8), 99).min(-1)  # even codes win ties
    code = np.where(code == 99, near.argmax(-1), code)
    sign = np.signbit(u)
    val = np.where(sign, -1.0, 1.0) * E2M1[code] * np.exp2(byte - 127.0)[..., None]
    val = np.where(fine[..., None], val, np.nan).reshape(R, kp)[:, :K]
    c = (code + 8 * sign).reshape(R, kp)
    return (c[:, 0::2] | c[:, 1::2] << 4).astype(np.uint8), byte.astype(np.uint8), val
