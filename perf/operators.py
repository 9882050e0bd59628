"""Cases for the operators around the experts' products: microscaled 4-bit quantisation (blocks of 32 elements along a
row, e2m1 elements, one power-of-two scale byte per block), products of 4-bit operands -- dense and grouped by expert -- and
the 16-bit products grouped by expert with their gradients.

Each case is one call of a public entry point (with its backward pass where the case says `train`).  `run` computes the same
from elementary torch operations while `own` is false."""
import math
import random

import torch

own = False

_TYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a handful of pooled tokens: the call's latency
        dict(name='quantise_small', op='quantize', rows=16, k=96, dtype='bf16'),
        # the GELU output of a stage-0 FFN, two images of 1024 x 1024
        dict(name='quantise_large', op='quantize', rows=131072, k=384, dtype='fp16'),
        # first FFN linear for a single token
        dict(name='linear_token', op='linear', m=1, n=4096, k=1024, dtype='bf16', gelu=True),
        # first FFN linear of a stage-3 dense block, two images of 1024 x 1024, fp32 activations
        dict(name='linear_stage3', op='linear', m=2048, n=4096, k=1024, dtype='fp32', gelu=True),
        # no size a multiple of anything the hardware likes
        dict(name='linear_odd', op='linear', m=1021, n=250, k=603, dtype='fp16', gelu=False),
        # eight routed tokens, most experts with one or none
        dict(name='mx4_experts_tokens', op='mx4_experts', s=8, e=8, n=2048, k=512, tail=0, dtype='bf16', gelu=True),
        # first expert linear of stage 2, top-2 of eight experts, two images
        dict(name='mx4_experts_stage2', op='mx4_experts', s=16384, e=8, n=2048, k=512, tail=0, dtype='fp16', gelu=True),
        # second expert linear, sixteen experts, fp32 activations
        dict(name='mx4_experts_fc2', op='mx4_experts', s=16384, e=16, n=384, k=1536, tail=0, dtype='fp32', gelu=False),
        # forward only, few tokens: bound by the weights
        dict(name='experts_tokens', op='experts', s=24, e=8, n=4096, k=1024, tail=0, dtype='bf16'),
        # training step of a stage-1 expert linear: many rows, short reduction
        dict(name='experts_train_stage1', op='experts_train', s=65536, e=8, n=1024, k=256, tail=0, dtype='bf16'),
        # training step of a stage-3 expert linear, eight images: the largest products
        dict(name='experts_train_stage3', op='experts_train', s=16384, e=8, n=4096, k=1024, tail=0, dtype='bf16'),
        # odd sizes, slots behind the last expert's that belong to nobody
        dict(name='experts_train_odd', op='experts_train', s=1999, e=5, n=117, k=203, tail=37, dtype='fp16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """over the logarithm; half of them rounded to a multiple of 32, the others as they fall (odd ones among them)"""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 or v < 32 else v // 32 * 32


def draw(rng):
    op = rng.choice(['quantize', 'linear', 'mx4_experts', 'mx4_experts', 'experts', 'experts_train', 'experts_train'])
    top = [work(c) for c in listed() if c['op'] == op or (op == 'experts' and c['op'] == 'experts_train')]
    while True:
        if op == 'quantize':
            c = dict(op=op, rows=_size(rng, 1, 262144), k=_size(rng, 1, 4096), dtype=rng.choice(['fp32', 'fp16', 'bf16']))
        elif op == 'linear':
            c = dict(op=op, m=_size(rng, 1, 16384), n=_size(rng, 1, 4096), k=_size(rng, 16, 4096),
                     dtype=rng.choice(['fp32', 'fp16', 'bf16']), gelu=rng.random() < 0.5)
        else:
            s = _size(rng, 1, 65536)
            c = dict(op=op, s=s, e=_log(rng, 1, 32), n=_size(rng, 8, 4096), k=_size(rng, 16, 4096),
                     tail=rng.choice([0, 0, 0, s // 20]))
            if op == 'mx4_experts':
                c.update(dtype=rng.choice(['fp32', 'fp16', 'bf16']), gelu=rng.random() < 0.5)
            else:
                c.update(dtype=rng.choice(['fp16', 'bf16']))
        w = work(c)
        if w['bytes'] <= max(t['bytes'] for t in top) and w['flops'] <= max(t['flops'] for t in top):
            return c


# ------------------------------------------------------------------------------------------------------ inputs
def _tokens(g, rows, k, dtype):
    """layer-normed activations: channel gains, a few loud channels"""
    x = torch.randn(rows, k, generator=g, device='cuda')
    gain = 0.5 + torch.rand(k, generator=g, device='cuda')
    loud = torch.rand(k, generator=g, device='cuda') < 0.02
    return (x * torch.where(loud, gain * 8, gain)).to(dtype)


def _offsets(case, seed):
    """prefix of the experts' slot counts as a router leaves them: uneven, some experts empty; `tail` slots belong to none"""
    r = random.Random(seed)
    load = [r.random() ** 2 * (r.random() < 0.9) for _ in range(case['e'])]
    if not any(load):
        load[r.randrange(case['e'])] = 1.0
    rows = case['s'] - case['tail']
    ends, run_sum, total = [0], 0.0, sum(load)
    for v in load:
        run_sum += v
        ends.append(min(rows, int(round(rows * run_sum / total))))
    ends[-1] = rows
    return ends


def _pack(w):
    """(R, K) values -> the 4-bit form a program keeps its weights in: codes (R, Kp / 2) uint8, the even element in the low
    nibble, scales (R, Kp / 32) uint8 (exponent + 127), K padded with zeros to Kp, a multiple of 128"""
    rows, k = w.shape
    kp = (k + 127) // 128 * 128
    v, byte = _mx4_parts(torch.nn.functional.pad(w.float(), (0, kp - k)).view(rows, kp // 32, 32))
    a = v.abs()
    code = ((a >= 0.5).int() + (a >= 1).int() + (a >= 1.5).int() + (a >= 2).int() + (a >= 3).int() + (a >= 4).int()
            + (a >= 6).int() + 8 * torch.signbit(v).int()).view(rows, kp)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    dt = _TYPES[case['dtype']]
    if case['op'] == 'quantize':
        return dict(case=case, x=_tokens(g, case['rows'], case['k'], dt))
    n, k, e = case['n'], case['k'], case.get('e', 1)
    rows = case['m'] if case['op'] == 'linear' else case['s']
    st = dict(case=case, x=_tokens(g, rows, k, dt))
    w = 0.02 * torch.randn(e, n, k, generator=g, device='cuda')
    b = 0.02 * torch.randn(e, n, generator=g, device='cuda')
    if case['op'] in ('linear', 'mx4_experts'):
        codes, scales = _pack(w.view(e * n, k))
        if case['op'] == 'linear':
            st.update(codes=codes, scales=scales, b=b[0].contiguous())
        else:
            st.update(codes=codes.view(e, n, -1), scales=scales.view(e, n, -1), b=b)
    else:
        st.update(w=w.to(dt), b=b.to(dt))
    if case['op'] != 'linear':
        ends = _offsets(case, seed)
        st['offsets'] = torch.tensor(ends, dtype=torch.int32, device='cuda')
        st['longest'] = max(max(q - p for p, q in zip(ends, ends[1:])), 1)  # what a padded batch of the experts' slots needs
    if case['op'] == 'experts_train':
        st['dy'] = (1e-2 * torch.randn(rows, n, generator=g, device='cuda')).to(dt)
        st['x'].requires_grad_()
        st['w'].requires_grad_()
        st['b'].requires_grad_()
    return st


# ------------------------------------------------------------------------------------------------------ plain form
def _power(byte):
    """2^(byte - 127) as float32, byte 0 the subnormal 2^-127"""
    bits = torch.where(byte > 0, byte << 23, torch.full_like(byte, 0x00400000))
    return bits.view(torch.float32)


def _mx4_parts(x):
    """x (..., 32) float32 -> (e2m1 values, scale byte): shared exponent floor(log2 max|x|) - 2, elements rounded to the
    nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code, larger ones to 6; a block that is not finite gets byte 255"""
    m = x.abs().amax(-1)
    byte = ((m.view(torch.int32) >> 23) - 2).clamp(min=0)
    bad = ~torch.isfinite(m)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    inv = ((254 - byte.clamp(max=252)) << 23).view(torch.float32)
    v = x * inv.unsqueeze(-1)
    a = v.abs()
    q = (0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + 1.0 * (a > 2.5) + 1.0 * (a >= 3.5)
         + 2.0 * (a > 5))
    return torch.copysign(q, v), byte


def _mx4_round(x):
    """float32 values of the 4-bit form of the rows of x"""
    rows, k = x.shape
    kp = (k + 31) // 32 * 32
    q, byte = _mx4_parts(torch.nn.functional.pad(x.float(), (0, kp - k)).view(rows, kp // 32, 32))
    y = q * _power(byte.clamp(max=252)).unsqueeze(-1)
    y = torch.where((byte == 255).unsqueeze(-1), torch.full_like(y, math.nan), y)
    return y.view(rows, kp)[:, :k]


def _unpack(codes, scales, k):
    """float32 values of packed rows (..., Kp / 2) / (..., Kp / 32)"""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    c = codes.int()
    v = table[torch.stack((c & 15, c >> 4), dim=-1)].view(*scales.shape, 32)
    return (v * _power(scales.int()).unsqueeze(-1)).view(*scales.shape[:-1], -1)[..., :k]


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _places(offsets, longest, rows):
    """slot of each (expert, place) of a padded batch and whether it is one; expert and place of each slot, and whether it
    has an expert"""
    off = offsets.long()
    at = off[:-1, None] + torch.arange(longest, device=off.device)
    held = at < off[1:, None]
    slot = torch.arange(rows, device=off.device)
    expert = (slot[:, None] >= off[None, 1:]).sum(1)
    some = (slot >= off[0]) & (slot < off[-1])
    expert = expert.clamp(max=off.numel() - 2)
    return at.clamp(max=rows - 1), held, expert, (slot - off[expert]).clamp(0, longest - 1), some


def _to_experts(x, at, held):
    return torch.where(held[..., None], x[at], torch.zeros((), device=x.device))


def _from_experts(y, expert, place, some):
    return torch.where(some[:, None], y[expert, place], torch.zeros((), device=y.device))


def _plain(st):
    case, x = st['case'], st['x'].detach()
    dt = x.dtype
    if case['op'] == 'quantize':
        return _mx4_round(x).to(dt)
    if case['op'] == 'linear':
        y = _mx4_round(x) @ _unpack(st['codes'], st['scales'], case['k']).t() + st['b'].float()
        return (_gelu(y) if case['gelu'] else y).to(dt)
    at, held, expert, place, some = _places(st['offsets'], st['longest'], x.shape[0])
    if case['op'] == 'mx4_experts':
        w = _unpack(st['codes'], st['scales'], case['k'])
        y = torch.bmm(_to_experts(_mx4_round(x), at, held), w.transpose(1, 2)) + st['b'].float()[:, None]
        y = _gelu(y) if case['gelu'] else y
        return _from_experts(y, expert, place, some).to(dt)
    w, xe = st['w'].detach().float(), _to_experts(x.float(), at, held)
    y = torch.bmm(xe, w.transpose(1, 2)) + st['b'].detach().float()[:, None]
    y = _from_experts(y, expert, place, some).to(dt)
    if case['op'] == 'experts':
        return y
    de = _to_experts(st['dy'].float(), at, held)
    dx = _from_experts(torch.bmm(de, w), expert, place, some).to(dt)
    dw = torch.bmm(de.transpose(1, 2), xe).to(dt)
    return dict(y=y, dx=dx, dw=dw, db=de.sum(1).to(dt))


# ------------------------------------------------------------------------------------------------------ the calls
def _own(st):
    from sm3det_amd import expert_ops, mx4
    case, x = st['case'], st['x']
    if case['op'] == 'quantize':
        return mx4.quantize(x).dequantize(x.dtype)
    if case['op'] in ('linear', 'mx4_experts'):
        w = mx4.Mx4Tensor(st['codes'], st['scales'], case['k'])
        act = 'gelu' if case['gelu'] else None
        if case['op'] == 'linear':
            return mx4.linear(x, w, st['b'], act=act)
        return mx4.expert_linear(x, w, st['offsets'], st['b'], act=act)
    y = expert_ops.expert_linear(x, st['w'], st['offsets'], st['b'])
    if case['op'] == 'experts':
        return y
    dx, dw, db = torch.autograd.grad(y, (x, st['w'], st['b']), st['dy'])
    return dict(y=y.detach(), dx=dx, dw=dw, db=db)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------ floors
def work(case):
    es = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'quantize':
        return dict(bytes=2 * es * case['rows'] * case['k'], flops=4 * case['rows'] * case['k'])
    n, k, e = case['n'], case['k'], case.get('e', 1)
    rows = case['m'] if case['op'] == 'linear' else case['s']
    flops = 2 * rows * n * k
    io = es * rows * (n + k)
    if case['op'] in ('linear', 'mx4_experts'):
        return dict(bytes=io + e * n * k * 17 // 32 + 4 * e * n, flops=flops)
    if case['op'] == 'experts':
        return dict(bytes=io + es * e * n * (k + 1), flops=flops)
    return dict(bytes=2 * io + 2 * es * e * n * (k + 1), flops=3 * flops)


# ------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    x = st['x'].detach().double()

    def rounded(t):
        r, k = t.shape
        t = torch.cat([t, t.new_zeros(r, -k % 32)], 1).reshape(r, -1, 32)
        exp = torch.frexp(t.abs().max(-1, keepdim=True).values)[1].double() - 1  # floor(log2 max)
        scale = torch.exp2((exp - 2).clamp(min=-127))
        u = (t / scale).clamp(-6, 6)
        step = torch.where(u.abs() < 2, 0.5, torch.where(u.abs() < 4, 1.0, 2.0)).double()
        return (torch.round(u / step) * step * scale).reshape(r, -1)[:, :k]  # torch.round: halves to even

    def weights(codes, scales):
        low, high = codes.long() % 16, codes.long() // 16
        c = torch.stack([low, high], -1).reshape(codes.shape[0], -1)
        mag = c % 8
        val = torch.where(mag < 2, mag * 0.5, (1 + (mag % 2) * 0.5) * torch.exp2((mag // 2 - 1).double()))
        val = torch.where(c >= 8, -val, val).double()
        return (val * torch.exp2(scales.double() - 127).repeat_interleave(32, 1))[:, :case['k']]

    def act(v):
        return v * torch.special.ndtr(v) if case.get('gelu') else v

    if case['op'] == 'quantize':
        return rounded(x)
    if case['op'] == 'linear':
        return act(rounded(x) @ weights(st['codes'], st['scales']).T + st['b'].double())
    ends = _offsets(case, seed)
    y = torch.zeros(case['s'], case['n'], dtype=torch.float64, device=x.device)
    if case['op'] == 'mx4_experts':
        xq = rounded(x)
        for i in range(case['e']):
            p, q = ends[i], ends[i + 1]
            y[p:q] = act(xq[p:q] @ weights(st['codes'][i], st['scales'][i]).T + st['b'][i].double())
        return y
    w, b = st['w'].detach().double(), st['b'].detach().double()
    for i in range(case['e']):
        p, q = ends[i], ends[i + 1]
        y[p:q] = x[p:q] @ w[i].T + b[i]
    if case['op'] == 'experts':
        return y
    dy = st['dy'].double()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i in range(case['e']):
        p, q = ends[i], ends[i + 1]
        dx[p:q] = dy[p:q] @ w[i]
        dw[i] = dy[p:q].T @ x[p:q]
        db[i] = dy[p:q].sum(0)
    return dict(y=y, dx=dx, dw=dw, db=db)
