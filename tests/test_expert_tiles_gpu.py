"""The grouped products at the sizes that reach each of their ways (tests/expert_shapes.py): large tiles and the quarters that finish
them, several tiles per workgroup, whole and cut units of the weight gradient, sliced reductions; and the longest rows."""
import pytest
import torch

from tests.expert_common import HALF_STEP, assert_within, bound, spans
from tests.expert_shapes import COARSE, FEW, MX4, SEVERAL, WEIGHT
from tests.test_expert_ops_gpu import _check_all, _run
from tests.test_mx4_gpu import _check, _values

pytestmark = pytest.mark.gpu
DT = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}


def _randn(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, generator=g, device='cuda', dtype=torch.float32) * scale).to(dtype)


def _inputs(rows, e, n, k, dtype, bias=torch.float32):
    return (_randn(1, rows, k, dtype=dtype), _randn(2, e, n, k, dtype=dtype, scale=k ** -0.5), _randn(3, e, n, dtype=bias),
            _randn(4, rows, n, dtype=dtype))


SIZES = {**{'coarse_' + k: v[:4] for k, v in COARSE.items()}, **{'several_' + k: v[:4] for k, v in SEVERAL.items()},
         **{'weight_' + k: v[:4] for k, v in WEIGHT.items()}}


@pytest.mark.parametrize('name', SIZES)
@pytest.mark.parametrize('dtype', ('fp16', 'bf16'))
def test_forward_and_gradients(name, dtype):
    rows, offsets, n, k = SIZES[name]
    x, w, b, dy = _inputs(rows, len(offsets) - 1, n, k, DT[dtype], DT[dtype] if dtype == 'fp16' else torch.float32)
    _check_all(x, w, b, dy, offsets, _run(x, w, b, dy, offsets), DT[dtype])


@pytest.mark.parametrize('name', ('coarse_few_left', 'several_part_filled_steps_forward', 'weight_whole_experts'))
def test_the_same_call_gives_the_same_bits(name):
    rows, offsets, n, k = SIZES[name]
    x, w, b, dy = _inputs(rows, len(offsets) - 1, n, k, torch.bfloat16)
    first = _run(x, w, b, dy, offsets)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(_run(x, w, b, dy, offsets), first))


@pytest.mark.parametrize('name', ('coarse_few_left', 'coarse_quarters_alone'))
def test_nan_rows_of_no_expert_and_one_experts_infinities_stay_out(name):
    rows, offsets, n, k = SIZES[name]
    x, w, b, dy = _inputs(rows, len(offsets) - 1, n, k, torch.bfloat16)
    clean = _run(x, w, b, dy, offsets)
    held = torch.zeros(rows, dtype=torch.bool, device='cuda')
    held[offsets[0]:offsets[-1]] = True
    for t in (x, dy):
        t[~held] = float('nan')
    assert all(torch.equal(a, c) for a, c in zip(_run(x, w, b, dy, offsets), clean))
    p, q = max(spans(offsets, rows), key=lambda s: s[1] - s[0])
    x[p + 130, 5], dy[p + 3, 7] = float('inf'), float('nan')
    y, dx = _run(x, w, b, dy, offsets)[:2]
    other = held.clone()
    other[p:q] = False
    assert torch.equal(y[other], clean[0][other]) and torch.equal(dx[other], clean[1][other])
    mine = torch.arange(rows, device='cuda') == p + 130
    assert torch.equal(torch.isfinite(y).all(1), ~mine)
    assert torch.equal(torch.isfinite(dx).all(1), torch.arange(rows, device='cuda') != p + 3)


@pytest.mark.parametrize('act', (None, 'gelu'))
@pytest.mark.parametrize('bias', (False, True))
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('name', (*MX4, *FEW))
def test_4_bit_products(name, dtype, act, bias):
    from sm3det_amd import mx4
    rows, offsets, n, k = {**MX4, **FEW}[name][:4]
    dt, e = DT[dtype], len(offsets) - 1 if offsets else 1
    x = _randn(1, rows, k, dtype=dt)
    w = mx4.quantize(_randn(2, e, n, k, dtype=torch.float32, scale=k ** -0.5))
    b = _randn(3, e, n, dtype=torch.float32) if bias else None
    xq = mx4.quantize(x)
    xv, wv = _values(xq), _values(w)
    if offsets is None:
        wd = mx4.Mx4Tensor(w.codes[0], w.scales[0], k)
        y, packed = (mx4.linear(t, wd, None if b is None else b[0], act=act, out_dtype=dt) for t in (x, xq))
    else:
        off = torch.tensor(offsets, dtype=torch.int32, device='cuda')
        y, packed = (mx4.expert_linear(t, w, off, b, act=act, out_dtype=dt) for t in (x, xq))
    if name in MX4:  # (few rows per expert have a kernel of their own unless they come packed)
        assert torch.equal(y, packed)
    left = torch.ones(rows, dtype=torch.bool, device='cuda')
    for g, (p, q) in enumerate(spans(offsets or [0, rows], rows)):
        if q > p:
            add = b[g].double() if bias else torch.zeros(n, dtype=torch.float64, device='cuda')
            h, mag = xv[p:q] @ wv[g].t() + add, xv[p:q].abs() @ wv[g].abs().t() + add.abs()
            _check(y[p:q], h, mag, k, act, dt, f'expert {g}')
            left[p:q] = False
    assert not y[left].any()


@pytest.mark.parametrize('few', (False, True))
def test_gelu_of_the_4_bit_products(few):
    """rows of zeros: the result is GELU of the bias, which no quantisation touches.  2^p(a) is off from Phi(-a) by at most 4.5e-8
    (the committed coefficients, in 64 bits).  In fp32 the last steps of the polynomial are off by 2^-24 of |p| each, which
    the power turns into 2^p |p| ln 2 <= 1/e of that, the steps before by less than as much again where a < 1 and, where a > 1,
    2^p |p| is smaller than the a by which they grow; the power is off by 2^-24 (one step of at most 1/2), product and sum by 2^-24 of
    |h| and half a step of the result: together less than 2^-22 |h|.  Behind 6 the tail stays |Phi(-6)| * 6 < 6e-9."""
    from sm3det_amd import mx4
    b = torch.cat([torch.linspace(-8, 8, 4001, device='cuda'), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 60000.0, -60000.0, 3e38], device='cuda')])
    n = b.numel()
    w = mx4.quantize(_randn(1, n, 64, dtype=torch.float32))
    y = mx4.linear(torch.zeros(3 if few else 40, 64, device='cuda'), w, b, act='gelu')
    h = b.double()
    want = h * torch.special.ndtr(h)
    assert_within(y, want.expand_as(y), (2.0 ** -22 * h.abs().clamp(max=6.0) + HALF_STEP[torch.float32] * want.abs() + 6e-9).expand_as(y))
    odd = mx4.linear(torch.zeros(3 if few else 40, 64, device='cuda'), mx4.quantize(_randn(1, 2, 64, dtype=torch.float32)),
                     torch.tensor([float('inf'), float('nan')], device='cuda'), act='gelu')
    assert (odd[:, 0] == float('inf')).all() and torch.isnan(odd[:, 1]).all()


@pytest.mark.parametrize('red', ((1 << 22) - 8, (1 << 22) - 3, 1 << 22))
def test_the_longest_reductions(red):
    """4096 x 4096 results of operands of 32 GiB each, zero but for 64 elements at either end of the rows (and 64 in the middle)"""
    from sm3det_amd import expert_ops
    n, places = 4096, [0, red // 2, red - 64]
    off = torch.tensor([0, n], dtype=torch.int32, device='cuda')
    x = torch.zeros(n, red, dtype=torch.bfloat16, device='cuda')
    w = torch.zeros(1, n, red, dtype=torch.bfloat16, device='cuda')
    for i, c in enumerate(places):
        x[:, c:c + 64], w[0, :, c:c + 64] = _randn(i, n, 64, dtype=x.dtype), _randn(9 + i, n, 64, dtype=x.dtype, scale=0.1)
    y = expert_ops.expert_linear(x, w, off)
    X, W = (torch.cat([t[:, c:c + 64] for c in places], 1).double() for t in (x, w[0]))
    del x, w
    torch.cuda.empty_cache()
    ref = X @ W.t()
    assert_within(y, ref, bound(ref, X.abs() @ W.abs().t(), 3 * 64, torch.bfloat16))  # (added zeros are exact)


@pytest.mark.parametrize('bias', (torch.float32, torch.bfloat16))
def test_a_bias_row_of_2_to_the_32_bytes(bias):
    from sm3det_amd import expert_ops
    n = 1 << 30
    w = torch.zeros(1, n, 8, dtype=torch.bfloat16, device='cuda')
    b = torch.ones(1, n, dtype=bias, device='cuda')
    some = torch.cat([torch.arange(300), n // 2 + torch.arange(300), n - 300 + torch.arange(300)]).cuda()
    w[0, some], b[0, some] = _randn(1, 900, 8, dtype=w.dtype), _randn(2, 900, dtype=bias)
    x = _randn(3, 2, 8, dtype=w.dtype)
    y = expert_ops.expert_linear(x, w, torch.tensor([0, 2], dtype=torch.int32, device='cuda'), b)
    W, B = w[0, some].double(), b[0, some].double()
    ref = x.double() @ W.t() + B
    assert_within(y[:, some], ref, bound(ref, x.double().abs() @ W.abs().t() + B.abs(), 8, torch.bfloat16))
    rest = int((y == 1).sum()) - int((y[:, some] == 1).sum())
    del w, b, y
    torch.cuda.empty_cache()
    assert rest == 2 * (n - 900)


@pytest.mark.parametrize('n', ((1 << 28) - 16, 1 << 28, (1 << 28) + 40))
def test_few_rows_of_very_many_columns(n):
    """a launch holds fewer than 2^32 threads: behind 2^28 columns the one-launch kernel of few rows would need more"""
    from sm3det_amd import mx4
    codes = torch.zeros(n, 64, dtype=torch.uint8, device='cuda')
    scales = torch.full((n, 4), 127, dtype=torch.uint8, device='cuda')
    some = torch.cat([torch.arange(200), n // 2 + torch.arange(200), n - 200 + torch.arange(200)]).cuda()
    codes[some] = torch.randint(0, 256, (600, 64), generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').to(torch.uint8)
    w = mx4.Mx4Tensor(codes, scales, 128)
    x = _randn(2, 3, 128, dtype=torch.bfloat16)
    y = mx4.linear(x, w)
    X, W = _values(mx4.quantize(x)), _values(mx4.Mx4Tensor(codes[some], scales[some], 128))
    ref = X @ W.t()
    assert_within(y[:, some], ref, bound(ref, X.abs() @ W.abs().t(), 128, torch.bfloat16))
    rest = int(y.count_nonzero()) - int(y[:, some].count_nonzero())
    del w, codes, scales, y
    torch.cuda.empty_cache()
    assert rest == 0
