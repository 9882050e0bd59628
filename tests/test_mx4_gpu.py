"""Microscaled 4-bit quantisation and products against plain 64-bit restatements (sm3det_amd/mx4.py)."""
import numpy as np
import pytest
import torch

from tests.expert_common import HALF_STEP, SMALLEST, assert_within, bound, quantize_ref, ragged, spans

pytestmark = pytest.mark.gpu
DT = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}


def _rows(seed, rows, k, dtype, spread=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-spread, spread, (rows, 1), generator=g).float())
    return x.to(dtype).cuda()


def _same(q, ref):
    codes, scales, _ = ref
    assert np.array_equal(q.scales.cpu().numpy().reshape(scales.shape), scales)
    got = q.codes.cpu().numpy().reshape(codes.shape)
    bad = scales.repeat(16, 1) == 255  # the codes of a NaN block mean nothing
    assert np.array_equal(np.where(bad, 0, got), np.where(bad, 0, codes))


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('rows,k', [(1, 1), (1, 32), (3, 31), (5, 33), (2, 128), (7, 203), (64, 96), (33, 384), (300, 1000)])
def test_quantize_matches_the_definition_bit_for_bit(rows, k, dtype):
    from sm3det_amd import mx4
    x = _rows(rows * 7 + k, rows, k, DT[dtype])
    q = mx4.quantize(x)
    ref = quantize_ref(x.double().cpu().numpy())
    _same(q, ref)
    assert q.shape == (rows, k)
    assert np.array_equal(q.dequantize().double().cpu().numpy(), ref[2])


@pytest.mark.parametrize('dtype', DT)
def test_quantize_at_ties_saturation_and_the_ends_of_the_range(dtype):
    from sm3det_amd import mx4
    grid = torch.arange(-64, 65).double() / 8  # every tie and both sides of it, up to 8 > 6
    tiny, big = (2.0 ** -140, 2.0 ** 125) if dtype != 'fp16' else (2.0 ** -24, 2.0 ** 12)
    rows = [torch.cat([grid[i:i + 31], torch.tensor([7.99], dtype=torch.float64)]) for i in range(0, 96, 31)]
    x = torch.stack(rows + [rows[0] * tiny, rows[1] * big, rows[2] * 0, -rows[3] * tiny * 4])
    x = x.to(DT[dtype]).cuda()
    ref = quantize_ref(x.double().cpu().numpy())
    q = mx4.quantize(x)
    _same(q, ref)
    # (7.99 * 2^125 rounds to 2^128 in bfloat16: that block is infinite on the way in, NaN in both)
    assert np.array_equal(q.dequantize().double().cpu().numpy(), ref[2], equal_nan=True)


@pytest.mark.parametrize('dtype', DT)
def test_blocks_with_infinities_or_nans_are_nan_and_their_neighbours_are_not(dtype):
    from sm3det_amd import mx4
    x = _rows(3, 6, 100, DT[dtype])
    x[0, 5], x[1, 40], x[2, 99] = float('inf'), float('nan'), -float('inf')
    q = mx4.quantize(x)
    ref = quantize_ref(x.double().cpu().numpy())
    _same(q, ref)
    got = q.dequantize(DT[dtype]).double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref[2])) and np.isnan(got).sum() == 32 + 32 + 4
    ok = ~np.isnan(got)
    if dtype != 'fp16':
        assert np.array_equal(got[ok], ref[2][ok])


def test_quantize_reads_strided_rows_and_leading_dimensions():
    from sm3det_amd import mx4
    big = _rows(5, 40, 300, torch.bfloat16)
    for view in (big[:, 8:200], big[:, 3:202], big[::3, :128], big.t()[:200], big[1:2, 5:90], big[:1].expand(7, 300)):
        _same(mx4.quantize(view), quantize_ref(view.double().cpu().numpy()))
    q = mx4.quantize(big.view(4, 10, 300))
    assert q.shape == (4, 10, 300) and q.dequantize().shape == (4, 10, 300)
    _same(q, quantize_ref(big.double().cpu().numpy()))
    assert mx4.quantize(big[:0]).shape == (0, 300)
    assert mx4.quantize(big[:0]).dequantize().shape == (0, 300)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_dequantize_rounds_to_nearest(dtype):
    from sm3det_amd import mx4
    x = _rows(9, 16, 160, torch.float32, spread=30)
    q = mx4.quantize(x)
    want = q.dequantize().to(DT[dtype])  # (values beyond fp16's largest become infinite in both)
    assert torch.equal(q.dequantize(DT[dtype]).view(torch.int16), want.view(torch.int16))


def test_rows_beyond_32_bit_byte_offsets():
    from sm3det_amd import mx4
    rows, k = (1 << 21) + 3, 1040  # 4.06 GiB of bf16
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device='cuda')
    x[-2:] = _rows(1, 2, k, torch.bfloat16)
    q = mx4.quantize(x)
    ref = quantize_ref(x[-2:].double().cpu().numpy())
    assert np.array_equal(q.codes[-2:].cpu().numpy(), ref[0]) and np.array_equal(q.scales[-2:].cpu().numpy(), ref[1])
    assert not q.codes[:-2].any()
    y = mx4.linear(q, mx4.quantize(x[-1:].clone()), out_dtype=torch.bfloat16)
    v = torch.from_numpy(ref[2]).cuda()
    want = v @ v[1]
    assert_within(y[-2:, 0], want, bound(want, v.abs() @ v[1].abs(), k, torch.bfloat16))
    assert not y[:-2].any()


def _gelu(h):
    return h * torch.special.ndtr(h)


def _values(q):
    return q.dequantize(torch.float32).double()


def _check(y, h, mag, k, act, dtype, what=''):
    """h, mag: the sums (with bias) and sums of magnitudes in 64 bits"""
    if act is None:
        return assert_within(y, h, bound(h, mag, k, dtype), what)
    # |gelu'| <= 1.13; the operator's erfc is off by at most 1.5e-7 (Abramowitz & Stegun 7.1.26), its exponential and reciprocal by
    # a few steps of 2^-23 of a value of at most 1/2 (the argument h^2 / 2 times e^(-h^2 / 2) is below 1/2 too): 2^-20 |h| in all
    acc = 1.13 * (k + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * h.abs()
    g = _gelu(h)
    assert_within(y, g, acc + HALF_STEP[dtype] * (g.abs() + acc) + 0.5 * SMALLEST[dtype], what)


LINEAR = [(1, 1, 1), (1, 8, 32), (2, 130, 96), (17, 64, 128), (32, 257, 300), (33, 40, 256), (129, 128, 512), (200, 250, 603),
          (1, 4096, 1024), (5, 96, 4096), (300, 384, 96), (700, 130, 2000), (16, 17, 129), (15, 33, 1000), (3, 250, 603)]


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('m,n,k', LINEAR)
def test_linear(m, n, k, dtype):
    from sm3det_amd import mx4
    dt = DT[dtype]
    x = _rows(m + 3 * n + k, m, k, dt, spread=2)
    w = mx4.quantize(_rows(k, n, k, torch.float32, spread=2) * k ** -0.5)
    b = torch.linspace(-1, 1, n, device='cuda')
    xv, wv = _values(mx4.quantize(x)), _values(w)
    h, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    _check(mx4.linear(x, w), h, mag, k, None, dt, 'plain')
    hb, magb = h + b.double(), mag + b.abs().double()
    for act in (None, 'gelu'):
        _check(mx4.linear(x, w, b, act=act), hb, magb, k, act, dt, str(act))
    bh = b.to(torch.float16)
    _check(mx4.linear(x, w, bh), h + bh.double(), mag + bh.abs().double(), k, None, dt, 'fp16 bias')


def test_linear_of_packed_rows_and_other_result_types():
    from sm3det_amd import mx4
    x, w = _rows(1, 70, 224, torch.float16), mx4.quantize(_rows(2, 90, 224, torch.float32))
    xq = mx4.quantize(x)
    assert mx4.linear(xq, w).dtype == torch.float32
    for dt in DT.values():
        assert torch.equal(mx4.linear(xq, w, out_dtype=dt), mx4.linear(x, w, out_dtype=dt))
    assert mx4.linear(x[:0], w).shape == (0, 90)


def test_a_nan_block_poisons_its_row_and_its_column_alone():
    from sm3det_amd import mx4
    for m, n, k in ((40, 50, 200), (1, 50, 96), (300, 200, 640)):
        x, w = _rows(1, m, k, torch.bfloat16), _rows(2, n, k, torch.float32)
        x[m // 2, k - 1] = float('inf')
        w[3, 0] = float('nan')
        y = mx4.linear(x, mx4.quantize(w))
        want = torch.zeros(m, n, dtype=torch.bool, device='cuda')
        want[m // 2], want[:, 3] = True, True
        assert torch.equal(torch.isnan(y), want)


GROUPED = [  # rows, offsets, n, k
    (8, ragged(1, 8, 8), 64, 96),
    (1, [0, 0, 1, 1], 33, 40),
    (300, ragged(2, 300, 5), 130, 256),
    (300, ragged(3, 300, 5, head=20, tail=37), 130, 203),
    (500, [0, 0, 0, 500], 64, 128),
    (500, [500, 500, 500], 64, 128),   # nobody's rows
    (257, [0] + [257] * 70, 48, 64),   # more experts than lanes
    (1000, ragged(4, 1000, 130), 32, 96),
    (2000, ragged(5, 2000, 3, tail=1), 260, 1100),
    (640, [0, 128, 256, 384, 640], 128, 512),
    (100, [-5, 40, 30, 1000, 60], 40, 64),  # clamped and made monotone
]


@pytest.mark.parametrize('rows,offsets,n,k', GROUPED, ids=range(len(GROUPED)))
@pytest.mark.parametrize('dtype,act', [('bf16', 'gelu'), ('fp32', None), ('fp16', None)])
def test_expert_linear(rows, offsets, n, k, dtype, act):
    from sm3det_amd import mx4
    dt, e = DT[dtype], len(offsets) - 1
    x = _rows(rows + n, rows, k, dt, spread=2)
    w = mx4.quantize(_rows(k + e, e * n, k, torch.float32, spread=2).view(e, n, k) * k ** -0.5)
    b = torch.randn(e, n, generator=torch.Generator().manual_seed(1)).cuda()
    y = mx4.expert_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device='cuda'), b, act=act)
    xv, wv = _values(mx4.quantize(x)), _values(w)
    left = torch.ones(rows, dtype=torch.bool, device='cuda')
    for g, (p, q) in enumerate(spans(offsets, rows)):
        if q > p:
            h, mag = xv[p:q] @ wv[g].t() + b[g].double(), xv[p:q].abs() @ wv[g].abs().t() + b[g].abs().double()
            _check(y[p:q], h, mag, k, act, dt, f'expert {g}')
            left[p:q] = False
    assert not y[left].any()


def test_nan_rows_of_no_expert_stay_out():
    from sm3det_amd import mx4
    x = _rows(1, 90, 96, torch.bfloat16)
    off = torch.tensor([10, 30, 80], dtype=torch.int32, device='cuda')
    w = mx4.quantize(_rows(2, 2 * 40, 96, torch.float32).view(2, 40, 96))
    clean = mx4.expert_linear(x, w, off)
    x[:10], x[80:] = float('nan'), float('inf')
    assert torch.equal(mx4.expert_linear(x, w, off), clean)


def test_on_another_stream_and_replayed_from_a_graph():
    from sm3det_amd import mx4
    x = _rows(1, 400, 320, torch.bfloat16)
    off = torch.tensor(ragged(7, 400, 6, tail=11), dtype=torch.int32, device='cuda')
    w = mx4.quantize(_rows(2, 6 * 200, 320, torch.float32).view(6, 200, 320))
    few = x[:3].clone()
    wd = mx4.quantize(_rows(3, 200, 320, torch.float32))

    def both():
        return mx4.expert_linear(x, w, off, act='gelu'), mx4.linear(few, wd)
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (11, 12, 13):  # new inputs and new expert loads through the same graph, eager work in between
        x.copy_(_rows(seed, 400, 320, torch.bfloat16))
        few.copy_(x[5:8])
        off.copy_(torch.tensor(ragged(seed, 400, 6, head=3), dtype=torch.int32))
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_the_same_call_gives_the_same_bits():
    from sm3det_amd import mx4
    x, w = _rows(1, 6, 4000, torch.float32), mx4.quantize(_rows(2, 100, 4000, torch.float32))
    first = mx4.linear(x, w)
    assert all(torch.equal(mx4.linear(x, w), first) for _ in range(5))


# ---- the operators together: quantise, first product with GELU, second product, by expert -- and the backbone's MoE blocks
def _plain_ffn(x, w1, b1, w2, b2, offsets):
    """64-bit restatement of expert_ffn on the packed weights' values -> (y, sums of magnitudes, largest hidden value)"""
    e, c = w1.shape[0], x.shape[1]
    rows = x.shape[0]
    y = torch.zeros(rows, c, dtype=torch.float64, device='cuda')
    mag, top = torch.zeros_like(y), 0.0
    for g, (p, q) in enumerate(spans(offsets, rows)):
        if p == q:
            continue
        xv = torch.from_numpy(quantize_ref(x[p:q].double().cpu().numpy())[2]).cuda()
        h = _gelu(xv @ w1[g].t() + b1[g].double()).to(torch.bfloat16)
        hv = torch.from_numpy(quantize_ref(h.double().cpu().numpy())[2]).cuda()
        y[p:q] = hv @ w2[g].t() + b2[g].double()
        mag[p:q] = hv.abs() @ w2[g].abs().t() + b2[g].abs().double()
        top = max(top, h.abs().max().item())
    return y, mag, top


def _check_ffn(got, x, w1, b1, w2, b2, offsets):
    W1, W2 = _values(w1), _values(w2)
    y, mag, top = _plain_ffn(x, W1, b1, W2, b2, offsets)
    # hidden values next to a border of the 4-bit grid may round to its other side: each moves by at most half its block's
    # largest value; their share is the fp32 sums' error over the grid's spacing, about 1e-6: allow three in a row's reduction
    flips = 3 * W2.abs().max().item() * top / 2
    assert_within(got, y, bound(y, mag, W2.shape[2], torch.float32) + flips)


@pytest.mark.parametrize('rows,e,c,seed', [(700, 8, 96, 1), (12, 4, 64, 2), (2500, 3, 136, 3)])
@pytest.mark.parametrize('dtype', ['fp32', 'fp16'])
def test_expert_ffn(rows, e, c, seed, dtype):
    from sm3det_amd import mx4
    x = _rows(seed, rows, c, DT[dtype], spread=1)
    w1 = mx4.quantize(_rows(seed + 1, e * 4 * c, c, torch.float32, spread=1).view(e, 4 * c, c) * c ** -0.5)
    w2 = mx4.quantize(_rows(seed + 2, e * c, 4 * c, torch.float32, spread=1).view(e, c, 4 * c) * (4 * c) ** -0.5)
    b1, b2 = _rows(seed + 3, e, 4 * c, torch.float32, spread=1), _rows(seed + 4, e, c, torch.float32, spread=1)
    offsets = ragged(seed, rows, e, tail=rows // 20)
    off = torch.tensor(offsets, dtype=torch.int32, device='cuda')
    got = mx4.expert_ffn(x, w1, b1, w2, b2, off)
    assert got.dtype == torch.float32
    _check_ffn(got, x, w1, b1, w2, b2, offsets)


def test_backbone_with_quantised_experts(monkeypatch):
    """every MoE block of the fixture's backbone in evaluation: the experts' inputs and outputs are caught and checked, the
    rest of the forward is the full-precision one"""
    from sm3det_amd import mx4
    from sm3det_amd._lib import SM3Error
    from sm3det_amd.convnext_moe import ConvNeXt_moe_MultiInput, MoE_layer
    from tests.moe_common import load_fixture
    fx = load_fixture('moe_e4k2')
    net = ConvNeXt_moe_MultiInput(**fx['cfg'])
    net.load_state_dict(fx['state_dict'])
    net = net.cuda()
    with pytest.raises(SM3Error):
        mx4.quantize_experts(net.train())
    net.eval()
    x = fx['x'].cuda()
    with torch.no_grad():
        full = net(x, ['single'])
    layers = [m for m in net.modules() if isinstance(m, MoE_layer)]
    assert mx4.quantize_experts(net) == len(layers) > 0
    caught = []
    ffn = mx4.expert_ffn

    def spy(xs, w1, b1, w2, b2, offsets):
        y = ffn(xs, w1, b1, w2, b2, offsets)
        caught.append((xs, w1, b1, w2, b2, offsets, y))
        return y
    monkeypatch.setattr(mx4, 'expert_ffn', spy)
    with torch.no_grad():
        outs = net(x, ['single'])
    assert len(caught) == len(layers)
    for (xs, w1, b1, w2, b2, offsets, y), m in zip(caught, layers):
        assert w1.shape == m.w1.shape and w2.shape == m.w2.shape
        _check_ffn(y, xs, w1, b1, w2, b2, offsets.tolist())
    for a, b in zip(outs[0], full[0]):
        assert a.shape == b.shape and torch.isfinite(a).all()
    assert not torch.equal(outs[0][-1], full[0][-1])  # (stages without MoE blocks are the same)
    with pytest.raises(SM3Error):  # a gradient would be needed
        net(x, ['single'])
    for again in (lambda: mx4.restore_experts(net), lambda: net.load_state_dict(fx['state_dict']), lambda: net.train().eval(),
                  lambda: net.cuda()):
        mx4.quantize_experts(net)
        again()
        with torch.no_grad():
            back = net(x, ['single'])
        assert all(torch.equal(a, b) for a, b in zip(back[0], full[0]))
