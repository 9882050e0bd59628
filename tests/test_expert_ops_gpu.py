"""16-bit products grouped by expert and their gradients against 64-bit references (sm3det_amd/expert_ops.py)."""
import pytest
import torch

from tests.expert_common import assert_within, bound, ragged, spans

pytestmark = pytest.mark.gpu
DT = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _make(seed, rows, e, n, k, dtype, bias=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).to(dtype).cuda()
    w = (torch.randn(e, n, k, generator=g) * k ** -0.5).to(dtype).cuda()
    b = torch.randn(e, n, generator=g).to(bias).cuda()
    dy = torch.randn(rows, n, generator=g).to(dtype).cuda()
    return x, w, b, dy


def _check_all(x, w, b, dy, offsets, outs, dtype):
    y, dx, dw, db = outs
    rows, k = x.shape
    e, n = w.shape[:2]
    X, W, D = x.double(), w.double(), dy.double()
    left = torch.ones(rows, dtype=torch.bool, device='cuda')
    for g, (p, q) in enumerate(spans(offsets, rows)):
        left[p:q] = False
        c = q - p
        if c:
            ref = X[p:q] @ W[g].t() + (b[g].double() if b is not None else 0)
            mag = X[p:q].abs() @ W[g].abs().t() + (b[g].double().abs() if b is not None else 0)
            assert_within(y[p:q], ref, bound(ref, mag, k, dtype), f'y of expert {g}')
            ref = D[p:q] @ W[g]
            assert_within(dx[p:q], ref, bound(ref, D[p:q].abs() @ W[g].abs(), n, dtype), f'dx of expert {g}')
        ref = D[p:q].t() @ X[p:q]
        assert_within(dw[g], ref, bound(ref, D[p:q].abs().t() @ X[p:q].abs(), c, dtype), f'dw of expert {g}')
        if db is not None:
            ref = D[p:q].sum(0)
            assert_within(db[g], ref, bound(ref, D[p:q].abs().sum(0), c, db.dtype), f'db of expert {g}')
    assert not y[left].any() and not dx[left].any()


def _run(x, w, b, dy, offsets):
    from sm3det_amd import expert_ops
    off = torch.tensor(offsets, dtype=torch.int32, device='cuda')
    leaves = [t.detach().clone().requires_grad_() for t in ((x, w) if b is None else (x, w, b))]
    y = expert_ops.expert_linear(leaves[0], leaves[1], off, leaves[2] if b is not None else None)
    grads = torch.autograd.grad(y, leaves, dy)
    return (y.detach(), *grads) + (() if b is not None else (None,))


CASES = [  # rows, offsets, n, k
    (1, [0, 1], 1, 1),
    (1, [0, 0, 1, 1], 8, 8),
    (7, ragged(1, 7, 4), 33, 70),
    (24, ragged(2, 24, 8), 256, 128),
    (130, [0, 130], 128, 64),
    (300, ragged(3, 300, 5), 130, 96),
    (300, ragged(4, 300, 5, head=20, tail=37), 117, 203),
    (500, [0, 0, 0, 500], 64, 128),
    (500, [500, 500, 500], 64, 40),
    (257, [0] + [257] * 70, 48, 64),
    (1000, ragged(5, 1000, 130), 40, 72),
    (4000, ragged(6, 4000, 3, tail=1), 264, 136),
    (1500, ragged(7, 1500, 2), 520, 1032),
    (100, [-5, 40, 30, 1000, 60], 40, 64),
]


@pytest.mark.parametrize('rows,offsets,n,k', CASES, ids=range(len(CASES)))
@pytest.mark.parametrize('dtype', DT)
def test_forward_and_gradients(rows, offsets, n, k, dtype):
    dt = DT[dtype]
    for bias in (torch.float32, dt):
        x, w, b, dy = _make(rows + n, rows, len(offsets) - 1, n, k, dt, bias)
        _check_all(x, w, b, dy, offsets, _run(x, w, b, dy, offsets), dt)


@pytest.mark.parametrize('dtype', DT)
def test_without_bias_and_no_rows_at_all(dtype):
    dt = DT[dtype]
    x, w, b, dy = _make(3, 90, 3, 24, 48, dt)
    _check_all(x, w, None, dy, [0, 10, 10, 90], _run(x, w, None, dy, [0, 10, 10, 90]), dt)
    y, dx, dw, db = _run(x[:0], w, b, dy[:0], [0, 0, 0, 0])
    assert y.shape == (0, 24) and dx.shape == (0, 48) and not dw.any() and not db.any()


@pytest.mark.parametrize('dtype', DT)
def test_gradients_are_the_differences_of_the_function(dtype):
    """inputs are small integers: the products, their sums and the differences of the loss are exact"""
    from sm3det_amd import expert_ops
    dt, off = DT[dtype], torch.tensor([2, 9, 9, 20], dtype=torch.int32, device='cuda')
    g = torch.Generator().manual_seed(1)

    def ints(*shape, most):
        return torch.randint(-most, most + 1, shape, generator=g).to(dt).cuda()
    x, w, b, dy = ints(22, 6, most=3), ints(3, 5, 6, most=3), ints(3, 5, most=3), ints(22, 5, most=2)

    def loss(x, w, b):
        return (expert_ops.expert_linear(x, w, off, b).double() * dy.double()).sum()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(expert_ops.expert_linear(leaves[0], leaves[1], off, leaves[2]), leaves, dy)
    for i in range(3):
        for place in range(0, leaves[i].numel(), 7):
            bumped = [t.clone() for t in (x, w, b)]
            bumped[i].view(-1)[place] += 1
            assert (loss(*bumped) - loss(x, w, b)).item() == grads[i].reshape(-1)[place].item(), (i, place)


def test_views_strides_and_unaligned_rows():
    big = torch.randn(90, 400, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    _, w, b, dy = _make(3, 90, 3, 40, 64, torch.bfloat16)
    off = [0, 25, 25, 90]
    for x in (big[:, 8:72], big[:, 3:67], big[:, :128:2], big.t()[:90, :64], big[:1, :64].expand(90, 64)):
        for wv in (w, w.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([w, w], 2)[:, :, 64:]):
            for d in (dy, dy[:, :1].expand(90, 40), torch.cat([dy, dy], 1)[:, 40:]):
                _check_all(x, wv, b, d, off, _run_views(x, wv, b, d, off), torch.bfloat16)


def _run_views(x, w, b, dy, offsets):
    from sm3det_amd import expert_ops
    x, w, b = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
    y = expert_ops.expert_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device='cuda'), b)
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))


def test_only_the_gradients_asked_for():
    from sm3det_amd import expert_ops
    x, w, b, dy = _make(3, 90, 3, 40, 64, torch.float16)
    off = torch.tensor([0, 25, 25, 90], dtype=torch.int32, device='cuda')
    full = _run(x, w, b, dy, [0, 25, 25, 90])
    for need in range(1, 8):
        leaves = [t.detach().clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        y = expert_ops.expert_linear(leaves[0], leaves[1], off, leaves[2])
        asked = [t for t in leaves if t.requires_grad]
        for got, want in zip(torch.autograd.grad(y, asked, dy), [f for i, f in enumerate(full[1:]) if need >> i & 1]):
            assert torch.equal(got, want)


def test_nan_rows_of_no_expert_enter_nothing():
    x, w, b, dy = _make(5, 90, 2, 40, 64, torch.bfloat16)
    off = [10, 30, 80]
    clean = _run(x, w, b, dy, off)
    for t in (x, dy):
        t[:10], t[80:] = float('nan'), float('inf')
    for a, c in zip(_run(x, w, b, dy, off), clean):
        assert torch.equal(a, c)


def test_one_experts_infinities_stay_with_it():
    x, w, b, dy = _make(5, 90, 2, 40, 72, torch.bfloat16)
    off = [0, 37, 90]
    clean = _run(x, w, b, dy, off)
    x[40], dy[50], w[1, 3] = float('inf'), float('nan'), float('nan')
    y, dx, dw, db = _run(x, w, b, dy, off)
    assert torch.equal(y[:37], clean[0][:37]) and torch.equal(dx[:37], clean[1][:37])
    assert torch.equal(dw[0], clean[2][0]) and torch.equal(db[0], clean[3][0])


def test_rows_beyond_32_bit_byte_offsets():
    from sm3det_amd import expert_ops
    rows, k, n = (1 << 21) + 300, 1040, 16  # 4.06 GiB of activations
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device='cuda')
    dy = torch.zeros(rows, n, dtype=torch.bfloat16, device='cuda')
    xs, w, b, ds = _make(1, 500, 2, n, k, torch.bfloat16)
    x[-500:], dy[-500:] = xs, ds
    off = [0, rows - 500, rows]
    y, dx, dw, db = _run(x, w, b, dy, off)
    outs = (y[-500:], dx[-500:], dw, db)
    _check_all(xs, w, b, ds, [0, 0, 500], outs, torch.bfloat16)
    assert not dx[:-500].any() and torch.equal(y[:1].expand(rows - 500, n), y[:-500])


@pytest.mark.parametrize('experts', (63, 64, 65))
@pytest.mark.parametrize('rows', (90, 3000, 20000))
def test_as_many_experts_as_lanes(experts, rows):
    """up to 64 experts the job list is made by one wave's lanes, beyond by a loop; rows: empty experts, whole and cut ones"""
    off = ragged(experts, rows, experts, head=3, tail=4)
    x, w, b, dy = _make(experts, rows, experts, 72, 40, torch.bfloat16)
    _check_all(x, w, b, dy, off, _run(x, w, b, dy, off), torch.bfloat16)


def test_more_columns_than_a_tile_addresses():
    n = (1 << 20) + 8
    x, w, b, dy = _make(5, 5, 1, n, 32, torch.bfloat16)
    _check_all(x, w, b, dy, [0, 3], _run(x, w, b, dy, [0, 3]), torch.bfloat16)


def test_repeated_calls_other_streams_and_graph_replays_agree():
    from sm3det_amd import expert_ops
    x, w, b, dy = _make(5, 900, 6, 200, 136, torch.bfloat16)
    off = torch.tensor(ragged(7, 900, 6, tail=11), dtype=torch.int32, device='cuda')
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def step():
        y = expert_ops.expert_linear(x, w, off, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(step(), first))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(other, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        nx, _, _, nd = _make(seed, 900, 6, 200, 136, torch.bfloat16)
        with torch.no_grad():
            x.copy_(nx)
        dy.copy_(nd)
        off.copy_(torch.tensor(ragged(seed, 900, 6, head=3), dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_second_derivatives_are_refused():
    from sm3det_amd import expert_ops
    x, w, b, dy = _make(5, 20, 2, 8, 8, torch.bfloat16)
    off = torch.tensor([0, 5, 20], dtype=torch.int32, device='cuda')
    x = x.requires_grad_()
    (dx,) = torch.autograd.grad(expert_ops.expert_linear(x, w, off, b), x, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().sum(), dy)
