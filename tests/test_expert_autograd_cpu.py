"""CPU tier of what autograd may ask of the grouped and 4-bit products: the launches are replaced by torch products in 64 bits, so
that the Python side alone is at work."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests.expert_common import spans


def _view(t, rows, cols, ld):
    return t.as_strided((rows, cols), (ld, 1))


def launch(fn, device, mode, dtype, out, p, q, rows, red, cols, *, rows_out=0, ldp=0, ldq=0, groups=1, offsets=None, bias=None,
           bias_grad=None, **_):
    """what sm3_expert_gemm_h16 is asked for, on the CPU"""
    from sm3det_amd import _lib_backbone as LB
    assert fn == 'expert_gemm_h16'
    out.zero_()
    x = _view(p, rows, rows_out if mode == LB.TN else red, ldp).double()
    for g, (a, b) in enumerate(spans(offsets.tolist(), rows)):
        if mode == LB.TN:
            out[g] = (x[a:b].t() @ _view(q, rows, cols, ldq)[a:b].double()).to(out.dtype)
            if bias_grad is not None:
                bias_grad[g] = x[a:b].sum(0).to(bias_grad.dtype)
        else:
            y = x[a:b] @ (q[g].double().t() if mode == LB.NT else q[g].double())
            out[a:b] = (y + bias[g].double() if bias is not None else y).to(out.dtype)


@pytest.fixture
def ops(monkeypatch):
    from sm3det_amd import expert_ops
    monkeypatch.setattr(expert_ops, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(expert_ops, 'launch', launch)
    return expert_ops


def _inputs(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randint(-3, 4, s, generator=g).to(dtype) for s in ((9, 6), (2, 5, 6), (2, 5), (9, 5)))
    return x, w, b, dy, torch.tensor([1, 4, 8], dtype=torch.int32)


def _refused(call):
    with pytest.raises((RuntimeError, NotImplementedError)):
        call()


@pytest.mark.parametrize('which', (0, 1, 2))
@pytest.mark.parametrize('grad', (False, True))
def test_forward_mode_derivatives_are_refused(ops, which, grad):
    """a tangent on any input, with and without backward-mode gradients being recorded: never a result without one"""
    x, w, b, _, off = _inputs()
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        t = [x, w, b]
        plain = ops.expert_linear(t[0], t[1], off, t[2])  # (no tangent: a level alone refuses nothing)
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        _refused(lambda: ops.expert_linear(t[0], t[1], off, t[2]))
        assert torch.equal(plain, ops.expert_linear(x, w, off, b))
    _refused(lambda: torch.func.jvp(lambda v: ops.expert_linear(v, w, off, b), (x,), (torch.ones_like(x),)))


@pytest.mark.parametrize('grad', (False, True))
def test_forward_mode_derivatives_of_the_4_bit_calls_are_refused(monkeypatch, grad):
    from sm3det_amd import mx4
    monkeypatch.setattr(mx4, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(mx4, 'launch', lambda *a, **k: None)
    monkeypatch.setattr(mx4, '_call', lambda *a, **k: None)
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    w, we = mx4.Mx4Tensor(u(5, 64), u(5, 4), 6), mx4.Mx4Tensor(u(2, 5, 64), u(2, 5, 4), 6)
    xq = mx4.Mx4Tensor(u(9, 64), u(9, 4), 6)
    x, b, be, off = torch.ones(9, 6), torch.ones(5), torch.ones(2, 5), torch.tensor([0, 4, 9], dtype=torch.int32)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        d = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda f: mx4.quantize(f(x)), lambda f: mx4.linear(f(x), w, b), lambda f: mx4.linear(xq, w, f(b)),
                     lambda f: mx4.linear(x, w, f(b)), lambda f: mx4.expert_linear(f(x), we, off, be),
                     lambda f: mx4.expert_linear(x, we, off, f(be))):
            call(lambda t: t)
            _refused(lambda: call(d))


SECOND = [  # what needs a gradient of (x, w, b, dy); strided inputs are copied on their way in
    (which, strided) for which in ((0, 1), (1, 2), (0, 1, 2), (0,), (1,), (0, 1, 2, 3)) for strided in (False, True)]


@pytest.mark.parametrize('which,strided', SECOND, ids=str)
def test_a_second_derivative_is_refused_not_dropped(ops, which, strided):
    """loss = y . dy + |first gradient|^2: whatever input of the second term the caller differentiates with respect to, the
    call raises -- also where the gradient that came in carries no graph itself, and where the other input alone does"""
    x, w, b, dy, off = _inputs(torch.float16)
    if strided:  # unit stride along neither dimension
        x = torch.stack([x, x], -1)[..., 0]
        w = torch.stack([w, w], -1)[..., 0]
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(i in which) if not strided else t.requires_grad_(i in which)
              for i, t in enumerate((x, w, b, dy))]
    x, w, b, dy = leaves
    asked = [t for t in leaves[:3] if t.requires_grad]
    y = ops.expert_linear(x, w, off, b)
    firsts = torch.autograd.grad(y, asked, dy, create_graph=True)
    # dx depends on (dy, w), dw on (dy, x), db on dy
    depends = {id(x): [w, dy], id(w): [x, dy], id(b): [dy]}
    for leaf, first in zip(asked, firsts):
        for other in depends[id(leaf)]:
            if other.requires_grad:
                mixed = (y * dy.detach()).double().sum() + first.double().square().sum()
                _refused(lambda: torch.autograd.grad(mixed, other, retain_graph=True, allow_unused=True))


def test_first_derivatives_are_the_formulas_with_and_without_a_graph(ops):
    x, w, b, dy, off = _inputs(torch.float16)
    for graph in (False, True):
        for leaves in ([t.clone().requires_grad_() for t in (x, w, b)],
                       [torch.stack([t, t], -1)[..., 0].requires_grad_() for t in (x, w, b)]):
            y = ops.expert_linear(leaves[0], leaves[1], off, leaves[2])
            dx, dw, db = torch.autograd.grad(y, leaves, dy, create_graph=graph)
            for g, (p, q) in enumerate(((1, 4), (4, 8))):
                assert torch.equal(y[p:q].double(), x[p:q].double() @ w[g].double().t() + b[g].double())
                assert torch.equal(dx[p:q].double(), dy[p:q].double() @ w[g].double())
                assert torch.equal(dw[g].double(), dy[p:q].double().t() @ x[p:q].double())
                assert torch.equal(db[g].double(), dy[p:q].double().sum(0))
            assert not y[:1].any() and not y[8:].any() and not dx[:1].any() and not dx[8:].any()
            for leaf, got in zip(leaves, (dx, dw, db)):
                assert got.shape == leaf.shape and got.dtype == leaf.dtype
