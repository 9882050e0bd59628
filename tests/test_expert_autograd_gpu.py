"""What autograd may ask of the grouped products, on the device: a derivative that is not implemented raises, and is never left out."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _inputs():
    g = torch.Generator().manual_seed(5)
    x, w, b, dy = (torch.randn(*s, generator=g).to(torch.bfloat16).cuda() for s in ((20, 8), (2, 16, 8), (2, 16), (20, 16)))
    return x, w, b, dy, torch.tensor([0, 5, 20], dtype=torch.int32, device='cuda')


def test_a_second_derivative_in_a_mixed_loss():
    from sm3det_amd import expert_ops
    x, w, b, dy, off = _inputs()
    x, w = x.requires_grad_(), w.requires_grad_()
    y = expert_ops.expert_linear(x, w, off, b)
    plain = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    first = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    assert all(torch.equal(p, f) for p, f in zip(plain, first))
    for f, other in ((first[0], w), (first[1], x)):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.float().sum() + f.float().square().sum(), other, retain_graph=True)
    (y.float().sum()).backward()
    assert x.grad is not None and w.grad is not None


def test_forward_mode_derivatives():
    from sm3det_amd import expert_ops, mx4
    x, w, b, dy, off = _inputs()
    wq = mx4.quantize(w)
    with fwAD.dual_level(), torch.no_grad():
        plain = expert_ops.expert_linear(x, w, off, b)
        d = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda: expert_ops.expert_linear(d, w, off, b), lambda: mx4.expert_linear(d, wq, off), lambda: mx4.quantize(d),
                     lambda: mx4.expert_ffn(d, wq, b, wq, b, off)):
            with pytest.raises(RuntimeError):
                call()
    assert torch.equal(plain, expert_ops.expert_linear(x, w, off, b))
