"""CPU tier of mx4.quantize_experts: when a layer may use the experts it packed, and when their weights are no longer its own.  The
quantisation is replaced by a copy, so that a forward's operands show which values they were made from."""
import copy
import io

import pytest
import torch
from torch import nn


@pytest.fixture
def net(monkeypatch):
    from sm3det_amd import mx4
    from sm3det_amd.convnext_moe import MoE_layer
    monkeypatch.setattr(mx4, 'quantize', lambda w: w.clone())
    monkeypatch.setattr(mx4, 'expert_ffn', lambda xslot, w1, b1, w2, b2, offsets: (w1, b1, w2, b2))
    torch.manual_seed(1)
    cfg = dict(noisy_gating=False, num_experts=2, in_channels=4, mid_channels=16, top_k=1, gating='cosine')
    m = nn.ModuleList([MoE_layer(cfg), MoE_layer(cfg)]).eval()
    assert mx4.quantize_experts(m) == 2
    return m


NAMES = ('w1', 'b1', 'w2', 'b2')


def _used(layer):
    """the values the 4-bit experts of the next forward come from, or None: the full-precision experts run"""
    f = layer.experts()
    return None if f is None else f(None, None)


def _packed(layer):
    got = _used(layer)
    return got is not None and all(torch.equal(g, getattr(layer, n)) for g, n in zip(got, NAMES))


@torch.no_grad()
def _copy(p):
    p.copy_(torch.randn_like(p))


@torch.no_grad()
def _lerp(p):  # averaged weights
    p.lerp_(torch.randn_like(p), 0.1)


def _inference(p):
    with torch.inference_mode():
        p.mul_(2)


def _storage(p):
    p.data = torch.randn_like(p)


def _by_address(p):
    """what MultiTensorAdamW does: writes without moving the version, and counts its step"""
    from sm3det_amd.optim import MultiTensorAdamW
    opt = MultiTensorAdamW([p])
    p._sm3_writers = (opt._writer,)
    p.data.add_(1.0)
    opt._writer.steps += 1


@pytest.mark.parametrize('name', NAMES)
@pytest.mark.parametrize('write', (_copy, _lerp, _inference, _storage, _by_address), ids=lambda f: f.__name__)
def test_a_changed_parameter_ends_the_use_of_the_packed_experts(net, name, write):
    a, b = net
    assert _packed(a) and _packed(b)
    write(getattr(a, name))
    assert _used(a) is None and _packed(b)
    from sm3det_amd import mx4
    mx4.quantize_experts(net)
    assert _packed(a) and _packed(b)


def test_another_parameter_in_its_place_is_not_the_packed_one(net):
    a, b = net
    old, a.w1 = a.w1, nn.Parameter(torch.randn_like(a.w1))
    assert _used(a) is None and _packed(b)
    a.w1 = old
    assert _packed(a)
    assert torch.func.functional_call(_Call(b), {'layer.w2': torch.zeros_like(b.w2)}, ()) is None
    assert _packed(b)


class _Call(nn.Module):
    def __init__(self, layer):
        super().__init__()
        self.layer = layer

    def forward(self):
        return self.layer.experts()


def test_optimizer_steps_are_seen_before_and_after_packing(net):
    from sm3det_amd import mx4
    from sm3det_amd.optim import _Writer
    a, _ = net
    w = a.w1._sm3_writers = (_Writer(),)
    assert _used(a) is None  # an optimizer took the parameter over after it was packed
    mx4.quantize_experts(net)
    assert _packed(a)
    w[0].steps += 1
    a.w1.data.add_(1.0)
    assert _used(a) is None
    # a step inside a captured graph: replays change the weights, the host sees nothing of it
    mx4.quantize_experts(net)
    w[0].captured, w[0].steps = True, w[0].steps + 1
    assert _used(a) is None
    mx4.quantize_experts(net)
    for _ in range(3):
        a.w1.data.add_(1.0)
        assert _packed(a)


def test_parameters_without_a_version_are_packed_anew(net):
    from sm3det_amd import mx4
    from sm3det_amd.convnext_moe import MoE_layer
    with torch.inference_mode():
        m = MoE_layer(dict(noisy_gating=False, num_experts=2, in_channels=4, mid_channels=16, top_k=1, gating='linear')).eval()
        mx4.quantize_experts(m)
        for _ in range(2):
            m.w2.add_(1.0)
            assert _packed(m)


def test_training_loading_and_moving_end_it_too(net):
    from sm3det_amd import mx4
    a = net[0]
    for change in (lambda: net.train().eval(), lambda: net.load_state_dict(net.state_dict()), lambda: net.to(torch.float32),
                   lambda: mx4.restore_experts(net)):
        assert _packed(a)
        change()
        assert _used(a) is None
        mx4.quantize_experts(net)


@pytest.mark.parametrize('through', ('deepcopy', 'copy', 'pickle'))
def test_copies_take_the_packed_experts_along_while_they_are_current(net, through):
    def again(m):
        if through == 'pickle':
            f = io.BytesIO()
            torch.save(m, f)
            return torch.load(io.BytesIO(f.getvalue()), weights_only=False)
        return getattr(copy, through)(m)
    a = net[0]
    c = again(a)
    assert _packed(c) and _packed(a)
    _copy(c.w1)
    assert _used(c) is None and _packed(a) == (through != 'copy')  # (copy.copy shares the parameters)
    _copy(a.b2)
    assert _used(a) is None and _used(again(a)) is None
    from sm3det_amd import mx4
    mx4.quantize_experts(net)
    assert _packed(again(a))
    again(again(net))


def test_a_broadcast_moves_the_version_of_what_it_writes(monkeypatch):
    import torch.distributed as dist

    from sm3det_amd.data_parallel import BucketedGradReducer
    monkeypatch.setattr(dist, 'broadcast', lambda t, src, group: t.add_(1))
    red = BucketedGradReducer.__new__(BucketedGradReducer)
    p = nn.Parameter(torch.zeros(3))
    red.world, red.params, red.group = 2, [p], None
    before = p._version
    red.broadcast_parameters(0)
    assert p._version > before and p.detach().tolist() == [1.0] * 3


def test_layers_are_packed_together_or_not_at_all(net, monkeypatch):
    from sm3det_amd import mx4
    from sm3det_amd._lib import SM3Error
    mx4.restore_experts(net)
    last = net[1].w2

    def quantize(w):
        if w.data_ptr() == last.data_ptr():
            raise SM3Error('no')
        return w.clone()
    monkeypatch.setattr(mx4, 'quantize', quantize)
    with pytest.raises(SM3Error):
        mx4.quantize_experts(net)
    assert _used(net[0]) is None and _used(net[1]) is None
