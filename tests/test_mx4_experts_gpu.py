"""mx4.quantize_experts on the device: in mixed precision, in a detector, in graphs, and after the weights changed."""
import copy

import numpy as np
import pytest
import torch

from tests.moe_common import load_fixture
from tests.test_mx4_gpu import _check_ffn

pytestmark = pytest.mark.gpu


@pytest.fixture
def net():
    from sm3det_amd.convnext_moe import ConvNeXt_moe_MultiInput
    fx = load_fixture('moe_e4k2')
    m = ConvNeXt_moe_MultiInput(**fx['cfg'])
    m.load_state_dict(fx['state_dict'])
    m = m.cuda().eval()
    m.x = fx['x'].cuda()
    return m


def _layers(m):
    from sm3det_amd.convnext_moe import MoE_layer
    return [c for c in m.modules() if isinstance(c, MoE_layer)]


@torch.no_grad()
def _out(m):
    return m(m.x, ['single'])[0]


def _full(m):
    """the outputs of a copy with its full-precision experts"""
    from sm3det_amd import mx4
    c = copy.deepcopy(m)
    mx4.restore_experts(c)
    return _out(c)


def _four(m):
    """the outputs of a copy whose experts have just been packed"""
    from sm3det_amd import mx4
    c = copy.deepcopy(m)
    mx4.quantize_experts(c)
    return _out(c)


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def _caught(monkeypatch):
    from sm3det_amd import mx4
    seen, ffn = [], mx4.expert_ffn

    def spy(*args):
        seen.append((*args, ffn(*args)))
        return seen[-1][-1]
    monkeypatch.setattr(mx4, 'expert_ffn', spy)
    return seen


def _check_caught(seen, layers):
    assert len(seen) == len(layers) > 0
    for (xs, w1, b1, w2, b2, offsets, y), m in zip(seen, layers):
        assert w1.shape == m.w1.shape and w2.shape == m.w2.shape and torch.equal(b1, m.b1) and torch.equal(b2, m.b2)
        _check_ffn(y, xs, w1, b1, w2, b2, offsets.tolist())


def test_a_mixed_precision_backbone(net, monkeypatch):
    from sm3det_amd import amp, mx4
    amp.wrap_fp16_model(net)
    full = _out(net)
    mx4.quantize_experts(net)
    seen = _caught(monkeypatch)
    outs = _out(net)
    assert {s[0].dtype for s in seen} == {torch.float16}
    _check_caught(seen, _layers(net))
    assert all(torch.isfinite(o).all() and o.shape == f.shape for o, f in zip(outs, full)) and not _same(outs, full)
    mx4.restore_experts(net)
    assert _same(_out(net), full)


@pytest.mark.parametrize('half', (False, True))
def test_a_detector(monkeypatch, half):
    from sm3det_amd import amp, detector, mx4  # noqa: F401
    from sm3det_amd.registry import MODELS
    from tests.test_detector_gpu import _model_cfg
    torch.manual_seed(1)
    det = MODELS.build(_model_cfg()).cuda().eval()
    with torch.no_grad():
        for n, p in det.backbone.named_parameters():
            if n.endswith('gamma'):
                p.fill_(1.0)
    if half:
        amp.wrap_fp16_model(det)
    x = torch.randn(1, 3, 256, 256, device='cuda')
    meta = [dict(img_shape=(256, 256, 3), scale_factor=np.ones(4, np.float32))]
    full = det.simple_test(x, meta, [['sar']])
    layers = _layers(det)
    assert mx4.quantize_experts(det) == len(layers)
    seen = _caught(monkeypatch)
    res = det.simple_test(x, meta, [['sar']])
    _check_caught(seen, layers)
    assert len(res) == len(full) and len(res[0]) == det.sar_bbox_head.num_classes
    assert all(isinstance(a, np.ndarray) and a.ndim == 2 and a.shape[1] == 5 and np.isfinite(a).all() for a in res[0])


def test_weights_changed_in_place(net):
    from sm3det_amd import mx4
    mx4.quantize_experts(net)
    first = _out(net)
    assert _same(first, _four(net)) and not _same(first, _full(net))
    with torch.no_grad():
        for m in _layers(net):
            m.w1.mul_(0.5), m.b2.add_(1.0)
    assert _same(_out(net), _full(net)) and not _same(_out(net), first)
    mx4.quantize_experts(net)
    assert _same(_out(net), _four(net)) and not _same(_out(net), _full(net))


def _optimizer(net):
    from sm3det_amd.optim import MultiTensorAdamW
    ps = [p for m in _layers(net) for p in (m.w1, m.b1, m.w2, m.b2)]
    for p in ps:
        p.grad = torch.randn_like(p)
    return MultiTensorAdamW(ps, lr=1e-2)


def test_optimizer_steps_in_evaluation_mode(net):
    from sm3det_amd import mx4
    opt = _optimizer(net)
    mx4.quantize_experts(net)
    assert _same(_out(net), _four(net))
    for _ in range(2):
        opt.step()
        assert _same(_out(net), _full(net))
        mx4.quantize_experts(net)
        assert _same(_out(net), _four(net)) and not _same(_out(net), _full(net))


def test_optimizer_steps_replayed_from_a_graph(net):
    from sm3det_amd import mx4
    opt = _optimizer(net)
    opt.step()
    opt.refresh_grad_pointers()
    mx4.quantize_experts(net)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    assert _same(_out(net), _full(net))  # a step was captured after the experts were packed
    mx4.quantize_experts(net)
    last = _out(net)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        now = _out(net)
        assert _same(now, _four(net)) and not _same(now, last)
        last = now


def test_a_captured_forward_keeps_the_snapshot_it_was_captured_with(net):
    from sm3det_amd import mx4
    mx4.quantize_experts(net)
    want = [o.clone() for o in _out(net)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _out(net)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _out(net)
    for forget in (lambda: None, lambda: net.train().eval(), lambda: mx4.restore_experts(net), lambda: mx4.quantize_experts(net)):
        forget()
        junk = [torch.full((1 << 16,), 0x5a5a5a5a, dtype=torch.int32, device='cuda') for _ in range(64)]  # what was freed is written over
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        del junk
        assert _same(out, want)


def test_a_forward_on_another_stream_outlives_what_it_reads(net):
    """the packed experts are dropped and their memory is used again while a side stream has yet to run the forward"""
    from sm3det_amd import mx4
    mx4.quantize_experts(net)
    want = [o.clone() for o in _out(net)]
    sizes = [t.numel() for m in _layers(net) for t in (m._mx4.w1.codes, m._mx4.w1.scales, m._mx4.w2.codes, m._mx4.w2.scales)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _out(net)  # (allocations of the side stream, first launches)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(1_000_000_000)
        out = _out(net)
    net.train().eval()
    junk = [torch.full((n,), 0x11, dtype=torch.uint8, device='cuda') for n in sizes * 3]
    torch.cuda.current_stream().synchronize()
    assert not s.query()  # (the side stream still sleeps: what was written above, it finds)
    s.synchronize()
    del junk
    same = _same(out, want)
    assert same
