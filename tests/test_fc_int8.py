"""VGG16's fc6 / fc7 in 8 bits at test time (core/detector.py fc_int8): the detector must run exactly the
8-bit layers of ops/int8.py on the weights of the model it was built from."""
import pytest
import torch

from mx_rcnn_amd.core.detector import Detector
from mx_rcnn_amd.models import FasterRCNN
from mx_rcnn_amd.ops import int8_linear, quantize_rows
from tests.test_model import _cfg

ROIS = torch.tensor([[0., 10, 20, 180, 150], [0., 30, 30, 90, 120], [0., 60, 5, 200, 140], [0., 0, 0, 100, 60],
                     [0., 5, 5, 60, 50]])


def _model(net='vgg16'):
    torch.manual_seed(0)
    return FasterRCNN(net, 21, cfg=_cfg(), train_mode='test')


def _data(seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(1, 3, 160, 224, generator=gen) * 50, torch.tensor([[160., 224., 1.]])


@pytest.mark.parametrize('dev,dtype', [('cpu', 'fp32'), pytest.param('cuda', 'bf16', marks=pytest.mark.gpu),
                                       pytest.param('cuda', 'fp16', marks=pytest.mark.gpu)])
def test_head_runs_the_8bit_layers(request, dev, dtype):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    m = _model()
    before = {k: v.clone() for k, v in m.state_dict().items()}
    det = Detector(m, dev, compute_dtype=dtype, fc_int8=True)
    plain = Detector(m, dev, compute_dtype=dtype)
    assert m.head.fc6.int8 is None and det.model is not m
    assert all(torch.equal(v.cpu(), before[k]) for k, v in m.state_dict().items())
    # the head by hand: rows of the pooled map in (h, w, c) order
    pooled = (torch.randn(37, 512, 7, 7, generator=torch.Generator().manual_seed(3)).clamp(min=0) * 2)
    pooled = pooled.to(dev, det.dtype).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        cls, box = det.model.head(pooled)
        rows = pooled.permute(0, 2, 3, 1).reshape(37, -1)
        w6 = m.head.fc6.weight.detach().float().permute(0, 2, 3, 1).reshape(4096, -1).contiguous().to(dev)
        w7 = m.head.fc7.weight.detach().float().to(dev)
        h = int8_linear(rows, *quantize_rows(w6), m.head.fc6.bias.detach().float().to(dev), relu=True)
        h = int8_linear(h, *quantize_rows(w7), m.head.fc7.bias.detach().float().to(dev), relu=True)
        from mx_rcnn_amd.ops.head import fc_pair
        wc, wb = fc_pair(h, det.model.head.cls_score, det.model.head.bbox_pred)
    assert torch.equal(cls, wc) and torch.equal(box, wb)
    assert not torch.equal(cls, plain.model.head(pooled)[0])
    # and through the whole graph
    data, info = _data()
    r, p, b = det.forward(data, info, ROIS)
    assert p.shape == (5, 21) and b.shape == (5, 84) and bool(torch.isfinite(p).all())


def test_refusals_cpu():
    with pytest.raises(ValueError):
        Detector(_model('resnet18'), torch.device('cpu'), fc_int8=True)
    det = Detector(_model(), torch.device('cpu'), fc_int8=True)
    det.model.train()
    with pytest.raises(RuntimeError):
        det.model.head(torch.randn(2, 512, 7, 7))


@pytest.mark.gpu
def test_fp32_graph_is_refused(cuda):
    with pytest.raises(ValueError):
        Detector(_model(), cuda, compute_dtype='fp32', fc_int8=True)


@pytest.mark.gpu
def test_graph_replay_equals_eager(cuda):
    det = Detector(_model(), cuda, compute_dtype='bf16', fc_int8=True)
    xs = [det._prep(_data(k)[0]) for k in range(3)]
    info, rois = _data()[1].to(cuda), ROIS.to(cuda)
    want = [[t.clone() for t in det.detect(x, info, rois)] for x in xs]
    static = xs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        det.detect(static, info, rois)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = det.detect(static, info, rois)
    for k in (0, 1, 2, 0):
        static.copy_(xs[k])
        graph.replay()
        for a, b in zip(out, want[k]):
            assert torch.equal(a, b)
