"""BN calibration of a random-init trunk gives the same statistics in every process: it takes no vendor convolution
on the GPU, whose choice goes by timing."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from mx_rcnn_amd.models import FasterRCNN
from tests.test_model import _cfg


class _GpuConvs(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if 'conv' in str(func) and any(torch.is_tensor(a) and a.is_cuda for a in args):
            self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def _model(net):
    torch.manual_seed(0)
    return FasterRCNN(net, 21, cfg=_cfg())


@pytest.mark.parametrize('dev', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('net', ['resnet18', 'resnet50'])
def test_calibrate_bn(request, dev, net):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    data = torch.randn(1, 3, 160, 224, generator=torch.Generator().manual_seed(1)) * 50
    want = _model(net)
    want.calibrate_bn(data)
    m = _model(net).to(dev)
    where = {n: t.data_ptr() for n, t in m.state_dict(keep_vars=True).items()}
    with _GpuConvs() as convs:
        n = m.calibrate_bn(data.to(dev))
    assert convs.seen == []
    assert n == sum(hasattr(k, 'moving_var') for k in m.trunk.modules()) and m.training
    assert not any(getattr(k, '_calibrate', False) for k in m.modules())
    state = m.state_dict(keep_vars=True)
    assert where == {n: t.data_ptr() for n, t in state.items()}  # in place: a parameter store's views stay
    for k, v in want.state_dict().items():
        assert torch.equal(state[k].detach().cpu(), v), k
    assert not torch.equal(state['trunk.stage3.0.bn2.moving_mean'].cpu(), torch.zeros(1).expand_as(
        want.state_dict()['trunk.stage3.0.bn2.moving_mean']))
    m.calibrate_bn(data.to(dev))
    assert all(torch.equal(v, state[k]) for k, v in m.state_dict().items())


@pytest.mark.gpu
def test_calibration_sees_a_vendor_convolution(cuda):
    """The watch above does name one."""
    with _GpuConvs() as convs, torch.no_grad():
        torch.nn.functional.conv2d(torch.zeros(1, 3, 8, 8, device=cuda), torch.zeros(4, 3, 3, 3, device=cuda))
    assert convs.seen
