"""The 8-bit detector keeps the weights it was built from: a model that trains on does not reach it."""
import pytest
import torch

from mx_rcnn_amd.core.detector import Detector
from tests.test_fc_int8 import _model


@pytest.mark.parametrize('dev,dtype', [('cpu', 'fp32'), pytest.param('cuda', 'bf16', marks=pytest.mark.gpu)])
def test_source_model_may_change(request, dev, dtype):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    m = _model()
    det = Detector(m, dev, compute_dtype=dtype, fc_int8=True)
    gen = torch.Generator().manual_seed(0)
    pooled = torch.randn(7, 512, 7, 7, generator=gen).clamp(min=0).to(dev, det.dtype)
    pooled = pooled.contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        want = [t.clone() for t in det.model.head(pooled)]
        for p in m.parameters():
            p.add_(1.0)
        got = det.model.head(pooled)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = {t.untyped_storage().data_ptr() for t in m.state_dict().values()}
    for k in ('fc6', 'fc7'):
        assert not held & {t.untyped_storage().data_ptr() for t in getattr(det.model.head, k).int8}
