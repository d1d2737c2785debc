"""The gradient buffer that a Muon update clears, in every type that a gradient may have."""
import pytest
import torch

from mx_rcnn_amd import ops

MATS = ((3, 70, 90), (6400, 30, 20), (7001, 66, 130))  # by launches; BLOCK: in one block each
BLOCK = ((3, 16, 40), (700, 30, 20))


@pytest.mark.parametrize('dev', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('mats', [MATS, BLOCK])
@pytest.mark.parametrize('gdtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('zdtype', [torch.float32, torch.bfloat16, torch.float16, None])
def test_cleared_buffer(request, dev, mats, gdtype, zdtype):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    n = mats[-1][0] + mats[-1][1] * mats[-1][2] + 5
    gen = torch.Generator().manual_seed(2)
    w, mom, grad = ((torch.randn(n, generator=gen) * k).to(dev) for k in (0.02, 5e-3, 1e-3))
    grad = grad.to(gdtype)
    lr = torch.full((1,), 0.02, device=dev)
    want = [w.clone(), mom.clone()]
    ops.muon_update_(want[0], want[1], grad.clone(), mats, lr)
    before = grad.clone()
    zero = grad if zdtype is None else torch.ones(n, dtype=zdtype, device=dev)  # None: the gradient itself
    kept = zero.clone()
    ops.muon_update_(w, mom, grad, mats, lr, zero=zero)
    assert torch.equal(w, want[0]) and torch.equal(mom, want[1])
    inside = torch.zeros(n, dtype=torch.bool, device=dev)
    for o, r, c in mats:
        inside[o:o + r * c] = True
    assert bool((zero[inside] == 0).all()) and torch.equal(zero[~inside], kept[~inside])
    assert zdtype is None or torch.equal(grad, before)


@pytest.mark.gpu
def test_refused_buffers(cuda):
    w, mom, grad = (torch.randn(200, device=cuda) for _ in range(3))
    lr = torch.ones(1, device=cuda)
    for zero in (grad.double(), grad.int(), grad[:100], grad.cpu(), grad.expand(2, 200)[0:1].t()[::2]):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            ops.muon_update_(w, mom, grad, ((0, 10, 10),), lr, zero=zero)
