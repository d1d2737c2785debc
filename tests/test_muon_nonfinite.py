"""The Muon update where gradients are not finite: a NaN reaches its own matrix's weights whatever the clip, an infinity
is clipped like any large value; other matrices and what lies between them keep their values."""
import pytest
import torch

from mx_rcnn_amd import ops

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
# in one block each; by launches, straight and turned
SETS = {'blocks': [(16, 40), (30, 20), (64, 64)], 'launches': [(70, 90), (30, 20), (200, 66)]}


def _state(shapes, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    mats, at = [], 1
    for r, c in shapes:
        mats.append((at, r, c))
        at += r * c + 2
    w, mom, grad = (torch.randn(at, generator=gen) * k for k in (0.02, 5e-3, 1e-3))
    return [t.to(dev) for t in (w, mom, grad)], tuple(mats)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('which', sorted(SETS))
@pytest.mark.parametrize('clip', [-1.0, 1e-3, 1.0])
@pytest.mark.parametrize('nesterov', [True, False])
def test_nan_reaches_its_matrix(request, dev, which, clip, nesterov):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    lr = torch.full((1,), 0.02, device=dev)
    (w, mom, grad), mats = _state(SETS[which], dev)
    clean = [t.clone() for t in (w, mom)]
    ops.muon_update_(clean[0], clean[1], grad.clone(), mats, lr, clip=clip, nesterov=nesterov)
    o, r, c = mats[1]
    grad[o + 7] = float('nan')
    ops.muon_update_(w, mom, grad, mats, lr, clip=clip, nesterov=nesterov)
    hit = torch.zeros(w.numel(), dtype=torch.bool, device=dev)
    hit[o:o + r * c] = True
    assert bool(torch.isnan(w[hit]).all())
    assert torch.isnan(mom).nonzero().flatten().tolist() == [o + 7]
    assert torch.equal(w[~hit], clean[0][~hit]) and torch.equal(mom[~hit], clean[1][~hit])


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('which', sorted(SETS))
def test_infinity_is_clipped(request, dev, which):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    lr = torch.full((1,), 0.02, device=dev)
    (w, mom, grad), mats = _state(SETS[which], dev)
    at = mats[0][0] + 5
    grad[at], grad[at + 1] = float('inf'), -float('inf')
    same = [w.clone(), mom.clone(), grad.clone()]
    same[2][at], same[2][at + 1] = 2e-3, -2e-3
    ops.muon_update_(w, mom, grad, mats, lr, clip=2e-3)
    ops.muon_update_(same[0], same[1], same[2], mats, lr, clip=2e-3)
    assert bool(torch.isfinite(w).all()) and torch.equal(w, same[0]) and torch.equal(mom, same[1])
