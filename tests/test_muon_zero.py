"""Matrices of zeros stay zero for every positive eps, down to the smallest double."""
import pytest
import torch

from mx_rcnn_amd import ops


@pytest.mark.parametrize('dev', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('eps', [1e-7, 1e-300, 1e-306, 1e-310, 5e-324])
@pytest.mark.parametrize('r,c', [(8, 8), (64, 40), (70, 90), (200, 66)])
def test_zeros(request, dev, eps, r, c):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    g = torch.zeros(3, r, c, device=dev)
    g[1, 0, 0], g[1, 1, 1] = 1e-45, -1e-45  # the smallest fp32 values: a direction all the same
    out = ops.orthogonalize(g, eps=eps)
    assert bool((out[[0, 2]] == 0).all()) and bool(torch.isfinite(out).all())
    if eps < 1e-100:
        x = 2.0 ** -0.5  # both singular values of X0
        for _ in range(5):
            x = 3.4445 * x - 4.7750 * x ** 3 + 2.0315 * x ** 5
        assert abs(float(out[1, 0, 0]) - x) < 1e-5 and abs(float(out[1, 1, 1]) + x) < 1e-5
    w = torch.ones(2 * r * c, device=dev)
    mom, grad = torch.zeros_like(w), torch.zeros_like(w)
    ops.muon_update_(w, mom, grad, ((0, r, c), (r * c, c, r)), torch.ones(1, device=dev), eps=eps)
    assert bool((w == 1).all()) and bool((mom == 0).all())
