"""Large square matrices: sums of squares over many thousands of terms stay as exact as the plain recurrence's in fp32."""
import pytest
import torch

from mx_rcnn_amd import ops
from mx_rcnn_amd.ops.muon import newton_schulz_ref


@pytest.mark.gpu
@pytest.mark.parametrize('r,c', [(12288, 12288), (9001, 9100)])
def test_error_of_large_matrices(cuda, r, c):
    """At most 1.5 times the plain recurrence's error: the operands' 22 bits and sums in runs of 256 terms, each rounded
    some 100 times, leave less than a blocked fp32 product; one running sum of 12288 terms, rounded 4600 times, leaves
    about sqrt(4600 / 150) = 5.5 times the error on the diagonals of X X^T and A A, and 1.9 times in the result."""
    gen = torch.Generator(device='cuda').manual_seed(2)
    u, v = (torch.randn(1, *s, generator=gen, device=cuda) for s in ((r, 8), (8, c)))
    v *= torch.logspace(0, -1.5, 8, device=cuda)[None, :, None]
    g = (torch.randn(1, r, c, generator=gen, device=cuda) * 0.5 + torch.bmm(u, v)) * 1e-3
    out = ops.orthogonalize(g)
    x = g.double()
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        a = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = 3.4445 * x + torch.bmm(-4.7750 * a + 2.0315 * torch.bmm(a, a), x)
    del a
    plain = float((newton_schulz_ref(g).double() - x).norm())
    assert float((out.double() - x).norm()) <= 1.5 * plain
