"""quantize_rows of rows that are read twice (K > 32768), up to the longest that its 32-bit K admits, against the
definition: scale = max|row| * fp32(1 / 127) in fp32, values rounded to the nearest integer, ties to even."""
import pytest
import torch

from mx_rcnn_amd import ops


def _check(x, q, s):
    peak = x.float().abs().amax(1).double()
    want_s = (peak * torch.tensor(1.0 / 127).double().to(x.device)).float()
    assert torch.equal(s, want_s)
    # the quotient of two fp32 values, rounded from 64 bits, is the correctly rounded fp32 quotient
    want = torch.round((x.double() / s.double()[:, None]).float()).to(torch.int8)
    assert torch.equal(q, want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,K', [(3, 32769), (2, 33000), (5, 40961), (1, 100003)])
def test_rows_read_twice(cuda, dtype, M, K):
    gen = torch.Generator(device='cuda').manual_seed(K)
    x = (torch.randn(M, K, generator=gen, device=cuda) * (torch.rand(M, 1, generator=gen, device=cuda) * 10 + 0.1)).to(dtype)
    x[:, K - 1] = x.abs().amax() * 2  # the last value decides the scale
    q, s = ops.quantize_rows(x)
    _check(x, q, s)


@pytest.mark.gpu
def test_longest_row(cuda):
    """K = 2^31 - 1: the column numbers of the last step pass 32 bits."""
    K = (1 << 31) - 1
    gen = torch.Generator(device='cuda').manual_seed(0)
    part = torch.randn(1, 1 << 20, generator=gen, device=cuda).bfloat16()
    x = torch.empty(1, K, dtype=torch.bfloat16, device=cuda)
    for at in range(0, K, 1 << 20):
        n = min(1 << 20, K - at)
        x[:, at:at + n] = part[:, :n]
    x[0, K - 1] = 9.0
    q, s = ops.quantize_rows(x)
    want, want_s = ops.quantize_rows(torch.cat([part, x[:, K - 1:]], 1))
    assert torch.equal(s, want_s)
    for at in range(0, K - 1, 1 << 20):
        n = min(1 << 20, K - 1 - at)
        assert torch.equal(q[:, at:at + n], want[:, :n]), at
    assert int(q[0, K - 1]) == int(want[0, 1 << 20]) == 127
    _check(torch.cat([part, x[:, K - 1:]], 1), want, want_s)
