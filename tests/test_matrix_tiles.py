"""The kernels that real layers run on -- large tiles, runs of K on them, rows held by one wave or by a block -- at
sizes that are no multiple of a tile, against 64-bit computations on the device.  The comments name the kernels that the
sizes lead to.

8-bit sums are exact: with scales of 1 and an fp32 result the sum rounded once; else at most four fp32 roundings
(2^-24 of the terms each) and one of the result.  Tolerance of an orthogonalisation, of the result's norm: twice the error
that the plain recurrence has in fp32 on the same input, plus 16 * 2^-23 for the 22-bit operands, plus eps / 2 of the
output type; a weight moves by lr * scale times that and three fp32 roundings.
"""
import math

import pytest
import torch

from mx_rcnn_amd import ops
from mx_rcnn_amd.ops.muon import newton_schulz_ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24


# ---- rows to 8 bits ------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K', [
    (2048, 513), (2051, 1000), (2049, 2048),      # a wave per row, up to 32 values a lane
    (7, 513), (2047, 1001), (3, 4095),            # 256 threads
    (2, 4097), (5, 5003), (3, 8192),              # 512 threads, 16 values each
    (2, 8193), (3, 20001), (2, 32768)])           # 512 threads, 64 values each
def test_quantize_rows(cuda, dtype, M, K):
    gen = torch.Generator(device='cuda').manual_seed(M + K)
    x = (torch.randn(M, K, generator=gen, device=cuda) * (torch.rand(M, 1, generator=gen, device=cuda) * 100)).to(dtype)
    x[M // 2, K - 1] = 2 * x[M // 2].abs().amax()  # a row whose last value decides
    q, s = ops.quantize_rows(x)
    peak = x.float().abs().amax(1).double()
    want_s = torch.maximum((peak * torch.tensor(1.0 / 127).double()).float(), torch.tensor(2.0 ** -126))
    assert torch.equal(s, want_s)
    assert torch.equal(q, torch.round((x.double() / s.double()[:, None]).float()).to(torch.int8))


# ---- 8-bit products ------------------------------------------------------------------------------
INT8 = [
    (524, 3854, 128), (301, 4093, 25088), (77, 3458, 10944),  # 128 x 160 tiles: whole, in 4 and 8 runs
    (733, 2859, 148), (2214, 65, 16924),                      # .. of rows copied first, whole and in 12 runs
    (1710, 3184, 160), (2399, 4093, 1600), (253, 2731, 23552),  # 256 x 160 tiles: whole, whole, in 8 runs
    (3195, 1685, 132), (170, 3703, 22847),                    # .. of rows copied first, whole and in 8 runs
    (300, 4095, 4096), (38, 57, 17200), (45, 4379, 166)]      # 64 x 64 tiles: whole, in 12 runs, copied


@pytest.mark.parametrize('M,N,K', INT8)
def test_int8_sums(cuda, M, N, K):
    gen = torch.Generator(device='cuda').manual_seed(K)
    x, w = (torch.randint(-128, 128, (r, K), generator=gen, device=cuda, dtype=torch.int8) for r in (M, N))
    one = torch.ones(max(M, N), device=cuda)
    got = ops.int8_matmul(x, one[:M], w, one[:N], out_dtype=torch.float32)
    want = x.double() @ w.double().t().contiguous()
    assert torch.equal(got, want.float())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,N,K', [(301, 4093, 25088), (2399, 4093, 1600), (300, 4095, 4096), (170, 3703, 22847)])
def test_int8_results(cuda, dtype, M, N, K):
    gen = torch.Generator(device='cuda').manual_seed(K)
    x, w = (torch.randint(-127, 128, (r, K), generator=gen, device=cuda, dtype=torch.int8) for r in (M, N))
    xs = torch.rand(M, generator=gen, device=cuda) * 0.05 + 1e-3
    ws = torch.rand(N, generator=gen, device=cuda) * 1e-3 + 1e-5
    b = torch.randn(N, generator=gen, device=cuda)
    p = (x.double() @ w.double().t().contiguous()) * xs.double()[:, None] * ws.double()
    want = (p + b.double()).clamp(min=0)
    got = ops.int8_matmul(x, xs, w, ws, b, relu=True, out_dtype=dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of fp16's subnormals
    tol = 4 * U32 * (p.abs() + b.double().abs()) + torch.finfo(dtype).eps / 2 * want * 1.001 + tiny
    assert got.dtype == dtype and bool(((got.double() - want).abs() <= tol).all())


# ---- orthogonalisation ---------------------------------------------------------------------------
def _ns64(g, steps=5, eps=1e-7):
    """(b, r, c) in 64 bits, step by step in the smaller dimension."""
    x = g.double()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        a = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = 3.4445 * x + torch.bmm(-4.7750 * a + 2.0315 * torch.bmm(a, a), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _norm(x):
    return x.double().flatten(1).norm(dim=1)


def _tol(g, want, dtype=torch.float32):
    e32 = _norm(newton_schulz_ref(g.float()).double() - want)
    return 2 * e32 + (16 * 2.0 ** -23 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0)) * _norm(want)


def _gradients(b, r, c, dev, seed=0):
    """A few strong directions over noise."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    u, v = (torch.randn(b, *s, generator=gen, device=dev) for s in ((r, 8), (8, c)))
    v *= torch.logspace(0, -1.5, 8, device=dev)[None, :, None]
    return (torch.randn(b, r, c, generator=gen, device=dev) * 0.5 + torch.bmm(u, v)) * 1e-3


NS = [  # tiles of X X^T / of the m x m products / of Q X
    (1, 72, 66), (1, 133, 133), (23, 256, 2304),           # 64 / 64 / 64 and 128
    (8, 459, 540), (8, 540, 459), (1, 585, 8281),          # 128 / 128 / 128, tall, 128 in 13 runs / 64
    (8, 262, 2841), (2, 7986, 517), (1, 936, 14886),       # Q X 192, tall; X X^T 192 in 15 runs
    (8, 1465, 1343), (8, 1343, 1465),                      # 192 / 192 / 192, tall and wide
    (8, 1707, 2026), (8, 2026, 1707),                      # 256 / 256 / 256, wide and tall
    (1, 19103, 1202), (2, 679, 10166)]                     # X X^T 256 in 15 runs; Q X 256


@pytest.mark.parametrize('b,r,c', NS)
def test_orthogonalize(cuda, b, r, c):
    g = _gradients(b, r, c, cuda, seed=r)
    out = ops.orthogonalize(g)
    want = _ns64(g)
    assert float((_norm(out.double() - want) - _tol(g, want)).max()) <= 0


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('b,r,c', [(23, 256, 2304), (8, 540, 459), (8, 1343, 1465), (8, 2026, 1707)])
def test_orthogonalize_low_precision(cuda, dtype, b, r, c):
    g = _gradients(b, r, c, cuda, seed=r).to(dtype)
    out = ops.orthogonalize(g)
    want = _ns64(g)
    assert out.dtype == dtype and float((_norm(out.double() - want) - _tol(g, want, dtype)).max()) <= 0


@pytest.mark.parametrize('b,r,c,dtype', [(23, 256, 2304, torch.bfloat16), (1, 64, 576, torch.float32),
                                         (8, 540, 459, torch.float32), (1, 936, 14886, torch.float32),
                                         (8, 1343, 1465, torch.float32), (2, 2026, 1707, torch.bfloat16)])
def test_orthogonalize_repeats_its_bits(cuda, b, r, c, dtype):
    """The same input gives the same bits, whatever earlier calls and other tensors left in the memory of its
    workspace."""
    g = _gradients(b, r, c, cuda, seed=1).to(dtype)
    want = ops.orthogonalize(g)
    for k, fill in enumerate((float('nan'), 1e30, 0.0, -7.0)):
        held = [torch.full((1 << n,), fill, device=cuda) for n in range(8, 28)]
        del held
        assert torch.equal(ops.orthogonalize(g), want)
        ops.orthogonalize(_gradients(b, r, c, cuda, seed=k + 2).to(dtype))
        assert torch.equal(ops.orthogonalize(g), want)


MUON = [  # (count, rows, cols) of one call
    [(8, 489, 503), (1, 65, 52)],                          # 128 / 128 / 128
    [(1, 512, 9216), (3, 512, 4608), (5, 256, 2304), (2, 2048, 512), (4, 1024, 256)],  # 128 in runs
    [(2, 907, 6842), (8, 179, 209)],                       # X X^T 192 in runs, Q X 256
    [(8, 1617, 1319), (3, 80, 153)],                       # 192 / 192 / 192
    [(1, 959, 8347), (1, 322, 3260), (2, 984, 9114)],      # X X^T 256 in runs, Q X 256
    [(1, 215, 757), (8, 2043, 1677), (1, 784, 9107)]]      # m x m products 256


@pytest.mark.parametrize('gdtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shapes', MUON)
def test_muon_update(cuda, shapes, gdtype):
    mats, parts, at = [], [], 0
    for k, (n, r, c) in enumerate(shapes):
        parts.append(_gradients(n, r, c, cuda, seed=k).reshape(-1))
        for _ in range(n):
            mats.append((at, r, c))
            at += r * c
    grad = torch.cat(parts).to(gdtype)
    gen = torch.Generator(device='cuda').manual_seed(9)
    mom = torch.randn(at, generator=gen, device=cuda) * 2e-3
    w = torch.randn(at, generator=gen, device=cuda) * 0.02
    lr = torch.full((1,), 0.02, device=cuda)
    mwant = 0.95 * mom.double() + grad.double()
    u = grad.double() + 0.95 * mwant
    w0 = w.clone()
    mtol = 3 * U32 * (mom.double().abs() + grad.double().abs())
    shadow = torch.empty(at, dtype=torch.bfloat16, device=cuda)
    ops.muon_update_(w, mom, grad, mats, lr, wd=5e-4, w_bf16=shadow)
    assert bool(((mom.double() - mwant).abs() <= mtol).all())
    assert torch.equal(shadow, w.bfloat16())
    lr = float(lr)
    for o, r, c in mats:
        s = slice(o, o + r * c)
        g = u[s].view(1, r, c)
        d = _ns64(g)
        k = math.sqrt(max(1.0, r / c))
        want = w0[s].double() - lr * (k * d.reshape(-1) + 5e-4 * w0[s].double())
        tol = lr * k * float(_tol(g, d)[0]) + 3 * U32 * float(want.norm() + w0[s].double().norm())
        assert float((w[s].double() - want).norm()) <= tol, (o, r, c)
