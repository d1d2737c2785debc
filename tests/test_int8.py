"""8-bit rows and products (ops/int8.py) against 64-bit computations of the same definition.

Tolerances: the integer sum is exact; int -> fp32, the two scales and the bias round at most four
times (2^-24 of the terms each), the result once more to its type (eps / 2 of the value).
"""
import pytest
import torch

from mx_rcnn_amd import ops
from mx_rcnn_amd.ops import int8 as int8_ops

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.fixture
def dev(request):
    if request.param == 'cuda':
        return request.getfixturevalue('cuda')
    return torch.device('cpu')


on_both = pytest.mark.parametrize('dev', DEVICES, indirect=True)


def _quantize64(x):
    """(q, scale) by definition: scale in fp32, the quotient of two fp32 values rounded to fp32 and then to an
    integer.  (The quotient of 24-bit values, rounded from 64 bits, is the correctly rounded fp32 quotient.)"""
    x = x.detach().cpu().float()
    peak = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0])
    inv = torch.tensor(1.0 / 127).double()  # 1 / 127 rounded to fp32
    s = torch.maximum((peak.double() * inv).float(), torch.tensor(2.0 ** -126))
    q = (x.double() / s.double()[:, None]).float()
    return torch.round(q).to(torch.int8), s


def _product64(xq, xs, wq, ws, bias, relu):
    acc = xq.cpu().double() @ wq.cpu().double().t().contiguous()
    p = acc * xs.cpu().double()[:, None] * ws.cpu().double()
    y = p if bias is None else p + bias.cpu().double()
    mag = p.abs() if bias is None else p.abs() + bias.cpu().double().abs()
    return (y.clamp(min=0) if relu else y), mag


def _check_product(y, args, bias, relu, dtype):
    want, mag = _product64(*args, bias, relu)
    assert y.dtype == dtype and tuple(y.shape) == tuple(want.shape)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of fp16's subnormals
    tol = 4 * 2.0 ** -24 * mag + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + tiny
    over = (y.cpu().double() - want).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


def _operands(M, N, K, dev, seed=0, lo=-127, hi=127):
    g = torch.Generator().manual_seed(seed)
    xq = torch.randint(lo, hi + 1, (M, K), generator=g, dtype=torch.int8)
    wq = torch.randint(lo, hi + 1, (N, K), generator=g, dtype=torch.int8)
    xs = torch.rand(M, generator=g) * 0.05 + 1e-3
    ws = torch.rand(N, generator=g) * 1e-3 + 1e-5
    return [t.to(dev) for t in (xq, xs, wq, ws)]


@on_both
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K', [(1, 1), (1, 4096), (3, 7), (5, 127), (2, 2048), (4, 2056), (300, 513), (33, 25088)])
def test_quantize_rows(dev, dtype, M, K):
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) * (torch.rand(M, 1, generator=g) * 100)).to(dtype)
    q, s = ops.quantize_rows(x.to(dev))
    wq, ws = _quantize64(x)
    assert q.dtype == torch.int8 and torch.equal(q.cpu(), wq)
    assert s.dtype == torch.float32 and torch.equal(s.cpu(), ws)


@on_both
def test_quantize_rows_edges(dev):
    x = torch.randn(9, 40)
    x[0] = 0
    x[1, 3] = float('inf')
    x[2, 39] = float('nan')
    x[3] = 1e-40                      # below the smallest scale
    x[4] = 3e38
    x[5] = torch.arange(40) - 20.0    # the peak is 20, steps of 127 / 20
    x[6, 0], x[6, 1:] = -1.0, 0.5     # -127 and a tie-free half
    x[7] = -float('inf')
    # a scale of exactly 2^-7 * fl(1 / 127) * 128, a power of two apart from 127's: ties go to even
    x[8] = torch.tensor([1.0] + [k + 0.5 for k in range(39)])
    x[8, 1:] *= float(torch.tensor(1.0 / 127))
    q, s = ops.quantize_rows(x.to(dev))
    q, s = q.cpu(), s.cpu()
    wq, ws = _quantize64(x)
    bad = torch.tensor([1, 2, 7])
    good = torch.tensor([0, 3, 4, 5, 6, 8])
    assert torch.isnan(s[bad]).all() and (q[bad] == 0).all()
    assert torch.equal(s[good], ws[good]) and torch.equal(q[good], wq[good])
    assert int(q[6, 0]) == -127 and float(s[0]) == 2.0 ** -126
    assert float(s[8]) == float(torch.tensor(1.0 / 127)) and q[8, 1:].remainder(2).eq(0).sum() >= 20


@on_both
@pytest.mark.parametrize('dtype', DTYPES)
def test_quantize_rows_strided(dev, dtype):
    base = torch.randn(12, 64 + 24).to(dtype).to(dev)
    for x in (base[:, 8:72], base[:, 3:66], base[::3, :64], base.t()[:40], base[:, :64][:1]):
        q, s = ops.quantize_rows(x)
        wq, ws = _quantize64(x)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    for shape in ((0, 16), (4, 0), (0, 0)):
        q, s = ops.quantize_rows(torch.empty(shape, dtype=dtype, device=dev))
        assert tuple(q.shape) == shape and tuple(s.shape) == shape[:1]
        assert (s.cpu() == 2.0 ** -126).all()


@on_both
@pytest.mark.parametrize('M,N,K', [
    (1, 1, 1), (1, 4096, 64), (1, 5, 4096), (2, 64, 48), (7, 33, 130), (15, 100, 1024), (16, 64, 272), (17, 65, 80),
    (31, 129, 4099), (64, 64, 64), (65, 127, 63), (96, 324, 2048), (128, 128, 16), (130, 260, 640), (257, 84, 1000),
    (300, 512, 1568), (301, 325, 515), (513, 40, 96)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_int8_matmul(dev, M, N, K, dtype):
    args = _operands(M, N, K, dev, seed=M + N + K)
    bias = (torch.randn(N, generator=torch.Generator().manual_seed(1)) * 0.1).to(dev) if M % 2 else None
    relu = N % 2 == 1
    y = ops.int8_matmul(*args, bias, relu=relu, out_dtype=dtype)
    _check_product(y, args, bias, relu, dtype)


@on_both
def test_int8_matmul_empty(dev):
    xq, xs, wq, ws = _operands(4, 6, 32, dev)
    assert tuple(ops.int8_matmul(xq[:0], xs[:0], wq, ws).shape) == (0, 6)
    assert tuple(ops.int8_matmul(xq, xs, wq[:0], ws[:0]).shape) == (4, 0)
    b = torch.arange(6.0, device=dev) - 2
    y = ops.int8_matmul(xq[:, :0], xs, wq[:, :0], ws, b, out_dtype=torch.float32)
    assert torch.equal(y, b.expand(4, 6))
    y = ops.int8_matmul(xq[:, :0], xs, wq[:, :0], ws, b, relu=True, out_dtype=torch.float32)
    assert torch.equal(y, b.clamp(min=0).expand(4, 6))


@on_both
@pytest.mark.parametrize('M,N,K', [(20, 40, 96), (3, 70, 256), (140, 130, 144)])
def test_int8_matmul_strides(dev, M, N, K):
    """Row strides, addresses and orders other than contiguous rows."""
    g = torch.Generator().manual_seed(3)
    xs, ws = torch.rand(M, generator=g).to(dev), torch.rand(N, generator=g).to(dev)
    big = torch.randint(-127, 128, (2 * max(M, N), K + 64), generator=g, dtype=torch.int8).to(dev)
    views = [(big[:M, :K], big[:N, 16:K + 16]), (big[:M, 1:K + 1], big[:N, :K]), (big[:M, :K], big[:N, 7:K + 7]),
             (big[::2][:M, 32:K + 32], big[1::2][:N, 16:K + 16]),
             (big[:K, :M].t() if M <= K + 64 and K <= big.shape[0] else big[:M, :K], big[:N, :K]),
             (big[:1, :K].expand(M, K), big[:N, :K])]
    for xq, wq in views:
        y = ops.int8_matmul(xq, xs, wq, ws, out_dtype=torch.float32)
        _check_product(y, (xq, xs, wq, ws), None, False, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize('M,N', [(5, 20), (33, 17), (70, 130)])
def test_int8_matmul_any_address(cuda, M, N):
    """Rows that start at every byte of a dword and end at every place of a load: with scales of 1 and an fp32
    result, the sum rounded once.  What lies between and behind the rows is not zero."""
    gen = torch.Generator().manual_seed(3)
    one = torch.ones(max(M, N), device=cuda)
    for K in (1, 3, 15, 16, 17, 63, 64, 65, 79, 127, 129, 2047, 2048, 2049, 2064, 4111, 6200):
        for at, gap in ((0, 0), (1, 0), (2, 3), (3, 5), (0, 1), (4, 4)):
            flat = [torch.randint(-128, 128, (at + r * (K + gap),), generator=gen).to(torch.int8) for r in (M, N)]
            x, w = (torch.as_strided(f.to(cuda), (r, K), (K + gap, 1), at) for f, r in zip(flat, (M, N)))
            got = ops.int8_matmul(x, one[:M], w, one[:N], out_dtype=torch.float32)
            want = (x.cpu().to(torch.int64) @ w.cpu().to(torch.int64).t()).float()
            assert torch.equal(got.cpu(), want), (K, at, gap)


@pytest.mark.gpu
@pytest.mark.parametrize('M,N,K', [(1, 512, 25088), (15, 64, 21419), (20, 530, 7026), (40, 64, 20001), (33, 20, 30000),
                                   (16, 33, 16385), (2, 70, 131071)])
def test_int8_matmul_long_rows(cuda, M, N, K):
    """Few rows and a long K, which is cut into runs: the sums stay exact."""
    gen = torch.Generator().manual_seed(K)
    x, w = (torch.randint(-128, 128, (r, K), generator=gen).to(torch.int8) for r in (M, N))
    one = torch.ones(max(M, N), device=cuda)
    got = ops.int8_matmul(x.to(cuda), one[:M], w.to(cuda), one[:N], out_dtype=torch.float32)
    assert torch.equal(got.cpu(), (x.to(torch.int64) @ w.to(torch.int64).t()).float())


@pytest.mark.gpu
@pytest.mark.parametrize('K', [5, 9, 100])
def test_more_rows_than_one_launch_takes(cuda, K):
    """Rows past 2^21 (quantized, copied) and 2^22 blocks: the last ones are as if they were alone."""
    M = (1 << 22) + 77
    gen = torch.Generator(device='cuda').manual_seed(K)
    x = torch.randn(M, K, generator=gen, device=cuda, dtype=torch.bfloat16)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(torch.randn(40, K, generator=gen, device=cuda))
    y = ops.int8_matmul(q, s, wq, ws)
    y2 = ops.int8_linear(x, wq, ws)
    for at in (0, (1 << 21) - 3, (1 << 22) - 3, M - 30):
        part = slice(at, at + 30)
        q1, s1 = ops.quantize_rows(x[part])
        assert torch.equal(q[part], q1) and torch.equal(s[part], s1), at
        want = ops.int8_matmul(q1, s1, wq, ws)
        assert torch.equal(y[part], want) and torch.equal(y2[part], want), at


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_int8_linear_is_its_two_parts(cuda, dtype):
    gen = torch.Generator().manual_seed(4)
    for M, N, K in ((1, 9, 1), (1, 40, 7), (3, 8, 17), (20, 300, 1001), (300, 96, 515), (130, 257, 4096), (2, 5, 33000)):
        x = torch.randn(M, K, generator=gen).to(dtype).to(cuda)
        wq, ws = ops.quantize_rows(torch.randn(N, K, generator=gen).to(cuda))
        b = torch.randn(N, generator=gen).to(cuda)
        want = ops.int8_matmul(*ops.quantize_rows(x), wq, ws, b, relu=True, out_dtype=dtype)
        assert torch.equal(ops.int8_linear(x, wq, ws, b, relu=True), want), (M, N, K)


@on_both
def test_int8_matmul_extremes(dev):
    """The largest sums (K = 131071, all -128), single steps, and a NaN scale that stays in its row."""
    K = int8_ops.MAX_K
    xq = torch.full((3, K), -128, dtype=torch.int8, device=dev)
    wq = torch.full((5, K), -128, dtype=torch.int8, device=dev)
    xq[1] = 127
    xq[2] = 0
    xq[2, K - 1] = 1
    xs, ws = torch.ones(3, device=dev), torch.ones(5, device=dev)
    y = ops.int8_matmul(xq, xs, wq, ws, out_dtype=torch.float32).cpu().double()
    for r, v in enumerate((16384 * K, -16256 * K, -128)):
        assert (y[r] - v).abs().max() <= 2.0 ** -24 * abs(v)
    xs[1] = float('nan')
    for relu in (False, True):
        y = ops.int8_matmul(xq, xs, wq, ws, relu=relu).cpu()
        assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


@on_both
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,N,K', [(1, 256, 1568), (9, 65, 77), (300, 128, 512)])
def test_int8_linear(dev, dtype, M, N, K):
    """Two layers in a row, as the head runs them: each is its own rows quantized, then the product."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(M, K, generator=g).clamp(min=0).to(dtype).to(dev)
    w1 = ops.quantize_rows((torch.randn(N, K, generator=g) * 0.05).to(dev))
    w2 = ops.quantize_rows((torch.randn(24, N, generator=g) * 0.05).to(dev))
    b = torch.randn(N, generator=g).to(dev)
    h = ops.int8_linear(x, *w1, b, relu=True)
    xq, xs = _quantize64(x)
    _check_product(h, (xq, xs, *w1), b, True, dtype)
    y = ops.int8_linear(h, *w2)
    hq, hs = _quantize64(h)
    _check_product(y, (hq, hs, *w2), None, False, dtype)


@on_both
def test_int8_refusals(dev):
    xq, xs, wq, ws = _operands(4, 6, 32, dev)
    for bad in (xq, xs.double()[:, None], xs, xs.to(torch.int32)[:, None]):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            ops.quantize_rows(bad)
    f = torch.ones(4, 8, device=dev)
    cases = [(f, xs, wq, ws), (xq, xs, f, ws), (xq[0], xs, wq, ws), (xq, xs[:3], wq, ws), (xq, xs, wq, xs),
             (xq, xs.half(), wq, ws), (xq[:, :16], xs, wq, ws), (xq, xs, wq, ws[:, None])]
    for c in cases:
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            ops.int8_matmul(*c)
    for kw in ({'bias': xs}, {'bias': ws.half()}, {'out_dtype': torch.float64}, {'out_dtype': torch.int32}):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            ops.int8_matmul(xq, xs, wq, ws, **kw)
    long = torch.zeros(1, int8_ops.MAX_K + 1, dtype=torch.int8, device=dev)
    with pytest.raises(ValueError):
        ops.int8_matmul(long, xs[:1], long, ws[:1])


@pytest.mark.gpu
def test_int8_refuses_mixed_devices(cuda):
    xq, xs, wq, ws = _operands(4, 6, 32, cuda)
    for c in ((xq, xs.cpu(), wq, ws), (xq, xs, wq.cpu(), ws), (xq.cpu(), xs, wq, ws), (xq, xs, wq, ws.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.int8_matmul(*c)


@pytest.mark.gpu
@pytest.mark.parametrize('M,N,K', [(1, 512, 4096), (40, 96, 515), (300, 256, 2048)])
def test_int8_linear_graph_and_streams(cuda, M, N, K):
    """Captured on a side stream and replayed on new inputs: the eager result, every time; a second
    graph and eager work in between do not disturb it."""
    g = torch.Generator().manual_seed(7)
    w = ops.quantize_rows(torch.randn(N, K, generator=g).to(cuda))
    b = torch.randn(N, generator=g).to(cuda)
    xs = [torch.randn(M, K, generator=g).bfloat16().to(cuda) for _ in range(4)]
    want = [ops.int8_linear(x, *w, b) for x in xs]
    static = [xs[0].clone(), xs[0].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            assert torch.equal(ops.int8_linear(s, *w, b), want[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.int8_linear(s, *w, b))
        graphs.append(gr)
    for k in range(6):
        i, j = k % 4, (k + 1) % 4
        static[0].copy_(xs[i])
        static[1].copy_(xs[j])
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(ops.int8_linear(xs[j], *w, b), want[j])
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[j])
