"""8-bit products for serving: rows to int8 with one scale each, and the product of two such
matrices with bias and ReLU (csrc/hip/int8_gemm.hip).

A fully connected layer in this form keeps its weight as ``quantize_rows(weight)`` -- one scale per
output channel, laid out once -- and quantizes its input rows (one scale per RoI) in each call.  VGG16's
fc6 then reads 103 MB of weights instead of 205 MB of bf16, at twice the matrix-core rate.

None of them is differentiable: an input that records a gradient is refused.

CPU tensors run the PyTorch form below, which is also the oracle of the kernels.
"""
import torch

from ._ext import need_ext, refuse_grad

TINY = 2.0 ** -126
MAX_K = 131071  # int32 sums of 8-bit products are exact up to here, -128 included
OUT_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_float(x, what):
    if x.dtype not in OUT_CODES:
        raise TypeError('%s: fp32, bf16 or fp16, not %s' % (what, x.dtype))


def quantize_rows(x):
    """(M, K) fp32 / bf16 / fp16 -> (int8 (M, K), fp32 scales (M,)): scale = max|row| * (1 / 127) in fp32
    (at least 2^-126), values divided by it and rounded to the nearest integer, ties to even, so that ``q * scale`` stands
    for the row.  A row that holds an infinity or a NaN gets the scale NaN and zeros: what is computed from it is NaN."""
    if x.is_cuda:
        return tuple(need_ext().quantize_rows(_rows(x)))
    refuse_grad('quantize_rows', x)
    _check_float(x, 'quantize_rows')
    if x.dim() != 2:
        raise ValueError('quantize_rows: (M, K), not %s' % (tuple(x.shape),))
    xf = x.float()
    peak = xf.abs().amax(1) if x.shape[1] else xf.new_zeros(x.shape[0])
    bad = ~torch.isfinite(peak)
    s = (peak * torch.tensor(1.0 / 127.0)).clamp(min=TINY)  # (1 / 127 in fp32)
    q = torch.round(xf / s[:, None])
    q = torch.where(bad[:, None], torch.zeros_like(q), q).to(torch.int8)
    return q, torch.where(bad, torch.full_like(s, float('nan')), s)


def _rows(t):
    """``t`` with its columns contiguous (its rows any stride apart)."""
    return t if t.dim() != 2 or t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def int8_matmul(xq, xs, wq, ws, bias=None, relu=False, out_dtype=torch.bfloat16):
    """``relu(xs[:, None] * ws * (xq @ wq.T) + bias)`` of int8 ``xq`` (M, K) and ``wq`` (N, K) with fp32
    scales ``xs`` (M,) and ``ws`` (N,) and fp32 ``bias`` (N,): the sum exact in int32 (K <= 131071), the
    rest in fp32, rounded once to ``out_dtype`` (fp32, bf16 or fp16).  Rows may lie any stride apart, at any
    address; where there are many of them, those whose K, stride or address is no multiple of 16 are copied first."""
    if out_dtype not in OUT_CODES:
        raise TypeError('int8_matmul: out_dtype fp32, bf16 or fp16, not %s' % (out_dtype,))
    if xq.dim() == 2 and xq.shape[1] > MAX_K:
        raise ValueError('int8_matmul: K = %d (int32 sums are exact up to %d)' % (xq.shape[1], MAX_K))
    if xq.is_cuda:  # (the extension checks the rest)
        return need_ext().int8_matmul(_rows(xq), xs, _rows(wq), ws, bias, relu, OUT_CODES[out_dtype])
    refuse_grad('int8_matmul', xs, ws, bias)
    for t, what in ((xq, 'xq'), (wq, 'wq')):
        if t.dtype != torch.int8 or t.dim() != 2:
            raise TypeError('int8_matmul: %s must be a 2-D int8 tensor, not %s %s' % (what, t.dtype, tuple(t.shape)))
    M, K, N = xq.shape[0], xq.shape[1], wq.shape[0]
    if wq.shape[1] != K:
        raise ValueError('int8_matmul: K differs: xq %s, wq %s' % (tuple(xq.shape), tuple(wq.shape)))
    for t, n, what in [(xs, M, 'xs'), (ws, N, 'ws')] + ([] if bias is None else [(bias, N, 'bias')]):
        if t.dtype != torch.float32 or tuple(t.shape) != (n,):
            raise TypeError('int8_matmul: %s must be fp32 (%d,), not %s %s' % (what, n, t.dtype, tuple(t.shape)))
        if t.device != xq.device:
            raise ValueError('int8_matmul: tensors on %s and %s' % (xq.device, t.device))
    y = (xq.to(torch.int32) @ wq.to(torch.int32).t()).float()
    y = y * xs[:, None] * ws
    if bias is not None:
        y = y + bias
    if relu:
        y = torch.where(y < 0, torch.zeros_like(y), y)
    return y.to(out_dtype)


def int8_linear(x, wq, ws, bias=None, relu=False):
    """A fully connected layer on floating rows ``x`` (M, K) with an 8-bit weight (``quantize_rows`` of the
    (N, K) weight): the rows quantized, multiplied, scaled back; result in x's type."""
    if x.is_cuda:  # one call; the rows are quantized into the layout that the product reads
        if x.dim() == 2 and x.shape[1] > MAX_K:
            raise ValueError('int8_linear: K = %d (int32 sums are exact up to %d)' % (x.shape[1], MAX_K))
        return need_ext().int8_linear(_rows(x), _rows(wq), ws, bias, relu)
    refuse_grad('int8_linear', x, ws, bias)
    xq, xs = quantize_rows(x)
    return int8_matmul(xq, xs, wq, ws, bias, relu, x.dtype)
