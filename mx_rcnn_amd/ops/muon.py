"""Orthogonalised updates (Muon): Newton-Schulz orthogonalisation of weight-shaped matrices and the
weight update built on it, beside the fused SGD of ops/sgd.py (csrc/hip/newton_schulz.hip).

The update of an (out, in) matrix keeps a plain momentum of its gradient and steps along the
momentum's orthogonal factor, whose singular values all lie near 1 -- every direction of the matrix moves
by about the same amount.  Conv filters take part as (out, kh * kw * in) matrices (the order of the columns does
not matter); biases, BN parameters and the predictors stay with SGD.

CPU tensors run the PyTorch form below, which is also the oracle of the kernels.
"""
import math

import torch

from ._ext import need_ext, refuse_grad

NS_COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
MAX_STEPS = 16
MAX_SIDES = (16384, 1 << 20)  # of the smaller and the larger side


def newton_schulz_ref(g, steps=5, eps=EPS):
    """(b, r, c) -> (b, r, c) in g's own precision: X0 = G / (|G|_F + eps), then ``steps`` times
    X <- (a I + b A + c A^2) X with A = X X^T (of the smaller side)."""
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2) if tall else g
    x = (x.double() / (x.double().square().sum((1, 2), keepdim=True).sqrt() + eps)).to(g.dtype)
    a, b, c = NS_COEFFS
    for _ in range(steps):
        m = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * m + c * (m @ m)) @ x
    return (x.transpose(1, 2) if tall else x).contiguous()


def _check_steps(steps, eps):
    if int(steps) != steps or not 1 <= steps <= MAX_STEPS:
        raise ValueError('newton_schulz: 1 to %d steps, not %r' % (MAX_STEPS, steps))
    if not eps > 0:
        raise ValueError('newton_schulz: eps must be positive, not %r' % (eps,))


def _check_sides(r, c):
    if r < 1 or c < 1 or min(r, c) > MAX_SIDES[0] or max(r, c) > MAX_SIDES[1]:
        raise ValueError('newton_schulz: a matrix of %d x %d (the smaller side may be %d, the larger %d)' %
                         ((r, c) + MAX_SIDES))


def orthogonalize(g, steps=5, eps=EPS):
    """The Newton-Schulz orthogonalisation of a matrix (r, c) or of each of a batch (b, r, c), in g's
    type (fp32, bf16 or fp16): U V^T of G = U S V^T up to the iteration's own accuracy (singular values
    between about 0.7 and 1.2 after five steps, those far below |G|_F / 500 left smaller).  A matrix of zeros stays
    zero; one that holds an infinity or a NaN comes back as NaN.  Computed in 22-bit operands with fp32 sums
    whatever the type; where |G|_F is far below ``eps``, to an absolute accuracy of about 1e-9.  Not
    differentiable: an input that records a gradient is refused."""
    if g.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError('orthogonalize: fp32, bf16 or fp16, not %s' % g.dtype)
    if g.dim() not in (2, 3):
        raise ValueError('orthogonalize: (r, c) or (b, r, c), not %s' % (tuple(g.shape),))
    _check_steps(steps, eps)
    x = g.contiguous()
    x = x.unsqueeze(0) if g.dim() == 2 else x
    if x.numel() == 0:
        return torch.empty_like(x).reshape(g.shape)
    _check_sides(x.shape[1], x.shape[2])
    if x.is_cuda:
        return need_ext().ns_orthogonalize(x, int(steps), float(eps)).reshape(g.shape)
    refuse_grad('orthogonalize', g)
    return newton_schulz_ref(x.float(), steps, eps).reshape(g.shape).to(g.dtype)


def muon_update_(w, mom, grad, mats, lr, momentum=0.95, wd=0.0, rescale=1.0, clip=-1.0, nesterov=True, steps=5, eps=EPS,
                 w_bf16=None, planes=1, zero=None, plane_stride=0):
    """In-place Muon update of the matrices ``mats`` -- (element offset, rows, cols) each, disjoint -- of
    flat fp32 ``w`` / ``mom`` from ``grad`` (fp32, bf16 or fp16); elements outside them are not touched:

        g = clip(rescale * grad),  mom = momentum * mom + g,  u = g + momentum * mom (nesterov) or mom
        w -= lr * (sqrt(max(1, rows / cols)) * orthogonalize(u) + wd * w)

    A NaN in a matrix's gradient is not clipped away: that matrix's weights become NaN, the others' do not.
    ``lr``, ``w_bf16``, ``planes``, ``plane_stride`` and ``zero`` are those of :func:`sgd_momentum_`: a
    1-element fp32 device tensor, the low-precision copy of the new weights, its planes, and the gradient
    buffer to clear once read (the matrices' elements of it).  All matrices of a call share its launches, and
    the tiles are chosen for the call: the same call gives the same bits, a matrix among others may end in other
    last bits than alone."""
    _check_steps(steps, eps)
    mats = [(int(o), int(r), int(c)) for o, r, c in mats]
    for o, r, c in mats:
        _check_sides(r, c)
        if o < 0 or o + r * c > w.numel():
            raise ValueError('muon_update_: matrix at %d (%d x %d) reaches outside the buffer of %d' %
                             (o, r, c, w.numel()))
    if w.is_cuda:
        need_ext().muon_update(w, mom, grad, mats, lr, float(momentum), float(wd), float(rescale), float(clip),
                               bool(nesterov), int(steps), float(eps), w_bf16, int(planes), zero, int(plane_stride))
        return
    assert not plane_stride, 'plane_stride: GPU only'
    spans = sorted((o, o + r * c) for o, r, c in mats)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError('muon_update_: overlapping matrices')
    step = lr.float()
    for o, r, c in mats:
        s = slice(o, o + r * c)
        g = grad[s].float() * rescale
        if clip > 0:
            g = g.clamp(-clip, clip)
        if zero is not None:
            zero[s] = 0
        mom[s] = momentum * mom[s] + g
        u = g + momentum * mom[s] if nesterov else mom[s]
        d = newton_schulz_ref(u.view(1, r, c), steps, eps).reshape(-1)
        w[s] -= step * (math.sqrt(max(1.0, r / c)) * d + wd * w[s])
        if w_bf16 is not None:
            _write_shadow_span(w_bf16, w[s], planes, o)


def _write_shadow_span(w_bf16, w, planes, at):
    if planes <= 1:
        w_bf16[at:at + w.numel()].copy_(w)
        return
    from . import precision
    parts, n, pl = precision.split(w, planes), w.numel(), w_bf16.numel() // planes
    for k in range(planes):
        w_bf16[k * pl + at:k * pl + at + n].copy_(parts[k * n:(k + 1) * n])
