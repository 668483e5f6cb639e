"""64-bit definitions of the packed-sequence operators and the error bounds the tests hold the kernels to (test
infrastructure).

Bounds.  u = 2^-24 is half a step of f32, h half a step of the tensor's type relative to the value
(torch.finfo(t).eps / 2).  A stored result is rounded once: h |value|.  Everything before it is f32 (matrix products of
16-bit operands: exact products, f32 sums)."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound elementwise (NaN where and only where wanted)"""
    got, want, bound = got.detach().double().cpu(), want.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~(((got - want).abs() <= bound) | same)
    if bad.any():
        i = int(torch.nonzero(bad.flatten())[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: got {got.flatten()[i]}, "
                             f"want {want.flatten()[i]}, bound {bound.expand_as(got).flatten()[i]}")


# ------------------------------------------------------------------------------------------------ norm and rotation
def rotate(x, pos, freqs, interleaved, amplitude, inverse=False):
    """x (M, H, D) f64"""
    if freqs is None:
        return x
    rot = 2 * freqs.numel()
    t = pos.double()[:, None, None] * freqs.double()
    c, s = amplitude * torch.cos(t), amplitude * torch.sin(t) * (-1 if inverse else 1)
    if interleaved:
        lo, hi = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((lo * c - hi * s, hi * c + lo * s), -1).flatten(-2)
    else:
        lo, hi = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
    return torch.cat((y, x[..., rot:]), -1)


def norm_rotary(x, w, pos, freqs, eps, interleaved, amplitude):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return rotate(x, pos, freqs, interleaved, amplitude)


def pair_size(x, freqs, interleaved, amplitude):
    """|lo| + |hi| of a value's pair (the value itself where nothing turns): what the errors of a rotation scale with"""
    x = x.abs()
    if freqs is None:
        return x
    rot = 2 * freqs.numel()
    y = x.clone()
    if interleaved:
        m = amplitude * (x[..., 0:rot:2] + x[..., 1:rot:2])
        y[..., 0:rot:2] = m
        y[..., 1:rot:2] = m
    else:
        m = amplitude * (x[..., :rot // 2] + x[..., rot // 2:rot])
        y[..., :rot] = torch.cat((m, m), -1)
    return y


# Of the norm: the sum of squares is 16 sequential terms and 5 exchanges (21 u), the quotient, the sum with eps and the
# root (halved) and the two products come to < 16 u.  Of the rotation: sine and cosine of a fraction rounded to f32 before
# them (the 16-bit lane): |t| <= 1/2 turn rounded by 2^-26, pi at most 2 pi 2^-26 < 2 u radians, 2 u of the functions;
# two products and a sum 3 u.  Together < 32 u of the pair's size.
def rotary_bound(n, want, dtype, freqs, interleaved, amplitude):
    return half_step(dtype) * want.abs() + 32 * U * pair_size(n, freqs, interleaved, abs(amplitude))
