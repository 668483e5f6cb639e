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


# ---------------------------------------------------------------------------------------------------------- attention
def attention(q, k, v, scale, dout=None, sees=None):
    """one head of one sequence in 64 bits: q (nq, D), k, v (nk, D) -> dict of o, lse and, with dout, dq, dk, dv, and for each
    the size its f32 errors scale with (s_*)"""
    nq, nk = q.shape[0], k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    if sees is None:
        sees = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)
    s = scale * q @ k.t()
    s = s.masked_fill(~sees, -math.inf)
    lse = torch.logsumexp(s, -1) if nk else torch.full((nq,), -math.inf, dtype=torch.float64)
    some = lse > -math.inf
    p = torch.where(some[:, None], torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
    r = dict(o=p @ v, lse=lse, p=p, s_o=p @ v.abs(), s_score=(abs(scale) * q.abs() @ k.abs().t()).masked_fill(~sees, 0).amax(-1) if nk else torch.zeros(nq).double())
    if dout is not None:
        g = dout.double()
        dp = g @ v.t()
        delta = (g * r["o"]).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        r.update(dq=scale * ds @ k, dk=scale * ds.t() @ q, dv=p.t() @ g)
        sds = p * (g.abs() @ v.abs().t() + (g.abs() * r["s_o"]).sum(-1, keepdim=True))
        r.update(s_ds=sds, s_dq=abs(scale) * sds @ k.abs(), s_dk=abs(scale) * sds.t() @ q.abs(), s_dv=p.t() @ g.abs())
        one = sees.double()
        sdp = one * (1 + g.abs() @ v.abs().t() + (g.abs() * r["s_o"]).sum(-1, keepdim=True))
        r.update(a_dq=abs(scale) * sdp @ k.abs(), a_dk=abs(scale) * sdp.t() @ q.abs(), a_dv=one.t() @ g.abs())
    r["a_o"] = sees.double() @ v.abs()
    return r


def smallest(dtype):
    """absolute error of a probability, of ds or of a result below the normal range: the exponential's subnormal results are
    flushed (2^-126, f32 and bf16); IEEE half rounds there by half its smallest step, 2^-25.  The a_* sums carry it through
    the second product."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


# Attention.  A score is a product of D <= 128 terms summed in f32 by matrix instructions: |error| <= D u times the sum of
# sizes (s_score), so an exponential carries e = D u s_score + 4 u relative, and so does the sum of exponentials.
# Probabilities (and ds) are rounded to the tensors' type before the second product: h each relative; its sum over n keys
# is n u at worst.  The output is rounded once.  A relative error common to numerator and denominator only cancels in part:
# both are counted.
def attention_relative(D, s_score, n, dtype):
    """of a probability-weighted sum of n terms against its sum of sizes, in front of the last rounding"""
    h = half_step(dtype) if dtype != torch.float32 else 0.0
    return h + 2 * (D * U * s_score + 4 * U) + n * U
