"""Differentiable operators for packed sequences of different lengths, over the kernels of ops.py: what a transformer with
rotary positions, normed queries and keys and shared key heads needs between its projections.  The serving forms
(ops.kv_append, ops.paged_attn_decode) stand in ops.py; they have no gradient.  Gradients are reverse mode, once: second
derivatives and forward mode raise.

A captured backward pass (HIP graph): call ops.*_fwd / ops.*_bwd directly, or capture forward and backward together with
torch.autograd.grad on leaves that no live eager graph holds - autograd's leaf nodes remember the stream they were made on."""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops


def rotary_freqs(rot, base=10000.0, *, stretch=1.0, base_stretch=1.0, ramp=None, device="cuda"):
    """-> (rot / 2,) f64 radians per position: base^(-2 i / rot), for longer contexts than trained on optionally scaled.
      stretch       positions divided by it (every frequency / stretch)
      base_stretch  the base raised so that the slowest frequency shrinks by it and the fastest keeps its own
      ramp          (trained length, slow turns, fast turns): `stretch` applies in full to frequencies that make fewer than
                    `slow` turns over the trained length, not at all to those of more than `fast`, linearly between"""
    assert rot > 0 and rot % 2 == 0
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    if base_stretch != 1.0:
        assert rot > 2
        base = base * base_stretch ** (rot / (rot - 2))
    f = base ** (-i)
    if stretch != 1.0:
        if ramp is None:
            f = f / stretch
        else:
            trained, slow, fast = ramp
            keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
            f = f * keep + f / stretch * (1 - keep)
    return f.to(device)


_tracing = torch._C._get_tracing_state


def _differentiated(*tensors):
    """whether one of them wants a gradient or carries a tangent of forward-mode differentiation"""
    grad, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if grad or dual:
        for t in tensors:
            if t is not None and ((grad and t.requires_grad) or (dual and forward_ad.unpack_dual(t).tangent is not None)):
                return True
    return False


def _through_autograd(*tensors):
    """whether a call goes through its autograd function: for a gradient; with a tangent, which the function refuses and the
    bare kernel would drop; and in a trace, which holds the function and not the kernel"""
    return _differentiated(*tensors) or _tracing() is not None


class _QkNormRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freqs, eps, interleaved, amplitude):
        kw = dict(q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved, amplitude=amplitude)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, freqs)
        ctx.cfg = (eps, interleaved, amplitude)
        return ops.qk_norm_rotary_fwd(q, k, positions, freqs, **kw)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, freqs = ctx.saved_tensors
        eps, interleaved, amplitude = ctx.cfg
        dq, dk, dqw, dkw = ops.qk_norm_rotary_bwd(dq_out, dk_out, q, k, positions, freqs, q_weight=q_weight, k_weight=k_weight,
                                                  eps=eps, interleaved=interleaved, amplitude=amplitude)
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rotary(q, k, positions, freqs, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, amplitude=1.0):
    """ops.qk_norm_rotary_fwd with gradients for q, k and both weights (not for freqs)."""
    if freqs is not None and (freqs.requires_grad or forward_ad._current_level >= 0):
        assert not _differentiated(freqs), "the frequencies have no gradient: give them detached"
    if not _through_autograd(q, k, q_weight, k_weight):
        return ops.qk_norm_rotary_fwd(q, k, positions, freqs, q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved,
                                      amplitude=amplitude)
    return _QkNormRotaryFn.apply(q, k, q_weight, k_weight, positions, freqs, float(eps), bool(interleaved), float(amplitude))


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale):
        out, lse, low = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, scale=scale, want_low=True)
        ctx.save_for_backward(q, k, v, out, lse, low, cu_q, cu_k)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, low, cu_q, cu_k = ctx.saved_tensors
        return ops.packed_attn_bwd(q, k, v, out, dout, lse, cu_q, cu_k, scale=ctx.scale, low=low) + (None, None, None)


def packed_attention(q, k, v, cu_q, cu_k=None, *, scale=None, max_length=None):
    """ops.packed_attn_fwd's output with gradients for q, k and v (those of a key head summed over its query heads).
    max_length: as there (a call with gradients does not share keys out)."""
    if not _through_autograd(q, k, v):
        return ops.packed_attn_fwd(q, k, v, cu_q, cu_k, scale=scale, max_length=max_length)[0]
    return _PackedAttentionFn.apply(q, k, v, cu_q, cu_k, scale)
