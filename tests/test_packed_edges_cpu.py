"""Packed and cached sequence operators at the edges of what their documentation allows, without a GPU (stand-ins in place of
the kernels where a call is needed)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


# ------------------------------------------------------------------------------------ derivatives other than .backward()'s
def _opaque(monkeypatch):
    """the kernels' wrappers replaced by host code that torch does not see: (2 q + mean v), (2 q, 3 k)"""
    from melspec_gpt_vqvae_amd import ops

    def host(x, f):
        return torch.from_numpy(f(x.detach().numpy()).copy())

    def attention(q, k, v, cu_q, cu_k=None, *, scale=None, out=None, want_low=False):
        o = host(q, lambda a: 2 * a + v.detach().numpy().mean())
        return (o, o[..., 0].t().contiguous(), None) if want_low else (o, o[..., 0])

    def rotary(q, k, positions, freqs, **kw):
        return host(q, lambda a: 2 * a), host(k, lambda a: 3 * a)

    monkeypatch.setattr(ops, "packed_attn_fwd", attention)
    monkeypatch.setattr(ops, "qk_norm_rotary_fwd", rotary)


@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused_not_dropped(which, grad_mode, monkeypatch):
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    _opaque(monkeypatch)
    x = [torch.randn(5, 2, 64) for _ in range(3)]
    w = [torch.ones(64), torch.ones(64)]
    pos, cu = torch.arange(5, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        pk.packed_attention(*x, cu)                                # (a level alone is no tangent)
        pk.qk_norm_rotary(x[0], x[1], pos, None, q_weight=w[0], k_weight=w[1])
        if which < 3:
            d = list(x)
            d[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
            with pytest.raises(NotImplementedError):
                pk.packed_attention(*d, cu)
        d = x[:2] + w
        d[which] = forward_ad.make_dual(d[which], torch.ones_like(d[which]))
        with pytest.raises(NotImplementedError):
            pk.qk_norm_rotary(d[0], d[1], pos, None, q_weight=d[2], k_weight=d[3])


@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_trace_holds_the_operator(requires_grad, monkeypatch):
    """replayed with other inputs it computes them, and does not repeat what it saw"""
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    _opaque(monkeypatch)
    q, k, v = [torch.randn(5, 2, 64) for _ in range(3)]
    cu, pos = torch.tensor([0, 5], dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    q.requires_grad_(requires_grad)
    attention = torch.jit.trace(lambda a, b, c: pk.packed_attention(a, b, c, cu), (q, k, v), check_trace=False)
    rotary = torch.jit.trace(lambda a, b: pk.qk_norm_rotary(a, b, pos, None), (q, k), check_trace=False)
    q2, k2, v2 = [torch.randn(5, 2, 64) for _ in range(3)]
    assert torch.equal(attention(q2, k2, v2), 2 * q2 + v2.numpy().mean())
    a, b = rotary(q2, k2)
    assert torch.equal(a, 2 * q2) and torch.equal(b, 3 * k2)


def test_frequencies_that_want_a_gradient_are_refused(monkeypatch):
    """the rotation has no gradient for its frequencies: they are refused rather than left without one"""
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    _opaque(monkeypatch)
    q, k = [torch.randn(5, 2, 64) for _ in range(2)]
    pos, f = torch.arange(5, dtype=torch.int32), pk.rotary_freqs(64, device="cpu").requires_grad_(True)
    for a in (q, q.clone().requires_grad_(True)):
        with pytest.raises(AssertionError):
            pk.qk_norm_rotary(a, k, pos, f)
        with torch.no_grad():
            pk.qk_norm_rotary(a, k, pos, f)
    pk.qk_norm_rotary(q, k, pos, f.detach())
    with forward_ad.dual_level(), pytest.raises(AssertionError):
        pk.qk_norm_rotary(q, k, pos, forward_ad.make_dual(f.detach(), torch.ones(32, dtype=torch.float64)))
