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

    def attention(q, k, v, cu_q, cu_k=None, *, want_low=False, **kw):
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


# ------------------------------------------------------------------------------------------------------ results apart
def _elements(x):
    """byte addresses of a tensor's elements, one by one"""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(x.shape, x.stride()):
        at = at[..., None] + torch.arange(n) * s
    return set((x.data_ptr() + x.element_size() * at.flatten()).tolist())


def test_results_that_overlap_inputs_at_any_offset_are_refused():
    from melspec_gpt_vqvae_amd.ops import _apart

    room = torch.zeros(40000)
    rows = lambda at, M, H, D=64: room[at:at + M * H * D].view(M, H, D)
    fused = room[:6 * 12 * 64].view(6, 12, 64)                     # q | k | v of 4 heads each, row by row
    heads = room[:12 * 6 * 64].view(12, 6, 64).transpose(0, 1)     # the same heads outermost
    good = [(rows(0, 6, 4), rows(6 * 256, 6, 4)), (fused[:, :4], fused[:, 4:8]), (fused[:, 8:], fused[:, :4]), (fused[:, 4:8], fused[:, 8:]),
            (heads[:, :4], heads[:, 4:]), (heads[:, 1::2], heads[:, ::2]), (fused[:, ::2], fused[:, 1::2]), (fused[:3], fused[3:]),
            (rows(0, 0, 4), rows(0, 6, 4)), (fused[:1, :4], fused[1:, :4]), (fused[..., :32], fused[..., 32:]), (rows(0, 6, 4), None)]
    for x, y in good:
        _apart(x, y)
        if y is not None:
            _apart(y, x)
    bad = [(rows(0, 6, 4), rows(64, 6, 4)), (rows(64, 6, 4), rows(0, 6, 4)), (fused[:, :4], fused[:, 3:7]), (fused[:, 4:8], fused),
           (heads[:, :4], heads[:, 3:]), (fused[:, :4], heads[:, :4]), (fused[..., :32], fused[..., 24:56]), (rows(0, 6, 4), rows(5 * 256 + 192, 1, 1)),
           (fused[:, :4], rows(12 * 64 * 5 + 64, 2, 2)), (fused[1:3, :4], fused[2:4, 2:6]), (rows(0, 6, 4), room[100:108].view(torch.int32))]
    for x, y in bad:
        for a, b in ((x, y), (y, x)):
            with pytest.raises(AssertionError):
                _apart(a, None, rows(30000, 2, 2), b)


def test_results_apart_against_every_element():
    import random

    from melspec_gpt_vqvae_amd.ops import _apart

    room, rng, seen = torch.zeros(6000), random.Random(1), [0, 0]
    for _ in range(3000):
        pair = []
        for _ in range(2):
            M, H, D = rng.randint(1, 5), rng.randint(1, 4), 4 * rng.randint(1, 3)
            h = 4 * rng.choice([0, D // 4, D // 4 + rng.randint(0, 3), rng.randint(1, 40)])
            r = 4 * rng.choice([0, H * h // 4 + D // 4, 24, rng.randint(1, 60)])
            pair.append(room.as_strided((M, H, D), (r, h, 1), 4 * rng.randint(0, 120)))
        x, y = pair
        apart = _elements(x).isdisjoint(_elements(y))
        seen[apart] += 1
        if apart:
            _apart(x, y)
        else:
            with pytest.raises(AssertionError):
                _apart(x, y)
    assert min(seen) > 500


# ------------------------------------------------------------------------------------------------------- shares
def test_shares_of_a_long_sequence_in_a_large_batch():
    from melspec_gpt_vqvae_amd import _ffi

    f = _ffi.lib().melgpt_paged_attn_splits
    assert f(256, 32, 8, 100000) == 25 and f(512, 32, 8, 100000) == 25 and f(64, 32, 8, 100000) == 25     # 4096 keys each
    assert f(256, 32, 8, 4096) == f(256, 32, 8, 16384) == 1 and f(64, 32, 8, 8192) == 4 and f(3, 32, 4, 131072) == 128   # as without
    assert f(513, 32, 8, 100000) == 1
    for S in (1, 64, 1000, 5000, 100000):
        for Hq, Hk in ((32, 8), (16, 16), (1, 1)):
            n, usual = f(S, Hq, Hk, 1 << 30), -(-2048 // (S * Hk))
            assert 1 <= n <= 128 and S * Hq * n <= max(1 << 19, S * Hq * usual)                           # room for partial results


def test_shares_of_a_long_sequence_in_a_packed_batch():
    from melspec_gpt_vqvae_amd import _ffi

    lib, H = _ffi.lib(), _ffi.BF16
    f, g = lib.melgpt_packed_attn_splits, lib.melgpt_packed_attn_splits_for
    for n in (63, 255):                                            # 128 queries over 16000 keys among tokens over 64
        a = (128 + n, 16000 + 64 * n, n + 1, 8, 128, H)
        assert f(*a) == 1 and g(*a, 16000) == 16 and g(*a, 64) == g(*a, 0) == 1
    assert g(2000, 2000, 8, 16, 64, H, 2000) == f(2000, 2000, 8, 16, 64, H) == 1                          # nothing to gain
    for a in ((1500, 16001, 1, 32, 128, H), (100, 100, 1, 16, 64, H), (1, 16000, 1, 32, 128, H), (200, 16000, 9, 8, 128, _ffi.F32), (0, 5, 3, 1, 64, H)):
        assert g(*a, a[1]) == f(*a)                                # one sequence, the f32 lane, no rows: as before
    for rows in (64, 4000, 100000):                                # room for partial results
        assert g(rows, 10 ** 6, 60, 32, 128, H, 500000) * rows * 32 <= max(1 << 19, rows * 32)
