"""Refusals of the packed / cached sequence entry points (arguments are checked on the host before anything is launched, so
made-up addresses do) and the rotation frequencies, without a GPU."""
import math

import pytest
import torch

OK, BAD, UNSUPPORTED, ALIGN = 0, -1, -2, -4
P = 1 << 20        # a made-up, aligned address
F32, HALF = 0, 1


def _lib():
    from melspec_gpt_vqvae_amd import _ffi

    return _ffi.lib()


def norm_rotary(q=P, qr=512, qh=64, k=P, kr=512, kh=64, pos=P, freqs=P, rot=64, il=0, amp=1.0, wq=P, wk=P, eps=1e-6, qo=P, ko=P,
                M=3, Hq=8, Hk=8, D=64, dt=HALF):
    return _lib().melgpt_qk_norm_rotary_fwd(q, qr, qh, k, kr, kh, pos, freqs, rot, il, amp, wq, wk, eps, qo, ko, M, Hq, Hk, D, dt, None)


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), OK), (dict(q=None), BAD), (dict(k=None), BAD), (dict(pos=None), BAD), (dict(freqs=None), BAD), (dict(qo=None), BAD),
    (dict(ko=None), BAD), (dict(Hq=0), BAD), (dict(Hk=-1), BAD), (dict(M=-1), BAD), (dict(wq=None), BAD), (dict(wk=None), BAD),
    (dict(rot=-16), BAD), (dict(dt=2), UNSUPPORTED), (dict(D=72, rot=16), UNSUPPORTED), (dict(D=272), UNSUPPORTED),
    (dict(rot=24), UNSUPPORTED), (dict(rot=80), UNSUPPORTED), (dict(q=P + 8), ALIGN), (dict(k=P + 2), ALIGN), (dict(qr=513), ALIGN),
    (dict(kh=66), ALIGN), (dict(qo=P + 4), ALIGN)])
def test_norm_rotary_refusals(kw, code):
    assert norm_rotary(**kw) == code


def norm_rotary_bwd(gq=P, gqr=512, gqh=64, gk=P, gkr=512, gkh=64, q=P, k=P, pos=P, freqs=P, rot=64, wq=P, wk=P, dq=P, dk=P, part=P,
                    M=3, Hq=8, Hk=8, D=64, dt=HALF, xr=512):
    return _lib().melgpt_qk_norm_rotary_bwd(gq, gqr, gqh, gk, gkr, gkh, q, xr, 64, k, xr, 64, pos, freqs, rot, 0, 1.0, wq, wk, 1e-6,
                                            dq, dk, part, M, Hq, Hk, D, dt, None)


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), OK), (dict(gq=None), BAD), (dict(gk=None), BAD), (dict(dq=None), BAD), (dict(dk=None), BAD), (dict(part=None), BAD),
    (dict(q=None), BAD), (dict(wk=None), BAD), (dict(gq=P + 8), ALIGN), (dict(dk=P + 8), ALIGN), (dict(gkr=510), ALIGN),
    (dict(xr=500), ALIGN), (dict(D=24), UNSUPPORTED), (dict(dt=9), UNSUPPORTED)])
def test_norm_rotary_bwd_refusals(kw, code):
    assert norm_rotary_bwd(**kw) == code


def append(q=P, k=P, kr=512, v=P, vr=512, seq=P, pos=P, table=P, S=2, width=4, freqs=P, rot=64, wq=P, wk=P, qo=P, kp=P, vp=P,
           pages=9, page=16, M=3, Hq=8, Hk=8, D=64, dt=HALF):
    return _lib().melgpt_kv_append(q, 512, 64, k, kr, 64, v, vr, 64, seq, pos, table, width, S, width, freqs, rot, 0, 1.0, wq, wk, 1e-6,
                                   qo, 1, kp, vp, pages, page, M, Hq, Hk, D, dt, None)


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), OK), (dict(k=None), BAD), (dict(v=None), BAD), (dict(seq=None), BAD), (dict(pos=None), BAD), (dict(table=None), BAD),
    (dict(S=0), BAD), (dict(width=0), BAD), (dict(kp=None), BAD), (dict(vp=None), BAD), (dict(pages=0), BAD), (dict(qo=None), BAD),
    (dict(wk=None), BAD), (dict(page=0), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(page=-16), UNSUPPORTED),
    (dict(pages=1 << 31), UNSUPPORTED), (dict(D=40), UNSUPPORTED), (dict(rot=8), UNSUPPORTED), (dict(dt=3), UNSUPPORTED),
    (dict(kp=P + 8), ALIGN), (dict(v=P + 8), ALIGN), (dict(vr=100), ALIGN), (dict(q=P + 4), ALIGN)])
def test_append_refusals(kw, code):
    assert append(**kw) == code


def packed(q=P, qr=512, k=P, kr=512, v=P, vr=512, cq=P, ck=P, S=2, o=P, orow=512, lse=P, Mq=100, Mk=100, Hq=8, Hk=4, D=64, dt=HALF,
           low=None, splits=1, ws=None, scale=0.125):
    return _lib().melgpt_packed_attn_fwd(q, qr, 64, k, kr, 64, v, vr, 64, cq, ck, S, o, orow, 64, low, lse, 1, splits, ws, Mq, Mk, Hq,
                                         Hk, D, scale, dt, None)


PACKED_REFUSALS = [
    (dict(q=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(cq=None), BAD), (dict(ck=None), BAD), (dict(S=-1), BAD),
    (dict(o=None), BAD), (dict(lse=None), BAD), (dict(Mq=-1), BAD), (dict(Mk=-1), BAD), (dict(Hq=0), BAD), (dict(Hk=0), BAD),
    (dict(Hq=9), UNSUPPORTED), (dict(D=96), UNSUPPORTED), (dict(D=32), UNSUPPORTED), (dict(dt=2), UNSUPPORTED),
    (dict(kr=56), UNSUPPORTED), (dict(vr=0), UNSUPPORTED), (dict(qr=8), UNSUPPORTED), (dict(kr=1 << 25), UNSUPPORTED),
    (dict(Mq=1 << 23), UNSUPPORTED), (dict(S=1 << 20), UNSUPPORTED), (dict(Mk=1 << 31), UNSUPPORTED), (dict(q=P + 8), ALIGN),
    (dict(v=P + 2), ALIGN), (dict(orow=100), ALIGN), (dict(qr=516), ALIGN), (dict(low=P + 8), ALIGN), (dict(low=P, dt=F32), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", PACKED_REFUSALS + [
    (dict(Mq=0), OK), (dict(splits=0), BAD), (dict(splits=2), BAD), (dict(splits=2, ws=P, dt=F32), UNSUPPORTED),
    (dict(splits=2, ws=P, low=P), UNSUPPORTED), (dict(splits=2000, ws=P), UNSUPPORTED), (dict(splits=2, ws=P + 4), ALIGN)])
def test_packed_refusals(kw, code):
    assert packed(**kw) == code


def packed_bwd(q=P, qr=512, k=P, kr=512, v=P, vr=512, cq=P, ck=P, S=2, o=P, orow=512, lse=P, Mq=100, Mk=100, Hq=8, Hk=4, D=64, dt=HALF,
               do=P, dor=512, delta=P, dq=P, dqr=512, dk=P, dv=P, low=P, scale=0.125, splits=1, ws=None):
    return _lib().melgpt_packed_attn_bwd(q, qr, 64, k, kr, 64, v, vr, 64, cq, ck, S, o, orow, 64, low, do, dor, 64, lse, delta, dq, dqr, 64,
                                         dk, 256, 64, dv, 256, 64, 1, splits, ws, Mq, Mk, Hq, Hk, D, scale, dt, None)


@pytest.mark.parametrize("kw,code", [r for r in PACKED_REFUSALS if "Mq" not in r[0] or r[0]["Mq"] < 0] + [
    (dict(do=None), BAD), (dict(delta=None), BAD), (dict(dq=None), BAD), (dict(dk=None), BAD), (dict(dv=None), BAD),
    (dict(dor=32), UNSUPPORTED), (dict(Mq=1 << 23), UNSUPPORTED), (dict(dq=P + 8), ALIGN), (dict(dqr=513), ALIGN), (dict(do=P + 4), ALIGN),
    (dict(splits=0), BAD), (dict(splits=2), BAD), (dict(splits=2, ws=P, dt=F32, low=None), UNSUPPORTED), (dict(splits=2000, ws=P), UNSUPPORTED),
    (dict(splits=2, ws=P + 4), ALIGN)])
def test_packed_bwd_refusals(kw, code):
    assert packed_bwd(**kw) == code


def decode(q=P, qr=512, kp=P, vp=P, pages=9, page=16, table=P, width=4, lens=P, S=2, o=P, orow=512, lse=P, splits=1, ws=None, Hq=8,
           Hk=4, D=64, dt=HALF, scale=0.125):
    return _lib().melgpt_paged_attn_decode(q, qr, 64, kp, vp, pages, page, table, width, width, lens, S, o, orow, 64, lse, splits, ws, Hq,
                                           Hk, D, scale, dt, None)


@pytest.mark.parametrize("kw,code", [
    (dict(S=0), OK), (dict(S=-1), BAD), (dict(q=None), BAD), (dict(kp=None), BAD), (dict(vp=None), BAD), (dict(table=None), BAD),
    (dict(lens=None), BAD), (dict(o=None), BAD), (dict(lse=None), BAD), (dict(splits=2), BAD), (dict(splits=0), BAD), (dict(width=0), BAD),
    (dict(pages=0), BAD), (dict(Hk=0), BAD), (dict(page=24), UNSUPPORTED), (dict(Hq=6), UNSUPPORTED), (dict(D=256), UNSUPPORTED),
    (dict(dt=2), UNSUPPORTED), (dict(pages=1 << 31), UNSUPPORTED), (dict(S=1 << 22), UNSUPPORTED), (dict(Hq=1 << 13), UNSUPPORTED),
    (dict(q=P + 8), ALIGN), (dict(orow=4), ALIGN), (dict(vp=P + 8), ALIGN)])
def test_decode_refusals(kw, code):
    assert decode(**kw) == code


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan])
def test_scales_that_are_not_finite_are_refused(scale):
    assert packed(scale=scale) == packed_bwd(scale=scale) == decode(scale=scale) == BAD


def test_splits():
    f = _lib().melgpt_paged_attn_splits
    for S, Hq, Hk, n in ((1, 16, 16, 1), (1, 16, 16, 265), (64, 32, 8, 8192), (3, 32, 4, 131072), (1, 1, 1, 10 ** 9), (4096, 32, 8, 8192)):
        s = f(S, Hq, Hk, n)
        assert 1 <= s <= 128 and (s == 1 or n >= 256 * (s - 1))
    assert f(1, 16, 16, 200) == 1 and f(0, 1, 1, 5) == 1 and f(1, 1, 1, 0) == 1


def test_packed_splits():
    f = _lib().melgpt_packed_attn_splits
    assert f(1500, 16001, 1, 32, 128, F32) == 1 and f(100, 100, 1, 16, 64, HALF) == 1 and f(30000, 30000, 1, 32, 128, HALF) == 1
    assert f(1, 16000, 1, 32, 128, HALF) > 4 and 1 < f(1500, 16001, 1, 32, 128, HALF) <= 16 and f(0, 5, 1, 1, 64, HALF) == 1


def test_packed_bwd_splits():
    f = _lib().melgpt_packed_attn_bwd_splits
    assert f(4000, 1, 8, 8, HALF) == f(4000, 1, 8, 1, F32) == f(0, 1, 8, 1, HALF) == f(100000, 1, 8, 1, HALF) == 1
    assert f(4000, 1, 8, 1, HALF) == 8 and f(200, 3, 7, 1, HALF) == 7 and 1 < f(4000, 1, 32, 2, HALF) < 16


def test_cpu_tensors_and_wrong_arguments_are_refused():
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd._ffi import MelgptError
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    q = torch.zeros(4, 2, 64)
    i = torch.zeros(4, dtype=torch.int32)
    f = pk.rotary_freqs(64, device="cpu")
    pages = torch.zeros(2, 2, 16, 64)
    for call in (lambda: pk.qk_norm_rotary(q, q, i, f), lambda: pk.packed_attention(q, q, q, i[:2]),
                 lambda: pk.packed_attention(q.requires_grad_(True), q, q, i[:2]),
                 lambda: ops.kv_append(q, q, pages, pages, i.view(1, 4), i, i),
                 lambda: ops.paged_attn_decode(q, pages, pages, i.view(4, 1), i),
                 lambda: ops.qk_norm_rotary_bwd(q, q, q, q, i, f), lambda: ops.packed_attn_bwd(q, q, q, q, q, q, i[:2])):
        with pytest.raises(MelgptError):
            call()


def test_result_buffers_that_overlap_are_refused():
    from melspec_gpt_vqvae_amd.ops import _into

    x = torch.zeros(6, 4, 64)
    fused = torch.zeros(6, 3, 4, 64)
    good = [torch.empty(6, 4, 64), fused[:, 1], torch.empty(4, 6, 64).transpose(0, 1), torch.empty(6, 4, 96)[..., 16:80]]
    for y in good:
        _into(y, x, x, fused)
    _into(torch.empty(0, 4, 64), torch.empty(0, 4, 64), torch.empty(0, 4, 64))
    _into(torch.zeros(1, 1, 64).expand(1, 1, 64), torch.zeros(1, 1, 64))
    bad = [x, torch.empty(1, 4, 64).expand(6, 4, 64), torch.empty(6, 1, 64).expand(6, 4, 64), torch.empty(6, 4, 128)[..., ::2],
           torch.empty(6, 64, 4).transpose(1, 2), torch.empty(6, 4, 32), torch.empty(6, 4, 64, dtype=torch.float64),
           torch.empty(4000).as_strided((6, 4, 64), (128, 64, 1)), torch.empty(4000).as_strided((6, 4, 64), (64, 128, 1))]
    for y in bad:
        with pytest.raises(AssertionError):
            _into(y, x, x)


def test_rotary_freqs():
    from melspec_gpt_vqvae_amd.transformer.packed import rotary_freqs

    f = rotary_freqs(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 1, 17, 31):
        assert abs(float(f[i]) - 10000.0 ** (-2 * i / 64)) <= 1e-15 * float(f[i]) * 8
    assert torch.allclose(rotary_freqs(64, stretch=4.0, device="cpu"), f / 4, rtol=1e-15, atol=0)
    g = rotary_freqs(64, base_stretch=8.0, device="cpu")
    assert abs(float(g[0]) - 1) < 1e-15 and abs(float(g[-1]) * 8 / float(f[-1]) - 1) < 1e-12    # fastest kept, slowest by 8
    r = rotary_freqs(64, stretch=4.0, ramp=(4096, 1, 32), device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(r[turns >= 32], f[turns >= 32]) and torch.allclose(r[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (r[mid] < f[mid]).all() and (r[mid] > f[mid] / 4).all()
    with pytest.raises(AssertionError):
        rotary_freqs(63, device="cpu")
