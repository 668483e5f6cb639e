"""Per-head norm and rotation of queries and keys (melgpt_qk_norm_rotary_*) and the paged append (melgpt_kv_append) against
their definitions in 64 bits."""
import pytest
import torch

import packed_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _half():
    from melspec_gpt_vqvae_amd import _ffi

    return _ffi.HALF_DTYPE


def _dt(name):
    return torch.float32 if name == "f32" else _half()


def _freqs(rot, base=10000.0):
    from melspec_gpt_vqvae_amd.transformer.packed import rotary_freqs

    return rotary_freqs(rot, base, device=DEV) if rot else None


def _inputs(M, Hq, Hk, D, dtype, seed, norm=True):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(M, (Hq + 2 * Hk) * D, generator=g) * 3 - 0.5).to(dtype).to(DEV)
    q = qkv[:, :Hq * D].unflatten(1, (Hq, D))
    k = qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    v = qkv[:, (Hq + Hk) * D:].unflatten(1, (Hk, D))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g)).to(DEV), (1 + 0.3 * torch.randn(D, generator=g)).to(DEV)
    return q, k, v, (wq if norm else None), (wk if norm else None), g


def check_forward(M, Hq, Hk, D, rot, interleaved, dtype, norm=True, first=0, amplitude=1.0, seed=0):
    from melspec_gpt_vqvae_amd import ops

    q, k, _, wq, wk, _ = _inputs(M, Hq, Hk, D, dtype, seed, norm)
    pos = (first + 17 * torch.arange(M)).to(torch.int32).to(DEV)
    f = _freqs(rot)
    got = ops.qk_norm_rotary_fwd(q, k, pos, f, q_weight=wq, k_weight=wk, eps=1e-6, interleaved=interleaved, amplitude=amplitude)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        assert y.dtype == dtype and y.is_contiguous()
        x, w, fc = x.double().cpu(), None if w is None else w.cpu(), None if f is None else f.cpu()
        n = R.norm_rotary(x, w, pos.cpu(), None, 1e-6, interleaved, 1.0)
        want = R.rotate(n, pos.cpu(), fc, interleaved, amplitude)
        R.assert_within(y, want, R.rotary_bound(n, want, dtype, fc, interleaved, amplitude), "forward")


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,Hq,Hk,D,rot", [(1, 1, 1, 16, 16), (1, 16, 16, 64, 64), (3, 7, 1, 80, 32), (65, 32, 8, 128, 128),
                                           (5, 5, 5, 96, 48), (2, 3, 2, 256, 256), (7, 1, 1, 240, 16), (4, 4, 2, 32, 0),
                                           (9001, 2, 1, 64, 64)])
def test_forward(M, Hq, Hk, D, rot, interleaved, dtype):
    check_forward(M, Hq, Hk, D, rot, interleaved, _dt(dtype))


@pytest.mark.parametrize("dtype", ["f32", "half"])
def test_forward_without_norm_far_positions_and_amplitude(dtype):
    check_forward(33, 8, 2, 64, 64, False, _dt(dtype), norm=False)
    check_forward(3, 8, 2, 128, 64, True, _dt(dtype), first=2 ** 31 - 100)
    check_forward(3, 8, 2, 128, 64, False, _dt(dtype), first=-50)
    check_forward(9, 4, 4, 64, 32, False, _dt(dtype), amplitude=1.25)


def test_forward_rows_of_zeros_infinities_and_strides():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    q = torch.randn(4, 3, 64, device=DEV).to(dt)
    q[1] = 0
    q[2, 0, 5] = float("inf")
    w = torch.ones(64, device=DEV)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    f = _freqs(64)
    base, _ = ops.qk_norm_rotary_fwd(q, q, pos, f, q_weight=w, k_weight=w)
    assert float(base[1].abs().max()) == 0.0                                    # eps keeps a row of zeros at zero
    assert not torch.isfinite(base[2, 0].float()).all() and torch.isfinite(base[2, 1:].float()).all()
    assert torch.isfinite(base[3].float()).all()
    # heads outermost, an unaligned view and a broadcast head give the same bits
    ht = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(4 * 3 * 64 + 1, dtype=dt, device=DEV)[1:].view(4, 3, 64)
    odd.copy_(q)
    for z in (ht, odd):
        got, _ = ops.qk_norm_rotary_fwd(z, z, pos, f, q_weight=w, k_weight=w)
        assert torch.equal(got.view(torch.int16), base.view(torch.int16))
    one = q[:, :1].expand(4, 3, 64)
    got, _ = ops.qk_norm_rotary_fwd(one, q, pos, f, q_weight=w, k_weight=w)
    assert torch.equal(got[:, 2].contiguous().view(torch.int16), base[:, 0].contiguous().view(torch.int16))


def test_no_rows():
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import qk_norm_rotary

    q = torch.zeros(0, 4, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    pos = torch.zeros(0, dtype=torch.int32, device=DEV)
    a, b = qk_norm_rotary(q, q, pos, _freqs(64), q_weight=w, k_weight=w)
    gq, gw = torch.autograd.grad((a, b), (q, w), (torch.zeros_like(a), torch.zeros_like(b)))
    assert a.shape == (0, 4, 64) and gq.shape == (0, 4, 64) and float(gw.abs().max()) == 0.0


def check_backward(M, Hq, Hk, D, rot, interleaved, dtype, norm=True, amplitude=1.0, seed=3):
    from melspec_gpt_vqvae_amd.transformer.packed import qk_norm_rotary

    q, k, _, wq, wk, g = _inputs(M, Hq, Hk, D, dtype, seed, norm)
    pos = (5 + torch.arange(M)).to(torch.int32).to(DEV)
    f = _freqs(rot)
    dq = torch.randn(M, Hq, D, generator=g).to(dtype).to(DEV)
    dk = torch.randn(Hk, M, D, generator=g).to(dtype).to(DEV).transpose(0, 1)          # heads outermost
    leaves = [t_.detach().requires_grad_(True) for t_ in ((q, k, wq, wk) if norm else (q, k))]
    out = qk_norm_rotary(leaves[0], leaves[1], pos, f, q_weight=leaves[2] if norm else None, k_weight=leaves[3] if norm else None,
                         interleaved=interleaved, amplitude=amplitude)
    got = torch.autograd.grad(out, leaves, (dq, dk))
    fc = None if f is None else f.cpu()
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        x, dy = x.double().cpu(), dy.double().cpu()
        u = R.rotate(dy, pos.cpu(), fc, interleaved, amplitude, inverse=True)
        pair = R.pair_size(dy, fc, interleaved, abs(amplitude))
        if not norm:
            R.assert_within(got[i], u, R.half_step(dtype) * u.abs() + 32 * R.U * pair, "dx")
            continue
        w = w.double().cpu()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xh = x * r
        m = (u * w * xh).mean(-1, keepdim=True)
        want = r * (u * w - xh * m)
        # u carries 32 u of its pair, x^ and w u another 16; the mean sums D such terms (21 u more of their sizes)
        size = r * (pair * w.abs() + xh.abs() * (pair * w.abs() * xh.abs()).mean(-1, keepdim=True))
        R.assert_within(got[i], want, R.half_step(dtype) * want.abs() + 96 * R.U * size, "dx")
        # a lane adds ceil(rows of its wave) * steps terms in sequence, a workgroup <= 256 lane sums, then <= 1024 / 16 + 16 rows
        terms = (u * xh)
        depth = 48 + (M // 4096 + 1) * 64 + 256 + 80
        R.assert_within(got[2 + i], terms.sum((0, 1)), depth * R.U * (pair * xh.abs()).sum((0, 1)), "dw")


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,Hq,Hk,D,rot", [(1, 1, 1, 16, 16), (3, 7, 1, 80, 32), (65, 32, 8, 128, 128), (2, 3, 2, 256, 256),
                                           (4, 4, 2, 32, 0), (9001, 2, 1, 64, 32)])
def test_backward(M, Hq, Hk, D, rot, interleaved, dtype):
    check_backward(M, Hq, Hk, D, rot, interleaved, _dt(dtype))


def test_backward_without_norm_and_reproducible():
    from melspec_gpt_vqvae_amd import ops

    check_backward(37, 4, 2, 64, 64, False, _half(), norm=False)
    check_backward(37, 4, 2, 64, 32, True, torch.float32, norm=False, amplitude=0.5)
    q, k, _, wq, wk, _ = _inputs(5000, 8, 2, 64, _half(), 9)
    pos = torch.arange(5000, dtype=torch.int32, device=DEV)
    first = ops.qk_norm_rotary_bwd(q, k, q, k, pos, _freqs(64), q_weight=wq, k_weight=wk)
    for _ in range(3):
        again = ops.qk_norm_rotary_bwd(q, k, q, k, pos, _freqs(64), q_weight=wq, k_weight=wk)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradient_against_differences():
    """central differences of the 64-bit definition along random directions"""
    from melspec_gpt_vqvae_amd.transformer.packed import qk_norm_rotary

    q, k, _, wq, wk, g = _inputs(6, 4, 2, 64, torch.float32, 21)
    pos = torch.tensor([0, 1, 5, 100, 4095, 70000], dtype=torch.int32, device=DEV)
    f = _freqs(32)
    dq, dk = torch.randn(6, 4, 64, generator=g).to(DEV), torch.randn(6, 2, 64, generator=g).to(DEV)
    leaves = [t_.detach().requires_grad_(True) for t_ in (q, k, wq, wk)]
    out = qk_norm_rotary(leaves[0], leaves[1], pos, f, q_weight=leaves[2], k_weight=leaves[3], interleaved=True)
    got = torch.autograd.grad(out, leaves, (dq, dk))

    def value(x):
        y = [R.norm_rotary(a, w, pos.cpu(), f.cpu(), 1e-6, True, 1.0) for a, w in ((x[0], x[2]), (x[1], x[3]))]
        return float((y[0] * dq.double().cpu()).sum() + (y[1] * dk.double().cpu()).sum())

    base = [t_.detach().double().cpu() for t_ in leaves]
    for i in range(4):
        d = torch.randn(base[i].shape, generator=g).double()
        e = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + e * d, base[i] - e * d
        slope = (value(up) - value(down)) / (2 * e)
        mine = float((got[i].double().cpu() * d).sum())
        # the difference's own error is O(e^2); the gradients' f32 error is below 400 u of the sum of sizes (see above)
        size = float((got[i].double().cpu().abs() * d.abs()).sum())
        assert abs(mine - slope) <= 1e-6 * size, (i, mine, slope, size)


# ------------------------------------------------------------------------------------------------------------- append
def check_append(dtype, Hq, Hk, D, rot, interleaved, norm, page, new, old, with_q=True, seed=1):
    from melspec_gpt_vqvae_amd import ops

    M = sum(new)
    q, k, v, wq, wk, g = _inputs(M, Hq, Hk, D, dtype, seed, norm)
    need = [max(1, -(-(a + b) // page)) for a, b in zip(new, old)]
    P = sum(need) + 2
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(new)]).to(torch.int32)
    pos = torch.cat([torch.arange(o, o + n) for n, o in zip(new, old)]).to(torch.int32)
    kp = torch.randn(P, Hk, page, D, generator=g).to(dtype)
    vp = torch.randn(P, Hk, page, D, generator=g).to(dtype)
    f = _freqs(rot)
    kd, vd = kp.to(DEV), vp.to(DEV)
    qo = ops.kv_append(k, v, kd, vd, table.to(DEV), seq.to(DEV), pos.to(DEV), q=q if with_q else None, freqs=f,
                       q_weight=wq if with_q else None, k_weight=wk, interleaved=interleaved)
    # the same rotation and norm as the operator without a cache, bit for bit; the rest of the cache as it was
    ref_q, ref_k = ops.qk_norm_rotary_fwd(q, k, pos.to(DEV), f, q_weight=wq, k_weight=wk, interleaved=interleaved)
    if with_q:
        assert torch.equal(qo, ref_q)
    else:
        assert qo is None
    for r in range(M):
        pg, slot = int(table[seq[r], pos[r] // page]), int(pos[r]) % page
        kp[pg, :, slot], vp[pg, :, slot] = ref_k[r].cpu(), v[r].cpu()
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("Hq,Hk,D,rot,interleaved,norm,page,new,old", [
    (32, 8, 128, 128, False, True, 16, [1] * 9, [0, 1, 15, 16, 17, 31, 32, 250, 1000]),
    (16, 4, 64, 32, True, False, 64, [70, 1, 129, 3], [0, 100, 63, 64]),
    (3, 1, 80, 16, False, True, 1, [5, 2], [0, 3]),
    (2, 2, 256, 256, True, True, 8, [17], [7]),
    (7, 7, 32, 0, False, False, 128, [1, 300], [127, 0])])
def test_append(dtype, Hq, Hk, D, rot, interleaved, norm, page, new, old):
    check_append(_dt(dtype), Hq, Hk, D, rot, interleaved, norm, page, new, old)


def test_append_without_queries():
    check_append(_half(), 4, 2, 64, 64, False, True, 16, [20, 1], [0, 40], with_q=False)


def test_append_skips_padding_and_pages_outside():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    q, k, v, _, _, _ = _inputs(8, 4, 2, 64, dt, 4, norm=False)
    kp, vp = torch.full((3, 2, 16, 64), 7.0, dtype=dt, device=DEV), torch.full((3, 2, 16, 64), 7.0, dtype=dt, device=DEV)
    table = torch.tensor([[2, 3], [-1, 0]], dtype=torch.int32, device=DEV)      # page 3 and page -1 do not exist
    seq = torch.tensor([0, 0, 1, 1, -1, 0, 2, 0], dtype=torch.int32, device=DEV)
    pos = torch.tensor([4, 16, 4, 31, 4, -1, 4, 32], dtype=torch.int32, device=DEV)   # rows 0 and 3 have a slot
    f = _freqs(64)
    qo = ops.kv_append(k, v, kp, vp, table, seq, pos, q=q, freqs=f)
    want_k, want_v = torch.full_like(kp, 7.0), torch.full_like(vp, 7.0)
    rq, rk = ops.qk_norm_rotary_fwd(q, k, pos, f)
    want_k[2, :, 4], want_v[2, :, 4] = rk[0], v[0]
    want_k[0, :, 15], want_v[0, :, 15] = rk[3], v[3]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    pad = torch.tensor([4, 5], device=DEV)                                      # negative sequence, negative position
    rq[pad] = 0
    assert torch.equal(qo, rq)
    given = torch.full_like(qo, 3.0)
    ops.kv_append(k, v, kp, vp, table, seq, pos, q=q, freqs=f, q_out=given)
    rq[pad] = 3.0
    assert torch.equal(given, rq)


def test_captured_and_replayed_append():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    q, k, v, wq, wk, _ = _inputs(4, 4, 2, 64, dt, 6)
    kp, vp = torch.zeros(8, 2, 16, 64, dtype=dt, device=DEV), torch.zeros(8, 2, 16, 64, dtype=dt, device=DEV)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(4, 2)
    seq, pos = torch.arange(4, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    f = _freqs(64)

    def step():
        return ops.kv_append(k, v, kp, vp, table, seq, pos, q=q, freqs=f, q_weight=wq, k_weight=wk)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        pos.fill_(3 * i + 1)
        g.replay()
        ref_q, ref_k = ops.qk_norm_rotary_fwd(q, k, pos, f, q_weight=wq, k_weight=wk)
        assert torch.equal(out, ref_q)
        assert torch.equal(kp[0, :, 3 * i + 1], ref_k[0]) and torch.equal(vp[6, :, 3 * i + 1], v[3])


def test_captured_forward_and_backward_and_two_streams():
    """a captured pass replayed with new inputs, and the same pass on two streams side by side: the eager bits every time"""
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import rotary_freqs

    M, Hq, Hk, D = 700, 8, 2, 64
    g = torch.Generator().manual_seed(11)
    q, k, dq, dk = [torch.randn(M, h, D, generator=g).to(_half()).to(DEV) for h in (Hq, Hk, Hq, Hk)]
    w = [torch.rand(D, generator=g).to(DEV) + 0.5 for _ in range(2)]
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    f = rotary_freqs(D, device=DEV)

    def run():
        kw = dict(q_weight=w[0], k_weight=w[1])
        return ops.qk_norm_rotary_fwd(q, k, pos, f, **kw) + ops.qk_norm_rotary_bwd(dq, dk, q, k, pos, f, **kw)

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(run())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(3):
        q.mul_(0.5)
        pos.add_(100000)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


# few heads and many rows: a wave takes several rows at once (the last one fewer than it could)
FEW_HEADS = [(4097, 1, 1, 128, 128), (8203, 2, 1, 80, 32), (16385, 1, 1, 32, 16), (4099, 16, 16, 32, 32), (4096, 1, 1, 256, 64),
             (8195, 3, 3, 16, 16)]


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,Hq,Hk,D,rot", FEW_HEADS)
def test_few_heads_many_rows(M, Hq, Hk, D, rot, interleaved, dtype):
    check_forward(M, Hq, Hk, D, rot, interleaved, _dt(dtype), norm=not interleaved or D != 80)
    check_backward(M, Hq, Hk, D, rot, interleaved, _dt(dtype), norm=not interleaved or D != 80)


@pytest.mark.parametrize("dtype", ["f32", "half"])
def test_append_few_heads_many_rows(dtype):
    check_append(_dt(dtype), 1, 1, 64, 64, False, True, 16, [4000, 1, 300], [0, 100, 7])
    check_append(_dt(dtype), 2, 1, 128, 32, True, True, 64, [8300], [3])
    check_append(_dt(dtype), 1, 1, 80, 32, True, False, 32, [5000, 77], [1, 0], with_q=False)


@pytest.mark.parametrize("dtype", ["f32", "half"])
def test_append_few_heads_padding_among_rows(dtype):
    """padding and rows that point outside, in the same wave as rows that do not"""
    from melspec_gpt_vqvae_amd import ops

    dt, M, D, page = _dt(dtype), 9000, 64, 16
    g = torch.Generator().manual_seed(2)
    q, k, v = [torch.randn(M, 1, D, generator=g).to(dt).to(DEV) for _ in range(3)]
    P = -(-M // page)
    kp, vp = [torch.randn(P, 1, page, D, generator=g).to(dt).to(DEV) for _ in range(2)]
    table = torch.randperm(P, generator=g).to(torch.int32).view(1, P).to(DEV)
    pos = torch.arange(M, dtype=torch.int32)
    seq = torch.zeros(M, dtype=torch.int32)
    pos[::7], seq[3::11], seq[5::13] = -1, -2, 9                     # padding, padding, no such sequence
    pad = (pos < 0) | (seq < 0)
    stored = ~pad & (seq == 0)
    full_q, full_k = ops.qk_norm_rotary_fwd(q, k, pos.to(DEV), _freqs(64))
    q_out = torch.full_like(q, 3.0)
    want_k, want_v = kp.clone(), vp.clone()
    at = pos[stored].long().to(DEV)
    want_k[table[0].long()[at // page], 0, at % page] = full_k[stored.to(DEV), 0]
    want_v[table[0].long()[at // page], 0, at % page] = v[stored.to(DEV), 0]
    k1, v1 = kp.clone(), vp.clone()
    ops.kv_append(k, v, k1, v1, table, seq.to(DEV), pos.to(DEV), q=q, freqs=_freqs(64), q_out=q_out)
    assert torch.equal(k1, want_k) and torch.equal(v1, want_v)
    p = pad.to(DEV)
    assert torch.equal(q_out[~p], full_q[~p]) and (q_out[p] == 3.0).all()
    new = ops.kv_append(k, v, kp, vp, table, seq.to(DEV), pos.to(DEV), q=q, freqs=_freqs(64))
    assert torch.equal(new[~p], full_q[~p]) and (new[p] == 0).all()
