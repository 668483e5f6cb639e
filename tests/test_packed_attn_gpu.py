"""Causal attention over packed sequences (melgpt_packed_attn_*) against its definition in 64 bits."""
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


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def make(lens_q, lens_k, Hq, Hk, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(lens_q), Hq, D, generator=g) * std).to(dtype)
    kv = torch.randn(sum(lens_k), 2, Hk, D, generator=g).to(dtype)
    do = torch.randn(sum(lens_q), Hq, D, generator=g).to(dtype)
    return q, kv[:, 0], kv[:, 1], do


def reference(q, k, v, lens_q, lens_k, scale, do=None):
    """per (sequence, query head) results of packed_ref.attention"""
    Hq, Hk = q.shape[1], k.shape[1]
    cq, ck = _cu(lens_q).tolist(), _cu(lens_k).tolist()
    for s in range(len(lens_q)):
        a, b = slice(cq[s], cq[s + 1]), slice(ck[s], ck[s + 1])
        for h in range(Hq):
            yield a, b, h, h // (Hq // Hk), R.attention(q[a, h], k[b, h // (Hq // Hk)], v[b, h // (Hq // Hk)], scale,
                                                        None if do is None else do[a, h])


def check(lens_q, lens_k, Hq, Hk, D, dtype, backward=True, seed=0, scale=None, std=1.0):
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention

    q, k, v, do = make(lens_q, lens_k, Hq, Hk, D, dtype, seed, std)
    sc = D ** -0.5 if scale is None else scale
    leaves = [x.to(DEV).requires_grad_(backward) for x in (q, k, v)]
    cu_q = _cu(lens_q).to(DEV)
    cu_k = None if lens_k == lens_q else _cu(lens_k).to(DEV)
    out = packed_attention(*leaves, cu_q, cu_k, scale=scale)
    _, lse = ops.packed_attn_fwd(*[x.detach() for x in leaves], cu_q, cu_k, scale=scale)
    assert out.dtype == dtype and out.shape == q.shape
    if backward:
        dq, dk, dv = torch.autograd.grad(out, leaves, do.to(DEV))
        want_dk, want_dv = torch.zeros(k.shape).double(), torch.zeros(v.shape).double()
        tol_dk, tol_dv = torch.zeros(k.shape).double(), torch.zeros(v.shape).double()
    h2, tiny = R.half_step(dtype), R.smallest(dtype)
    for a, b, h, hk, r in reference(q, k, v, lens_q, lens_k, sc, do if backward else None):
        n = b.stop - b.start
        rel = R.attention_relative(D, r["s_score"], n, dtype)[:, None]
        what = f"rows {a.start}.. head {h}"
        R.assert_within(out[a, h], r["o"], h2 * r["o"].abs() + rel * r["s_o"] + tiny * (1 + r["a_o"]), "out " + what)
        R.assert_within(lse[h, a], r["lse"], (D + 4) * R.U * r["s_score"] + (n + 4) * R.U + 4 * R.U * r["lse"].abs().nan_to_num(posinf=0), "lse " + what)
        if backward:
            # delta is formed with the stored output (h |o| more), the scores against the stored log-sum (its error, as above):
            # twice the forward's relative error, and once more h for ds and p
            rel = 3 * rel + 8 * R.U + 2 * R.U * r["lse"].abs().nan_to_num(posinf=0)[:, None]
            R.assert_within(dq[a, h], r["dq"], h2 * r["dq"].abs() + _max(rel) * r["s_dq"] + tiny * (1 + r["a_dq"]), "dq " + what)
            want_dk[b, hk] += r["dk"]
            want_dv[b, hk] += r["dv"]
            m = _max(rel) + (a.stop - a.start) * (Hq // Hk) * R.U
            tol_dk[b, hk] += m * r["s_dk"] + tiny * (1 + r["a_dk"])
            tol_dv[b, hk] += m * r["s_dv"] + tiny * (1 + r["a_dv"])
    if backward:
        R.assert_within(dk, want_dk, h2 * want_dk.abs() + tol_dk, "dk")
        R.assert_within(dv, want_dv, h2 * want_dv.abs() + tol_dv, "dv")


def _max(x):
    return float(x.max()) if x.numel() else 0.0


LENS = [([1], [1]), ([266], [266]), ([64, 1, 63, 65, 31, 32, 33, 128], None), ([5, 300, 129], [40, 301, 129]), ([1, 1, 1], [513, 7, 64]),
        ([70, 33, 3], [10, 0, 3]), ([0, 40, 0, 0, 17], [5, 40, 0, 3, 17]), ([129], [1000])]


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", range(len(LENS)))
def test_lengths(lens, D, dtype):
    lq, lk = LENS[lens]
    check(lq, lk or lq, 4, 2, D, _dt(dtype), seed=lens)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (16, 16), (7, 1), (24, 8), (32, 2)])
def test_heads(Hq, Hk, dtype):
    check([100, 37], [100, 37], Hq, Hk, 64, _dt(dtype), seed=5)


def test_scale_and_large_scores():
    check([130], [130], 2, 1, 64, _half(), scale=0.5, std=4.0)
    check([130], [130], 2, 1, 128, torch.float32, scale=1.0, std=3.0)
    check([50], [50], 2, 2, 64, torch.float32, scale=-0.125)
    check([150, 20], [170, 20], 4, 2, 128, _half(), scale=-0.125)
    for dt in (torch.float32, _half()):                            # every visible key alike
        check([70, 3], [70, 5], 2, 1, 64, dt, scale=0.0)


def test_few_queries_over_many_keys():
    """the keys of a row tile shared by several workgroups"""
    from melspec_gpt_vqvae_amd import _ffi, ops

    split = _ffi.lib().melgpt_packed_attn_splits
    for lq, lk, Hq, Hk, D in (([3], [3000], 4, 2, 64), ([130], [1500], 2, 1, 128), ([1, 20, 5], [700, 2000, 3], 4, 1, 128), ([40, 0, 200], [2900, 7, 180], 2, 2, 64)):
        assert split(sum(lq), sum(lk), len(lq), Hq, D, _ffi.BF16) > 1
        check(lq, lk, Hq, Hk, D, _half(), backward=False, seed=4)
        check(lq, lk, Hq, Hk, D, _half(), seed=4)                  # (with gradients: in one piece)
    # rows of nobody, in a new and a given output
    q, k, v, _ = [x.to(DEV) for x in make([30], [2100], 4, 2, 64, _half(), 4)]
    cu_q = torch.tensor([4, 20], dtype=torch.int32, device=DEV)
    cu_k = torch.tensor([50, 2080], dtype=torch.int32, device=DEV)
    assert split(30, 2100, 1, 4, 64, _ffi.BF16) > 1
    out, lse = ops.packed_attn_fwd(q, k, v, cu_q, cu_k)
    given = torch.full_like(out, 5.0)
    ops.packed_attn_fwd(q, k, v, cu_q, cu_k, out=given)
    assert torch.equal(given[4:20], out[4:20]) and (given[:4] == 5).all() and (given[20:] == 5).all()
    assert (out[:4] == 0).all() and (out[20:] == 0).all() and torch.isinf(lse[:, 20:]).all()
    want, _, _ = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, want_low=True)
    assert float((want.float() - out.float()).abs().max()) <= 4 * R.half_step(_half()) * float(want.float().abs().max())


def test_many_short_sequences():
    lens = [(7 * i) % 5 for i in range(5000)]                     # more sequences than one 64-way step of the search covers
    check(lens[:300], lens[:300], 2, 1, 64, _half(), seed=2)
    from melspec_gpt_vqvae_amd import ops

    q, k, v, _ = make(lens, lens, 2, 1, 64, _half(), 3)
    out, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens).to(DEV))
    first = _cu(lens)[:-1].long()[torch.tensor(lens) > 0]         # the first query of a sequence sees its own key alone
    assert torch.equal(out.cpu()[first], v[first].expand(-1, 2, -1))


def test_rows_behind_the_last_sequence():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    q, k, v, do = [x.to(DEV) for x in make([200], [200], 4, 2, 64, dt, 4)]
    q, k, v, do = q.clone(), k.clone(), v.clone(), do.clone()
    cu = torch.tensor([10, 50, 131], dtype=torch.int32, device=DEV)             # rows 0..9 and 131..199 belong to nobody
    for x in (q, k, v, do):
        x[:10] = float("nan")
        x[131:] = float("nan")
    out, lse = ops.packed_attn_fwd(q, k, v, cu)
    grads = ops.packed_attn_bwd(q, k, v, out, do, lse, cu)
    base, _ = ops.packed_attn_fwd(q[10:131], k[10:131], v[10:131], cu - 10)
    assert torch.equal(out[10:131], base)
    for x in (out,) + grads:
        assert float(x[:10].abs().max()) == 0.0 and float(x[131:].abs().max()) == 0.0
        assert torch.isfinite(x.float()).all()
    assert torch.isinf(lse[:, 131:]).all()
    given = torch.full_like(out, 5.0)
    left = [torch.full_like(g, 5.0) for g in grads]
    ops.packed_attn_fwd(q, k, v, cu, out=given)
    ops.packed_attn_bwd(q, k, v, given, do, lse, cu, grads=left)
    for x, y in zip((given, *left), (out, *grads)):
        assert torch.equal(x[10:131], y[10:131])
        assert (x[:10] == 5).all() and (x[131:] == 5).all()


def test_offsets_out_of_range_stay_inside():
    from melspec_gpt_vqvae_amd import ops

    q, k, v, do = [x.to(DEV) for x in make([100], [100], 2, 1, 64, _half(), 4)]
    for cu in ([0, 60, 4000], [-5, 60, 100], [0, 80, 20, 100], [100, 50, 0], [0, 0, 0]):
        cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        out, lse = ops.packed_attn_fwd(q, k, v, cu)
        ops.packed_attn_bwd(q, k, v, out, do, lse, cu)
    cu = torch.tensor([0, 60, 4000], dtype=torch.int32, device=DEV)             # the last offset stands for the end
    good = torch.tensor([0, 60, 100], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.packed_attn_fwd(q, k, v, cu)[0], ops.packed_attn_fwd(q, k, v, good)[0])


def test_strides_broadcast_and_no_rows():
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention

    dt = _half()
    q, k, v, do = [x.to(DEV) for x in make([77, 20], [77, 20], 4, 2, 64, dt, 8)]
    cu = _cu([77, 20]).to(DEV)
    base, lse = ops.packed_attn_fwd(q, k, v, cu)
    heads_out = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(97 * 4 * 64 + 1, dtype=dt, device=DEV)[1:].view(97, 4, 64)
    odd.copy_(q)
    assert torch.equal(ops.packed_attn_fwd(heads_out(q), heads_out(k), heads_out(v), cu)[0], base)
    assert torch.equal(ops.packed_attn_fwd(odd, k, v, cu)[0], base)
    g0 = ops.packed_attn_bwd(q, k, v, base, do, lse, cu)
    block = torch.empty(97, 8 * 64, dtype=dt, device=DEV)          # q | k | v gradients side by side
    views = (block[:, :256].unflatten(1, (4, 64)), block[:, 256:384].unflatten(1, (2, 64)), block[:, 384:].unflatten(1, (2, 64)))
    ops.packed_attn_bwd(heads_out(q), heads_out(k), v, heads_out(base), heads_out(do), lse, cu, grads=views)
    assert all(torch.equal(a, b) for a, b in zip(g0, views))
    # one key head broadcast to two by the caller: its gradient is the sum of both
    k1, v1 = k[:, :1].clone().requires_grad_(True), v[:, :1].clone().requires_grad_(True)
    out = packed_attention(q, k1.expand(-1, 2, -1), v1.expand(-1, 2, -1), cu)
    gk, gv = torch.autograd.grad(out, (k1, v1), do)
    out2 = packed_attention(q, k1, v1, cu)
    assert torch.equal(out, out2)
    hk, hv = torch.autograd.grad(out2, (k1, v1), do)
    # two halves each rounded, then their rounded sum, against one rounding
    for a, b in ((gk, hk), (gv, hv)):
        assert float((a.float() - b.float()).abs().max()) <= 4 * R.half_step(dt) * float(b.float().abs().max())
    none = torch.zeros(0, 4, 64, dtype=dt, device=DEV)
    assert packed_attention(none, none[:, :2], none[:, :2], _cu([0, 0]).to(DEV)).shape == (0, 4, 64)
    o, l = ops.packed_attn_fwd(q, none[:, :2], none[:, :2], cu, _cu([0, 0]).to(DEV))
    assert float(o.abs().max()) == 0.0 and torch.isinf(l).all()
    dq, dk, dv = ops.packed_attn_bwd(q, none[:, :2], none[:, :2], o, do, l, cu, _cu([0, 0]).to(DEV))
    assert float(dq.abs().max()) == 0.0 and dk.shape == (0, 2, 64)


def test_gradient_against_differences_and_reproducible():
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention

    lens = [40, 1, 75]
    q, k, v, do = make(lens, lens, 4, 2, 64, torch.float32, 12)
    cu = _cu(lens).to(DEV)
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, cu), leaves, do.to(DEV))
    for _ in range(3):
        again = torch.autograd.grad(packed_attention(*leaves, cu), leaves, do.to(DEV))
        assert all(torch.equal(a, b) for a, b in zip(grads, again))

    def value(x):
        return sum(float((r["o"] * do[a, h].double()).sum()) for a, b, h, hk, r in reference(*x, lens, lens, 0.125))

    g = torch.Generator().manual_seed(1)
    base = [x.double() for x in (q, k, v)]
    for i in range(3):
        d = torch.randn(base[i].shape, generator=g).double()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        slope = (value(up) - value(down)) / 2e-5
        mine = float((grads[i].double().cpu() * d).sum())
        size = float((grads[i].double().cpu().abs() * d.abs()).sum())
        assert abs(mine - slope) <= 1e-5 * size, (i, mine, slope, size)   # f32 gradients: D u s_score ~ 128 * 6e-8 relative


def test_captured_and_replayed():
    """forward and backward in a graph, replayed with new inputs and new lengths; other work between the replays"""
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    q, k, v, do = [x.to(DEV).clone() for x in make([150], [150], 4, 2, 128, dt, 1)]
    cu = torch.tensor([0, 70, 150], dtype=torch.int32, device=DEV)

    def step():
        out, lse = ops.packed_attn_fwd(q, k, v, cu)
        return (out, lse) + ops.packed_attn_bwd(q, k, v, out, do, lse, cu)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        q.mul_(0.9)
        v.add_(0.1 * i)
        cu[1] = 1 + 40 * i
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once():
    """forward and backward on two streams side by side, over and over, against the same calls one after the other"""
    from melspec_gpt_vqvae_amd import ops

    a = [x.to(DEV) for x in make([900, 40], [900, 40], 4, 2, 128, _half(), 1)]
    b = [x.to(DEV) for x in make([20], [3000], 8, 2, 128, _half(), 2)]
    cu_a, cu_q, cu_k = _cu([900, 40]).to(DEV), _cu([20]).to(DEV), _cu([3000]).to(DEV)

    def first():
        out, lse = ops.packed_attn_fwd(*a[:3], cu_a)
        return (out, lse) + ops.packed_attn_bwd(*a[:3], out, a[3], lse, cu_a)

    def other():
        out, lse = ops.packed_attn_fwd(*b[:3], cu_q, cu_k)         # (keys shared by several workgroups)
        return (out, lse) + ops.packed_attn_bwd(*b[:3], out, b[3], lse, cu_q, cu_k)

    want_a, want_b = first(), other()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            x = first()
        with torch.cuda.stream(streams[1]):
            y = other()
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert all(torch.equal(p, q) for p, q in zip(x, want_a)) and all(torch.equal(p, q) for p, q in zip(y, want_b))


def test_backward_through_a_broadcast_sum_and_one_input():
    """a gradient that is one value expanded, and inputs of which only one wants a gradient"""
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention

    q, k, v, _ = [x.to(DEV) for x in make([90], [90], 4, 2, 64, _half(), 3)]
    cu = _cu([90]).to(DEV)
    v = v.detach().clone().requires_grad_(True)
    packed_attention(q, k, v, cu).sum().backward()
    one = v.grad.clone()
    v.grad = None
    packed_attention(q, k, v, cu).backward(torch.ones_like(q))
    assert torch.equal(v.grad, one) and q.grad is None
    # every query hands out a total weight of 1: the values' gradients of a column add up to the queries (rounded once each,
    # probabilities to the tensors' type before)
    total = v.grad.double().sum((0, 1))
    assert float((total - 4 * 90).abs().max()) <= 4 * 90 * 2 * R.half_step(_half())


@pytest.mark.parametrize("D", [64, 128])
def test_output_in_two_halves(D):
    """out + low of sequences of up to 64 keys: probabilities and output in two 16-bit halves each (what the first half left
    out rounded once more: h^2 of the sum of sizes and of the output), f32 otherwise"""
    from melspec_gpt_vqvae_amd import ops

    dt, lens, scale = _half(), [1, 2, 3, 4, 7, 33, 64, 64, 50], D ** -0.5
    q, k, v, _ = make(lens, lens, 4, 2, D, dt, 8)
    out, _, low = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens).to(DEV), want_low=True)
    plain, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens).to(DEV))
    both, tiny = out.double().cpu() + low.double().cpu(), R.smallest(dt)
    h = R.half_step(dt)
    for a, b, head, _, r in reference(q, k, v, lens, lens, scale):
        rel = R.attention_relative(D, r["s_score"], b.stop - b.start, torch.float32)[:, None] + h * h
        R.assert_within(both[a, head], r["o"], (h * h + 4 * R.U) * r["o"].abs() + rel * r["s_o"] + tiny * (2 + r["a_o"]), f"{a} {head}")
    assert (out - plain).abs().max() <= 4 * h * v.abs().max()       # (two roundings of probabilities, two of the output)


@pytest.mark.parametrize("Hq,Hk,D", [(7, 1, 64), (8, 2, 128), (5, 1, 128)])
def test_backward_with_few_key_heads(Hq, Hk, D):
    """query heads of a key head shared out over workgroups; rows no sequence owns; a given buffer with strides"""
    from melspec_gpt_vqvae_amd import _ffi, ops

    lens_q, lens_k = [130, 1, 64, 0, 20], [150, 3, 64, 70, 10]
    check(lens_q, lens_k, Hq, Hk, D, _half(), seed=9)
    assert _ffi.lib().melgpt_packed_attn_bwd_splits(sum(lens_k), len(lens_k), Hq, Hk, 1) > 1
    q, k, v, do = [x.to(DEV) for x in make(lens_q + [9], lens_k + [33], Hq, Hk, D, _half(), 9)]
    cu_q, cu_k = _cu(lens_q).to(DEV), _cu(lens_k).to(DEV)            # 9 and 33 rows behind the last sequence
    for x, n in ((q, 9), (k, 33), (v, 33), (do, 9)):
        x[-n:] = float("nan")
    out, lse = ops.packed_attn_fwd(q, k, v, cu_q, cu_k)
    new = ops.packed_attn_bwd(q, k, v, out, do, lse, cu_q, cu_k)
    room = torch.full((k.shape[0], 2, Hk, D), 3.0, dtype=q.dtype, device=DEV)
    given = ops.packed_attn_bwd(q, k, v, out, do, lse, cu_q, cu_k, grads=(torch.empty_like(q), room[:, 0], room[:, 1]))
    for a, b in zip(new[1:], given[1:]):
        assert torch.isfinite(a).all() and torch.equal(a[:-33], b[:-33]) and (a[-33:] == 0).all() and (b[-33:] == 3.0).all()


def test_rows_far_apart():
    """rows whose offsets pass 2^32 bytes: the same bits as from tensors side by side"""
    from melspec_gpt_vqvae_amd import ops

    D, M, far = 64, 2500, 1 << 20                                   # (2500 rows of 2^20 values: 5.2 GB)
    cu = _cu([1100, 1400]).to(DEV)
    near = [x.to(DEV) for x in make([1100, 1400], [1100, 1400], 2, 1, D, _half(), 7)]
    room = torch.empty(M * far, dtype=_half(), device=DEV).view(M, far)
    q, k, v, dout, out, dq, dk, dv = [room[:, 128 * i:128 * i + D * h].view(M, h, D) for i, h in enumerate((2, 1, 1, 2, 2, 2, 1, 1))]
    for x, y in zip((q, k, v, dout), near):
        x.copy_(y)
    want, lse = ops.packed_attn_fwd(*near[:3], cu)
    got, lse_far = ops.packed_attn_fwd(q, k, v, cu, out=out)
    assert torch.equal(got, want) and torch.equal(lse, lse_far)
    for a, b in zip(ops.packed_attn_bwd(q, k, v, out, dout, lse, cu, grads=(dq, dk, dv)),
                    ops.packed_attn_bwd(*near[:3], want, near[3], lse, cu)):
        assert torch.equal(a, b)


def test_other_stream():
    from melspec_gpt_vqvae_amd import ops

    q, k, v, do = [x.to(DEV) for x in make([300], [300], 4, 2, 64, _half(), 1)]
    cu = _cu([300]).to(DEV)
    want = ops.packed_attn_fwd(q, k, v, cu)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, lse = ops.packed_attn_fwd(q, k, v, cu)
        grads = ops.packed_attn_bwd(q, k, v, got, do, lse, cu)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and all(torch.isfinite(x.float()).all() for x in grads)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("n,D", [(200, 64), (200, 128), (130, 128)])
def test_values_that_are_not_finite_reach_only_the_queries_that_see_them(n, D, dtype):
    from melspec_gpt_vqvae_amd import ops

    dt = _dt(dtype)
    more = 40
    q, k, v, _ = make([n], [n + more], 4, 2, D, dt, 6)
    cu_q, cu_k = _cu([n]).to(DEV), _cu([n + more]).to(DEV)
    base, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k)
    bad_v, bad_k = v.clone(), k.clone()
    bad_v[more + 100, 0, 3] = float("nan")
    bad_v[more + 64, 1, D - 1] = float("inf")
    bad_v[more + 120, 1, 7] = float("-inf")
    out, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), bad_v.to(DEV), cu_q, cu_k)
    want = base.clone()
    want[100:, :2, 3] = float("nan")                     # key 40 + 100 is the last key of query 100
    want[64:, 2:, D - 1] = float("inf")
    want[120:, 2:, 7] = float("-inf")
    same = (out == want) | (torch.isnan(out) & torch.isnan(want))
    assert same.all(), torch.nonzero(~same)[:5]
    bad_k[more + 90, 0, 0] = float("nan")
    out, lse = ops.packed_attn_fwd(q.to(DEV), bad_k.to(DEV), v.to(DEV), cu_q, cu_k)
    assert torch.equal(out[:90], base[:90]) and torch.equal(out[:, 2:], base[:, 2:]) and torch.isnan(out[90:, :2]).all()
    assert torch.isnan(lse[:2, 90:]).all()
    # a value that is not finite in front of every border: all queries of its key head see it
    bad_v = v.clone()
    bad_v[0, 0, 5] = float("inf")
    out, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), bad_v.to(DEV), cu_q, cu_k)
    assert torch.isinf(out[:, :2, 5]).all() and torch.equal(out[:, 2:], base[:, 2:])
