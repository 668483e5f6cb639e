"""Attention of single tokens over a paged cache (melgpt_paged_attn_decode) against its definition in 64 bits, and the whole
run of the packed-sequence operators as a model uses them."""
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


def make(lens, Hq, Hk, D, page, dtype, seed, std=1.0, extra_width=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 2
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1) + extra_width), -7, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    kp = torch.randn(P, Hk, page, D, generator=g).to(dtype)
    vp = torch.randn(P, Hk, page, D, generator=g).to(dtype)
    q = (torch.randn(len(lens), Hq, D, generator=g) * std).to(dtype)
    return q, kp, vp, table


def rows_of(pages, table, s, n, h):
    page = pages.shape[2]
    j = torch.arange(n)
    return pages[table[s].long()[j // page], h, j % page]


def compare(out, lse, q, kp, vp, table, lens, scale, dtype, visible=None):
    D, Hq, Hk = q.shape[2], q.shape[1], kp.shape[1]
    h2, tiny = R.half_step(dtype), R.smallest(dtype)
    for s, n in enumerate(lens):
        for h in range(Hq):
            k, v = rows_of(kp, table, s, n, h // (Hq // Hk)), rows_of(vp, table, s, n, h // (Hq // Hk))
            if visible is not None:
                k, v = k[visible[s]], v[visible[s]]
            r = R.attention(q[s, h][None], k, v, scale, sees=torch.ones(1, k.shape[0], dtype=torch.bool))
            rel = R.attention_relative(D, r["s_score"], n + 300, dtype)[:, None]      # (the joins add up to 4 + 128 parts)
            R.assert_within(out[s, h][None], r["o"], h2 * r["o"].abs() + rel * r["s_o"] + tiny * (1 + r["a_o"]), f"out {s} {h}")
            bound = (D + 4) * R.U * r["s_score"] + (n + 300) * R.U + 4 * R.U * r["lse"].abs().nan_to_num(posinf=0)
            R.assert_within(lse[s, h][None], r["lse"], bound, f"lse {s} {h}")


def check(lens, Hq, Hk, D, page, dtype, seed=0, scale=None, std=1.0, max_length=None, extra_width=0):
    from melspec_gpt_vqvae_amd import ops

    q, kp, vp, table = make(lens, Hq, Hk, D, page, dtype, seed, std, extra_width)
    out, lse = ops.paged_attn_decode(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                     scale=scale, max_length=max_length)
    assert out.dtype == dtype
    compare(out.cpu(), lse.cpu(), q, kp, vp, table, lens, D ** -0.5 if scale is None else scale, dtype)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,page", [([1], 16), ([265], 16), ([0, 1, 31, 32, 33, 127, 128, 129, 0, 500], 16), ([513, 3], 1),
                                       ([700, 64, 65], 64), ([3000, 2999], 256), ([40, 7], 4)])
def test_lengths(lens, page, D, dtype):
    check(lens, 4, 2, D, page, _dt(dtype), seed=len(lens))


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (16, 16), (7, 1), (16, 1), (17, 1), (40, 2), (32, 8)])
def test_heads(Hq, Hk, dtype):
    check([100, 37, 300], Hq, Hk, 64, 32, _dt(dtype), seed=3)


def test_split_lengths_and_scales():
    check([9000], 8, 2, 128, 16, _half(), seed=1)
    check([9000, 1, 200], 2, 2, 64, 16, torch.float32, seed=1, scale=0.5, std=2.0)
    check([100, 50], 4, 2, 64, 16, _half(), seed=2, extra_width=600)              # a wide table, short sequences: empty splits
    check([100, 2050], 4, 2, 64, 16, _half(), seed=2, max_length=64)              # a wrong hint changes the split alone
    check([50], 2, 2, 64, 16, torch.float32, scale=-0.125)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 64), (7, 1, 128), (17, 1, 64), (40, 2, 64), (8, 8, 128)])
def test_split_heads(Hq, Hk, D, dtype):
    """few pairs: shares of 128 keys, sequences that fill some, one or none of the splits, shares that end inside a page"""
    check([300, 0, 128, 129, 1, 1100, 256], Hq, Hk, D, 32, _dt(dtype), seed=3, extra_width=100)


@pytest.mark.parametrize("dtype", ["f32", "half"])
def test_split_many_sequences(dtype):
    """256 pairs of sequence and key head or more: shares of 512 keys"""
    lens = [0, 1, 511, 512, 513, 1025, 2100] + [7 * i % 90 for i in range(60)]
    check(lens, 4, 4, 64, 16, _dt(dtype), seed=4)
    check(lens, 8, 4, 128, 64, _dt(dtype), seed=5)


def test_no_sequences_strides_and_given_out():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    lens = [70, 33]
    q, kp, vp, table = make(lens, 4, 2, 64, 16, dt, 5)
    args = [kp.to(DEV), vp.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)]
    base, lse = ops.paged_attn_decode(q.to(DEV), *args)
    wide = torch.zeros(2, 8, 64, dtype=dt, device=DEV)
    wide[:, ::2] = q.to(DEV)
    got, _ = ops.paged_attn_decode(wide[:, ::2], *args)
    assert torch.equal(got, base)
    room = torch.full((3, 4, 64), 9.0, dtype=dt, device=DEV)
    got, _ = ops.paged_attn_decode(q.to(DEV), *args, out=room[:2])
    assert torch.equal(room[:2], base) and (room[2] == 9).all()
    tab = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)
    tab[:, :table.shape[1]] = table.to(DEV)
    got, _ = ops.paged_attn_decode(q.to(DEV), args[0], args[1], tab[:, :table.shape[1]], args[3])
    assert torch.equal(got, base)
    o, l = ops.paged_attn_decode(q[:0].to(DEV), args[0], args[1], args[2][:0], args[3][:0])
    assert o.shape == (0, 4, 64) and l.shape == (0, 4)


def test_pages_outside_and_what_lies_behind_a_sequence():
    """keys of pages outside the cache are left out; NaN and infinities in the unused slots of the last page reach nothing"""
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    lens = [100, 45, 60]
    q, kp, vp, table = make(lens, 4, 2, 64, 16, dt, 5)
    for s, n in enumerate(lens):
        if n % 16:
            pg = int(table[s, n // 16])
            kp[pg, :, n % 16:] = float("nan")
            vp[pg, :, n % 16:] = float("inf")
    table[0, 2], table[0, 4] = -1, kp.shape[0]                                     # keys 32..47 and 64..79
    table[2, :] = 2 ** 31 - 1                                                      # no page at all
    out, lse = ops.paged_attn_decode(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), torch.tensor(lens + [], dtype=torch.int32, device=DEV))
    j = torch.arange(100)
    vis = [~(((j >= 32) & (j < 48)) | ((j >= 64) & (j < 80))), torch.ones(45, dtype=torch.bool), torch.zeros(60, dtype=torch.bool)]
    safe = table.clone()
    safe[0, 2] = safe[0, 4] = 0
    safe[2, :] = 0
    compare(out.cpu(), lse.cpu(), q, kp, vp, safe, lens, 0.125, dt, vis)
    assert float(out[2].abs().max()) == 0.0 and torch.isinf(lse[2]).all()
    # lengths beyond the table or below zero
    l2 = torch.tensor([10 ** 6, -4, 45], dtype=torch.int32, device=DEV)
    t2 = table[1:2].repeat(3, 1).to(DEV)
    kp[~torch.isfinite(kp)] = 0
    vp[~torch.isfinite(vp)] = 0
    o2, _ = ops.paged_attn_decode(q[1:2].repeat(3, 1, 1).to(DEV), kp.to(DEV), vp.to(DEV), t2, l2)
    assert float(o2[1].abs().max()) == 0.0 and torch.isfinite(o2.float()).all()


def test_cache_larger_than_two_to_the_32_bytes():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    P = 70000                                                                      # 70000 * 2 * 256 * 64 * 2 bytes = 4.6 GB each
    kp = torch.zeros(P, 2, 256, 64, dtype=dt, device=DEV)
    vp = torch.zeros(P, 2, 256, 64, dtype=dt, device=DEV)
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[P - 1, 3, P - 5]], dtype=torch.int32)
    k, v = torch.randn(700, 2, 64, generator=g).to(dt), torch.randn(700, 2, 64, generator=g).to(dt)
    ops.kv_append(k.to(DEV), v.to(DEV), kp, vp, table.to(DEV), torch.zeros(700, dtype=torch.int32, device=DEV),
                  torch.arange(700, dtype=torch.int32, device=DEV))
    assert torch.equal(kp[P - 1, :, 5].cpu(), k[5]) and torch.equal(vp[P - 5, :, 699 - 512].cpu(), v[699])
    q = torch.randn(1, 4, 64, generator=g).to(dt)
    out, lse = ops.paged_attn_decode(q.to(DEV), kp, vp, table.to(DEV), torch.tensor([700], dtype=torch.int32, device=DEV))
    r = [R.attention(q[0, h][None], k[:, h // 2], v[:, h // 2], 0.125, sees=torch.ones(1, 700, dtype=torch.bool)) for h in range(4)]
    for h in range(4):
        rel = R.attention_relative(64, r[h]["s_score"], 1000, dt)[:, None]
        R.assert_within(out[0, h][None], r[h]["o"], R.half_step(dt) * r[h]["o"].abs() + rel * r[h]["s_o"] + R.smallest(dt) * (1 + r[h]["a_o"]))


def test_captured_graphs_do_not_share_scratch():
    from melspec_gpt_vqvae_amd import ops

    dt = _half()
    lens = [3000, 100]
    q, kp, vp, table = [x.to(DEV) for x in make([3100, 3100], 8, 2, 64, 16, dt, 5)]
    length = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q2 = -q

    def capture(x):
        ops.paged_attn_decode(x, kp, vp, table, length)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.paged_attn_decode(x, kp, vp, table, length)
        return g, r

    (g1, r1), (g2, r2) = capture(q), capture(q2)
    s = torch.cuda.Stream()
    for i in range(4):
        length[0] = 3000 - 700 * i
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        for r, x in ((r1, q), (r2, q2)):
            want = ops.paged_attn_decode(x, kp, vp, table, length)
            assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])


@pytest.mark.parametrize("dtype", ["f32", "half"])
def test_prompt_then_tokens(dtype):
    """A layer's life: prompts of different lengths normed, rotated, attended and stored; then token by token over the cache.
    Every token's output is the row that packed attention over the whole sequence gives."""
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention, qk_norm_rotary, rotary_freqs

    dt = _dt(dtype)
    Hq, Hk, D, page, more = 8, 2, 64, 16, 5
    lens = [33, 1, 70]
    total = [n + more for n in lens]
    g = torch.Generator().manual_seed(7)
    q, k, v = [torch.randn(sum(total), H, D, generator=g).to(dt).to(DEV) for H in (Hq, Hk, Hk)]
    wq, wk = [(1 + 0.2 * torch.randn(D, generator=g)).to(DEV) for _ in range(2)]
    f = rotary_freqs(D, device=DEV)
    cu_all = torch.tensor([0] + total).cumsum(0)
    pos_all = torch.cat([torch.arange(n) for n in total]).to(torch.int32).to(DEV)
    qr, kr = qk_norm_rotary(q, k, pos_all, f, q_weight=wq, k_weight=wk)
    whole = packed_attention(qr, kr, v, cu_all.to(torch.int32).to(DEV))
    # prompts
    rows = torch.cat([torch.arange(cu_all[s], cu_all[s] + n) for s, n in enumerate(lens)]).to(DEV)
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(lens)]).to(torch.int32).to(DEV)
    table = torch.randperm(3 * 6, generator=g).view(3, 6).to(torch.int32).to(DEV)
    kp, vp = [torch.zeros(18, Hk, page, D, dtype=dt, device=DEV) for _ in range(2)]
    qp = ops.kv_append(k[rows], v[rows], kp, vp, table, seq, pos_all[rows], q=q[rows], freqs=f, q_weight=wq, k_weight=wk)
    assert torch.equal(qp, qr[rows])
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    assert torch.equal(packed_attention(qp, kr[rows], v[rows], cu), whole[rows])
    # tokens
    every = torch.arange(3, dtype=torch.int32, device=DEV)
    for i in range(more):
        at = torch.tensor([int(cu_all[s]) + n + i for s, n in enumerate(lens)], device=DEV)
        length = torch.tensor([n + i for n in lens], dtype=torch.int32, device=DEV)
        qt = ops.kv_append(k[at], v[at], kp, vp, table, every, length, q=q[at], freqs=f, q_weight=wq, k_weight=wk)
        out, _ = ops.paged_attn_decode(qt, kp, vp, table, length + 1)
        # both sides within their bounds of the same definition: |p| <= 1, values below 5
        tol = 2 * (R.half_step(dt) * 5 + 2 * R.half_step(dt) * 5 + 1e-5)
        assert float((out.float() - whole[at].float()).abs().max()) <= tol
        for s in range(3):
            r = R.attention(qr[at[s], 0][None].cpu(), kr[cu_all[s]:at[s] + 1, 0].cpu(), v[cu_all[s]:at[s] + 1, 0].cpu(), D ** -0.5)
            rel = R.attention_relative(D, r["s_score"], 400, dt)[:, None]
            R.assert_within(out[s, 0][None], r["o"], R.half_step(dt) * r["o"].abs() + rel * r["s_o"] + R.smallest(dt) * (1 + r["a_o"]))
