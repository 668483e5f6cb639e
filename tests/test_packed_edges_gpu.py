"""Packed and cached sequence operators at the edges of what their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _dt(name):
    from melspec_gpt_vqvae_amd import _ffi

    return torch.float32 if name == "f32" else _ffi.HALF_DTYPE


def _bits(x):
    """bits of a tensor, every NaN alike (its payload is the conversion's)"""
    x = torch.where(torch.isnan(x), torch.full_like(x, float("nan")), x).contiguous()
    return x.view(torch.int16 if x.element_size() == 2 else torch.int32)


# ------------------------------------------------------------------------------- values beyond the rotated part of a head
def _with_odd_values(M, H, D, rot, dtype, seed):
    """-> a finite tensor and the same with infinities, NaN and negative zeros scattered over the values beyond `rot`"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, H, D, generator=g)
    y = x.clone()
    where = torch.rand(M, H, D, generator=g) < 0.1
    where[..., :rot] = False
    where[0, 0, D - 1] = where[M - 1, H - 1, rot] = True
    odd = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0])
    y[where] = odd[torch.randint(0, 4, (int(where.sum()),), generator=g)]
    return x.to(dtype).to(DEV), y.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,Hq,Hk,D,rot", [(5, 3, 2, 64, 32), (5, 3, 2, 64, 0), (4, 2, 1, 128, 16), (3, 1, 1, 80, 48), (8200, 1, 1, 64, 32)])
def test_values_beyond_the_rotation_pass_unchanged(M, Hq, Hk, D, rot, interleaved, dtype):
    """without a norm: the bits of every value beyond `rot`, whatever lies beside it, and the rotated values as if the others
    were finite; forward, backward and on the way into a cache"""
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer.packed import rotary_freqs

    dt, page = _dt(dtype), 16
    f = rotary_freqs(rot, device=DEV) if rot else None
    pos = (3 + torch.arange(M, device=DEV)).to(torch.int32)
    (q, q_odd), (k, k_odd) = _with_odd_values(M, Hq, D, rot, dt, 1), _with_odd_values(M, Hk, D, rot, dt, 2)

    def right(got, x, finite):
        assert torch.equal(_bits(got[..., rot:]), _bits(x[..., rot:]))
        assert torch.equal(_bits(got[..., :rot]), _bits(finite[..., :rot]))

    base = ops.qk_norm_rotary_fwd(q, k, pos, f, interleaved=interleaved)
    got = ops.qk_norm_rotary_fwd(q_odd, k_odd, pos, f, interleaved=interleaved)
    for a, b, c in zip(got, (q_odd, k_odd), base):
        right(a, b, c)
    base_g = ops.qk_norm_rotary_bwd(q, k, q, k, pos, f, interleaved=interleaved)
    got_g = ops.qk_norm_rotary_bwd(q_odd, k_odd, q, k, pos, f, interleaved=interleaved)
    for a, b, c in zip(got_g[:2], (q_odd, k_odd), base_g):
        right(a, b, c)
    pages = -(-(M + 3) // page)
    kp, vp = [torch.zeros(pages, Hk, page, D, dtype=dt, device=DEV) for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    qo = ops.kv_append(k_odd, k_odd, kp, vp, table, torch.zeros(M, dtype=torch.int32, device=DEV), pos, q=q_odd, freqs=f,
                       interleaved=interleaved)
    right(qo, q_odd, base[0])
    p = pos.long()
    right(kp[p // page, :, p % page], k_odd, base[1])
    assert torch.equal(_bits(vp[p // page, :, p % page]), _bits(k_odd))


# --------------------------------------------------------------------------------------- rows that no sequence owns
def _poisoned(*shapes_and_types):
    """leaves freed blocks of these sizes, full of sevens, to the allocator"""
    keep = [torch.full(s, 7.0, dtype=t, device=DEV) for s, t in shapes_and_types for _ in range(3)]
    del keep
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("lens_q,lens_k", [([10, 50, 131], [10, 50, 131]), ([4, 20], [50, 2080])])   # (the second: keys shared)
def test_log_sums_of_rows_that_no_sequence_owns(lens_q, lens_k, dtype):
    """with a buffer for the output its rows of nobody stay as they were; the new tensors beside it are defined there too"""
    from melspec_gpt_vqvae_amd import ops

    dt, Mq, Mk = _dt(dtype), lens_q[-1] + 69, lens_k[-1] + 20
    g = torch.Generator().manual_seed(3)
    q = torch.randn(Mq, 4, 64, generator=g).to(dt).to(DEV)
    k, v = [torch.randn(Mk, 2, 64, generator=g).to(dt).to(DEV) for _ in range(2)]
    cu_q, cu_k = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens_q, lens_k)]
    mine = torch.zeros(Mq, dtype=torch.bool, device=DEV)
    mine[lens_q[0]:lens_q[-1]] = True
    for low in (False, True):
        want = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, want_low=low)
        out = torch.full_like(q, 5.0)
        _poisoned((want[1].shape, torch.float32), (q.shape, dt))
        got = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, out=out, want_low=low)
        assert got[0] is out and (out[~mine] == 5).all() and torch.equal(out[mine], want[0][mine])
        assert (got[1][:, ~mine] == -float("inf")).all() and torch.equal(got[1], want[1])
        if low and dt != torch.float32:
            assert (got[2][~mine] == 0).all() and torch.equal(got[2], want[2])


# ------------------------------------------------------------------------------------------ forward mode, traces
def test_forward_mode_is_refused_and_a_trace_replays():
    import torch.autograd.forward_ad as forward_ad
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    dt = _dt("half")
    g = torch.Generator().manual_seed(5)
    q, q2 = [torch.randn(30, 4, 64, generator=g).to(dt).to(DEV) for _ in range(2)]
    k, k2 = [torch.randn(30, 2, 64, generator=g).to(dt).to(DEV) for _ in range(2)]
    cu, pos = torch.tensor([0, 30], dtype=torch.int32, device=DEV), torch.arange(30, dtype=torch.int32, device=DEV)
    f = pk.rotary_freqs(64, device=DEV)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            pk.packed_attention(d, k, k, cu)
        with pytest.raises(NotImplementedError):
            pk.qk_norm_rotary(d, k, pos, f)
    layer = lambda a, b: pk.packed_attention(*pk.qk_norm_rotary(a, b, pos, f), b, cu)
    traced = torch.jit.trace(layer, (q, k), check_trace=False)
    # (a trace goes through the autograd functions, as a call with gradients does)
    a, b = q2.clone().requires_grad_(True), k2
    assert torch.equal(traced(q2, k2), layer(a, b).detach())


# --------------------------------------------------------------------------------------------------- results apart
def test_results_that_share_memory_with_inputs_are_refused():
    from melspec_gpt_vqvae_amd import ops

    dt, M = _dt("half"), 40
    room = torch.zeros(1 << 20, dtype=dt, device=DEV)
    rows = lambda at, H: room[at:at + M * H * 64].view(M, H, 64)
    q, k, v, do = rows(0, 4), rows(20000, 2), rows(30000, 2), rows(40000, 4)
    cu = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    fused = torch.zeros(M, 8, 64, dtype=dt, device=DEV)            # (side by side in rows: apart)
    out, lse = ops.packed_attn_fwd(fused[:, :4], fused[:, 4:6], fused[:, 6:], cu, out=rows(0, 4))
    for at in (64, 20000 - 64, 30000 + 128):
        with pytest.raises(AssertionError):
            ops.packed_attn_fwd(q, k, v, cu, out=rows(at, 4))
    out, lse = ops.packed_attn_fwd(q, k, v, cu)
    free = 100000
    ops.packed_attn_bwd(q, k, v, out, do, lse, cu, grads=(rows(free, 4), rows(free + 20000, 2), rows(free + 30000, 2)))
    for at in ((64, free, free + 10000), (free, 30000 - 64, free + 20000), (free, free + 20000, 40000 + 64), (free, free + 64, free + 20000),
               (free, free + 20000, free + 20000 + 64)):
        with pytest.raises(AssertionError):
            ops.packed_attn_bwd(q, k, v, out, do, lse, cu, grads=(rows(at[0], 4), rows(at[1], 2), rows(at[2], 2)))
    # the cache: pages as parts of one buffer
    page = lambda at: room[at:at + 8 * 2 * 16 * 64].view(8, 2, 16, 64)
    kp, vp = page(200000), page(300000)
    seq, pos = torch.zeros(M, dtype=torch.int32, device=DEV), torch.arange(M, dtype=torch.int32, device=DEV)
    table = torch.arange(8, dtype=torch.int32, device=DEV)[None]
    ops.kv_append(k, v, kp, vp, table, seq, pos, q=q, q_out=rows(free, 4))
    for at in (64, 20000 - 64, 30000 + 64, 200000 + 64, 300000 - 64):
        with pytest.raises(AssertionError):
            ops.kv_append(k, v, kp, vp, table, seq, pos, q=q, q_out=rows(at, 4))
    with pytest.raises(AssertionError):
        ops.kv_append(k, v, kp, page(200000 + 1024), table, seq, pos, q=q)
    lengths = torch.tensor([M], dtype=torch.int32, device=DEV)
    ops.paged_attn_decode(q[:1], kp, vp, table, lengths, out=rows(free, 4)[:1])
    for at in (64, 200000 + 64, 300000 + 16 * 64 * 4):
        with pytest.raises(AssertionError):
            ops.paged_attn_decode(q[:1], kp, vp, table, lengths, out=rows(at, 4)[:1])


def test_append_of_no_rows_with_a_given_buffer():
    from melspec_gpt_vqvae_amd import ops

    q = torch.zeros(0, 2, 64, device=DEV)
    pages = [torch.zeros(1, 2, 16, 64, device=DEV) for _ in range(2)]
    none, table = torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    room = torch.empty(0, 2, 64, device=DEV)
    assert ops.kv_append(q, q, *pages, table, none, none, q=q, q_out=room) is room


# ------------------------------------------------------------------------------------------------- rows far apart
@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("M", [1, 3])
def test_rows_more_than_2_24_values_apart(M, dtype):
    """views of one position of a (rows, positions, heads, D) buffer: the same bits as from tensors side by side"""
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer import packed as pk

    dt, D, far = _dt(dtype), 64, (1 << 24) + 64
    room = torch.zeros((M - 1) * far + 4096, dtype=dt, device=DEV)
    view = lambda H, at: room.as_strided((M, H, D), (far if M > 1 else 1 << 27, D, 1), at)
    g = torch.Generator().manual_seed(2)
    near = [torch.randn(M, H, D, generator=g).to(dt).to(DEV) for H in (4, 2, 2, 4)]
    q, k, v, do = [view(x.shape[1], 512 * i) for i, x in enumerate(near)]
    for x, y in zip((q, k, v, do), near):
        x.copy_(y)
    cu = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    out, lse = ops.packed_attn_fwd(*near[:3], cu)
    got, got_lse = ops.packed_attn_fwd(q, k, v, cu)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    given = view(4, 512 * 4)
    ops.packed_attn_fwd(q, k, v, cu, out=given)
    assert torch.equal(given, out)
    grads = ops.packed_attn_bwd(*near[:3], out, near[3], lse, cu)
    places = tuple(view(H, 512 * i) for H, i in ((4, 5), (2, 6), (2, 7)))
    for a, b, c in zip(ops.packed_attn_bwd(q, k, v, given, do, lse, cu), grads, ops.packed_attn_bwd(q, k, v, given, do, lse, cu, grads=places)):
        assert torch.equal(a, b) and torch.equal(c, b)
    # one far tensor among near ones, each in turn, through the differentiable form
    for i, x in enumerate((q, k, v)):
        leaves = [(x if j == i else y).detach().requires_grad_(True) for j, y in enumerate(near[:3])]
        o = pk.packed_attention(*leaves, cu)
        plain = [y.detach().requires_grad_(True) for y in near[:3]]
        o2 = pk.packed_attention(*plain, cu)
        assert torch.equal(o, o2)
        for a, b in zip(torch.autograd.grad(o, leaves, do), torch.autograd.grad(o2, plain, near[3])):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------- the output's two halves fit
@pytest.mark.parametrize("D", [64, 128])
def test_output_and_its_remainder_fit_each_other(D):
    """enough values (10 sequences of 64, 8 heads) that dozens of them lie on a tie of the 16-bit format"""
    import packed_ref as R
    from melspec_gpt_vqvae_amd import ops

    dt, n, H = _dt("half"), 64, 8
    g = torch.Generator().manual_seed(9)
    q, k, v = [torch.randn(10 * n, H, D, generator=g).to(dt) for _ in range(3)]
    cu = torch.arange(0, 10 * n + 1, n, dtype=torch.int32, device=DEV)
    out, _, low = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), cu, want_low=True)
    both, h = out.double().cpu() + low.double().cpu(), R.half_step(dt)
    for s in range(10):
        a = slice(n * s, n * s + n)
        for i in range(H):
            r = R.attention(q[a, i], k[a, i], v[a, i], D ** -0.5)
            # probabilities and output each in two halves: what the first left out is rounded once more
            rel = R.attention_relative(D, r["s_score"], n, torch.float32)[:, None] + h * h
            bound = (h * h + 4 * R.U) * r["o"].abs() + rel * r["s_o"] + R.smallest(dt) * (2 + r["a_o"])
            R.assert_within(both[a, i], r["o"], bound, f"sequence {s} head {i}")


# ------------------------------------------------------------------- a few long sequences in a large batch: decode
def _cached(lens, Hq, Hk, D, page, dtype, seed, width=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    need = [-(-n // page) for n in lens]
    kp, vp = [torch.randn(sum(need) + 1, Hk, page, D, generator=g, device=DEV).to(dtype) for _ in range(2)]
    order = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    table, at = torch.full((len(lens), max(max(need), width // page)), -1, dtype=torch.int32, device=DEV), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return torch.randn(len(lens), Hq, D, generator=g, device=DEV).to(dtype), kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _decode_reference(q, kp, vp, table, lens, which):
    """for the sequences of `which`: (output, log sum, sizes of the output's terms, of the scores) in 64 bits, elementwise products"""
    Hq, Hk, D, page = q.shape[1], kp.shape[1], q.shape[2], kp.shape[2]
    for s in which:
        j = torch.arange(lens[s], device=DEV)
        at = table[s].long()[j // page], j % page
        k, v = [x[at[0], :, at[1]].double().repeat_interleave(Hq // Hk, 1) for x in (kp, vp)]      # (keys, Hq, D)
        w = (k * q[s].double()).sum(-1) * D ** -0.5
        size = (k * q[s].double()).abs().sum(-1).amax(0) * D ** -0.5 if lens[s] else torch.zeros(Hq, device=DEV).double()
        lse = torch.logsumexp(w, 0) if lens[s] else torch.full((Hq,), -float("inf"), device=DEV).double()
        p = torch.exp(w - lse)[..., None]
        yield s, (p * v).sum(0), lse, (p * v.abs()).sum(0), size


def _check_decode(lens, Hq, Hk, D, page, dtype, seed, which=None, max_length=None, width=0):
    import packed_ref as R
    from melspec_gpt_vqvae_amd import ops

    args = _cached(lens, Hq, Hk, D, page, dtype, seed, width)
    out, lse = ops.paged_attn_decode(*args, max_length=max_length)
    h = R.half_step(dtype)
    for s, o, l, size, score in _decode_reference(*args[:4], lens, range(len(lens)) if which is None else which):
        n = lens[s]
        rel = R.attention_relative(D, score, n + 300, dtype)[:, None]
        R.assert_within(out[s], o, h * o.abs() + rel * size + R.smallest(dtype) * (1 + n * 5), f"out {s}")
        R.assert_within(lse[s], l, (D + 4) * R.U * score + (n + 300) * R.U + 4 * R.U * l.abs().nan_to_num(posinf=0), f"lse {s}")
    return args, out, lse


@pytest.mark.parametrize("dtype", ["f32", "half"])
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 64), (8, 8, 128)])
def test_long_sequences_in_a_large_batch_of_short_ones(Hq, Hk, D, dtype):
    from melspec_gpt_vqvae_amd import _ffi

    lens = [7 * i % 90 for i in range(300)]
    for s, n in ((0, 4097), (5, 9000), (64, 4096), (127, 18000), (299, 8193)):      # (first, last, at a wave's end, two in one wave)
        lens[s] = n
    assert _ffi.lib().melgpt_paged_attn_splits(300, Hq, Hk, 18000) == 5 and 300 * Hk >= 2048
    _check_decode(lens, Hq, Hk, D, 16, _dt(dtype), 1)
    _check_decode(lens, Hq, Hk, D, 16, _dt(dtype), 1, which=[0, 5, 127, 299], max_length=5000)      # (wrong hints: one share each,
    _check_decode(lens[:128] + [60000] + lens[129:], Hq, Hk, D, 16, _dt(dtype), 1, which=[5, 127, 128], max_length=17000)   # larger ones)


def test_more_long_shares_than_workgroups_that_look_for_them():
    lens = [4500 + i for i in range(130)]                          # 130 sequences of 16 heads, a second share each: 2080
    _check_decode(lens, 16, 16, 64, 64, _dt("half"), 2, which=[0, 1, 63, 64, 65, 100, 128, 129], max_length=20000, width=20000)


def test_long_sequences_with_two_groups_of_heads():
    lens = [50] * 70
    lens[3] = lens[69] = 5000
    _check_decode(lens, 17 * 16, 16, 64, 32, _dt("half"), 3, which=[0, 3, 68, 69], width=20000)


def test_captured_decode_of_growing_lengths():
    """one graph, lengths on either side of a share of 4096 keys from replay to replay"""
    from melspec_gpt_vqvae_amd import ops

    (q, kp, vp, table, lengths), _, _ = _check_decode([9000] * 3 + [100] * 300, 8, 8, 64, 64, _dt("half"), 4, which=[1, 200], width=20000)
    step = lambda: ops.paged_attn_decode(q, kp, vp, table, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for a, b, c in ((4096, 1, 0), (4097, 9000, 8192), (0, 0, 0), (8193, 64, 4160), (9000, 9000, 9000)):
        lengths[:3] = torch.tensor([a, b, c], dtype=torch.int32, device=DEV)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        for s, o, l, size, score in _decode_reference(q, kp, vp, table, lengths.tolist(), range(3)):
            # (half a bf16 step of values up to 5, the largest of these; the bits are held to the eager call's above)
            assert float((got[0][s].double() - o).abs().max()) <= 0.02 and (lengths[s] > 0 or torch.isinf(got[1][s]).all())


# ------------------------------------------------------ a few long sequences in a batch of short ones: packed forward
def _shares(lens_q, lens_k, Hq, D, max_length=None):
    """(usual, with room for long ones) as ops.packed_attn_fwd asks for them"""
    from melspec_gpt_vqvae_amd import _ffi

    a = (sum(lens_q), sum(lens_k), len(lens_q), Hq, D, _ffi.BF16)
    longest = max_length if max_length is not None else a[1] // 2 if a[1] > a[0] and len(lens_q) >= 32 else 0
    return _ffi.lib().melgpt_packed_attn_splits(*a), _ffi.lib().melgpt_packed_attn_splits_for(*a, longest)


def _packed_check(lens_q, lens_k, Hq, Hk, D, seed, max_length=None, ahead=0, behind=0):
    """against 64 bits, with rows of nobody in front and behind; a new and a given output"""
    import packed_ref as R
    import test_packed_attn_gpu as pa
    from melspec_gpt_vqvae_amd import ops

    dt = _dt("half")
    q, k, v, _ = pa.make([ahead] + lens_q + [behind], [ahead] + lens_k + [behind], Hq, Hk, D, dt, seed)
    for x in (q, k, v):
        x[:ahead] = float("nan")
        x[len(x) - behind:] = float("nan")
    cu_q, cu_k = [(torch.tensor([0] + l).cumsum(0) + ahead).to(torch.int32).to(DEV) for l in (lens_q, lens_k)]
    out, lse = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k, max_length=max_length)
    end = ahead + sum(lens_q)
    mine = slice(ahead, end)
    h, own = R.half_step(dt), [x[ahead:len(x) - behind] for x in (q, k, v)]
    o, l = out[mine].cpu(), lse[:, mine].cpu()
    for a, b, head, _, r in pa.reference(*own, lens_q, lens_k, D ** -0.5):
        n = b.stop - b.start
        rel = R.attention_relative(D, r["s_score"], n + 40, dt)[:, None]         # (the joins add up to 16 shares)
        R.assert_within(o[a, head], r["o"], h * r["o"].abs() + rel * r["s_o"] + R.smallest(dt) * (1 + r["a_o"]), f"out {a} head {head}")
        bound = (D + 4) * R.U * r["s_score"] + (n + 40) * R.U + 4 * R.U * r["lse"].abs().nan_to_num(posinf=0)
        R.assert_within(l[head, a], r["lse"], bound, f"lse {a} head {head}")
    for part in (slice(0, ahead), slice(end, end + behind)):
        assert (out[part] == 0).all() and (lse[:, part] == -float("inf")).all()
    given = torch.full_like(out, 5.0)
    _poisoned((lse.shape, torch.float32))
    _, lse2 = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k, max_length=max_length, out=given)
    assert torch.equal(given[mine], out[mine]) and torch.equal(lse2, lse) and (given[:ahead] == 5).all() and (given[end:] == 5).all()


@pytest.mark.parametrize("where", [0, 31, 69])
@pytest.mark.parametrize("D", [64, 128])
def test_one_long_sequence_in_a_packed_batch(D, where):
    lens_q, lens_k = [1 + i % 3 for i in range(70)], [1 + 7 * i % 90 for i in range(70)]
    lens_q[5], lens_k[6], lens_q[7] = 0, 0, 100                     # no queries; no keys; queries that see none
    lens_q[where], lens_k[where] = 128, 16001
    usual, room = _shares(lens_q, lens_k, 4, D)
    assert room > usual
    _packed_check(lens_q, lens_k, 4, 2, D, 5, ahead=3, behind=40)


def test_long_sequences_of_several_row_tiles_and_more_shares_than_workgroups_that_look_for_them():
    lens_q, lens_k = [3] * 66, [40] * 66
    for s, n, m in ((2, 300, 4000), (63, 1, 9000), (64, 140, 2300), (65, 129, 6001)):
        lens_q[s], lens_k[s] = n, m
    usual, room = _shares(lens_q, lens_k, 32, 64, 9000)
    assert room > usual
    _packed_check(lens_q, lens_k, 32, 8, 64, 6, max_length=9000)    # 32 heads x (3 + 1 + 2 + 2 row tiles) x up to 7 shares


def test_one_long_prompt_among_tokens():
    lens = [4001] + [1] * 63
    usual, room = _shares(lens, lens, 2, 128, 4001)
    assert usual == 1 < room and _shares(lens, lens, 2, 128) == (1, 1)
    _packed_check(lens, lens, 2, 1, 128, 7, max_length=4001, behind=5)
    _packed_check(lens, lens, 2, 1, 128, 7, max_length=100000)      # (a wrong hint decides the shares alone)


def test_captured_packed_batch_whose_long_sequence_changes():
    from melspec_gpt_vqvae_amd import ops
    import test_packed_attn_gpu as pa

    lens_q, lens_k = [2] * 70, [200] * 70
    q, k, v, _ = [x.to(DEV) for x in pa.make(lens_q, lens_k, 8, 2, 64, _dt("half"), 8)]
    cu_q, cu_k = pa._cu(lens_q).to(DEV), pa._cu(lens_k).to(DEV)
    usual, room = _shares(lens_q, lens_k, 8, 64, 14000)
    assert room > usual
    step = lambda: ops.packed_attn_fwd(q, k, v, cu_q, cu_k, max_length=14000)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    even = cu_k.clone()
    for first, last in ((0, 0), (13000, 0), (0, 13000), (5000, 8000)):
        cu_k.copy_(even)                                            # keys moved to the first or the last sequence
        cu_k[1:70] = torch.maximum(cu_k[1:70], torch.full_like(cu_k[1:70], first)).clamp(max=14000 - last)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        plain = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, max_length=0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # both round probabilities and output: two half steps each of the sizes (values up to 5 in few keys, weights that add to 1)
        assert float((got[0].float() - plain[0].float()).abs().max()) <= 4 * 5 * 2.0 ** -8
        assert torch.allclose(got[1], plain[1], rtol=0, atol=1e-4)


def test_values_that_are_not_finite_in_a_long_sequence_of_a_batch():
    from melspec_gpt_vqvae_amd import ops
    import test_packed_attn_gpu as pa

    lens_q, lens_k = [2] * 40 + [100], [20] * 40 + [16000]
    q, k, v, _ = pa.make(lens_q, lens_k, 4, 2, 128, _dt("half"), 9)
    cu_q, cu_k = pa._cu(lens_q).to(DEV), pa._cu(lens_k).to(DEV)
    usual, room = _shares(lens_q, lens_k, 4, 128)
    assert room > usual
    base, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k)
    bad = v.clone()
    bad[800 + 15900 + 60, 0, 3] = float("nan")                      # key 15960 of the long one: its queries 60 and on see it
    bad[800 + 15999, 1, 7] = float("inf")                           # its last query alone
    out, _ = ops.packed_attn_fwd(q.to(DEV), k.to(DEV), bad.to(DEV), cu_q, cu_k)
    want = base.clone()
    want[80 + 60:, :2, 3] = float("nan")
    want[80 + 99, 2:, 7] = float("inf")
    assert ((out == want) | (torch.isnan(out) & torch.isnan(want))).all()
