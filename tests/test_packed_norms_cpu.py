"""The bound of packed_norms on the CPU: it holds for the kernels' roundings and no longer for small mistakes beside them."""
import pytest
import torch

import packed_norms as N
import packed_ref as R


def rounded(lens_q, lens_k, q, k, v, do, scale, dtype):
    """gradients and output with the kernels' roundings, all else in 64 bits"""
    to = lambda x: x.to(dtype).double()
    Hq, Hk = q.shape[1], k.shape[1]
    out = [torch.zeros(x.shape, dtype=torch.float64) for x in (q, k, v, q)]
    a0 = b0 = 0
    for nq, nk in zip(lens_q, lens_k):
        a, b = slice(a0, a0 + nq), slice(b0, b0 + nk)
        a0, b0 = a0 + nq, b0 + nk
        for h in range(Hq):
            hk = h // (Hq // Hk)
            qq, kk, vv, gg = q[a, h].double(), k[b, hk].double(), v[b, hk].double(), do[a, h].double()
            p = R.attention(qq, kk, vv, scale)["p"]
            pr = to(p)
            o = torch.cat((p[:, :64], pr[:, 64:]), 1) @ vv
            ds = to(p * (gg @ vv.t() - (gg * o).sum(-1, keepdim=True)))
            out[0][a, h] = scale * ds @ kk
            out[1][b, hk] += scale * ds.t() @ qq
            out[2][b, hk] += pr.t() @ gg
            out[3][a, h] = pr @ vv
    return [to(x) for x in out]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(N.CASES)))
def test_bound_holds_for_roundings_and_not_for_mistakes(case, dtype):
    lq, lk, Hq, Hk, D = N.CASES[case]
    x = N.inputs(lq, lk, Hq, Hk, D, dtype, case)
    scale = D ** -0.5
    want = N.results(*x, lq, lk, scale, dtype)
    got = dict(zip(("dq", "dk", "dv", "o"), rounded(lq, lk, *x, scale, dtype)))
    for n in want:
        g, bounds = want[n]
        N.assert_near(got[n], g, bounds, n)
        # at most four half steps of the gradient: five too many everywhere do not pass (two hundredths in bf16)
        for rows, bound in bounds:
            assert bound <= 4 * R.half_step(dtype) * float(g[rows].norm())
        wrong = got[n] * (1 + 5 * R.half_step(dtype))
        with pytest.raises(AssertionError):
            N.assert_near(wrong, g, bounds, n)
        for rows, bound in bounds:                                 # one head of a sequence lost
            lost = got[n].clone()
            lost[rows, 0] = 0
            with pytest.raises(AssertionError):
                N.assert_near(lost, g, [(rows, bound)], n)
