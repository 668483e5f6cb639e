"""The 16-bit output and gradients of packed attention as norms, against what their roundings allow (packed_norms)."""
import pytest
import torch

import packed_norms as N

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(lens_q, lens_k, Hq, Hk, D, dtype, seed):
    from melspec_gpt_vqvae_amd.transformer.packed import packed_attention

    x = N.inputs(lens_q, lens_k, Hq, Hk, D, dtype, seed)
    cu = [torch.tensor([0] + l).cumsum(0).to(torch.int32).to(DEV) for l in (lens_q, lens_k)]
    leaves = [t.to(DEV).requires_grad_(True) for t in x[:3]]
    out = packed_attention(*leaves, *cu)
    got = torch.autograd.grad(out, leaves, x[3].to(DEV))
    want = N.results(*x, lens_q, lens_k, D ** -0.5, dtype)
    plain = packed_attention(*[t.detach() for t in leaves], *cu)    # (keys shared by workgroups where rows are few)
    for n, g in zip(("dq", "dk", "dv", "o", "o"), got + (out, plain)):
        N.assert_near(g, *want[n], n)


@pytest.mark.parametrize("case", range(len(N.CASES)))
def test_gradients(case):
    from melspec_gpt_vqvae_amd import _ffi

    check(*N.CASES[case], _ffi.HALF_DTYPE, case)
