"""How far the packed attention's 16-bit output and gradients may be from their definition, as norms (test infrastructure).

A rounding to 16 bits is off by at most half a step, h |x|, and evenly spread within it: its square is at most h^2 x^2 / 3 on
average, and roundings of different values are independent, so the squares of what they add to a gradient add up.  The kernels
round (everything else is f32, below h / 100)
  the gradient itself                                 h^2 / 3 |g|^2
  dq, dk: ds_ij in front of the product with k, q     h^2 / 3 scale^2 sum_ij ds_ij^2 |k_j|^2   (|q_i|^2)
          delta_i = do_i . o_i, through the forward's probabilities of keys 64 and on (out + low is f32 otherwise):
          var_i = h^2 / 3 sum_(j >= 64) p_ij^2 (do_i . v_j)^2, on ds_ij as p_ij delta_i:
                                                      scale^2 sum_i var_i |sum_j p_ij k_j|^2   (sum_ij var_i p_ij^2 |q_i|^2)
  dv:     p_ij in front of the product with do        h^2 / 3 sum_ij p_ij^2 |do_i|^2
  output: p_ij in front of the product with v         h^2 / 3 sum_ij p_ij^2 |v_j|^2
A result's error may be twice the root of its sum."""
import torch

import packed_ref as R


def squares(q, k, v, do, scale, dtype):
    """one head of one sequence -> (packed_ref.attention's results, expected squares of the errors of dq, dk, dv and the output
    without the last rounding's)"""
    r = R.attention(q, k, v, scale, do)
    q, k, v, do = q.double(), k.double(), v.double(), do.double()
    e, p = R.half_step(dtype) ** 2 / 3, r["p"]
    dp = do @ v.t()
    ds2 = (p * (dp - (do * r["o"]).sum(-1, keepdim=True))) ** 2
    var = e * (p[:, 64:] ** 2 * dp[:, 64:] ** 2).sum(-1)
    k2, q2 = (k * k).sum(-1), (q * q).sum(-1)
    s2 = scale * scale
    dq = s2 * (e * (ds2 @ k2).sum() + (var * ((p @ k) ** 2).sum(-1)).sum())
    dk = s2 * (e * (ds2.t() @ q2).sum() + (var * (p * p).sum(-1) * q2).sum())
    dv = e * ((p * p).t() @ (do * do).sum(-1)).sum()
    o = e * ((p * p) @ (v * v).sum(-1)).sum()
    return r, (float(dq), float(dk), float(dv), float(o))


def results(q, k, v, do, lens_q, lens_k, scale, dtype):
    """all heads and sequences -> {name: (result in 64 bits, [(rows, allowed norm of the error) of every sequence])}"""
    Hq, Hk = q.shape[1], k.shape[1]
    want = {n: torch.zeros(x.shape, dtype=torch.float64) for n, x in (("dq", q), ("dk", k), ("dv", v), ("o", q))}
    bounds = {n: [] for n in want}
    a0 = b0 = 0
    e = R.half_step(dtype) ** 2 / 3
    for nq, nk in zip(lens_q, lens_k):
        a, b = slice(a0, a0 + nq), slice(b0, b0 + nk)
        a0, b0 = a0 + nq, b0 + nk
        sums = [0.0] * 4
        for h in range(Hq):
            hk = h // (Hq // Hk)
            r, s = squares(q[a, h], k[b, hk], v[b, hk], do[a, h], scale, dtype)
            want["dq"][a, h] = r["dq"]
            want["dk"][b, hk] += r["dk"]
            want["dv"][b, hk] += r["dv"]
            want["o"][a, h] = r["o"]
            sums = [x + y for x, y in zip(sums, s)]
        for (n, rows), s in zip((("dq", a), ("dk", b), ("dv", b), ("o", a)), sums):
            bounds[n].append((rows, 2 * float(torch.sqrt(s + e * want[n][rows].square().sum()))))
    return {n: (want[n], bounds[n]) for n in want}


def assert_near(got, want, bounds, what=""):
    """the error of every sequence's gradient as a norm"""
    got = got.detach().double().cpu()
    for rows, bound in bounds:
        err = float((got[rows] - want[rows]).norm())
        assert err <= bound, f"{what} rows {rows.start}..{rows.stop}: error {err:.3e} of {float(want[rows].norm()):.3e}, allowed {bound:.3e}"


# (lens_q, lens_k, Hq, Hk, D)
CASES = [([4] * 24, [4] * 24, 4, 2, 64), ([4] * 24, [4] * 24, 4, 2, 128), ([266], [266], 4, 4, 64), ([266, 265], [266, 265], 4, 2, 128),
         ([2000], [2000], 2, 2, 64), ([2000], [2000], 2, 1, 128), ([150, 300], [700, 300], 7, 1, 64), ([150, 300], [700, 300], 8, 1, 128)]


def inputs(lens_q, lens_k, Hq, Hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lens_q), Hq, D, generator=g).to(dtype)
    k = torch.randn(sum(lens_k), Hk, D, generator=g).to(dtype)
    v = torch.randn(sum(lens_k), Hk, D, generator=g).to(dtype)
    do = torch.randn(sum(lens_q), Hq, D, generator=g).to(dtype)
    return q, k, v, do
