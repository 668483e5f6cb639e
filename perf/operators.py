"""The language-model operators beside the fixed-length GPT path, as workloads: what each case stands for, its inputs, one
pass through it, what that pass has to move and compute, and its value in 64 bits.

  qk_norm_rotary    RMS norm of every query and key head and the position rotation, one pass (forward, and with gradients)
  packed_attention  causal attention with grouped heads over packed sequences of different lengths (forward, and with gradients)
  kv_append         the same norm and rotation on the way into a paged key / value cache
  paged_decode      attention of one query token per sequence over that cache

`own` False: plain torch operations in 32 bits (64 for angles).  `own` True: the framework's operators."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
BASE = 10000.0


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(x)) for x in values)


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a small batch with the repository's 16 heads of 64: launch latency
        dict(name="norm_rotary_step", op="qk_norm_rotary", dtype="bf16", rows=4, heads_q=16, heads_k=16, dim=64, rot=64,
             interleaved=False, train=False, first=265),
        # a long prompt with grouped heads
        dict(name="norm_rotary_prompt", op="qk_norm_rotary", dtype="bf16", rows=16385, heads_q=32, heads_k=8, dim=128, rot=128,
             interleaved=False, train=False, first=0),
        # a training batch of the repository's size, 128 sequences of 265 codes; part of the head rotated, pairs side by side
        dict(name="norm_rotary_train", op="qk_norm_rotary", dtype="bf16", rows=33920, heads_q=16, heads_k=16, dim=64, rot=32,
             interleaved=True, train=True, first=0),
        # one sequence of the repository's block size, 32-bit lane
        dict(name="attention_one_f32", op="packed_attention", dtype="f32", heads_q=16, heads_k=16, dim=64, lens_q="266",
             lens_k="266", train=False),
        # prompts of different lengths prefilled together
        dict(name="attention_prompts", op="packed_attention", dtype="bf16", heads_q=32, heads_k=8, dim=128,
             lens_q="4097,1,257,1023,64,2048,777,3000", lens_k="4097,1,257,1023,64,2048,777,3000", train=False),
        # one long prompt continued: its last 1500 tokens against all the keys so far
        dict(name="attention_continued", op="packed_attention", dtype="bf16", heads_q=32, heads_k=8, dim=128, lens_q="1500",
             lens_k="16001", train=False),
        # a packed training batch with its backward pass
        dict(name="attention_train", op="packed_attention", dtype="bf16", heads_q=16, heads_k=4, dim=128,
             lens_q="4096,265,1999,1,800,2050", lens_k="4096,265,1999,1,800,2050", train=True),
        # a decode step of a full serving batch
        dict(name="append_step", op="kv_append", dtype="bf16", heads_q=32, heads_k=8, dim=128, rot=128, interleaved=False,
             norm=True, page=16, lens_new=_text([1] * 64), lens_old=_text([37 * i * i % 8000 for i in range(64)])),
        # whole prompts into the cache, no norm, heads partly rotated
        dict(name="append_prompts", op="kv_append", dtype="bf16", heads_q=16, heads_k=4, dim=64, rot=32, interleaved=True,
             norm=False, page=64, lens_new="8191,1,4000,333,2065", lens_old="0,100000,17,0,255"),
        # one sequence of the repository's sampling loop
        dict(name="decode_one", op="paged_decode", dtype="bf16", heads_q=16, heads_k=16, dim=64, page=16, lens="265"),
        # a ragged serving batch
        dict(name="decode_batch", op="paged_decode", dtype="bf16", heads_q=32, heads_k=8, dim=128, page=16,
             lens=_text([1 + 131 * i * i % 8192 for i in range(64)])),
        # few very long contexts
        dict(name="decode_long", op="paged_decode", dtype="bf16", heads_q=32, heads_k=4, dim=128, page=64,
             lens="131071,65537,100000"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 16])
    return kv * rng.choice([1, 2, 3, 4, 7, 8]), kv


def _lens(rng, total, most):
    """1 .. `most` lengths whose sum is at most `total`"""
    n = _log_int(rng, 1, most)
    w = [rng.random() ** 2 + 1e-3 for _ in range(n)]
    return [max(1, int(total * x / sum(w)) - 1) for x in w]


def draw(rng):
    op = rng.choice(["qk_norm_rotary", "packed_attention", "kv_append", "paged_decode"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "qk_norm_rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        hq, hk = _heads(rng)
        rows = max(1, min(_log_int(rng, 1, 33920), (1 << 26) // ((hq + hk) * dim)))
        return dict(op=op, dtype=dtype, rows=rows, heads_q=hq, heads_k=hk, dim=dim, rot=16 * rng.randint(1, dim // 16),
                    interleaved=rng.random() < 0.5, train=rng.random() < 0.5, first=_log_int(rng, 1, 1000000))
    if op == "packed_attention":
        dim = rng.choice([64, 128])
        hq, hk = _heads(rng)
        train = rng.random() < 0.5
        total = _log_int(rng, 16, 4000 if train or dtype == "f32" else 8000)
        if hq > 32:
            total = min(total, 2000)
        lens_q = _lens(rng, total, 12)
        more = rng.random() < 0.3
        lens_k = [n + (_log_int(rng, 1, 2000) if more else 0) for n in lens_q]
        return dict(op=op, dtype=dtype, heads_q=hq, heads_k=hk, dim=dim, lens_q=_text(lens_q), lens_k=_text(lens_k), train=train)
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "kv_append":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        hq, hk = _heads(rng)
        lens_new = _lens(rng, min(_log_int(rng, 1, 16000), (1 << 25) // ((hq + 2 * hk) * dim)), 64)
        lens_old = [_log_int(rng, 1, 20000) - 1 for _ in lens_new]
        if sum(lens_new) + sum(lens_old) > 200000:
            lens_old = [x // 8 for x in lens_old]
        return dict(op=op, dtype=dtype, heads_q=hq, heads_k=hk, dim=dim, rot=16 * rng.randint(1, dim // 16),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, page=page, lens_new=_text(lens_new),
                    lens_old=_text(lens_old))
    dim = rng.choice([64, 128])
    hq, hk = _heads(rng)
    lens = _lens(rng, min(_log_int(rng, 64, 290000), (1 << 27) // (hk * dim)), 64)
    return dict(op=op, dtype=dtype, heads_q=hq, heads_k=hk, dim=dim, page=page, lens=_text(lens))


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _freqs(rot):
    """radians per position of each pair, in 64 bits"""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    return (BASE ** (-i / rot)).cuda()


def _offsets(lens):
    o = [0]
    for n in lens:
        o.append(o[-1] + n)
    return o


def _pages(g, lens, page):
    """a page table whose pages lie in random order, and the number of pages: (S, most pages of a sequence)"""
    need = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), 0, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    st = dict(case=case)
    if case["op"] == "qk_norm_rotary":
        m = case["rows"]
        qkv = _randn(g, (m, (hq + 2 * hk) * d), dt)                 # q, k and v side by side, as the projection leaves them
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        st["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        st["wq"] = 1 + 0.2 * _randn(g, (d,), torch.float32)
        st["wk"] = 1 + 0.2 * _randn(g, (d,), torch.float32)
        st["pos"] = (case["first"] + torch.arange(m, device="cuda") % 4096).to(torch.int32)
        st["freqs"] = _freqs(case["rot"])
        if case["train"]:
            st["dq"], st["dk"] = _randn(g, (m, hq, d), dt), _randn(g, (m, hk, d), dt)
            for n in ("q", "k", "wq", "wk"):
                st[n] = st[n].detach().requires_grad_(True)
    elif case["op"] == "packed_attention":
        oq, ok = _offsets(_ints(case["lens_q"])), _offsets(_ints(case["lens_k"]))
        st["oq"], st["ok"] = oq, ok
        st["cu_q"] = torch.tensor(oq, dtype=torch.int32, device="cuda")
        st["cu_k"] = torch.tensor(ok, dtype=torch.int32, device="cuda") if ok != oq else st["cu_q"]
        st["q"] = _randn(g, (oq[-1], hq, d), dt)
        kv = _randn(g, (ok[-1], 2, hk, d), dt)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]
        if case["train"]:
            st["do"] = _randn(g, (oq[-1], hq, d), dt)
            for n in ("q", "k", "v"):
                st[n] = st[n].detach().requires_grad_(True)
    elif case["op"] == "kv_append":
        new, old = _ints(case["lens_new"]), _ints(case["lens_old"])
        m = sum(new)
        st["table"], n_pages = _pages(g, [a + b for a, b in zip(new, old)], case["page"])
        st["k_pages"] = _randn(g, (n_pages, hk, case["page"], d), dt)
        st["v_pages"] = _randn(g, (n_pages, hk, case["page"], d), dt)
        st["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda")).to(torch.int32)
        off = torch.tensor(_offsets(new), device="cuda")
        st["pos"] = (torch.arange(m, device="cuda") - off[st["seq"].long()]
                     + torch.tensor(old, device="cuda")[st["seq"].long()]).to(torch.int32)
        qkv = _randn(g, (m, (hq + 2 * hk) * d), dt)
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        st["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        st["v"] = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
        st["wq"] = 1 + 0.2 * _randn(g, (d,), torch.float32) if case["norm"] else None
        st["wk"] = 1 + 0.2 * _randn(g, (d,), torch.float32) if case["norm"] else None
        st["freqs"] = _freqs(case["rot"])
    else:
        lens = _ints(case["lens"])
        st["lens"] = lens
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["table"], n_pages = _pages(g, lens, case["page"])
        st["k_pages"] = _randn(g, (n_pages, hk, case["page"], d), dt)
        st["v_pages"] = _randn(g, (n_pages, hk, case["page"], d), dt)
        st["q"] = _randn(g, (len(lens), hq, d), dt)
    return st


# ------------------------------------------------------------------------------------------------------- plain forms
def _cos_sin(pos, freqs):
    a = pos.double()[:, None] * freqs[None]
    return torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]          # (rows, 1, rot / 2)


def _turn(x, cos, sin, rot, interleaved):
    """rotates the pairs of the first `rot` values of x (rows, heads, dim) f32"""
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rot:]), -1) if rot < x.shape[-1] else y


def _norm(x, w):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_norm_rotary(st):
    c = st["case"]
    cos, sin = _cos_sin(st["pos"], st["freqs"])
    out, grads, wgrads = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk"))):
        dt = x.dtype
        x, w = x.detach().float(), w.detach()
        n, r = _norm(x, w)
        out.append(_turn(n * w, cos, sin, c["rot"], c["interleaved"]).to(dt))
        if c["train"]:
            g = _turn(dy.float(), cos, -sin, c["rot"], c["interleaved"])
            wgrads.append((g * n).sum((0, 1)))
            g = g * w
            grads.append((r * (g - n * (g * n).mean(-1, keepdim=True))).to(dt))
    return tuple(out + grads + wgrads)


def _plain_append(st):
    c = st["case"]
    cos, sin = _cos_sin(st["pos"], st["freqs"])
    res = []
    for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
        y = x.float()
        if w is not None:
            y = _norm(y, w)[0] * w
        res.append(_turn(y, cos, sin, c["rot"], c["interleaved"]).to(x.dtype))
    pos = st["pos"].long()
    page = st["table"][st["seq"].long(), pos // c["page"]].long()
    st["k_pages"][page, :, pos % c["page"]] = res[1]
    st["v_pages"][page, :, pos % c["page"]] = st["v"]
    return res[0], st["k_pages"], st["v_pages"]


def _plain_packed(st):
    c = st["case"]
    hq, hk, d = c["heads_q"], c["heads_k"], c["dim"]
    grp, scale = hq // hk, 1.0 / math.sqrt(d)
    q, k, v = st["q"].detach(), st["k"].detach(), st["v"].detach()
    out = torch.empty_like(q)
    if c["train"]:
        dq, dk, dv = torch.empty_like(q), torch.empty(k.shape, dtype=k.dtype, device="cuda"), torch.empty(v.shape, dtype=v.dtype, device="cuda")
    for q0, q1, k0, k1 in zip(st["oq"][:-1], st["oq"][1:], st["ok"][:-1], st["ok"][1:]):
        nq, nk = q1 - q0, k1 - k0
        hidden = (torch.arange(nk, device="cuda")[None] > torch.arange(nq, device="cuda")[:, None] + (nk - nq))
        for h in range(hk):                                        # one shared key head and its queries at a time
            qs = q[q0:q1, h * grp:(h + 1) * grp].float().transpose(0, 1)         # (grp, nq, d)
            ks, vs = k[k0:k1, h].float(), v[k0:k1, h].float()
            s = (qs @ ks.t()) * scale
            s.masked_fill_(hidden, float("-inf"))
            s = torch.exp(s - s.amax(-1, keepdim=True))
            p = s / s.sum(-1, keepdim=True)
            o = p @ vs
            out[q0:q1, h * grp:(h + 1) * grp] = o.transpose(0, 1).to(out.dtype)
            if c["train"]:
                do = st["do"][q0:q1, h * grp:(h + 1) * grp].float().transpose(0, 1)
                dv[k0:k1, h] = (p.transpose(1, 2) @ do).sum(0).to(dv.dtype)
                ds = p * (do @ vs.t() - (do * o).sum(-1, keepdim=True))
                dq[q0:q1, h * grp:(h + 1) * grp] = ((ds @ ks) * scale).transpose(0, 1).to(dq.dtype)
                dk[k0:k1, h] = ((ds.transpose(1, 2) @ qs).sum(0) * scale).to(dk.dtype)
    return (out, dq, dk, dv) if c["train"] else out


def _plain_decode(st):
    c = st["case"]
    hq, hk, d, page = c["heads_q"], c["heads_k"], c["dim"], c["page"]
    out = torch.empty_like(st["q"])
    lse = torch.empty(len(st["lens"]), hq, dtype=torch.float32, device="cuda")
    for s, n in enumerate(st["lens"]):
        ids = st["table"][s, :-(-n // page)].long()
        ks = st["k_pages"][ids].transpose(0, 1).reshape(hk, -1, d)[:, :n].float()
        vs = st["v_pages"][ids].transpose(0, 1).reshape(hk, -1, d)[:, :n].float()
        w = (st["q"][s].float().view(hk, hq // hk, d) @ ks.transpose(1, 2)) / math.sqrt(d)
        top = w.amax(-1, keepdim=True)
        w = torch.exp(w - top)
        total = w.sum(-1, keepdim=True)
        out[s] = ((w @ vs) / total).reshape(hq, d).to(out.dtype)
        lse[s] = (top + torch.log(total)).reshape(hq)
    return out, lse


# ------------------------------------------------------------------------------------------------------------- a pass
def run(st):
    c = st["case"]
    if not own:
        return {"qk_norm_rotary": _plain_norm_rotary, "packed_attention": _plain_packed, "kv_append": _plain_append,
                "paged_decode": _plain_decode}[c["op"]](st)
    from melspec_gpt_vqvae_amd import ops
    from melspec_gpt_vqvae_amd.transformer import packed

    if c["op"] == "qk_norm_rotary":
        q, k = packed.qk_norm_rotary(st["q"], st["k"], st["pos"], st["freqs"], q_weight=st["wq"], k_weight=st["wk"], eps=EPS,
                                     interleaved=c["interleaved"])
        if not c["train"]:
            return q, k
        grads = torch.autograd.grad((q, k), (st["q"], st["k"], st["wq"], st["wk"]), (st["dq"], st["dk"]))
        return (q.detach(), k.detach()) + grads
    if c["op"] == "packed_attention":
        o = packed.packed_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"])
        if not c["train"]:
            return o
        return (o.detach(),) + torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])
    if c["op"] == "kv_append":
        q = ops.kv_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["seq"], st["pos"], q=st["q"],
                          freqs=st["freqs"], q_weight=st["wq"], k_weight=st["wk"], eps=EPS, interleaved=c["interleaved"])
        return q, st["k_pages"], st["v_pages"]
    return ops.paged_attn_decode(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"])


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    if case["op"] == "qk_norm_rotary":
        m, n = case["rows"], case["rows"] * (hq + hk) * d
        if case["train"]:
            return {"bytes": 4 * n * es + 4 * m + 4 * case["rot"] + 16 * d, "flops": 24 * n}
        return {"bytes": 2 * n * es + 4 * m + 4 * case["rot"] + 8 * d, "flops": 8 * n}
    if case["op"] == "packed_attention":
        lq, lk = _ints(case["lens_q"]), _ints(case["lens_k"])
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(lq, lk))
        nq, nk = sum(lq) * hq * d, sum(lk) * hk * d
        if case["train"]:
            return {"bytes": es * (4 * nq + 4 * nk) + 8 * (len(lq) + 1), "flops": 14 * pairs * hq * d}
        return {"bytes": es * (2 * nq + 2 * nk) + 8 * (len(lq) + 1), "flops": 4 * pairs * hq * d}
    if case["op"] == "kv_append":
        m = sum(_ints(case["lens_new"]))
        return {"bytes": 2 * m * (hq + 2 * hk) * d * es + 12 * m, "flops": (8 if case["norm"] else 4) * m * (hq + hk) * d}
    lens = _ints(case["lens"])
    return {"bytes": es * (2 * sum(lens) * hk * d + 2 * len(lens) * hq * d) + 4 * len(lens) * hq + 4 * sum(-(-n // case["page"]) for n in lens) + 4 * len(lens),
            "flops": 4 * sum(lens) * hq * d}


# --------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_turn(x, pos, freqs, interleaved):
    """x (rows, heads, dim) f64: the pairs as complex numbers times exp(i angle)"""
    rot = 2 * freqs.numel()
    z = x[..., :rot].unflatten(-1, (-1, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = torch.outer(pos.double(), freqs)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
    y = torch.view_as_real(z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _exact_norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def exact(case, seed):
    st = prepare(case, seed)
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    if case["op"] in ("qk_norm_rotary", "kv_append"):
        x = [st[n].detach().double().requires_grad_(True) if st[n] is not None else None for n in ("q", "k", "wq", "wk")]
        with torch.set_grad_enabled(case.get("train", False)):
            y = [_exact_turn(a if w is None else _exact_norm(a, w), st["pos"], st["freqs"], case["interleaved"])
                 for a, w in ((x[0], x[2]), (x[1], x[3]))]
        if case["op"] == "qk_norm_rotary":
            if not case["train"]:
                return tuple(y)
            return tuple(z.detach() for z in y) + torch.autograd.grad(y, x, (st["dq"].double(), st["dk"].double()))
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        flat = st["table"][st["seq"].long(), torch.div(st["pos"], case["page"], rounding_mode="floor").long()].long()
        slot = (st["pos"] % case["page"]).long()
        for h in range(hk):
            kp[flat, h, slot] = y[1][:, h]
            vp[flat, h, slot] = st["v"][:, h].double()
        return y[0], kp, vp
    if case["op"] == "packed_attention":
        names = ("q", "k", "v")
        x = [st[n].detach().double() for n in names]
        out = torch.zeros_like(x[0])
        grads = [torch.zeros_like(a) for a in x]
        for s in range(len(st["oq"]) - 1):
            a, b = slice(st["oq"][s], st["oq"][s + 1]), slice(st["ok"][s], st["ok"][s + 1])
            nq, nk = a.stop - a.start, b.stop - b.start
            seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
            for h in range(hq):
                part = [x[0][a, h].contiguous(), x[1][b, h // (hq // hk)].contiguous(), x[2][b, h // (hq // hk)].contiguous()]
                with torch.set_grad_enabled(case["train"]):
                    if case["train"]:
                        part = [z.requires_grad_(True) for z in part]
                    w = torch.mm(part[0], part[1].t()).div(math.sqrt(d)).where(seen, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
                    o = torch.mm(w.softmax(-1), part[2])
                out[a, h] = o.detach()
                if case["train"]:
                    gq, gk, gv = torch.autograd.grad(o, part, st["do"][a, h].double())
                    grads[0][a, h] = gq
                    grads[1][b, h // (hq // hk)] += gk
                    grads[2][b, h // (hq // hk)] += gv
        return (out, *grads) if case["train"] else out
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    for s, n in enumerate(st["lens"]):
        at = torch.arange(n, device="cuda")
        page, slot = st["table"][s].long()[at // case["page"]], at % case["page"]
        for h in range(hk):
            rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
            w = torch.mm(st["q"][s, rows].double(), st["k_pages"][page, h, slot].double().t()) * d ** -0.5
            out[s, rows] = torch.mm(torch.softmax(w, -1), st["v_pages"][page, h, slot].double())
            lse[s, rows] = torch.logsumexp(w, -1)
    return out, lse
