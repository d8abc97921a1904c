"""Workloads for the transformer-training operators: attention whose backward
recomputes the probabilities, the per-head query/key norm with the position
rotation, and the AdamW step over flat parameter storage.

`own` False runs the plain form (elementary torch operations, 32 bits, one
rounding at the end); True runs the framework's kernels. `exact` is the
definition in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}
ALIGN = 64  # flat storage: every parameter starts at a multiple of 64


def _attn(name, dtype, b, sq, sk, h, hk, hd, causal, ragged, grad, packed):
    return {"name": name, "op": "attention", "dtype": dtype, "b": b,
            "sq": sq, "sk": sk, "h": h, "hk": hk, "hd": hd,
            "causal": causal, "ragged": ragged, "grad": grad,
            "packed": packed}


def _qknr(name, dtype, b, s, h, hk, hd, rot, interleaved, positions, grad):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "b": b,
            "s": s, "h": h, "hk": hk, "hd": hd, "rot": rot,
            "interleaved": interleaved, "positions": positions, "grad": grad}


def _adamw(name, tensors, largest, bits, decay_some):
    return {"name": name, "op": "adamw", "tensors": tensors,
            "largest": largest, "bits": bits, "decay_some": decay_some}


def listed():
    return [
        # a CIFAR-sized image in 4x4 patches and a class token: latency
        _attn("attn_train_tiny", "fp16", 4, 65, 65, 3, 3, 64, False, False,
              True, True),
        # the repository's ViT-B/16 step: batch 128, 197 tokens, 12 heads
        _attn("attn_train_vit", "bf16", 128, 197, 197, 12, 12, 64, False,
              False, True, True),
        # a causal language model's step, four query heads to a key head
        _attn("attn_train_causal", "bf16", 4, 2048, 2048, 16, 4, 128, True,
              False, True, True),
        # one long document
        _attn("attn_train_long", "bf16", 1, 16384, 16384, 16, 2, 128, True,
              False, True, True),
        # images of many sizes padded to the longest, an empty one among
        # them, with a head that fills no tile
        _attn("attn_train_ragged", "fp16", 16, 777, 777, 10, 10, 80, False,
              True, True, True),
        # one new token against caches of many lengths
        _attn("attn_one_query", "bf16", 32, 1, 8191, 16, 4, 128, True, True,
              False, False),
        # the same ViT step: queries and keys between projection and
        # attention
        _qknr("qknr_train_vit", "bf16", 128, 197, 12, 12, 64, 64, False,
              False, True),
        # long sequences, neighbouring elements rotated, half of the head
        _qknr("qknr_train_long", "bf16", 2, 16384, 32, 8, 128, 64, True,
              False, True),
        # one new token a sequence, each at its own position
        _qknr("qknr_one_token", "fp16", 32, 1, 16, 4, 128, 128, False, True,
              False),
        # a small head being tuned: latency
        _adamw("adamw32_small", 12, 40000, 32, False),
        # a transformer of some 90 million parameters, biases and norms
        # without decay
        _adamw("adamw32_large", 150, 8000000, 32, True),
        # the same with states in 8 bits
        _adamw("adamw8_large", 150, 8000000, 8, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "qk_norm_rope", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    hk = rng.choice([1, 2, 3, 4, 8])
    h = hk * rng.choice([1, 1, 2, 3, 4, 8])
    hd = rng.choice([64, 64, 128, 128, 32, 72, 80, 96, 112])
    if op == "attention":
        sk = _log(rng, 1, 12000)
        grad = rng.random() < 0.7
        causal = rng.random() < 0.5
        sq = sk
        if not grad:
            sq = rng.choice([1, 1, min(sk, 4), min(sk, 7), sk])
        elif not causal and rng.random() < 0.3:
            sq = _log(rng, 1, 4000)
        b = _log(rng, 1, 64)
        while b > 1 and (b * sk * hk * hd > 1.2e8
                         or b * h * sq * sk > 1.5e9):
            b = b // 2
        while b * h * sq * sk > 3.0e9:
            hk, h = max(1, hk // 2), max(1, hk // 2) * (h // hk)
            if hk == 1:
                h = max(1, h // 2)
        c = _attn("", dtype, b, sq, sk, h, hk, hd, causal,
                  b > 1 and rng.random() < 0.4, grad, sq == sk)
    elif op == "qk_norm_rope":
        b, s = _log(rng, 1, 128), _log(rng, 1, 16384)
        while b > 1 and b * s * (h + hk) * hd > 0.8e8:
            b = b // 2
        rot = rng.choice([hd, hd, hd // 2 // 16 * 16 or 16])
        if rot % 16:
            rot = hd // 16 * 16
        c = _qknr("", rng.choice([dtype, dtype, "fp32"]), b, s, h, hk, hd,
                  rot, rng.random() < 0.5, rng.random() < 0.5,
                  rng.random() < 0.7)
    else:
        c = _adamw("", rng.randint(1, 200), _log(rng, 64, 2000000),
                   rng.choice([32, 8]), rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _lens(case):
    """Lengths of the sequences, from 0 to the longest."""
    b, sk = case["b"], case["sk"]
    return [i * sk // (b - 1) for i in range(b)]


def _sizes(case):
    """Element counts of the parameters: from one to the largest, spread
    over their logarithm."""
    t, top = case["tensors"], case["largest"]
    return [max(1, int(top ** ((i * 0.6180339887498949) % 1.0)))
            if i else top for i in range(t)]


def _prepare_attention(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    b, sq, sk, h, hk, hd = (case[x] for x in
                            ("b", "sq", "sk", "h", "hk", "hd"))
    if case["packed"]:  # views of one projection's output
        qkv = _randn(g, b, sq, h + 2 * hk, hd, dtype=dt)
        q, k, v = qkv.split([h, hk, hk], dim=2)
    else:
        q = _randn(g, b, sq, h, hd, dtype=dt)
        k = _randn(g, b, sk, hk, hd, dtype=dt)
        v = _randn(g, b, sk, hk, hd, dtype=dt)
    st = {"case": case, "q": q.detach(), "k": k.detach(), "v": v.detach(),
          "q_lens": None, "kv_lens": None}
    if case["ragged"]:
        st["kv_lens"] = torch.tensor(_lens(case), dtype=torch.int32,
                                     device="cuda")
        if sq == sk:  # the same sequences on both sides
            st["q_lens"] = st["kv_lens"]
    if case["grad"]:
        st["dout"] = _randn(g, b, sq, h, hd, dtype=dt)
        for x in ("q", "k", "v"):
            st[x].requires_grad_(True)
    return st


def _tables(n, rot):
    """cos, sin [n, rot/2] of the angles position * 10000^(-2i/rot)."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64,
                                  device="cuda") / rot)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float(), a.sin().float()


def _prepare_qknr(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    b, s, h, hk, hd = (case[x] for x in ("b", "s", "h", "hk", "hd"))
    qkv = _randn(g, b, s, h + 2 * hk, hd, dtype=dt, std=1.7)
    st = {"case": case, "q": qkv[:, :, :h].detach(),
          "k": qkv[:, :, h:h + hk].detach(),
          "wq": 1.0 + _randn(g, hd, std=0.1),
          "wk": 1.0 + _randn(g, hd, std=0.1), "positions": None}
    top = s
    if case["positions"]:
        top = max(s, 8192)
        st["positions"] = torch.randint(0, top, (b, s), generator=g,
                                        device="cuda")
    st["cos"], st["sin"] = _tables(top, case["rot"])
    if case["grad"]:
        st["dq"] = _randn(g, b, s, h, hd, dtype=dt)
        st["dk"] = _randn(g, b, s, hk, hd, dtype=dt)
        for x in ("q", "k", "wq", "wk"):
            st[x].requires_grad_(True)
    return st


def _prepare_adamw(case, seed):
    g = _gen(seed)
    sizes = _sizes(case)
    aligned = [-(-n // ALIGN) * ALIGN for n in sizes]
    total = sum(aligned)
    # gradients of one parameter are alike, of two may be far apart; the
    # gaps between parameters hold zeros
    span = torch.tensor(aligned, device="cuda")
    mag = torch.exp(torch.rand(len(sizes), generator=g, device="cuda") * 6
                    - 9).repeat_interleave(span)
    live = torch.ones(total, device="cuda")
    off, keep = 0, []
    for i, (n, a) in enumerate(zip(sizes, aligned)):
        live[off + n:off + a] = 0
        keep.append(0 if case["decay_some"] and n < 1024 else 1)
        off += a
    mag *= live
    p = _randn(g, total, std=0.02) * live
    grad = _randn(g, total) * mag
    m = _randn(g, total, std=0.3) * mag
    v = mag * mag * (0.2 + torch.rand(total, generator=g, device="cuda"))
    st = {"case": case, "p": p, "g": grad,
          "step": torch.full((1,), 1000 + seed % 1000, dtype=torch.int64,
                             device="cuda"),
          "lr": torch.full((1,), 3e-4, device="cuda"),
          "seed": seed % 2147483647, "decay": None}
    if case["decay_some"]:
        st["decay"] = torch.tensor(keep, dtype=torch.uint8, device="cuda") \
            .repeat_interleave(span // ALIGN)
    if case["bits"] == 8:
        st["m"], st["m_scale"] = _to8(m)
        st["v"], st["v_scale"] = _to8(v.sqrt())
    else:
        st["m"], st["v"] = m, v
    return st


def prepare(case, seed):
    if case["op"] == "attention":
        return _prepare_attention(case, seed)
    if case["op"] == "qk_norm_rope":
        return _prepare_qknr(case, seed)
    return _prepare_adamw(case, seed)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _mask(st):
    """True where a query may see a key: [b, 1, 1, sq, sk], or None."""
    c = st["case"]
    dev = st["q"].device
    if not c["causal"] and st["kv_lens"] is None:
        return None
    i = torch.arange(c["sq"], device=dev)[:, None]
    j = torch.arange(c["sk"], device=dev)[None, :]
    shape = (-1, 1, 1, 1, 1)
    kl = torch.full((1,), c["sk"], device=dev) if st["kv_lens"] is None \
        else st["kv_lens"]
    ql = torch.full((1,), c["sq"], device=dev) if st["q_lens"] is None \
        else st["q_lens"]
    kl, ql = kl.view(shape), ql.view(shape)
    ok = (j < kl) & (i < ql)
    if c["causal"]:
        ok = ok & (j <= i + kl - ql)
    return ok


def _plain_attention(st):
    c = st["case"]
    b, sq, sk, h, hk, hd = (c[x] for x in
                            ("b", "sq", "sk", "h", "hk", "hd"))
    scale = 1.0 / math.sqrt(hd)
    dt = st["q"].dtype
    with torch.no_grad():
        q = st["q"].float().view(b, sq, hk, h // hk, hd) \
            .permute(0, 2, 3, 1, 4)                      # b hk g sq hd
        k = st["k"].float().permute(0, 2, 1, 3)[:, :, None]  # b hk 1 sk hd
        v = st["v"].float().permute(0, 2, 1, 3)[:, :, None]
        p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
        ok = _mask(st)
        if ok is not None:
            p.masked_fill_(~ok, float("-inf"))
        top = p.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        p.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total > 0, total, torch.ones_like(total)))
        out = torch.matmul(p, v)                         # b hk g sq hd

        def back(x):
            return x.permute(0, 3, 1, 2, 4).reshape(b, sq, h, hd).to(dt)

        res = {"out": back(out)}
        if c["grad"]:
            do = st["dout"].float().view(b, sq, hk, h // hk, hd) \
                .permute(0, 2, 3, 1, 4)
            dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
            ds = torch.matmul(do, v.transpose(-1, -2))
            ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p)
            dq = torch.matmul(ds, k) * scale
            dk = (torch.matmul(ds.transpose(-1, -2), q) * scale).sum(2)
            res["dq"] = back(dq)
            res["dk"] = dk.permute(0, 2, 1, 3).to(dt)
            res["dv"] = dv.permute(0, 2, 1, 3).to(dt)
    return res


def _own_attention(st):
    from pytorch_distributed_train_amd.ops import functional as OF
    out = OF.attention_recompute(st["q"], st["k"], st["v"],
                                 causal=st["case"]["causal"],
                                 q_lens=st["q_lens"], kv_lens=st["kv_lens"])
    res = {"out": out.detach()}
    if st["case"]["grad"]:
        res["dq"], res["dk"], res["dv"] = torch.autograd.grad(
            out, (st["q"], st["k"], st["v"]), st["dout"])
    return res


def _exact_attention(case, seed):
    st = _prepare_attention(case, seed)
    h, hk = case["h"], case["hk"]
    scale = case["hd"] ** -0.5
    q, k, v = (st[x].detach().double() for x in ("q", "k", "v"))
    res = {"out": torch.zeros_like(q)}
    if case["grad"]:
        res |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k),
                "dv": torch.zeros_like(v)}
    lens = _lens(case) if case["ragged"] else [case["sk"]] * case["b"]
    for b, n in enumerate(lens):
        m = n if st["q_lens"] is not None else case["sq"]
        for head in range(h):
            if n == 0 or m == 0:
                continue
            qq, kk, vv = (x.clone().requires_grad_(case["grad"]) for x in (
                q[b, :m, head], k[b, :n, head // (h // hk)],
                v[b, :n, head // (h // hk)]))
            s = (qq * scale) @ kk.t()
            if case["causal"]:
                s = s + torch.full((m, n), float("-inf"), device="cuda",
                                   dtype=torch.float64).triu(n - m + 1)
            o = torch.softmax(s, -1) @ vv
            res["out"][b, :m, head] = o.detach()
            if case["grad"]:
                gq, gk, gv = torch.autograd.grad(
                    o, (qq, kk, vv), st["dout"][b, :m, head].double())
                res["dq"][b, :m, head] = gq
                res["dk"][b, :n, head // (h // hk)] += gk
                res["dv"][b, :n, head // (h // hk)] += gv
            del s, o
    return res


# ---------------------------------------------------------------------------
# query/key norm and rotation
# ---------------------------------------------------------------------------

def _halves(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _turn(x, cos, sin, rot, interleaved):
    """x with its rotated part turned by the angles of cos and sin."""
    a, b = _halves(x, rot, interleaved)
    y = torch.empty_like(x)
    c, d = _halves(y, rot, interleaved)
    c.copy_(a * cos - b * sin)
    d.copy_(b * cos + a * sin)
    y[..., rot:] = x[..., rot:]
    return y


def _plain_qknr(st):
    c = st["case"]
    rot, inter = c["rot"], c["interleaved"]
    res = {}
    with torch.no_grad():
        pos = st["positions"]
        if pos is None:
            cos, sin = st["cos"][:c["s"], None], st["sin"][:c["s"], None]
        else:
            cos, sin = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]

        def one(x, w, dy):
            x32 = x.float()
            r = (x32.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            xhat = x32 * r
            y = _turn(xhat * w, cos, sin, rot, inter).to(x.dtype)
            if dy is None:
                return y, None, None
            g = _turn(dy.float(), cos, -sin, rot, inter)
            dw = (g * xhat).double().sum((0, 1, 2)).float()
            gw = g * w
            dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
            return y, dx.to(x.dtype), dw

        res["q"], dq, dwq = one(st["q"], st["wq"], st.get("dq"))
        res["k"], dk, dwk = one(st["k"], st["wk"], st.get("dk"))
        if c["grad"]:
            res |= {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    return res


def _own_qknr(st):
    from pytorch_distributed_train_amd.ops import functional as OF
    q, k = OF.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"],
                           st["sin"], positions=st["positions"],
                           interleaved=st["case"]["interleaved"])
    res = {"q": q.detach(), "k": k.detach()}
    if st["case"]["grad"]:
        res["dq"], res["dk"], res["dwq"], res["dwk"] = torch.autograd.grad(
            (q, k), (st["q"], st["k"], st["wq"], st["wk"]),
            (st["dq"], st["dk"]))
    return res


def _exact_qknr(case, seed):
    st = _prepare_qknr(case, seed)
    pos = st["positions"]
    if pos is None:
        pos = torch.arange(case["s"], device="cuda").expand(case["b"], -1)
    # the tables are inputs of 32 bits; complex numbers turn the pairs
    e = torch.complex(st["cos"].double(), st["sin"].double())[pos]
    e = e[:, :, None]
    rot, n = case["rot"], case["hd"]
    order = torch.arange(n, device="cuda")
    if not case["interleaved"]:  # pair i with i + rot/2
        order[:rot] = order[:rot].view(2, rot // 2).t().reshape(-1)
    back = torch.empty_like(order)
    back[order] = torch.arange(n, device="cuda")
    res = {}
    for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
        xx = st[x].detach().double().requires_grad_(case["grad"])
        ww = st[w].detach().double().requires_grad_(case["grad"])
        y = xx / torch.sqrt((xx ** 2).sum(-1, keepdim=True) / n + 1e-6) * ww
        y = y[..., order]
        z = torch.view_as_complex(
            y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2)) * e
        y = torch.cat([torch.view_as_real(z).flatten(-2), y[..., rot:]], -1)
        y = y[..., back]
        res[x] = y.detach()
        if case["grad"]:
            gx, gw = torch.autograd.grad(y, (xx, ww), st[dy].double())
            res["d" + x], res["dw" + x] = gx, gw
    return res


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

BETA1, BETA2, EPS, DECAY = 0.9, 0.999, 1e-8, 0.05
TINY = 2.0 ** -100  # a block below this is stored as zeros
U32 = 0xFFFFFFFF


def _scale8(x):
    """Per 64 values: the scale that takes the largest to 448, and its
    inverse (both 0 for a block of nothing)."""
    top = x.abs().view(-1, ALIGN).amax(1)
    live = top >= TINY
    scale = torch.where(live, top * (1.0 / 448.0), torch.zeros_like(top))
    inv = torch.where(live, 448.0 / top, torch.zeros_like(top))
    return scale, inv.repeat_interleave(ALIGN)


def _to8(x):
    """(e4m3, scale) of x, to the nearest."""
    scale, inv = _scale8(x)
    return (x * inv).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _noise(n, step, seed, device):
    """16 random bits a value: both halves of a 32-bit mix of the pair's
    index, the step and the seed."""
    x = torch.arange((n + 1) // 2, dtype=torch.int64, device=device)
    # multipliers: the fractions of the golden ratio and of the roots of
    # 2, 3, 5 and 7 in 32 bits, all but the first cut to 31 and made odd
    x = (x * 0x9E3779B1 + step * 0x6A09E667 + seed * 0x3B67AE85) & U32
    x = ((x ^ (x >> 16)) * 0x3C6EF373) & U32
    x = ((x ^ (x >> 15)) * 0x254FF53B) & U32
    x = x ^ (x >> 16)
    return torch.stack([x & 0xFFFF, x >> 16], 1).view(-1)[:n].float()


def _to8_random(x, step, seed):
    """(e4m3, scale) of x >= 0, up or down at random so that the mean is x;
    never down to zero."""
    scale, inv = _scale8(x)
    y = (x * inv).clamp(max=448.0)
    # the distance of neighbouring e4m3 values: 2^(exponent - 3), 2^-9 least
    unit = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    z = torch.floor(y / unit + _noise(x.numel(), step, seed, x.device)
                    * 2.0 ** -16) * unit
    z = z.clamp(max=448.0)
    z = torch.where(y > 0, z.clamp(min=2.0 ** -9), torch.zeros_like(z))
    return z.to(torch.float8_e4m3fn), scale


def _plain_adamw(st):
    c, p, g, lr = st["case"], st["p"], st["g"], st["lr"]
    st["step"] += 1
    t = st["step"]
    bc1 = (1.0 - BETA1 ** t.double()).float()
    bc2 = (1.0 - BETA2 ** t.double()).float()
    if c["bits"] == 8:
        m = st["m"].float() * st["m_scale"].repeat_interleave(ALIGN)
        v = st["v"].float() * st["v_scale"].repeat_interleave(ALIGN)
        v.mul_(v)
    else:
        m, v = st["m"], st["v"]
    m.mul_(BETA1).add_(g * (1.0 - BETA1))
    v.mul_(BETA2).add_(g * g * (1.0 - BETA2))
    if st["decay"] is None:
        p.mul_(1.0 - lr * DECAY)
    else:
        p.mul_(1.0 - lr * DECAY
               * st["decay"].repeat_interleave(ALIGN).float())
    p.sub_(lr / bc1 * m / (v.sqrt() / bc2.sqrt() + EPS))
    if c["bits"] == 32:
        return {"p": p, "m": m, "v": v}
    q, s = _to8(m)
    st["m"].copy_(q)
    st["m_scale"].copy_(s)
    q, s = _to8_random(v.sqrt(), t, st["seed"])
    st["v"].copy_(q)
    st["v_scale"].copy_(s)
    return {"p": p, "m": st["m"], "m_scale": st["m_scale"], "v": st["v"],
            "v_scale": st["v_scale"]}


def _own_adamw(st):
    from pytorch_distributed_train_amd.ops import functional as OF
    eight = st["case"]["bits"] == 8
    OF.adamw_step(st["p"], st["g"], st["m"], st["v"], st["step"], st["lr"],
                  beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY,
                  decay=st["decay"],
                  m_scale=st["m_scale"] if eight else None,
                  v_scale=st["v_scale"] if eight else None, seed=st["seed"])
    return {x: st[x] for x in (("p", "m", "m_scale", "v", "v_scale")
                               if eight else ("p", "m", "v"))}


def _exact_adamw(case, seed):
    st = _prepare_adamw(case, seed)
    g, t = st["g"].double(), int(st["step"]) + 1
    lr = float(st["lr"])
    if case["bits"] == 8:
        def wide(x, s):
            return (x.double().view(-1, ALIGN) * s.double()[:, None]) \
                .view(-1)
        m = wide(st["m"], st["m_scale"])
        v = wide(st["v"], st["v_scale"]) ** 2
    else:
        m, v = st["m"].double(), st["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    on = torch.ones_like(g) if st["decay"] is None \
        else st["decay"].double()[:, None].expand(-1, ALIGN).reshape(-1)
    p = st["p"].double()
    p = p - lr * DECAY * on * p - lr * (m / (1 - BETA1 ** t)) / (
        torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v}

    def scale(x):
        return x.abs().view(-1, ALIGN).max(1).values / 448

    return {"p": p, "m": None, "m_scale": scale(m), "v": None,
            "v_scale": scale(torch.sqrt(v))}


# ---------------------------------------------------------------------------
# what is measured
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return (_own_attention if own else _plain_attention)(state)
    if op == "qk_norm_rope":
        return (_own_qknr if own else _plain_qknr)(state)
    return (_own_adamw if own else _plain_adamw)(state)


def exact(case, seed):
    if case["op"] == "attention":
        pairs = case["b"] * case["h"] * case["sq"] * case["sk"]
        if pairs > 8e9:
            return None
        return _exact_attention(case, seed)
    if case["op"] == "qk_norm_rope":
        return _exact_qknr(case, seed)
    return _exact_adamw(case, seed)


def work(case):
    if case["op"] == "attention":
        b, sq, sk, h, hk, hd = (case[x] for x in
                                ("b", "sq", "sk", "h", "hk", "hd"))
        lens = _lens(case) if case["ragged"] else [sk] * b
        pairs = rows = keys = 0
        for n in lens:
            m = n if case["ragged"] and sq == sk else sq
            rows += m
            keys += n
            if case["causal"]:
                # row i sees i + n - m + 1 keys
                lo, hi = max(0, n - m + 1), n
                pairs += max(0, hi - lo + 1) * (lo + hi) // 2
            else:
                pairs += m * n
        q, kv = rows * h * hd * 2, keys * hk * hd * 2
        if not case["grad"]:
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * h * hd}
        # q, out, dout and dq; k, v, dk and dv
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * h * hd}
    if case["op"] == "qk_norm_rope":
        n = case["b"] * case["s"] * (case["h"] + case["hk"]) * case["hd"]
        size = 4 if case["dtype"] == "fp32" else 2
        passes = 4 if case["grad"] else 2
        return {"bytes": passes * n * size, "flops": 8 * passes * n}
    n = sum(_sizes(case))
    return {"bytes": n * (28 if case["bits"] == 32 else 16.25),
            "flops": 16 * n}
