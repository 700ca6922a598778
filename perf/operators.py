"""The attention block's operators as measurable cases.

Three operators that a layer runs in a row between its projections:

* ``rope``: per-head RMSNorm of q and k with rotary positions of several axes
  (time, height, width), ``fused_qk_norm_mrope`` / ``apply_mrope_qk``;
* ``fwd``: attention, ``fused_attention`` without gradients: whole sequences,
  chunks after a cache, single tokens;
* ``train``: attention and its backward pass, which recomputes the
  probabilities.

``own = False`` computes them in plain torch operations in 32 bits; ``own =
True`` calls the package. ``exact`` is each operator's definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases
def _rope(name, B, S, Hq, Hk, D, dtype, norm=True, train=True, interleaved=False, heads_first=False,
          axes=3):
    return {"name": name, "op": "rope", "B": B, "S": S, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype,
            "norm": norm, "train": train, "interleaved": interleaved, "heads_first": heads_first,
            "axes": axes}


def _attn(name, op, B, Sq, Sk, Hq, Hk, D, dtype, causal=True, window=0, docs=0, ragged=False,
          heads_first=False):
    return {"name": name, "op": op, "B": B, "Sq": Sq, "Sk": Sk, "Hq": Hq, "Hk": Hk, "D": D,
            "dtype": dtype, "causal": causal, "window": window, "docs": docs, "ragged": ragged,
            "heads_first": heads_first}


def listed():
    return [
        # one new token of a chat: the launch is all there is
        _rope("rope token", 1, 1, 32, 8, 128, "bf16", train=False),
        # a small vision-language batch without q/k norms, interleaved axes,
        # q and k as the transposed views that attention modules pass on
        _rope("rope views", 4, 2048, 32, 8, 64, "f16", norm=False, interleaved=True,
              heads_first=True),
        # odd everything, in full precision: a numerics check of a small model
        _rope("rope odd f32", 3, 257, 5, 1, 256, "f32", axes=4),
        # a training batch of video and text
        _rope("rope train", 8, 4096, 32, 8, 128, "bf16"),
        # the smallest prompt
        _attn("fwd prompt", "fwd", 1, 37, 37, 4, 2, 64, "bf16"),
        # one new token for each of sixteen conversations over their caches
        _attn("fwd decode", "fwd", 16, 1, 8192, 32, 8, 128, "bf16", ragged=True),
        # a chunk of a long prompt after what the cache already holds
        _attn("fwd chunk", "fwd", 2, 509, 8192, 32, 8, 128, "bf16"),
        # evaluation of whole sequences
        _attn("fwd batch", "fwd", 4, 4096, 4096, 32, 8, 128, "bf16"),
        # full precision, a length that fills no tile: a numerics check
        _attn("train odd f32", "train", 2, 100, 100, 4, 2, 64, "f32"),
        # a small model with a sliding window, heads before the sequence
        _attn("train window", "train", 2, 2048, 2048, 32, 8, 64, "f16", window=1000,
              heads_first=True),
        # packed documents of uneven lengths
        _attn("train packed", "train", 1, 8192, 8192, 32, 8, 128, "bf16", docs=9),
        # long-context fine-tuning
        _attn("train long", "train", 1, 8192, 8192, 32, 8, 128, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "fwd", "fwd", "train", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([64, 128, 128, 256])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq = Hk * rng.choice([1, 2, 4, 5, 8])
    if op == "rope":
        tokens = _log_int(rng, 1, 32768 * 40 * 128 // ((Hq + Hk) * D * (_BYTES[dtype] // 2)))
        tokens = min(tokens, 65536)
        B = rng.choice([b for b in (1, 2, 3, 8) if b <= tokens])
        c = _rope("", B, max(1, tokens // B), Hq, Hk, D, dtype, norm=rng.random() < 0.6,
                  train=rng.random() < 0.7, interleaved=rng.random() < 0.5,
                  heads_first=rng.random() < 0.3, axes=rng.choice([2, 3, 3, 4]))
        del c["name"]
        return c
    # pairs of query and key rows over all heads, at most the largest listed
    # case's; the 32-bit and 256-wide ones smaller (they run on fewer units)
    most = 32 * 8192 * 8192
    if dtype == "f32" or D == 256:
        most //= 16
    kind = rng.choice(["whole", "whole", "packed", "chunk", "token"] if op == "fwd"
                      else ["whole", "whole", "packed"])
    B = 1 if kind == "packed" else rng.choice([1, 2, 3, 7])
    if kind == "token":
        Sq = rng.choice([1, 1, 2, 4])
        Sk = _log_int(rng, 1, 16384)
        Sk = max(Sk, Sq)
        B = _log_int(rng, 1, 32)
    elif kind == "chunk":
        Sk = _log_int(rng, 64, 8192)
        Sq = _log_int(rng, 1, Sk)
    else:
        Sq = Sk = _log_int(rng, 1, 8192)
    while B * Hq * Sq * Sk > most:
        if kind == "token" or kind == "chunk":
            Sk = max(Sq, Sk // 2)
            Sq = max(1, Sq // 2)
        else:
            Sq = Sk = Sk // 2
    causal = rng.random() < 0.75
    window = _log_int(rng, 1, Sk) if causal and rng.random() < 0.25 else 0
    docs = min(Sk, rng.choice([2, 5, 17])) if kind == "packed" else 0
    c = _attn("", op, B, Sq, Sk, Hq, Hk, D, dtype, causal, window, docs,
              ragged=docs == 0 and rng.random() < 0.3,
              heads_first=docs == 0 and rng.random() < 0.3)
    del c["name"]
    return c


def _shape_rng(case):
    """What the lengths inside a case come from: they belong to the case, not to its seed."""
    return random.Random(",".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def _lengths(case):
    """Lengths of the packed documents, of the padded batch's sequences or caches; None: all full."""
    r = _shape_rng(case)
    if case["docs"]:
        cuts = sorted(r.randrange(case["Sk"] + 1) for _ in range(case["docs"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [case["Sk"]])]
    if case["ragged"]:
        lo = case["Sk"] // 4 if case["Sq"] < case["Sk"] else 0
        least = case["Sq"] if case["Sq"] < case["Sk"] else 0
        return [case["Sk"]] + [max(least, r.randint(lo, case["Sk"])) for _ in range(case["B"] - 1)]
    return None


def _sections(case):
    """Frequencies of each axis, time first."""
    half, n = case["D"] // 2, case["axes"]
    rest = half // (n + 1)
    return [half - (n - 1) * rest] + [rest] * (n - 1)


# ------------------------------------------------------------------ inputs
def _normal(shape, dtype, gen, heads_first=False):
    """A [B, S, H, D] tensor; heads_first: a view of memory laid out [B, H, S, D]."""
    if heads_first:
        b, s, h, d = shape
        return torch.randn(b, h, s, d, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    c = dict(case)
    if case["op"] == "rope":
        B, S, D = case["B"], case["S"], case["D"]
        st = {"case": c}
        for n, h in (("q", case["Hq"]), ("k", case["Hk"])):
            st[n] = _normal((B, S, h, D), dt, gen, case["heads_first"])
            if case["train"]:
                st["d" + n] = _normal((B, S, h, D), dt, gen, case["heads_first"])
            if case["norm"]:
                st["w" + n] = (1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(dt)
        # time runs on; the other axes walk over frames of 24 by 32 patches
        start = torch.randint(0, 1000, (B, 1), generator=gen, device="cuda")
        t = torch.arange(S, device="cuda").unsqueeze(0) + start
        st["pos"] = torch.stack([t, t // 32 % 24, t % 32, t // 768][: case["axes"]]).contiguous()
        half = D // 2
        st["inv_freq"] = 1.0 / (1e6 ** (torch.arange(half, device="cuda", dtype=torch.float32)
                                        / half))
        if case["train"]:
            for n in ("q", "k") + (("wq", "wk") if case["norm"] else ()):
                st[n].requires_grad_(True)
        return st
    B, Sq, Sk, Hq, Hk, D = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D"))
    hf = case["heads_first"]
    st = {"case": c, "q": _normal((B, Sq, Hq, D), dt, gen, hf),
          "k": _normal((B, Sk, Hk, D), dt, gen, hf), "v": _normal((B, Sk, Hk, D), dt, gen, hf)}
    lens = _lengths(case)
    st["lens"] = lens
    if case["docs"]:
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
        for n in ("q", "k", "v"):
            st[n] = st[n][0]
    elif lens:
        st["k_lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        if Sq == Sk:
            st["q_lens"] = st["k_lens"]
    if case["op"] == "train":
        st["do"] = _normal((B, Sq, Hq, D), dt, gen, hf)
        if case["docs"]:
            st["do"] = st["do"][0]
        for n in ("q", "k", "v"):
            st[n].requires_grad_(True)
    return st


# --------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own_rope(state) if op == "rope" else _own_attention(state)
    with torch.no_grad():
        return _plain_rope(state) if op == "rope" else _plain_attention(state)


def _own_rope(st):
    import bloth_b200
    c = st["case"]
    axes = bloth_b200.mrope_axes(_sections(c), interleaved=c["interleaved"])
    if c["norm"]:
        q, k = bloth_b200.fused_qk_norm_mrope(st["q"], st["k"], st["wq"], st["wk"], st["pos"],
                                              st["inv_freq"], axes, eps=1e-6)
    else:
        q, k = bloth_b200.apply_mrope_qk(st["q"], st["k"], st["pos"], st["inv_freq"], axes)
    if not c["train"]:
        return {"q": q, "k": k}
    names = ["q", "k"] + (["wq", "wk"] if c["norm"] else [])
    grads = torch.autograd.grad([q, k], [st[n] for n in names], [st["dq"], st["dk"]])
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _own_attention(st):
    import bloth_b200
    c = st["case"]
    how = {"causal": c["causal"], "window": c["window"] or None}
    if c["docs"]:
        how["cu_seqlens"] = st["cu"]
    elif st["lens"]:
        how["k_lens"] = st["k_lens"]
        how["q_lens"] = st.get("q_lens")
    o = bloth_b200.fused_attention(st["q"], st["k"], st["v"], **how)
    if c["op"] == "fwd":
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


# -------------------------------------------------------- the plain forms
def _axis_of(case):
    """The axis of each frequency: runs of the sections' lengths, or, interleaved, the axes in
    turn while an axis other than time has frequencies left, and time for the rest."""
    sec = _sections(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    n = len(sec)
    return [i % n if i % n and i // n < sec[i % n] else 0 for i in range(sum(sec))]


def _plain_cos_sin(st):
    axis = torch.tensor(_axis_of(st["case"]), device="cuda")
    ang = st["pos"].float()[axis].permute(1, 2, 0) * st["inv_freq"]  # [B, S, D/2]
    return ang.cos().unsqueeze(2), ang.sin().unsqueeze(2)


def _plain_rope(st):
    c = st["case"]
    cos, sin = _plain_cos_sin(st)
    half = c["D"] // 2
    out = {}
    for n in ("q", "k"):
        x = st[n].float()
        if c["norm"]:
            rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            xh = x * rstd
            w = st["w" + n].float()
            x = xh * w
        a, b = x[..., :half], x[..., half:]
        out[n] = torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(st[n].dtype)
        if not c["train"]:
            continue
        g = st["d" + n].float()
        a, b = g[..., :half], g[..., half:]
        d = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
        if c["norm"]:
            out["dw" + n] = (d * xh).sum((0, 1, 2)).to(st[n].dtype)
            d = d * w
            d = rstd * (d - xh * (d * xh).mean(-1, keepdim=True))
        out["d" + n] = d.to(st[n].dtype)
    return out


def _plain_visible(st, Sq, Sk):
    """[B or 1, 1, 1, Sq, Sk]: which keys each query sees."""
    c = st["case"]
    i = torch.arange(Sq, device="cuda").view(1, Sq, 1)
    j = torch.arange(Sk, device="cuda").view(1, 1, Sk)
    if c["docs"]:
        doc = torch.bucketize(torch.arange(Sk, device="cuda"), st["cu"][1:], right=True)
        see = (doc.view(1, Sq, 1) == doc.view(1, 1, Sk))
        off = torch.zeros(1, 1, 1, device="cuda", dtype=torch.long)
    elif st["lens"]:
        kl = st["k_lens"].long().view(-1, 1, 1)
        ql = st["q_lens"].long().view(-1, 1, 1) if "q_lens" in st else torch.full_like(kl, Sq)
        see = (j < kl) & (i < ql)
        off = kl - ql
    else:
        see = torch.ones(1, Sq, Sk, device="cuda", dtype=torch.bool)
        off = torch.full((1, 1, 1), Sk - Sq, device="cuda", dtype=torch.long)
    if c["causal"]:
        see = see & (j <= i + off)
    if c["window"]:
        see = see & (j > i + off - c["window"])
    return see.unsqueeze(1).unsqueeze(1)


def _plain_attention(st):
    c = st["case"]
    q, k, v = (st[n].unsqueeze(0) if c["docs"] else st[n] for n in ("q", "k", "v"))
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    dt = q.dtype
    scale = 1.0 / math.sqrt(D)

    def grouped(x):  # [B, Hk, G, Sq, D]
        return x.float().view(B, Sq, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4)

    def rows(x):  # back to [B, Sq, Hq, D]
        x = x.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(dt)
        return x[0] if c["docs"] else x

    qf = grouped(q.reshape(B, Sq, Hq, D))
    kf = k.float().permute(0, 2, 1, 3).unsqueeze(2)
    vf = v.float().permute(0, 2, 1, 3).unsqueeze(2)
    see = _plain_visible(st, Sq, Sk)
    p = qf @ kf.transpose(-1, -2)
    p.mul_(scale).masked_fill_(~see, -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)  # a row that sees nothing: zeros
    p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p.div_(torch.where(l == 0, torch.ones_like(l), l))
    o = p @ vf
    out = {"o": rows(o)}
    if c["op"] == "fwd":
        return out
    do = grouped((st["do"].unsqueeze(0) if c["docs"] else st["do"]).reshape(B, Sq, Hq, D))
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = do @ vf.transpose(-1, -2)
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    out["dq"] = rows(ds @ kf * scale)
    dk = (ds.transpose(-1, -2) @ qf).sum(2) * scale
    out["dk"], out["dv"] = ((x.permute(0, 2, 1, 3).to(dt)[0] if c["docs"]
                             else x.permute(0, 2, 1, 3).to(dt)) for x in (dk, dv))
    return out


# -------------------------------------------------------------------- work
def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, and the query and key rows in use."""
    lens = _lengths(case)
    Sq, Sk = case["Sq"], case["Sk"]
    if case["docs"]:
        seqs = [(n, n) for n in lens]
    elif lens:
        seqs = [(n if Sq == Sk else Sq, n) for n in lens]
    else:
        seqs = [(Sq, Sk)] * case["B"]
    n = 0
    for a, b in seqs:
        if not case["causal"]:
            n += a * b
            continue
        for_row = lambda i: min(b - 1, i + b - a) + 1 - (  # noqa: E731
            max(0, i + b - a - case["window"] + 1) if case["window"] else 0)
        n += sum(max(0, for_row(i)) for i in range(a))
    return n, sum(a for a, _ in seqs), sum(b for _, b in seqs)


def work(case):
    e = _BYTES[case["dtype"]]
    D, Hq, Hk = case["D"], case["Hq"], case["Hk"]
    if case["op"] == "rope":
        rows = case["B"] * case["S"] * (Hq + Hk)
        # read x, write y; and with gradients read dy and x, write dx
        passes = 5 if case["train"] else 2
        if case["train"] and not case["norm"]:
            passes = 4
        pos = case["axes"] * case["B"] * case["S"] * 8
        return {"bytes": rows * D * e * passes + pos * (2 if case["train"] else 1),
                "flops": rows * D * (20 if case["train"] else 8)}
    pairs, nq, nk = _pairs(case)
    q, kv = nq * Hq * D * e, nk * Hk * D * e
    if case["op"] == "fwd":
        # read q, k, v, write o; two products
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * Hq * pairs}
    # the forward; then read q, k, v, o, do, write dq, dk, dv: two products and five
    return {"bytes": 2 * q + 2 * kv + 4 * q + 4 * kv, "flops": 14 * D * Hq * pairs}


# ------------------------------------------------------------- in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return _exact_rope(st) if case["op"] == "rope" else _exact_attention(st)


def _exact_rope(st):
    """Complex form: pair (x[i], x[i + D/2]) is a number turned by its axis' angle, which is
    the 32-bit product of position and frequency."""
    c = st["case"]
    half = c["D"] // 2
    turn = torch.empty(c["B"], c["S"], half, device="cuda", dtype=torch.complex128)
    for i, a in enumerate(_axis_of(c)):
        ang = (st["pos"][a].to(torch.float32) * st["inv_freq"][i]).double()
        turn[:, :, i] = torch.polar(torch.ones_like(ang), ang)
    out = {}
    for n in ("q", "k"):
        res, grads, dws = [], [], torch.zeros(c["D"], device="cuda", dtype=torch.float64)
        for b in range(c["B"]):
            x = st[n][b].detach().double().requires_grad_(True)
            y = x
            leaves = [x]
            if c["norm"]:
                w = st["w" + n].detach().double().requires_grad_(True)
                y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
                leaves.append(w)
            z = torch.complex(y[..., :half], y[..., half:]) * turn[b].unsqueeze(1)
            y = torch.cat([z.real, z.imag], -1)
            res.append(y.detach())
            if c["train"]:
                g = torch.autograd.grad(y, leaves, st["d" + n][b].double())
                grads.append(g[0])
                if c["norm"]:
                    dws += g[1]
        out[n] = torch.stack(res)
        if c["train"]:
            out["d" + n] = torch.stack(grads)
            if c["norm"]:
                out["dw" + n] = dws
    return out


def _exact_attention(st):
    """Sequence by sequence and head by head, gradients by differentiation of the formula."""
    c = st["case"]
    train = c["op"] == "train"
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    out = {"o": torch.zeros(q.shape, device="cuda", dtype=torch.float64)}
    if train:
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            out[n] = torch.zeros(x.shape, device="cuda", dtype=torch.float64)
    lens = st["lens"]
    seqs = []  # (where its queries are, where its keys are, how many of each)
    if c["docs"]:
        at = 0
        for n in lens:
            seqs.append(((slice(at, at + n),), (slice(at, at + n),), n, n))
            at += n
    else:
        for b in range(c["B"]):
            nk = lens[b] if lens else c["Sk"]
            nq = nk if lens and c["Sq"] == c["Sk"] else c["Sq"]
            seqs.append(((b, slice(0, nq)), (b, slice(0, nk)), nq, nk))
    for iq, ik, nq, nk in seqs:
        if not nq or not nk:
            continue
        i = torch.arange(nq, device="cuda").unsqueeze(1) + (nk - nq)
        j = torch.arange(nk, device="cuda").unsqueeze(0)
        hide = torch.zeros(nq, nk, device="cuda", dtype=torch.bool)
        if c["causal"]:
            hide |= j > i
        if c["window"]:
            hide |= j <= i - c["window"]
        none = hide.all(1, keepdim=True)
        for h in range(c["Hq"]):
            g = h // (c["Hq"] // c["Hk"])
            a, b, d = (x.double().requires_grad_(train)
                       for x in (q[iq][:, h], k[ik][:, g], v[ik][:, g]))
            s = torch.where(hide, -math.inf, a @ b.T / math.sqrt(c["D"]))
            p = torch.softmax(torch.where(none, torch.zeros_like(s), s), -1)
            o = torch.where(none, torch.zeros((), device="cuda", dtype=torch.float64), p @ d)
            out["o"][iq][:, h] = o.detach()
            if train:
                ga, gb, gd = torch.autograd.grad(o, (a, b, d), st["do"][iq][:, h].double())
                out["dq"][iq][:, h] = ga
                out["dk"][ik][:, g] += gb
                out["dv"][ik][:, g] += gd
    return out
