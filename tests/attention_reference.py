"""Attention and its gradients in 64 bits, sequence by sequence and head by
head, with a bound on what a kernel with fp32 arithmetic and probabilities
(and ds) rounded to the tensors' type may be off by, element for element.

The bounds, from u the unit roundoff of the tensors' type (2^-8 bf16, 2^-11
fp16, 2^-24 fp32), w = 2^-24 and t the largest absolute error of rounding a
number of the type's subnormal range (2^-25 for fp16, else 0):

* a score is a sum of D products, then scaled: |ds| <= e = (D + 2) w scale |q|.|k|;
* a probability, from score and row statistic, an exponential good to 2^-22 and
  a few fp32 roundings: relative error at most r = 2 max_j e + 64 w;
* o: (u + r + (n + 2) w) sum p|v| + t sum|v| + u|o|, n the row's keys;
* delta = do.o from the rounded o: d = (D + 2) w |do|.|o| + |do|.|err o|;
* ds = p (dp - delta): p (r |dp - delta| + (D + 2) w |do|.|v| + d) + u |ds| + t;
* dq, dk: scale times the sum of the errors of ds against |k| or |q|, plus
  (n + 2) w of the sum of absolute products, plus the result's own rounding;
* dv: (u + r + (n + 2) w) sum p|do| + t sum|do| + u|dv|.

Where p and ds are two terms (and o in delta too), u is u^2 (`inner`) but for
the results' own rounding.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
W = 2.0 ** -24


def sequences(B, Sq, Sk, q_lens=None, k_lens=None, cu_q=None, cu_k=None):
    """[(batch row, first query, queries, first key, keys)]"""
    if cu_q is not None:
        cu_k = cu_q if cu_k is None else cu_k
        return [(0, a, b - a, c, d - c)
                for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:])]
    return [(b, 0, Sq if q_lens is None else q_lens[b], 0, Sk if k_lens is None else k_lens[b])
            for b in range(B)]


def visible(nq, nk, causal, window, device):
    at = torch.arange(nq, device=device).unsqueeze(1) + (nk - nq)
    j = torch.arange(nk, device=device).unsqueeze(0)
    see = torch.ones(nq, nk, dtype=torch.bool, device=device)
    if causal:
        see &= j <= at
    if window:
        see &= j > at - window
    return see


def attention(q, k, v, do, seqs, causal=True, window=None, scale=None, inner=None):
    """{name: (value, bound)} of o, lse, dq, dk, dv for [B, S, H, D] tensors."""
    B, Sq, Hq, D = q.shape
    Hk = k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, t = U[q.dtype], 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    ui = u if inner is None else inner
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=q.device)  # noqa: E731
    val = {"o": z(q), "dq": z(q), "dk": z(k), "dv": z(v),
           "lse": torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device=q.device)}
    err = {n: torch.zeros_like(x) for n, x in val.items()}
    for b, q0, nq, k0, nk in seqs:
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, causal, window, q.device)
        none = ~see.any(1, keepdim=True)
        for h in range(Hq):
            g = h // (Hq // Hk)
            a, da = (x[b, q0:q0 + nq, h].double() for x in (q, do))
            c, d = (x[b, k0:k0 + nk, g].double() for x in (k, v))
            s = (a @ c.T * scale).masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(none, 0.0, torch.exp(s - torch.where(none, 0.0, lse)))
            e = ((D + 2) * W * scale * (a.abs() @ c.abs().T)).masked_fill(~see, 0.0)
            r = 2 * e.amax(1, keepdim=True) + 64 * W
            pe = p * r  # error of the probabilities in fp32
            seen = see.double()
            o = p @ d
            oe = (p * (ui + r + (nk + 2) * W)) @ d.abs() + t * (seen @ d.abs())
            dp = da @ d.T
            delta = (da * o).sum(1, keepdim=True)
            de = (da.abs() * ((D + 2) * W * o.abs() + oe + ui * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dse = pe * (dp - delta).abs() + p * ((D + 2) * W * (da.abs() @ d.abs().T) + de) \
                + ui * ds.abs() + t * seen
            qs, ks = slice(q0, q0 + nq), slice(k0, k0 + nk)
            val["o"][b, qs, h], err["o"][b, qs, h] = o, oe + u * o.abs()
            val["lse"][b, h, qs] = lse[:, 0]
            err["lse"][b, h, qs] = (r + 4 * W * lse.abs().clamp(max=1e300))[:, 0]
            dq = ds @ c * scale
            val["dq"][b, qs, h] = dq
            err["dq"][b, qs, h] = scale * (dse @ c.abs() + (nk + 2) * W * (ds.abs() @ c.abs())) \
                + u * dq.abs()
            # the group's heads add up: (the own rounding of the sum is added below)
            val["dk"][b, ks, g] += ds.T @ a * scale
            err["dk"][b, ks, g] += scale * (dse.T @ a.abs()
                                            + (nq * (Hq // Hk) + 2) * W * (ds.abs().T @ a.abs()))
            val["dv"][b, ks, g] += p.T @ da
            err["dv"][b, ks, g] += (p * (ui + r + (nq * (Hq // Hk) + 2) * W)).T @ da.abs() \
                + t * (seen.T @ da.abs())
    for n in ("dk", "dv"):
        err[n] += u * val[n].abs()
    # results below the type's normal range are rounded absolutely
    if q.dtype == torch.float16:
        for n in ("o", "dq", "dk", "dv"):
            err[n] += t
    return {n: (val[n], err[n]) for n in val}


def check(got, want, name):
    """Every element of `got` within the bound of `want` = (value, bound)."""
    val, err = want
    x = got.double()
    assert x.shape == val.shape, (name, x.shape, val.shape)
    inf = torch.isinf(val)
    assert torch.equal(x[inf], val[inf]), f"{name}: infinities differ"
    assert torch.isfinite(x[~inf]).all(), f"{name}: not finite"
    off = (x - val).abs()[~inf] - err[~inf]
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1e-30, f"{name}: off by {worst:.3e} more than the bound"
