"""Attention over sequences in 64 bits, from its definition, with a bound on
what rounding may do to each element of the result.

Bound for one output element o = sum_j w_j v_j (w the softmax weights), u the
half step of the output type, u_w that of the type the weights are held in
(both finfo.eps / 2; u_w = 0 where weights stay in 32 bits):

    |error| <= u |o|  +  (u_w + 2 d + (L + 8) 2^-23) * sum_j w_j |v_j|

d bounds a score's error: D products summed in 32 bits, (D + 8) 2^-23 of
scale * sum_d max|q| |k_jd|, and the exponent's argument rounded once, 2^-22 of
|s_j|, plus 2^-21 for the exponential itself; a weight's relative error is
twice that (numerator and denominator) to first order.  (L + 8) 2^-23 covers
the sums over L keys."""
import math

import torch

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def attend(q, k, v, scale, causal, u_w=0.0, u=0.0):
    """One sequence: q [n, Hq, D], k / v [L, Hkv, D] (any dtype).  (o, bound)
    in 64 bits, [n, Hq, D]; keys no query sees never enter."""
    n, hq, d = q.shape
    length, hkv = k.shape[0], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    o = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for i in range(n):
        lim = max(0, min(length, length - n + i + 1)) if causal else length
        if lim == 0:
            continue
        kk = k[:lim].repeat_interleave(hq // hkv, 1)
        vv = v[:lim].repeat_interleave(hq // hkv, 1)
        s = torch.einsum("hd,jhd->hj", q[i], kk) * scale
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total == 0, 1.0, total)
        o[i] = torch.einsum("hj,jhd->hd", w, vv)
        size = abs(scale) * (q[i].abs().amax(-1) * kk.abs().sum(-1)).amax(0)
        delta = (d + 8) * 2.0**-23 * size + 2.0**-22 * s.abs().amax(-1) + 2.0**-21
        spread = torch.einsum("hj,jhd->hd", w, vv.abs())
        tol[i] = u * o[i].abs() + (u_w + 2 * delta + (lim + 8) * 2.0**-23).unsqueeze(-1) * spread
    return o, tol


def check(got, want, tol, what=""):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities in other places"
    fine = want.isfinite()
    off = ((got - want).abs() - tol)[fine]
    if off.numel():
        worst = off.max().item()
        assert worst <= 1e-30, f"{what}: {worst:.3e} over the bound"


def e8m0(byte):
    return torch.where(byte == 255, math.nan, torch.exp2(byte.double() - 127))


def quantise(x):
    """(values e4m3 holds, scale byte) of vectors along the last axis, in 64 bits from the definition."""
    x = x.double()
    a = x.abs().amax(-1)
    e = torch.full(a.shape, 0.0, dtype=torch.float64, device=x.device)
    pos = (a > 0) & a.isfinite()
    guess = torch.ceil(torch.log2(torch.where(pos, a, 1.0) / 448))
    for step in (1, 0, -1):  # the smallest of the candidates that holds
        e = torch.where(pos & (a <= 448 * torch.exp2(guess + step)), guess + step, e)
    e = e.clamp(min=-127)
    y = x * torch.exp2(-e).unsqueeze(-1)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    y = torch.round(y / step) * step
    bad = ~a.isfinite()
    y = torch.where(bad.unsqueeze(-1), math.nan, y)
    return y, torch.where(bad, 255.0, e + 127).to(torch.uint8)
