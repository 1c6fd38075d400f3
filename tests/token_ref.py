"""Plain 64-bit restatements of the token operators (layer norm, dropout, attention) with the error bounds their tests use.

The bounds count roundings: u = eps / 2 of the element type per rounding to it (bf16 2^-8, fp32 2^-24), f = 2^-24 per fp32 operation.  They are
computed per element from the same inputs, before any kernel has run."""
import math

import numpy as np
import torch

F = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def keep_mask(n, p, seed, step, layer=0):
    """Philox2x32-10 keep mask of n elements (numpy)."""
    M = np.uint64(0xFFFFFFFF)
    quad = np.arange((n + 3) // 4, dtype=np.uint64)
    a, b = quad & M, np.uint64(step & 0xFFFFFFFF) ^ ((quad >> np.uint64(32)) * np.uint64(0x85EBCA6B) & M)
    key = (seed ^ ((seed >> 32) * 0xC2B2AE35) ^ (layer * 0x27D4EB2F)) & 0xFFFFFFFF
    for _ in range(10):
        prod = a * np.uint64(0xD256D193)
        a, b = (prod >> np.uint64(32)) ^ np.uint64(key) ^ b, prod & M
        key = (key + 0x9E3779B9) & 0xFFFFFFFF
    u = np.stack([a & np.uint64(0xFFFF), a >> np.uint64(16), b & np.uint64(0xFFFF), b >> np.uint64(16)], 1).reshape(-1)[:n]
    return torch.from_numpy(u >= np.uint64(int(np.float32(p) * np.float32(65536.0) + np.float32(0.5))))


def layer_norm(x, gamma, beta, eps, dy=None, add=None):
    """Returns {name: (value, bound)}; x, dy, add in their element type, the rest fp32.
    fp32 sums of a row: at most 128 sequential additions and tree levels below C = 32768 -> 128 f of the sum of magnitudes."""
    dt = x.dtype
    u = U[dt]
    x, C = x.double(), x.shape[1]
    g = torch.ones(C, dtype=torch.double) if gamma is None else gamma.double()
    b = torch.zeros(C, dtype=torch.double) if beta is None else beta.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    e_mean = 130 * F * x.abs().mean(1, keepdim=True)                    # error of the mean
    # the variance moves by e_mean^2 (its slope in the mean is zero) and by 130 f of itself; rstd by half of that, and by its own operations
    r_rstd = 70 * F + 0.5 * (e_mean * rstd) ** 2
    xh = d * rstd
    e_xh = e_mean * rstd + xh.abs() * (r_rstd + 4 * F)
    y = xh * g + b
    out = dict(y=(y, e_xh * g.abs() + 4 * F * ((xh * g).abs() + b.abs()) + u * y.abs()), mean=(mean[:, 0], e_mean[:, 0] + F * mean[:, 0].abs()),
               rstd=(rstd[:, 0], (rstd * r_rstd)[:, 0] + 2 * F * rstd[:, 0]))
    if dy is not None:
        dy = dy.double()
        w = dy * g
        m1, m2 = w.mean(1, keepdim=True), (w * xh).mean(1, keepdim=True)
        e1 = 130 * F * w.abs().mean(1, keepdim=True)
        e2 = (134 * F * (w * xh).abs() + w.abs() * e_xh).mean(1, keepdim=True)
        dx = rstd * (w - m1 - xh * m2)
        mag = rstd * (w.abs() + m1.abs() + (xh * m2).abs())
        e_dx = rstd * (e1 + xh.abs() * e2 + m2.abs() * e_xh) + mag * (r_rstd + 8 * F)
        if add is not None:
            dx = dx + add.double()
            e_dx = e_dx + F * add.double().abs()
        # a weight gradient: every block adds its rows one after another, then the partial rows: at most R additions
        n = min(x.shape[0], 4096) + 64
        out.update(dx=(dx, e_dx + u * dx.abs()), dgamma=((dy * xh).sum(0), n * F * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)),
                   dbeta=(dy.sum(0), n * F * dy.abs().sum(0)))
    return out


def attention(q, k, v, q_len=None, k_len=None, causal=False, scale=None, d_o=None):
    """q [B,Tq,Hq,D], k / v [B,Tk,Hkv,D] on the CPU.  Returns {name: (value, bound)} for o, lse (and dq, dk, dv when d_o is given).

    s: fp32 products in bf16 tensors are exact in pairs and summed over D: (D + 4) f of sum |q||k|; fp32 tensors also drop products of planes,
    2^-20 of |q||k| (2 x 2^-7 x 2^-14, planes by truncation).  p = 2^(..) moves by the error of its exponent and 4 f.
    bf16 tensors round p and ds to bf16 before the second product (u each), and every output once (u)."""
    dt = q.dtype
    u = U[dt]
    up = u if dt == torch.bfloat16 else 2.0 ** -20                       # rounding (or dropped planes) of the second product's operands
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    z = lambda t: torch.zeros(t.shape, dtype=torch.double)
    val = dict(o=z(q), lse=torch.full((B, Hq, Tq), -math.inf, dtype=torch.double))
    err = dict(o=z(q), lse=torch.zeros(B, Hq, Tq, dtype=torch.double))
    if d_o is not None:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            val[n], err[n] = z(t), z(t)
    for b in range(B):
        n = Tq if q_len is None else max(0, min(Tq, int(q_len[b])))
        m = Tk if k_len is None else max(0, min(Tk, int(k_len[b])))
        lo = max(0, n - m) if causal else 0                               # rows before see no key
        if n <= lo or m == 0:
            continue
        hide = torch.ones(n, m, dtype=torch.bool).triu(m - n + 1)[lo:] if causal else torch.zeros(n - lo, m, dtype=torch.bool)
        for h in range(Hq):
            Q, K, V = q[b, lo:n, h].double(), k[b, :m, h // G].double(), v[b, :m, h // G].double()
            s = (Q @ K.T * scale).masked_fill(hide, -math.inf)
            es = ((D + 4) * F + (2.0 ** -20 if dt == torch.float32 else 0.0)) * (Q.abs() @ K.abs().T) * scale + 6 * F * s.abs().masked_fill(hide, 0.0)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            # a row's common shift cancels; both the weight and the normalisation move by at most the row's largest score error
            rp = 2 * es.masked_fill(hide, 0.0).amax(1, keepdim=True) + (8 + min(m, 1024)) * F
            o = p @ V
            A = p @ V.abs()
            val["o"][b, lo:n, h], err["o"][b, lo:n, h] = o, (up + rp + 40 * F) * A + u * o.abs()
            val["lse"][b, h, lo:n], err["lse"][b, h, lo:n] = lse[:, 0], rp[:, 0] + 8 * F * lse[:, 0].abs() + 8 * F
            if d_o is None:
                continue
            g = d_o[b, lo:n, h].double()
            dp = g @ V.T
            delta = (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_dp = ((D + 4) * F + (2.0 ** -20 if dt == torch.float32 else 0.0)) * (g.abs() @ V.abs().T)
            e_delta = (g.abs() * err["o"][b, lo:n, h]).sum(1, keepdim=True) + (D + 4) * F * (g * o).abs().sum(1, keepdim=True)
            # the backward's p is 2^(s - lse): lse is a rounded fp32 number
            rb = rp + 10 * F * lse.abs() + 10 * F
            e_ds = ds.abs() * (up + rb + 4 * F) + p * (e_dp + e_delta)
            ep = p * (up + rb)
            sums = (8 + min(n + m, 1024)) * F
            dq = scale * ds @ K
            val["dq"][b, lo:n, h], err["dq"][b, lo:n, h] = dq, scale * (e_ds + sums * ds.abs()) @ K.abs() + u * dq.abs()
            val["dk"][b, :m, h // G] += scale * ds.T @ Q
            err["dk"][b, :m, h // G] += scale * (e_ds + G * sums * ds.abs()).T @ Q.abs()
            val["dv"][b, :m, h // G] += p.T @ g
            err["dv"][b, :m, h // G] += (ep + G * sums * p).T @ g.abs()
    if d_o is not None:
        for n in ("dk", "dv"):
            err[n] += u * val[n].abs()
    return {n: (val[n], err[n]) for n in val}


def within(got, ref, name=""):
    """Every element inside its bound; infinities equal."""
    want, bound = ref
    got = got.detach().double().cpu()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), name
    d = (got - want).masked_fill(inf, 0.0).abs()
    assert torch.isfinite(got[~inf]).all(), (name, "non-finite")
    over = d > bound + 1e-30
    assert not over.any(), (name, int(over.sum()), float((d / (bound + 1e-30)).max()), float(d.max()))
