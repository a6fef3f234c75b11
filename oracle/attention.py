"""Sink attention in float64, one head at a time, with element-wise error bounds.

``attention(...)`` is the definition (causal, sliding window, kept first tokens,
learned sink logits, packed rows or key ranges); with ``dout`` also its
gradients.  ``bounds=True`` adds how far an implementation may be off that takes
its operands in bf16, sums in fp32, and rounds to bf16 four things: p (as an
operand), dz (as an operand), the output and the results.  A first delta0 = do .
out gives dz0 = p (g - delta0), g = do . v; the fp32 sums of dz0 and of p k then
give delta = delta0 (1 - p_sink) + sum dz0 and dq = scale (sum dz0 k - (delta -
delta0) sum p k).  A rounding to bf16 is off by at most u = 2^-8 of the value.  With
e_z the error of z (fp32 sum of D products, relative to the sum of magnitudes,
and the scaling before the exponential) p has the relative error r = e_z + 2^-21:

    |out|     u |out| + (u + r) p |v|
    |delta0|  d0 = |do| . |out error|                 (+ its own fp32 sum)
    |delta|   d1 = r sum p (|do| |v| + |delta| + d0)  (p_sink among the p, + the fp32 sums)
    |dz|      (u + r) |dz| + p d1 + r p (|do| |v| + |delta|)
    |dv|      u |dv| + (u + r) p^T |do|
    |dk|      u |dk| + scale (dz error)^T |q|
    |dq|      u |dq| + scale ((u + r) (|dz| + 2 p d0) + p d1 + r p (|do| |v| + |delta| + d0)) |k|  (+ fp32 sums)
    |dsink|   sum p_sink (d1 + r |delta|) (+ u |dsink| in bf16)
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -8
U32 = 2.0 ** -24


def visible(Sq, Sk, window=0, first=0, starts=None, kv_range=None):
    """[Sq, Sk] truth values; ``starts`` [Sk] or ``kv_range`` (begin, end) as in the operator."""
    pos = torch.arange(Sq)[:, None] + (Sk - Sq)
    key = torch.arange(Sk)[None, :]
    lo = torch.zeros_like(pos)
    hi = Sk
    if starts is not None:
        lo = starts.cpu().long()[:, None]
    if kv_range is not None:
        lo = torch.full_like(pos, min(max(int(kv_range[0]), 0), Sk))
        hi = min(max(int(kv_range[1]), 0), Sk)
    ok = (key >= lo) & (key < hi) & (key <= pos)
    if window:
        ok &= (key > pos - window) | (key < lo + first)
    return ok


def starts_of(cu, n):
    """Start of each token's sequence; t + 1 for a token in none."""
    s = torch.arange(n) + 1
    for a, b in zip(cu, cu[1:]):
        s[max(a, 0):b] = max(a, 0)
    return s


def attention(q, k, v, sinks=None, *, scale=None, window=0, first=0, cu_seqlens=None, kv_range=None, dout=None,
              bounds=False):
    """q [B, Hq, Sq, D], k, v [B, Hkv, Sk, D], dout [B, Sq, Hq, D] -> dict of float64 CPU tensors
    (out [B, Sq, Hq, D], dq, dk, dv, dsinks) and, with ``bounds``, ``name + "_tol"`` of each."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    (B, Hq, Sq, D), (Hkv, Sk) = q.shape, k.shape[1:3]
    G = Hq // Hkv
    c = D ** -0.5 if scale is None else scale
    starts = starts_of(cu_seqlens, Sk) if cu_seqlens is not None else None
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64)
    res = {"out": out}
    if bounds:
        res["out_tol"] = torch.zeros_like(out)
    if dout is not None:
        dout = dout.detach().cpu().double()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            res[n] = torch.zeros_like(t)
            if bounds:
                res[n + "_tol"] = torch.zeros_like(t)
        if sinks is not None:
            res["dsinks"] = torch.zeros(Hq, dtype=torch.float64)
            res["dsinks_tol"] = torch.zeros(Hq, dtype=torch.float64)
    u_sink = U if sinks is not None and sinks.dtype == torch.bfloat16 else 0.0
    for b in range(B):
        ok = visible(Sq, Sk, window, first, starts, None if kv_range is None else kv_range[b])
        # keys no query sees have no influence, whatever they hold
        used = ok.any(0)[:, None]
        kb = torch.where(used, k[b], 0.0)
        vb = torch.where(used, v[b], 0.0)
        for h in range(Hq):
            qh, kh, vh = q[b, h], kb[h // G], vb[h // G]
            z = torch.where(ok, c * (qh @ kh.T), -math.inf)
            top = z.amax(1, keepdim=True) if Sk else torch.full((Sq, 1), -math.inf, dtype=torch.float64)
            if sinks is not None:
                sink = sinks[h].detach().cpu().double()
                top = top.clamp(min=sink)
            top = torch.where(top == -math.inf, 0.0, top)
            e = torch.exp(z - top)
            den = e.sum(1, keepdim=True)
            if sinks is not None:
                den = den + torch.exp(sink - top)
            den = torch.where(den == 0, 1.0, den)
            p = e / den
            o = p @ vh
            out[b, :, h] = o
            if bounds:
                # z: an fp32 sum of D exact products, and z log2(e) - max rounded once (|argument| of the exponential)
                ez = c * 2 * math.sqrt(D) * U32 * (qh.abs() @ kh.abs().T) + 4 * U32 * (torch.where(ok, z, 0.0).abs() + top.abs())
                r = torch.where(ok, ez, 0.0) + 2.0 ** -21
                o_tol = U * o.abs() * 1.01 + ((U + r) * p) @ vh.abs() * 1.01 + 1e-30
                res["out_tol"][b, :, h] = o_tol
            if dout is None:
                continue
            do = dout[b, :, h]
            delta = (do * o).sum(1, keepdim=True)
            g = do @ vh.T
            dz = p * (g - delta)
            res["dv"][b, h // G] += p.T @ do
            res["dq"][b, h] = c * (dz @ kh)
            res["dk"][b, h // G] += c * (dz.T @ qh)
            if sinks is not None:
                ps = torch.exp(sink - top) / den
                res["dsinks"][h] -= (ps * delta).sum()
            if not bounds:
                continue
            d_tol = (do.abs() * o_tol).sum(1, keepdim=True) + 2 * math.sqrt(D) * U32 * (do * o).abs().sum(1, keepdim=True)
            g_mag = do.abs() @ vh.abs().T + delta.abs()
            rd, n32 = r + 2 * math.sqrt(D) * U32, 2 * math.sqrt(max(Sk, 1)) * U32
            d1 = (rd * p * (g_mag + d_tol) + n32 * (dz.abs() + p * d_tol)).sum(1, keepdim=True) + 8 * U32 * (delta.abs() + d_tol)
            if sinks is not None:
                d1 = d1 + (r.amax(1, keepdim=True) if Sk else 2.0 ** -21) * ps * (delta.abs() + d_tol)
            z_tol = (U + r) * dz.abs() + p * d1 + rd * p * g_mag
            q_tol = (U + r + n32) * (dz.abs() + 2 * p * d_tol) + p * d1 + rd * p * (g_mag + d_tol)
            res["dv_tol"][b, h // G] += 1.01 * ((U + r) * p).T @ do.abs()
            res["dq_tol"][b, h] = 1.01 * c * (q_tol @ kh.abs()) + 1e-30
            res["dk_tol"][b, h // G] += 1.01 * c * (z_tol.T @ qh.abs())
            if sinks is not None:
                res["dsinks_tol"][h] += 1.01 * (ps * (d1 + (r.max() if Sk else 2.0 ** -21) * delta.abs())).sum() + \
                    2 * math.sqrt(B * Sq) * U32 * (ps * delta.abs()).sum() + 1e-30
    if bounds and dout is not None:
        for n in ("dq", "dk", "dv"):
            res[n + "_tol"] += 1.01 * U * res[n].abs() + 1e-30
        if sinks is not None:
            res["dsinks_tol"] += 1.01 * u_sink * res["dsinks"].abs()
    return res
