"""Residual norms in float64: values, gradients by the formulas, and error bounds of an
implementation that works in fp32, stores r and rounds each result once."""
import torch


def _rms(v, eps):
    return 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def half_step(dtype):
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def residual_norm(x, residual=None, weight=None, *, eps=1e-5, post=None, gate=None, scale=1.0, dr=None, dh=None):
    """Tensors on the CPU in their own types, x [rows, H], gate broadcast to x.  A dict of float64 results
    (r, h; with dr or dh the gradients) and, as name + "_tol", their bounds:

    fp32 steps are 2^-24 each.  A sum over H (at most 32 additions in a lane, 9 across lanes and waves) makes a
    root mean square's reciprocal off by 2^-19 of it, a dot product by 2^-18 of the sum of its magnitudes; products
    of a few factors by 2^-21.  Sums over rows: at most 1000 additions in a chain are 2^-14 of the sum of magnitudes.
    """
    u_x = half_step(x.dtype)
    u_r = half_step(residual.dtype if residual is not None else x.dtype)
    types = {"dweight": weight, "dpost_weight": post, "dgate": gate}
    types = {k: v.dtype for k, v in types.items() if v is not None}
    gate_shape = None if gate is None else gate.shape
    x = x.double()
    w, p, g, dr, dh, res = (None if t is None else t.double() for t in (weight, post, gate, dr, dh, residual))
    o = {}
    e_r = torch.zeros_like(x)
    r = x
    if res is not None:
        sx = _rms(x, eps) if p is not None else None
        u = x if p is None else x * sx * p
        k = scale * (g if g is not None else 1.0) * torch.ones_like(x)
        r = res + k * u
        e_r = 2.0 ** -21 * (res.abs() + (k * u).abs()) + (2.0 ** -19 * (k * u).abs() if p is not None else 0)
        o["r"], o["r_tol"] = r, u_r * r.abs() + e_r
    s = _rms(r, eps)
    e_s = 2.0 ** -19 + e_r.norm(dim=-1, keepdim=True) / r.norm(dim=-1, keepdim=True).clamp(min=1e-300)  # relative
    if w is not None:
        o["h"] = w * r * s
        o["h_tol"] = u_x * o["h"].abs() + o["h"].abs() * (e_s + 2.0 ** -21) + (w * s).abs() * e_r
    if dr is None and dh is None:
        return o
    G, e_g = torch.zeros_like(x), torch.zeros_like(x)
    if dr is not None:
        G, e_g = G + dr, e_g + 2.0 ** -23 * dr.abs()
    if dh is not None:
        d_r = (u_r * r.abs() + e_r) if res is not None else e_r   # r is read as it was stored
        dw = dh * w
        m, am = (dw * r).mean(-1, keepdim=True), (dw * r).abs().mean(-1, keepdim=True)
        G = G + s * (dw - r * s * s * m)
        e_m = (dw.abs() * d_r).mean(-1, keepdim=True) + 2.0 ** -18 * am
        e_g = e_g + s ** 3 * (r.abs() * e_m + d_r * m.abs()) + (3 * e_s + 2.0 ** -20) * (s * dw.abs() + s ** 3 * r.abs() * am)
        o["dweight"] = (dh * r * s).sum(0)
        # (over a bf16 stream r is made again for it)
        o["dweight_tol"] = ((dh * s).abs() * (e_r if u_r > 2.0 ** -20 else d_r) + (e_s + 2.0 ** -14) * (dh * r * s).abs()).sum(0)
    if res is None:
        o["dx"], o["dx_tol"] = G, u_x * G.abs() + e_g
    else:
        o["dresidual"], o["dresidual_tol"] = G, u_r * G.abs() + e_g
        du, e_du = k * G, k.abs() * (e_g + 2.0 ** -21 * G.abs())
        if g is not None:
            dg, e_dg = scale * G * u, abs(scale) * (u.abs() * e_g + 2.0 ** -14 * (G * u).abs())
            o["dgate"], o["dgate_tol"] = dg.sum_to_size(gate_shape), e_dg.sum_to_size(gate_shape)
        if p is not None:
            t, e_t = du * p, e_du * p.abs()
            m, am = (t * x).mean(-1, keepdim=True), (t * x).abs().mean(-1, keepdim=True)
            e_m = (e_t * x.abs()).mean(-1, keepdim=True) + 2.0 ** -18 * am
            o["dx"] = sx * (t - x * sx * sx * m)
            o["dx_tol"] = (u_x * o["dx"].abs() + sx * e_t + sx ** 3 * x.abs() * e_m
                           + 2.0 ** -17 * (sx * t.abs() + sx ** 3 * x.abs() * am))
            o["dpost_weight"] = (du * x * sx).sum(0)
            o["dpost_weight_tol"] = ((x * sx).abs() * e_du + 2.0 ** -14 * (du * x * sx).abs()).sum(0)
        else:
            o["dx"], o["dx_tol"] = du, u_x * du.abs() + e_du
    for n, t in types.items():
        if n in o:
            o[n + "_tol"] = o[n + "_tol"] + half_step(t) * o[n].abs()
    return o
