"""A projection with bias, activation and residual in float64: values, gradients by the formulas, and
error bounds of an implementation with fp32 sums that rounds each result once, keeps the activation's
argument in bf16 and rounds the gradient behind it to bf16."""
import math

import torch

BF = 2.0 ** -8    # one rounding to bf16, relative


def act(z, name):
    """The activation, its derivative, and a bound of the second derivative's magnitude."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 0.5
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 0.134145 * z * z), 0.8
    return z, torch.ones_like(z), 0.0


def linear(x, weight, bias=None, activation=None, residual=None, dy=None):
    """[T, K], [N, K] tensors on the CPU.  A dict of float64 results and, as name + "_tol", their bounds: a sum of n
    products in fp32 is off by at most 2^-24 times its number of additions in a row (a matrix instruction adds 16 or
    32 products, then one of n / 16 results; up to 16 partial sums) of the sum of magnitudes: n / 16 + 48 of them."""
    types = None if bias is None else bias.dtype
    x, weight, bias, residual, dy = (None if t is None else t.double() for t in (x, weight, bias, residual, dy))
    n = lambda k: 2.0 ** -24 * (k / 16 + 48)  # noqa: E731
    z = x @ weight.t()
    e_z = n(x.shape[1]) * (x.abs() @ weight.abs().t())
    if bias is not None:
        z, e_z = z + bias, e_z + 2.0 ** -24 * (z.abs() + bias.abs())
    y, slope, curve = act(z, activation)
    # fp32 activations: an exponential of up to 88 after five roundings, 5 * 88 * 2^-24 < 2^-15 of the value, and as
    # much for the rest; 0 where the exponential leaves fp32 (values below |z| e^-87 < 2^-118)
    e_y = e_z if activation is None else 1.2 * e_z + 2.0 ** -14 * y.abs() + 2.0 ** -118
    if residual is not None:
        y, e_y = y + residual, e_y + 2.0 ** -24 * (y.abs() + residual.abs())
    o = {"y": y, "y_tol": BF * y.abs() + e_y}
    if dy is None:
        return o
    dz, e_dz, e_db = dy, torch.zeros_like(dy), torch.zeros_like(dy)
    if activation is not None:
        d_z = BF * z.abs() + e_z     # z is kept in bf16
        dz = dy * slope
        e_db = dy.abs() * (curve * d_z + 2.0 ** -18)
        if activation == "relu":     # a sum within its error of 0 may fall on either side
            e_db = dy.abs() * (z.abs() <= e_z)
        e_dz = e_db + BF * dz.abs()
    if residual is not None:
        o["dresidual"], o["dresidual_tol"] = dy, torch.zeros_like(dy)
    T, N = dy.shape
    o["dx"] = dz @ weight
    o["dx_tol"] = BF * o["dx"].abs() + e_dz @ weight.abs() + n(N) * (dz.abs() @ weight.abs())
    o["dweight"] = dz.t() @ x
    o["dweight_tol"] = BF * o["dweight"].abs() + e_dz.t() @ x.abs() + n(T) * (dz.abs().t() @ x.abs())
    if bias is not None:
        o["dbias"] = dz.sum(0)
        half = torch.finfo(types).eps / 2
        o["dbias_tol"] = half * o["dbias"].abs() + e_db.sum(0) + 2.0 ** -24 * (T / 8 + 1100) * dz.abs().sum(0)
    return o
