"""Projections on the MI355X: a matrix product with bias, activation and residual in its epilogue.

``linear`` is ``act(x W^T + b) + residual`` rounded once, differentiable in x, the
weight, the bias and the residual; gpt-oss's attention projections are calls of
nn.functional.linear, with the residual's add a pass of its own.  The HIP kernels
(one for the three products of a step, a weight-streaming one for a few rows) are
behind ``af3_linear`` and ``af3_linear_dz``; there is no CPU fallback.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _capi
from .routing import _device_of, _no_forward_mode, _once

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
SKINNY_ROWS = 32     # rows of x up to which the forward streams the weight (any alignment)
_MAX_STRIDE = 1 << 22


def _rows(t: torch.Tensor):
    """[..., C] as [rows, C] with contiguous rows."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _aligned(t: torch.Tensor):
    """(tensor, row stride) of [rows, C] as the tiled kernel reads it: rows at 16-byte
    aligned addresses that reach the next multiple of 8 elements, zeros there.  Others are copied."""
    C, ld = t.shape[1], t.stride(0)
    if C % 8 == 0 and t.data_ptr() % 16 == 0:
        if t.shape[0] == 1:
            return t, C
        if ld % 8 == 0 and C <= ld < _MAX_STRIDE:
            return t, ld
    width = (C + 7) // 8 * 8
    c = torch.empty((t.shape[0], width), dtype=t.dtype, device=t.device)
    _capi.call("af3_linear_dz", t.data_ptr(), ld, None, 0, t.shape[0], C, c.data_ptr(), width, None, 0, None, 0,
               _capi.stream_of(t.device))   # (without an activation: a copy with zeros after each row)
    return c, width


@functools.lru_cache(maxsize=256)
def _workspace(M, N, K) -> int:
    return int(_capi.load().af3_linear_workspace_bytes(M, N, K, 0, 0))


@functools.lru_cache(maxsize=256)
def _bwd_workspace(T, N, K, dx, dw, db) -> int:
    return int(_capi.load().af3_linear_bwd_workspace_bytes(T, N, K, dx, dw, db))


def _forward(x, weight, bias, act, residual, keep_z):
    """(y, z): the output, and the sums before the activation where they are kept."""
    N, K = weight.shape
    shape = (*x.shape[:-1], N)
    y = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    x2 = _rows(x)
    T = x2.shape[0]
    z = torch.empty(T, N, dtype=torch.bfloat16, device=x.device) if keep_z and act else None
    if T:
        w = weight if weight.stride(1) == 1 or K == 1 else weight.contiguous()
        if T <= SKINNY_ROWS:
            (p, ldp), (q, ldq) = (x2, x2.stride(0)), (w, w.stride(0))
        else:
            (p, ldp), (q, ldq) = _aligned(x2), _aligned(w)
        res = None if residual is None else _rows(residual)
        ws_n = _workspace(T, N, K)
        ws = torch.empty(ws_n, dtype=torch.uint8, device=x.device) if ws_n else None
        ptr = _capi.ptr
        _capi.call("af3_linear", p.data_ptr(), ldp, 0, q.data_ptr(), ldq, 0, T, N, K, ptr(bias),
                   int(bias is not None and bias.dtype == torch.float32), act, ptr(res),
                   0 if res is None else res.stride(0), y.data_ptr(), ptr(z), ptr(ws), ws_n, _capi.stream_of(x.device))
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = _forward(x, weight, bias, act, residual, True)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        ctx.save_for_backward(x if need_w else None, weight if need_x else None, z)
        ctx.args = (x.shape, tuple(weight.shape), None if bias is None else bias.dtype, act)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        _no_forward_mode("linear backward", dy)
        x, weight, z = ctx.saved_tensors
        x_shape, (N, K), bias_type, act = ctx.args
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        T = math.prod(x_shape[:-1])
        dx = dw = db = None
        if need_x or need_w or need_b:
            with _device_of(dy):
                new, dev = (torch.empty if T else torch.zeros), dy.device
                if need_x:
                    dx = new(x_shape, dtype=torch.bfloat16, device=dev)
                if need_w:
                    dw = new((N, K), dtype=torch.bfloat16, device=dev)
                if need_b:
                    db = new(N, dtype=bias_type, device=dev)
                if T:
                    _Linear._gradients(_rows(dy), x, weight, z, act, T, N, K, dx, dw, db)
        return dx, dw, db, dy if need_res else None, None

    @staticmethod
    def _gradients(dy, x, weight, z, act, T, N, K, dx, dw, db):
        dev = dy.device
        ldy = dy.stride(0) if T > 1 else N
        dz = ws = p_w = p_x = None
        ldz = ldw = ldx = 0
        # dz in a tensor of its own: behind an activation, or where dy's rows are not as the products read them
        if (dx is not None or dw is not None) and (act or N % 8 or ldy % 8 or dy.data_ptr() % 16
                                                   or not N <= ldy < _MAX_STRIDE):
            ldz = (N + 7) // 8 * 8
            dz = torch.empty((T, ldz), dtype=torch.bfloat16, device=dev)
        if dx is not None:
            weight, ldw = _aligned(_rows(weight))
            p_w = weight.data_ptr()
        if dw is not None:
            x, ldx = _aligned(_rows(x))
            p_x = x.data_ptr()
        z = z if z is None else z.contiguous()
        ws_n = _bwd_workspace(T, N, K, dx is not None, dw is not None, db is not None)
        if ws_n:
            ws = torch.empty(ws_n, dtype=torch.uint8, device=dev)
        ptr = _capi.ptr
        _capi.call("af3_linear_bwd", dy.data_ptr(), ldy, ptr(z), act, p_w, ldw, p_x, ldx, T, N, K, ptr(dz), ldz, ptr(dx),
                   ptr(dw), ptr(db), int(db is not None and db.dtype == torch.float32), ptr(ws), ws_n, _capi.stream_of(dev))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x W^T + b) + residual``, with fp32 sums and one rounding.

    For the backward of an activation its argument is kept in bf16, and the gradient that
    passes it is rounded to bf16 as the operand of its products (about one more rounding
    of dx, the weight's and the bias's gradient; none without an activation).  Every sum
    is in a fixed order.  Without an activation the residual's gradient is the one that
    arrives, unchanged.

    Args:
        x: [..., K] bf16
        weight: [N, K] bf16
        bias: [N] bf16 or fp32, or None
        activation: None, "relu", "silu", "gelu" (by the error function) or "gelu_tanh"
        residual: [..., N] bf16, added after the activation; or None
    Rows that are not 16-byte aligned, or whose length is not a multiple of 8, are copied
    to rows that are (past 32 rows of x, and in the backward).
    Returns:
        [..., N] bf16
    """
    _no_forward_mode("linear", x, weight, bias, residual)
    device = x.device
    for name, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None or (t.dtype is torch.bfloat16 and t.is_cuda and (t is x or t.device == device) and t.data_ptr()):
            continue
        if not t.is_cuda:
            raise RuntimeError(f"linear: {name} must be a GPU tensor (the MI355X path has no CPU implementation)")
        if t.dtype != torch.bfloat16 and not (name == "bias" and t.dtype == torch.float32):
            raise TypeError(f"linear: {name} must be bfloat16{' or float32' if name == 'bias' else ''} (got {t.dtype})")
        if t.device != device:
            raise ValueError(f"linear: {name} is on {t.device}, x on {device}")
        if not t.data_ptr() and t.numel():
            raise TypeError(f"linear: {name} is a {type(t).__name__} without memory of its own (of a DTensor, pass the "
                            "local tensor)")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    N, K = weight.shape
    if N == 0 or K == 0 or max(N, K) >= _MAX_STRIDE:
        raise ValueError(f"linear: a weight of shape {tuple(weight.shape)}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"linear: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise ValueError(f"linear: residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation {activation!r} is not one of {list(ACTIVATIONS)}")
    if x.numel() // K >= 1 << 30:
        raise ValueError("linear: too many rows")
    act = ACTIVATIONS[activation]
    with _device_of(x):
        bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                        or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad)):
            return _Linear.apply(x, weight, bias, residual, act)
        return _forward(x, weight, bias, act, residual, False)[0]
