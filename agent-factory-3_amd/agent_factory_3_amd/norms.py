"""Root-mean-square norms with the residual stream on the MI355X.

``residual_norm`` adds a block's output to the residual stream and normalises the
sum for the next block, in one pass over the data (gpt-oss's layers do it in
several: transformers' GptOssDecoderLayer adds, GptOssRMSNorm converts, squares,
scales and converts back); the block's output may have a norm of its own, a gate
and a scale.  ``rms_norm`` is the norm alone.  Both are differentiable in every
tensor.  The HIP kernels are behind ``af3_residual_norm_fwd`` / ``_bwd``; there is
no CPU fallback.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _capi
from .routing import _device_of, _no_forward_mode, _once

MIN_HIDDEN, MAX_HIDDEN = 8, 16384
_TYPES = (torch.bfloat16, torch.float32)


def _rows(t: torch.Tensor):
    """[..., H] as a tensor of contiguous rows evenly apart, and the rows' stride."""
    if t.is_contiguous():   # (as it is: only its address is used)
        return t, t.shape[-1]
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _like(t: torch.Tensor, shape, dtype):
    """A new contiguous tensor of that shape and type (of t's, where t has them: the shorter call)."""
    if t.dtype == dtype and t.shape == shape and t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(shape, dtype=dtype, device=t.device)


def _f32(t) -> int:
    return int(t is not None and t.dtype == torch.float32)


@functools.lru_cache(maxsize=64)
def _bwd_workspace(rows, H, full, gate_cols, gate_rows, w, post, gate) -> int:
    return int(_capi.load().af3_residual_norm_bwd_workspace_bytes(rows, H, full, gate_cols, gate_rows, w, post, gate))


def _forward(x, residual, weight, post, gate, gate_rows, scale, eps, stats):
    """(r, h, 1 / rms of r, 1 / rms of x); r None without a residual, h None without a weight."""
    H = x.shape[-1]
    n = x.numel() // H
    dev = x.device
    x2, ldx = _rows(x)
    r = h = rstd = rstd_x = None
    res, ldr = (None, 0) if residual is None else _rows(residual)
    if residual is not None:
        r = _like(residual, residual.shape, residual.dtype)
    if weight is not None:
        h = _like(x, x.shape, x.dtype)
        rstd = torch.empty(n, dtype=torch.float32, device=dev) if stats else None
    if post is not None and stats:
        rstd_x = torch.empty(n, dtype=torch.float32, device=dev)
    ptr = _capi.ptr
    _capi.call("af3_residual_norm_fwd", x2.data_ptr(), _f32(x), ldx, ptr(res), _f32(residual), ldr, ptr(weight),
               _f32(weight), ptr(post), _f32(post), ptr(gate), _f32(gate), _cols(gate),
               gate_rows, scale, eps, n, H, ptr(r), ptr(h), ptr(rstd), ptr(rstd_x), _capi.stream_of(dev))
    return r, h, rstd, rstd_x


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, post, gate, gate_rows, scale, eps):
        r, h, rstd, rstd_x = _forward(x, residual, weight, post, gate, gate_rows, scale, eps, True)
        # r for the backward: as stored, or, for a weight's gradient beside a bf16 stream, made again from x and residual
        again = residual is not None and ctx.needs_input_grad[2] and residual.dtype == torch.bfloat16
        keep_x = residual is None or again or post is not None or gate is not None
        ctx.save_for_backward(x if keep_x else None, None if weight is None else residual if again else r, weight, post,
                              gate, rstd, rstd_x)
        full = residual is not None and (post is not None or gate is not None)
        rt = None if residual is None else residual.dtype
        # without norm, gate and scale the branch has the stream's own gradient, returned for both
        same = not full and (rt is None or (scale == 1.0 and x.dtype == rt))
        ctx.args = (x.shape, x.numel() // x.shape[-1], x.dtype, rt, gate_rows, scale, full, same, again)
        ctx.set_materialize_grads(False)
        if residual is None:
            return h
        return (r, h) if weight is not None else r

    @staticmethod
    @_once
    def backward(ctx, *grads):
        _no_forward_mode("residual_norm backward", *grads)
        dr, dh = (None, grads[0]) if ctx.args[3] is None else grads if len(grads) == 2 else (grads[0], None)
        some = dr if dr is not None else dh
        if some is None:
            return (None,) * 8
        if some.get_device() == torch.cuda.current_device():
            return _ResidualNorm._gradients(ctx, dr, dh, some)
        with torch.cuda.device(some.device):
            return _ResidualNorm._gradients(ctx, dr, dh, some)

    @staticmethod
    def _gradients(ctx, dr, dh, some):
        x, r, weight, post, gate, rstd, rstd_x = ctx.saved_tensors
        shape, n, xt, rt, gate_rows, scale, full, same, again = ctx.args
        need_x, need_res, need_w, need_post, need_gate = ctx.needs_input_grad[:5]
        H = shape[-1]
        p_dr = p_dh = p_r = p_x = p_w = p_rstd = p_post = p_rstd_x = p_gate = p_dx = p_dres = p_dw = p_ws = None
        lddr = lddh = ldx = ldr = cols = w32 = ws_n = 0
        dx = dres = dw = dpost = dgate = None
        # (saved-tensor hooks, as those that keep them on the host, may give them other strides)
        if dr is not None:
            dr, lddr = _rows(dr)
            p_dr = dr.data_ptr()
        if dh is not None:
            dh, lddh = _rows(dh)
            weight, rstd = weight.contiguous(), rstd.contiguous()
            p_dh, p_w, p_rstd, w32 = dh.data_ptr(), weight.data_ptr(), rstd.data_ptr(), _f32(weight)
        else:
            need_w = again = False
        if x is not None:
            x, ldx = _rows(x)
            p_x = x.data_ptr()
        if rt is None:
            p_r, ldr = p_x, ldx
        elif r is not None:
            r, ldr = _rows(r)
            p_r = r.data_ptr()
        if full:
            if post is not None:
                post, rstd_x = post.contiguous(), rstd_x.contiguous()
                p_post, p_rstd_x = post.data_ptr(), rstd_x.data_ptr()
            if gate is not None:
                gate, cols = gate.contiguous(), _cols(gate)
                p_gate = gate.data_ptr()
        if need_res or (need_x and same):
            dres = _like(some, shape, rt or xt)
            p_dres = dres.data_ptr()
        if need_x:
            if same:
                dx = dres
            else:
                dx = _like(some, shape, xt)
                p_dx = dx.data_ptr()
        if not n:
            return (dx, dres if need_res else None, *(torch.zeros_like(t) if need else None for t, need in
                                                      ((weight, need_w), (post, need_post), (gate, need_gate))),
                    None, None, None)
        if need_w or again:
            dw = torch.empty_like(weight)
            p_dw = dw.data_ptr()
        if need_post:
            dpost = torch.empty_like(post)
        if need_gate:
            dgate = torch.empty_like(gate)
        if p_dw is not None or need_post or need_gate:
            ws_n = _bwd_workspace(n, H, int(full), cols, gate_rows, p_dw is not None, need_post, need_gate)
            if ws_n:
                ws = torch.empty(ws_n, dtype=torch.uint8, device=some.device)
                p_ws = ws.data_ptr()
        _capi.call("af3_residual_norm_bwd", p_dr, lddr, p_dh, lddh, p_r, int((rt or xt) == torch.float32), int(again), ldr,
                   p_x, int(xt == torch.float32), ldx, p_rstd, p_rstd_x, p_w, w32, p_post, _f32(post), p_gate,
                   _f32(gate), cols, gate_rows, scale, int(rt is not None), n, H, p_dx, p_dres, p_dw, _capi.ptr(dpost),
                   _capi.ptr(dgate), p_ws, ws_n, _capi.stream_of(some.device))
        return dx, dres if need_res else None, dw, dpost, dgate, None, None, None


def _check_tensor(who, name, t, device):
    if not t.is_cuda:
        raise RuntimeError(f"{who}: {name} must be a GPU tensor (the MI355X path has no CPU implementation)")
    if t.dtype not in _TYPES:
        raise TypeError(f"{who}: {name} must be bfloat16 or float32 (got {t.dtype})")
    if t.device != device:
        raise ValueError(f"{who}: {name} is on {t.device}, x on {device}")
    if not t.data_ptr() and t.numel():
        raise TypeError(f"{who}: {name} is a {type(t).__name__} without memory of its own (of a DTensor, pass the local tensor)")


def _check(who, x, weight, post, eps):
    device, shape = x.device, x.shape
    _check_tensor(who, "x", x, device)
    H = shape[-1] if shape else 0
    if not MIN_HIDDEN <= H <= MAX_HIDDEN:
        raise ValueError(f"{who}: x must be [..., H] with H from {MIN_HIDDEN} to {MAX_HIDDEN}, got {tuple(shape)}")
    if weight is not None:
        _check_weight(who, "weight", weight, device, H)
    if post is not None:
        _check_weight(who, "post_weight", post, device, H)
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"{who}: eps must not be negative, got {eps}")


def _check_weight(who, name, t, device, H):
    _check_tensor(who, name, t, device)
    if t.shape != (H,):
        raise ValueError(f"{who}: {name} must be [{H}], got {tuple(t.shape)}")


def _gate_rows(gate, shape):
    """The gate as rows of 1 or H in a row, and the rows of x that share each of its rows."""
    if gate.dim() > len(shape) or any(g not in (1, s) for g, s in zip(gate.shape[::-1], shape[::-1])):
        raise ValueError(f"residual_norm: a gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape)
    cols, lead = lead[-1], lead[:-1]
    k = len(lead)   # dimensions from k on are shared
    while k and lead[k - 1] == 1:
        k -= 1
    if any(g != s for g, s in zip(lead[:k], shape)):   # shared along outer dimensions only: a row for each,
        # in fp32, so that the gradient is rounded once, after torch's sum over them
        gate, k = gate.float().expand(*shape[:-1], cols), len(lead)
    return gate if gate.is_contiguous() else gate.contiguous(), math.prod(shape[k:-1])


def _cols(gate) -> int:
    return 0 if gate is None else gate.shape[-1] if gate.dim() else 1


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """``weight * x / sqrt(mean(x^2) + eps)`` over the last dimension, rounded once.

    Args:
        x: [..., H] bf16 or fp32, H from 8 to 16384; rows contiguous (others are copied)
        weight: [H] bf16 or fp32
    Returns:
        [..., H] in x's type
    """
    _no_forward_mode("rms_norm", x, weight)
    eps = float(eps)
    _check("rms_norm", x, weight, None, eps)
    with _device_of(x):
        weight = weight if weight.is_contiguous() else weight.contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
            return _ResidualNorm.apply(x, None, weight, None, None, 1, 1.0, eps)
        return _forward(x, None, weight, None, None, 1, 1.0, eps, False)[1]


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None, *, eps: float = 1e-5,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0):
    """A block's output joins the residual stream, and the next block's norm:

        u = x,  or  post_weight * x / sqrt(mean(x^2) + eps)
        r = residual + scale * gate * u
        h = weight * r / sqrt(mean(r^2) + eps)

    Statistics and products are fp32, h is made from r before its rounding, and each
    result is rounded once; sums over rows are in a fixed order.  Where x takes the
    stream's gradient as it is (no norm, gate or scale of its own, one type), both
    get the same tensor, as from torch's add.

    Args:
        x: [..., H] bf16 or fp32, H from 8 to 16384
        residual: the same shape, in x's type or fp32
        weight: [H] bf16 or fp32; None: only r is made
        post_weight: [H] of the block's own norm, or None
        gate: bf16 or fp32, broadcast to x: [H], [B, 1, H], [B, S, 1], ...; or None
    Returns:
        (r in residual's type, h in x's type or None)
    """
    _no_forward_mode("residual_norm", x, residual, weight, post_weight, gate)
    eps, scale = float(eps), float(scale)
    _check("residual_norm", x, weight, post_weight, eps)
    _check_tensor("residual_norm", "residual", residual, x.device)
    if residual.shape != x.shape:
        raise ValueError(f"residual_norm: x is {tuple(x.shape)}, the residual {tuple(residual.shape)}")
    if x.dtype == torch.float32 and residual.dtype != torch.float32:
        raise TypeError(f"residual_norm: a float32 x needs a float32 residual (got {residual.dtype})")
    if not math.isfinite(scale):
        raise ValueError(f"residual_norm: scale must be finite, got {scale}")
    if gate is not None:
        _check_tensor("residual_norm", "gate", gate, x.device)
    with _device_of(x):
        gate_rows = 1
        if gate is not None:
            gate, gate_rows = _gate_rows(gate, x.shape)
            gate_rows = max(gate_rows, 1)
        weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
        post_weight = post_weight if post_weight is None or post_weight.is_contiguous() else post_weight.contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad
                                        or (weight is not None and weight.requires_grad)
                                        or (post_weight is not None and post_weight.requires_grad)
                                        or (gate is not None and gate.requires_grad)):
            out = _ResidualNorm.apply(x, residual, weight, post_weight, gate, gate_rows, scale, eps)
            return out if weight is not None else (out, None)
        return _forward(x, residual, weight, post_weight, gate, gate_rows, scale, eps, False)[:2]
