"""gpt-oss attention on the MI355X: a sliding window, kept first tokens, learned sinks.

``sink_attention`` is causal attention with one learned logit per query head
added to the softmax's denominator (``GptOssAttention.sinks``), over every
earlier token or a sliding window, optionally keeping a sequence's first tokens
visible; differentiable in q, k, v and the sinks, over a batch, a packed row of
sequences (the reference's collator packs them, data_collator_with_packing.py:
5-93) or a few new tokens at the end of a cache.  The HIP kernels are behind
``af3_sink_attention_fwd`` / ``_bwd``; there is no CPU fallback.

``register`` makes it transformers' ``attn_implementation="af3_sink"`` (importing
``quantizer_config`` calls it): gpt-oss has no sdpa form there, its flash forms
with sinks are CUDA kernels, and its eager form holds the [heads, S, S] scores.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _capi
from .routing import _device_of, _no_forward_mode

HEAD_DIMS = (64, 128)
MAX_GROUP = 128       # query heads per key/value head
MAX_LEN = 1 << 29     # tokens of a batch row
MAX_STRIDE = 1 << 23  # elements between two tokens (and heads, of q and dout) read in place


def _rows(t: torch.Tensor, heads: bool = False):
    """[B, H, S, D] as the kernels read it, with its element strides (batch, head,
    token): contiguous head vectors at 16-byte aligned addresses, tokens (with
    ``heads``, heads too) less than MAX_STRIDE apart.  Other tensors are copied."""
    B, H, S, _ = t.shape
    sb, sh, st, sd = t.stride()
    sb, sh, st = sb if B > 1 else 0, sh if H > 1 else 0, st if S > 1 else 0
    if (sd == 1 and not (sb | sh | st) & 7 and st < MAX_STRIDE and (sh < MAX_STRIDE or not heads)
            and t.data_ptr() % 16 == 0):
        return t, (sb, sh, st)
    c = t.transpose(1, 2).contiguous()   # token-major: small strides whatever the length
    t = (c if c.data_ptr() % 16 == 0 else c.clone()).transpose(1, 2)
    return t, t.stride()[:3]


@functools.lru_cache(maxsize=64)
def _fwd_workspace(B, Hq, Hkv, Sq, Sk, D, window, first, ranges) -> int:
    return int(_capi.load().af3_sink_attention_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, window, first, ranges))


@functools.lru_cache(maxsize=64)
def _bwd_workspace(B, Hq, Hkv, Sq) -> int:
    return int(_capi.load().af3_sink_attention_bwd_workspace_bytes(B, Hq, Hkv, Sq))


@functools.lru_cache(maxsize=64)
def _c_strides(strides: tuple):
    """``strides`` as a C array (read by the call it is passed to, never written)."""
    return (ctypes.c_int64 * len(strides))(*strides)


def _forward(q, k, v, strides, sinks, scale, window, first, cu_seqlens, starts, kv_range, lse):
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    dev = q.device
    out = torch.empty((B, Sq, Hq, D), dtype=torch.bfloat16, device=dev)
    ws_n = _fwd_workspace(B, Hq, Hkv, Sq, Sk, D, window, first, int(kv_range is not None))
    ws = torch.empty(ws_n, dtype=torch.uint8, device=dev) if ws_n else None
    _capi.call("af3_sink_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _c_strides(strides),
               _capi.ptr(sinks), int(sinks is not None and sinks.dtype == torch.float32), _capi.ptr(cu_seqlens),
               B if cu_seqlens is None else cu_seqlens.numel() - 1, _capi.ptr(starts), _capi.ptr(kv_range), B, Hq,
               Hkv, Sq, Sk, D, window, first, scale, out.data_ptr(), _capi.ptr(lse), _capi.ptr(ws), ws_n,
               _capi.stream_of(dev))
    return out


class _SinkAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sinks, strides, scale, window, first, cu_seqlens, starts, kv_range):
        B, Hq, Sq, D = q.shape
        lse = torch.empty(B * Hq * Sq, dtype=torch.float32, device=q.device)
        out = _forward(q, k, v, strides, sinks, scale, window, first, cu_seqlens, starts, kv_range, lse)
        ctx.save_for_backward(q, k, v, sinks, starts, kv_range, out, lse)
        ctx.args = (scale, window, first)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _no_forward_mode("sink_attention backward", dout)
        q, k, v, sinks, starts, kv_range, out, lse = ctx.saved_tensors
        scale, window, first = ctx.args
        B, Hq, Sq, D = q.shape
        Hkv, Sk = k.shape[1], k.shape[2]
        dev = q.device
        with _device_of(q):
            # (saved-tensor hooks, as those that keep them on the host, may give them other strides)
            (q, sq), (k, sk), (v, sv) = _rows(q, heads=True), _rows(k), _rows(v)
            sinks, starts, kv_range, out, lse = (t if t is None else t.contiguous()
                                                 for t in (sinks, starts, kv_range, out, lse))
            do, st = _rows(dout.transpose(1, 2), heads=True)
            dq = torch.empty((B, Sq, Hq, D), dtype=torch.bfloat16, device=dev)
            dk = torch.empty((B, Sk, Hkv, D), dtype=torch.bfloat16, device=dev)
            dv = torch.empty((B, Sk, Hkv, D), dtype=torch.bfloat16, device=dev)
            dsinks = torch.empty_like(sinks) if sinks is not None else None
            ws_n = _bwd_workspace(B, Hq, Hkv, Sq)
            ws = torch.empty(ws_n, dtype=torch.uint8, device=dev)
            _capi.call("af3_sink_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), do.data_ptr(),
                       _c_strides(sq + sk + sv + st), _capi.ptr(sinks),
                       int(sinks is not None and sinks.dtype == torch.float32), _capi.ptr(starts),
                       _capi.ptr(kv_range), B, Hq, Hkv, Sq, Sk, D, window, first, scale, out.data_ptr(),
                       lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _capi.ptr(dsinks), ws.data_ptr(),
                       ws_n, _capi.stream_of(dev))
        return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), dsinks, *[None] * 7


def _check(q, k, v, sinks, scale, window, first):
    _no_forward_mode("sink_attention", q, k, v, sinks)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise RuntimeError(f"sink_attention: {name} must be a GPU tensor (the MI355X path has no CPU implementation)")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"sink_attention: {name} must be bfloat16 (got {t.dtype})")
        if t.dim() != 4:
            raise ValueError(f"sink_attention: {name} must be [batch, heads, tokens, dim], got {tuple(t.shape)}")
        if t.device != q.device:
            raise ValueError(f"sink_attention: {name} is on {t.device}, q on {q.device}")
    B, Hq, Sq, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"sink_attention: shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")
    Hkv = k.shape[1]
    if Hkv == 0 or Hq == 0 or Hq % Hkv or Hq // Hkv > MAX_GROUP:
        raise ValueError(f"sink_attention: {Hq} query heads cannot share {Hkv} key/value heads")
    if D not in HEAD_DIMS:
        raise ValueError(f"sink_attention: head dimension {D} is not one of {HEAD_DIMS}")
    if max(Sq, k.shape[2]) >= MAX_LEN:
        raise ValueError("sink_attention: too many tokens")
    if sinks is not None:
        if sinks.shape != (Hq,) or sinks.dtype not in (torch.bfloat16, torch.float32) or sinks.device != q.device:
            raise ValueError(f"sink_attention: sinks must be [{Hq}] bfloat16 or float32 on {q.device}, got "
                             f"{tuple(sinks.shape)} {sinks.dtype} on {sinks.device}")
    if not (0.0 < scale < math.inf):
        raise ValueError(f"sink_attention: scale must be positive and finite, got {scale}")
    if window < 0 or first < 0:
        raise ValueError(f"sink_attention: window and first must not be negative, got {window} and {first}")


def _run(q, k, v, sinks, scale, window, first, cu_seqlens, starts, kv_range):
    need = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                        or (sinks is not None and sinks.requires_grad))
    (q, sq), (k, sk), (v, sv) = _rows(q, heads=True), _rows(k), _rows(v)
    if sinks is not None and not sinks.is_contiguous():
        sinks = sinks.contiguous()
    args = (sq + sk + sv, sinks, scale, window, first, cu_seqlens, starts, kv_range)
    if not need:
        return _forward(q, k, v, *args, None)
    return _SinkAttention.apply(q, k, v, sinks, sq + sk + sv, *args[2:])


def _cu(cu_seqlens: torch.Tensor) -> torch.Tensor:
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.is_floating_point():
        raise ValueError(f"cu_seqlens must be a [sequences + 1] integer tensor, got {tuple(cu_seqlens.shape)} "
                         f"{cu_seqlens.dtype}")
    if not cu_seqlens.is_cuda:
        raise RuntimeError("cu_seqlens must be a GPU tensor (the MI355X path has no CPU implementation)")
    if cu_seqlens.dtype != torch.int32:
        cu_seqlens = cu_seqlens.to(torch.int64).clamp(-1, MAX_LEN).to(torch.int32)
    return cu_seqlens.contiguous()


def sequence_starts(cu_seqlens: torch.Tensor, n_tokens: int) -> torch.Tensor:
    """[n_tokens] int32: the first token of each token's sequence; t + 1 for a token in none."""
    cu = _cu(cu_seqlens)
    starts = torch.empty(n_tokens, dtype=torch.int32, device=cu.device)
    with _device_of(cu):
        _capi.call("af3_seq_starts", cu.data_ptr(), cu.numel() - 1, n_tokens, starts.data_ptr(),
                   _capi.stream_of(cu.device))
    return starts


def sequence_starts_of_positions(position_ids: torch.Tensor) -> torch.Tensor:
    """The same from a packed row's position ids [n_tokens] (a sequence starts where
    a position is not its predecessor's plus one, as transformers reads them)."""
    if not position_ids.is_cuda:
        raise RuntimeError("position_ids must be a GPU tensor (the MI355X path has no CPU implementation)")
    pos = position_ids.reshape(-1).to(torch.int64).contiguous()
    starts = torch.empty(pos.numel(), dtype=torch.int32, device=pos.device)
    with _device_of(pos):
        _capi.call("af3_seq_starts_positions", pos.data_ptr(), pos.numel(), starts.data_ptr(),
                   _capi.stream_of(pos.device))
    return starts


def sequence_starts_of_rows(position_ids: torch.Tensor, kv_range: torch.Tensor | None = None) -> torch.Tensor:
    """The same of a batch of packed rows: [B, S] int32, each counted in its own row, from
    position ids [B, S].  ``kv_range`` [B, 2] (begin, end) where the rows are padded: a
    sequence starts at begin too, and a token outside lies in no sequence."""
    if not position_ids.is_cuda:
        raise RuntimeError("position_ids must be a GPU tensor (the MI355X path has no CPU implementation)")
    if position_ids.dim() != 2 or position_ids.is_floating_point():
        raise ValueError(f"position_ids must be a [rows, tokens] integer tensor, got {tuple(position_ids.shape)} "
                         f"{position_ids.dtype}")
    B, S = position_ids.shape
    if kv_range is not None:
        kv_range = _ranges(kv_range, B, S, position_ids.device)
    with _device_of(position_ids):
        pos = position_ids.to(torch.int64).contiguous()
        starts = torch.empty((B, S), dtype=torch.int32, device=pos.device)
        _capi.call("af3_seq_starts_rows", pos.data_ptr(), S, B, S, _capi.ptr(kv_range), starts.data_ptr(),
                   _capi.stream_of(pos.device))
    return starts


def _ranges(kv_range, B, Sk, device):
    if kv_range.device != device:
        raise ValueError(f"kv_range is on {kv_range.device}, the rows on {device}")
    if kv_range.shape != (B, 2) or kv_range.is_floating_point():
        raise ValueError(f"kv_range must be a [{B}, 2] integer tensor, got {tuple(kv_range.shape)} {kv_range.dtype}")
    with _device_of(kv_range):
        if kv_range.dtype != torch.int32:
            kv_range = kv_range.to(torch.int64).clamp(0, Sk).to(torch.int32)
        return kv_range.contiguous()


def sink_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sinks: torch.Tensor | None = None, *,
                   scale: float | None = None, window: int = 0, first: int = 0,
                   cu_seqlens: torch.Tensor | None = None, kv_range: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention with a sliding window, kept first tokens and learned sinks.

    Query i stands at key position p = i + Sk - Sq (the last query is the last
    key) and sees the keys j <= p of its sequence with ``j > p - window`` (window
    0: all of them) or among the sequence's ``first`` tokens.  With z the scaled
    products, out = sum_j e^z_j v_j / (e^sink + sum_j e^z_j); a row that sees
    nothing gives 0, and zero gradients.

    Probabilities and their gradients are rounded to bf16 once, as operands of the
    next product (results are 1.2 to 1.45 times one bf16 rounding off); every sum is
    fp32 and in a fixed order.  Scores are fp32: a probability is off by its score's
    rounding (2^-24 of it), and scores past 2^29 overflow.  What stands outside a
    row's ``kv_range``, or in a packed row's tokens of no sequence, has no influence;
    a NaN or infinity inside can reach rows of the same tile (128 rows, 64 keys) that
    do not see it, as 0 times NaN does in any masked product.

    Args:
        q: [B, Hq, Sq, D] bf16, D 64 or 128; any strides (head vectors contiguous
            and 16-byte aligned are read in place, others copied)
        k, v: [B, Hkv, Sk, D] bf16; query head h reads head h // (Hq // Hkv)
        sinks: [Hq] bf16 or fp32 logits, or None
        scale: 1 / sqrt(D) when None
        window: keys of the sliding window, the query's own among them; 0 = no window
        first: tokens at the sequence's start that stay visible with a window
        cu_seqlens: [sequences + 1] integer cumulative lengths of a packed row (B = 1,
            Sq = Sk), on the GPU, not decreasing; tokens outside give 0
        kv_range: [B, 2] integer (begin, end) of each batch row's keys (padding on
            either side), on the GPU; values are clamped to [0, Sk]
    Returns:
        [B, Sq, Hq, D] bf16
    """
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    window, first = int(window), int(first)
    _check(q, k, v, sinks, scale, window, first)
    B, _, Sq, _ = q.shape
    Sk = k.shape[2]
    window, first = min(window, MAX_LEN), min(first, MAX_LEN)
    if cu_seqlens is not None and kv_range is not None:
        raise ValueError("sink_attention: cu_seqlens and kv_range exclude each other")
    for name, t in (("cu_seqlens", cu_seqlens), ("kv_range", kv_range)):
        if t is not None and t.device != q.device:
            raise ValueError(f"sink_attention: {name} is on {t.device}, q on {q.device}")
    with _device_of(q):
        starts = None
        if cu_seqlens is not None:
            if B != 1 or Sq != Sk:
                raise ValueError(f"sink_attention: a packed row has batch 1 and as many keys as queries, got q "
                                 f"{tuple(q.shape)}, k {tuple(k.shape)}")
            cu_seqlens = _cu(cu_seqlens)
            starts = torch.empty(Sk, dtype=torch.int32, device=q.device)
        if kv_range is not None:
            kv_range = _ranges(kv_range, B, Sk, q.device)
        return _run(q, k, v, sinks, scale, window, first, cu_seqlens, starts, kv_range)


# ---------------------------------------------------------------------------
# transformers: attn_implementation="af3_sink"
# ---------------------------------------------------------------------------

ATTN_IMPLEMENTATION = "af3_sink"


@functools.lru_cache(maxsize=1)
def _mask_codes():
    """Code objects of what transformers builds its mask functions from: joined by and,
    sliding window and causal order (honoured by the attention itself), packing, chunks."""
    from transformers import masking_utils as mu
    both = mu.sliding_window_causal_mask_function(1)
    return (both.__code__, {f.__code__ for f in _cells(both)["mask_functions"]},
            mu.packed_sequence_mask_function(None).__code__,
            {f.__code__ for f in _cells(mu.chunked_causal_mask_function(1, None))["mask_functions"]})


def _cells(f) -> dict:
    return dict(zip(f.__code__.co_freevars, (c.cell_contents for c in f.__closure__ or ())))


def _packing(f, kv_end: int):
    """The sequence numbers [rows, S] that a mask function keeps apart, or None.  What the
    attention cannot honour is refused."""
    joined, own, packed, chunks = _mask_codes()
    code = getattr(f, "__code__", None)
    if code is joined:
        parts = [p for p in (_packing(x, kv_end) for x in _cells(f)["mask_functions"]) if p is not None]
        if len(parts) < 2:
            return parts[0] if parts else None
    elif code is packed:
        return _cells(f)["packed_sequence_mask"]
    elif code in own or (code in chunks and kv_end <= _cells(f)["chunk_size"]):
        return None
    raise NotImplementedError(f"af3_sink: the mask function {getattr(f, '__qualname__', f)} is not supported (causal "
                              "order, a sliding window and packed sequences are)")


def attention_mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None, attention_mask=None,
                   use_vmap=False, **kwargs):
    """What transformers hands every layer as its mask (causal order and window are
    the attention's own): None; [B, 2] int32 key ranges of a batch padded on either
    side; or [B, S, 1] int64, where transformers found packed sequences (position ids
    that start again, which most of its models look for where neither padding nor a
    cache is given): each token's place in its own.  Other mask functions are refused.
    Reads the padding mask once per call (a host synchronisation): twice a forward for a
    model with sliding and full layers."""
    if use_vmap:
        raise NotImplementedError("af3_sink: custom mask functions are not supported")
    if isinstance(q_offset, torch.Tensor) or kv_offset + kv_length != q_offset + q_length:
        raise NotImplementedError("af3_sink: the last key must be the last query's (a cache that grows, "
                                  "not one of fixed length)")
    seq = _packing(mask_function, kv_offset + kv_length) if mask_function is not None else None
    if seq is not None:
        if attention_mask is not None or q_length != kv_length or seq.shape[-1] != kv_length:
            raise NotImplementedError("af3_sink: packed sequences with a padding mask or a cache are not supported")
        at = torch.arange(kv_length, device=seq.device).expand(batch_size, kv_length)
        new = torch.ones_like(at, dtype=torch.bool)
        new[:, 1:] = seq[:, 1:] != seq[:, :-1]
        return (at - torch.where(new, at, 0).cummax(1).values)[..., None]
    if attention_mask is None:
        return None
    m = attention_mask[:, kv_offset:kv_offset + kv_length].to(torch.int32)
    if m.shape[1] != kv_length:
        raise ValueError(f"af3_sink: the attention mask covers {attention_mask.shape[1]} tokens, the keys reach "
                         f"{kv_offset + kv_length}")
    n = m.sum(1)
    begin = m.argmax(1)
    end = kv_length - m.flip(1).argmax(1)
    end = torch.where(n == 0, begin, end)
    holes, full = torch.stack([(end - begin != n).any(), (n == kv_length).all()]).tolist()
    if holes:
        raise ValueError("af3_sink: a row of the attention mask must be one run of tokens (packed sequences go by "
                         "position_ids or cu_seq_lens_q)")
    return None if full else torch.stack([begin, end], 1).to(torch.int32)


def attention_forward(module, query, key, value, attention_mask, scaling=None, dropout=0.0, sliding_window=None,
                      s_aux=None, **kwargs):
    """transformers' attention interface over ``sink_attention``: query [B, Hq, Sq, D]
    -> ([B, Sq, Hq, D], None).  A packed row (B = 1) is read from ``cu_seq_lens_q``;
    one or a batch of them, padded or not, from position ids [B, S] that start again,
    or from what ``attention_mask`` made of the packing that transformers found."""
    if dropout:
        raise NotImplementedError("af3_sink: attention dropout is not supported")
    if kwargs.get("softcap") is not None:
        raise NotImplementedError("af3_sink: capped scores (softcap) are not supported")
    causal = kwargs.get("is_causal")
    if not (getattr(module, "is_causal", True) if causal is None else causal):
        raise NotImplementedError("af3_sink: only causal attention is supported")
    B, S, Sk = query.shape[0], query.shape[2], key.shape[2]
    cu, pos = kwargs.get("cu_seq_lens_q"), kwargs.get("position_ids")
    if attention_mask is not None:
        if S == Sk and attention_mask.shape == (B, S, 1):
            pos, attention_mask = attention_mask, None
        elif attention_mask.shape != (B, 2):
            raise ValueError("af3_sink: the mask must be the one that its own mask function makes (or None), got "
                             f"{tuple(attention_mask.shape)}")
    if s_aux is not None and s_aux.dtype not in (torch.bfloat16, torch.float32):
        s_aux = s_aux.float()
    args = dict(scale=scaling, window=sliding_window or 0, kv_range=attention_mask)
    if cu is not None:
        cu_k = kwargs.get("cu_seq_lens_k")
        if cu_k is not None and cu_k is not cu and cu_k.shape != cu.shape:
            raise ValueError("af3_sink: cu_seq_lens_q and cu_seq_lens_k differ")
        return sink_attention(query, key, value, s_aux, cu_seqlens=cu, **args), None
    if pos is not None and S == Sk > 1 and pos.numel() == B * S:
        starts = sequence_starts_of_rows(pos.to(query.device, torch.int64).reshape(B, S), attention_mask)
        scale = query.shape[-1] ** -0.5 if scaling is None else scaling
        _check(query, key, value, s_aux, scale, args["window"], 0)
        with _device_of(query):
            return _run(query, key, value, s_aux, scale, min(args["window"], MAX_LEN), 0, None, starts, None), None
    return sink_attention(query, key, value, s_aux, **args), None


def register() -> None:
    """Register with transformers as attn_implementation="af3_sink" (again is harmless)."""
    from transformers import AttentionInterface, AttentionMaskInterface
    AttentionInterface.register(ATTN_IMPLEMENTATION, attention_forward)
    AttentionMaskInterface.register(ATTN_IMPLEMENTATION, attention_mask)
