"""The router's load-balancing loss in float64: loss, tokens per expert and the logits gradient."""
from __future__ import annotations

import torch


def top_k(logits, k):
    """Top k ids per row: larger logit first, equal logits by lower id, NaN last."""
    z = torch.where(torch.isnan(logits), -torch.inf, logits.double())
    # NaN below -inf: a second key
    order = torch.argsort(torch.isnan(logits).to(torch.int8), dim=-1, stable=True)
    z2 = z.gather(-1, order)
    nan2 = torch.isnan(logits).gather(-1, order)
    n_ok = (~nan2).sum(-1, keepdim=True)
    pos = torch.arange(z.shape[-1])[None]
    key = torch.where(pos < n_ok, z2, -torch.inf)
    # stable descending sort of the finite part; the NaN tail keeps its place behind it
    idx = torch.argsort(key, dim=-1, descending=True, stable=True)
    return order.gather(-1, idx)[..., :k]


def balance_loss(logits, k, expt_indx=None, token_mask=None, dloss=1.0):
    """logits [T, E] -> (loss, counts [E] int64, dlogits [T, E]) on the CPU."""
    z = logits.detach().cpu().double()
    T, E = z.shape
    rows = torch.arange(T) if token_mask is None else torch.nonzero(token_mask.cpu().reshape(-1) != 0).reshape(-1)
    ids = top_k(z[rows], k) if expt_indx is None else expt_indx.cpu().reshape(T, k).long()[rows]
    ids = ids[(ids >= 0) & (ids < E)]
    counts = torch.bincount(ids.reshape(-1), minlength=E)
    n = rows.numel()
    grad = torch.zeros_like(z)
    if n == 0:
        return torch.tensor(0.0, dtype=torch.float64), counts, grad
    p = torch.softmax(z[rows], -1)
    f = counts.double() / n
    loss = E * (f * p.sum(0) / n).sum()
    grad[rows] = dloss * E / n * p * (f - (p * f).sum(-1, keepdim=True))
    return loss, counts, grad
