"""The global gradient norm and its clipping on the MI355X.

``clip_grad_norm_`` takes torch.nn.utils.clip_grad_norm_'s arguments (the
reference's training step calls that through accelerate) for the gradients that
LoRA training leaves: hundreds of bf16 and fp32 tensors, reached in a few launches
each way instead of some per tensor.  Sharded gradients (DTensor, as FSDP2 leaves
them) are counted once over their mesh.  The HIP kernels are behind
``af3_grad_norm`` and ``af3_grad_scale``; there is no CPU fallback.
"""
from __future__ import annotations

import math
from array import array
from operator import attrgetter

import torch
from torch.autograd.graph import increment_version

from . import _capi
from .routing import _device_of

_DTYPE = attrgetter("dtype")
_NORMS = {2.0: 2, 1.0: 1, math.inf: 0}


def _norm_code(norm_type) -> int:
    try:
        return _NORMS[float(norm_type)]
    except KeyError:
        raise NotImplementedError(f"grad_norm: norm_type {norm_type} is not one of 1, 2 and inf") from None


class _Tensors:
    """GPU tensors of one device as the kernels take them: addresses, lengths, types.
    Tensors that do not fill one run of memory are read (and scaled) through a copy."""

    def __init__(self, tensors, sizes=None):
        self.n = len(tensors)
        self.device = tensors[0].device
        dtypes = set(map(_DTYPE, tensors))
        _check([(self.device, dtypes)])
        self.copies = []
        if not all(map(torch.Tensor.is_contiguous, tensors)):
            tensors = [t if t.is_contiguous() else self._run(t) for t in tensors]
        self.kept = tensors
        f32 = array("B", [torch.float32 in dtypes]) * self.n
        if len(dtypes) > 1:
            f32 = array("B", [d is torch.float32 for d in map(_DTYPE, tensors)])
        # (host arrays: the calls read them before they return)
        self._arrays = (array("Q", map(torch.Tensor.data_ptr, tensors)), sizes or array("q", map(torch.Tensor.numel, tensors)), f32)
        self.ptrs, self.sizes, self.f32 = (a.buffer_info()[0] for a in self._arrays)

    def _run(self, t):
        if t.layout is not torch.strided:
            raise NotImplementedError("grad_norm: sparse gradients are not supported")
        order = sorted(range(t.dim()), key=t.stride, reverse=True)
        run = t.detach().permute(order)
        if run.is_contiguous():   # the same memory in another order
            return run
        if any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
            raise ValueError("grad_norm: a gradient whose elements share memory (an expanded tensor) cannot be clipped")
        c = t.detach().contiguous()
        self.copies.append((t, c))
        return c

    def norm(self, code, sum_out=None, norm_out=None):
        """The partials (and their sum, or the norm)."""
        n = int(_capi.load().af3_grad_norm_partials(self.sizes, self.n))
        partials = torch.empty(n, dtype=torch.float64, device=self.device)
        _capi.call("af3_grad_norm", self.ptrs, self.sizes, self.f32, self.n, code, partials.data_ptr(), n,
                   _capi.ptr(sum_out), _capi.ptr(norm_out), _capi.stream_of(self.device))
        return partials

    def scale(self, code, partials, max_norm, norm_out):
        _capi.call("af3_grad_scale", self.ptrs, self.sizes, self.f32, self.n, code, partials.data_ptr(),
                   partials.numel(), max_norm, _capi.ptr(norm_out), _capi.stream_of(self.device))
        increment_version(self.kept)   # (a graph that saved one of them must see that it changed)
        for t, c in self.copies:
            t.copy_(c)


def _local(t):
    """(the local tensor, process groups its elements are spread over)."""
    if type(t) is torch.Tensor or type(t) is torch.nn.Parameter or not hasattr(t, "device_mesh"):
        return t, ()
    groups = []
    for dim, p in enumerate(t.placements):
        if p.is_partial():
            raise NotImplementedError("grad_norm: a gradient that is still to be reduced (a Partial DTensor)")
        if not p.is_replicate():   # (is_shard leaves out the strided shards of FSDP2 over tensor parallelism)
            groups.append(t.device_mesh.get_group(dim))
    return t.to_local(), tuple(groups)


def _held(tensors):
    """Tensors by (device, process groups), in order of first appearance, as the kernels take them (None
    where all of them are empty)."""
    if (set(map(type, tensors)) == {torch.Tensor} and len(set(map(torch.Tensor.get_device, tensors))) == 1
            and len(set(map(id, tensors))) == len(tensors)):
        sizes = array("q", map(torch.Tensor.numel, tensors))
        if all(sizes):   # the common case, without a step per tensor
            one = _Tensors(tensors, sizes)
            return {(one.device, ()): one}
    buckets = _gather(tensors)
    _check([(device, set(map(_DTYPE, ts))) for (device, _), ts in buckets.items()])
    return {key: _Tensors(ts) if ts else None for key, ts in buckets.items()}


def _gather(tensors):
    """Tensors by (device, process groups); doubles and empty ones left out."""
    buckets, seen = {}, set()
    for t in tensors:
        if id(t) in seen:
            continue
        seen.add(id(t))
        groups = ()
        if type(t) is not torch.Tensor:
            t, groups = _local(t)
        bucket = buckets.get((t.device, groups))
        if bucket is None:
            bucket = buckets[t.device, groups] = []
        if t.numel():
            bucket.append(t)
    return buckets


def _check(types):
    for device, dtypes in types:
        if device.type != "cuda":
            raise RuntimeError("grad_norm: gradients must be GPU tensors (the MI355X path has no CPU implementation)")
        for dtype in dtypes:
            if dtype is not torch.float32 and dtype is not torch.bfloat16:
                raise TypeError(f"grad_norm: gradients must be bfloat16 or float32 (got {dtype})")


def _bucket_sum(tensors, code):
    """sum |g|^p (or the largest) of a bucket's tensors as a 64-bit scalar [1] on their device."""
    total = torch.empty(1, dtype=torch.float64, device=tensors.device)
    with _device_of(total):
        tensors.norm(code, sum_out=total)
    return total


def _join_ranks(total, groups, code):
    """A bucket's sum over the ranks that hold its other elements."""
    import torch.distributed as dist
    if code:
        for g in groups:
            dist.all_reduce(total, dist.ReduceOp.SUM, group=g)
        return total
    # (a reduction to the largest may drop a NaN: it goes along as a flag)
    nan = total.isnan()
    both = torch.cat([total.nan_to_num(nan=0.0, posinf=math.inf), nan.to(total.dtype)])
    for g in groups:
        dist.all_reduce(both, dist.ReduceOp.MAX, group=g)
    return torch.where(both[1:] > 0, math.nan, both[:1])


def _partials(held, code):
    """[(tensors of a device, partials on that device)], a device each; all partials together make the norm."""
    if len(held) == 1 and not next(iter(held))[1]:   # one GPU, nothing sharded: the partials as they are
        (t,) = held.values()
        if t is None:
            return []
        with _device_of(t.kept[0]):
            return [([t], t.norm(code))]
    sums = []
    for (device, groups), t in held.items():
        total = torch.zeros(1, dtype=torch.float64, device=device) if t is None else _bucket_sum(t, code)
        sums.append(_join_ranks(total, groups, code) if groups else total)
    by_device = {}
    for (device, _), t in held.items():
        by_device.setdefault(device, []).append(t)
    return [([t for t in ts if t is not None], torch.cat([s.to(device) for s in sums])) for device, ts in by_device.items()]


def _norm_of(partials, code):
    if code == 2:
        return partials.sum().sqrt().float()
    return (partials.sum() if code else partials.max()).float()   # (torch's max keeps a NaN)


def _grads(parameters):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [g for p in parameters if (g := p.grad) is not None]


@torch.no_grad()
def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """Norm of all tensors' elements taken as one vector: an fp32 scalar on the first one's
    device.  bf16 and fp32 tensors, DTensors among them; sums are 64 bits in a fixed order.

    Args:
        tensors: a tensor or several (a list of gradients); one listed twice counts once
        norm_type: 2, 1 or inf
    """
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    held = _held(tensors)
    if len(held) == 1 and not next(iter(held))[1]:   # one GPU, nothing sharded
        (t,) = held.values()
        if t is not None:
            out = torch.empty((), dtype=torch.float32, device=t.device)
            with _device_of(out):
                t.norm(code, norm_out=out)
            return out
    parts = _partials(held, code)
    if not parts:
        return torch.zeros((), device=tensors[0].device if tensors else None)
    return _norm_of(parts[0][1], code)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: bool | None = None) -> torch.Tensor:
    """Scale the parameters' gradients in place by min(1, max_norm / (norm + 1e-6)), with
    the norm over all of them together; torch.nn.utils.clip_grad_norm_'s arguments and
    result (a norm that is NaN makes every gradient NaN, an infinite one 0 and NaN).

    Within the limit the gradients are read once and not written.  The norm is summed in
    64 bits in a fixed order and returned in fp32 (torch takes a norm per tensor in the
    tensor's type, and a norm of those); the factor is formed from the 64-bit norm and
    rounded to fp32 once.  Nothing synchronises the host unless
    ``error_if_nonfinite``.

    Args:
        parameters: a tensor or several; those without a gradient are passed over, one
            listed twice counts once.  Gradients are bf16 or fp32 on the GPU; DTensors
            (FSDP2) are summed over the mesh dimensions that shard them, with one
            all-reduce per mesh dimension and no gathering.
        norm_type: 2, 1 or inf
        error_if_nonfinite: raise, before anything is scaled, if the norm is not finite
        foreach: taken for torch's signature; there is one form
    """
    grads = _grads(parameters)
    max_norm = float(max_norm)
    code = _norm_code(norm_type)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    if not grads:
        return torch.tensor(0.0)
    parts = _partials(_held(grads), code)
    if not parts:
        return torch.zeros((), device=grads[0].device)
    if error_if_nonfinite:
        norm = _norm_of(parts[0][1], code)
        if not math.isfinite(norm):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
                               "non-finite, so it cannot be clipped.")
    out = None
    for held, partials in parts:
        norm = None
        for t in held:
            norm = norm if norm is not None else torch.empty((), dtype=torch.float32, device=partials.device)
            with _device_of(norm):
                t.scale(code, partials, max_norm, norm)
        if norm is None:   # this rank holds no element of these gradients
            norm = _norm_of(partials, code)
        out = out if out is not None else norm
    return out
