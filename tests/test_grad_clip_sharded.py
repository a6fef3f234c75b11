"""Norm of sharded gradients over ranks (gloo, CPU): the grouping, the joins over ranks and the factor;
the kernels' two calls are stood in for by torch on the ranks' own tensors."""
import math
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp


def _stand_in(monkeypatch_target):
    """CPU forms of the two kernel calls."""
    gc = monkeypatch_target

    def norm(self, code, sum_out=None, norm_out=None):
        flat = torch.cat([t.double().abs().reshape(-1) for t in self.kept])
        s = (flat * flat).sum() if code == 2 else flat.sum() if code == 1 else flat.max()
        if sum_out is not None:
            sum_out.copy_(s)
        if norm_out is not None:
            norm_out.copy_(gc._norm_of(s[None], code))
        return s[None]

    def scale(self, code, partials, max_norm, norm_out):
        n = gc._norm_of(partials, code)
        norm_out.copy_(n)
        f = max_norm / (n + 1e-6)
        if not f >= 1:
            for t in self.kept:
                t.mul_(f)
        for t, c in self.copies:
            t.copy_(c)
    gc._Tensors.norm, gc._Tensors.scale = norm, scale
    gc._check = lambda buckets: None
    import contextlib
    gc._device_of = lambda t: contextlib.nullcontext()


def _rank(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Partial, Replicate, Shard, distribute_tensor, DTensor

    from agent_factory_3_amd import grad_clip as gc
    _stand_in(gc)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    mesh = init_device_mesh("cpu", (world,))
    g = torch.Generator().manual_seed(0)
    full = [torch.randn(6, 5, generator=g), torch.randn(3, generator=g), torch.randn(1, 4, generator=g),
            torch.randn(7, generator=g)]
    for p in (2.0, 1.0, math.inf):
        for max_norm in (0.5, 1e6):
            for bad in (None, float("nan")):
                src = [t.clone() for t in full]
                if bad is not None:
                    src[0][5, 4] = bad   # held by the last rank alone
                grads = [distribute_tensor(src[0].clone(), mesh, [Shard(0)]), distribute_tensor(src[1].clone(), mesh, [Replicate()]),
                         distribute_tensor(src[2].clone(), mesh, [Shard(0)]),   # (one row: no element on the other rank)
                         src[3].clone()]
                ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in grads]
                for q, t in zip(ps, grads):
                    q.grad = t
                norm = gc.clip_grad_norm_(ps + [ps[0]], max_norm, p)
                flat = torch.cat([t.double().abs().reshape(-1) for t in src])
                want = {2.0: (flat * flat).sum().sqrt(), 1.0: flat.sum(), math.inf: flat.max()}[p]
                if bad is not None:
                    assert norm.isnan() and all(q.grad.full_tensor().isnan().all() if isinstance(q.grad, DTensor)
                                                else q.grad.isnan().all() for q in ps)
                    continue
                assert abs(float(norm) - float(want)) < 1e-6 * float(want), (p, norm, want)
                assert abs(float(gc.grad_norm(grads, p)) - min(float(want), max_norm)) < 2e-6 * float(want)
                f = min(1.0, max_norm / (float(want) + 1e-6))
                for q, t in zip(ps, src):
                    got = q.grad.full_tensor() if isinstance(q.grad, DTensor) else q.grad
                    assert torch.allclose(got, t * f, rtol=1e-5)
    part = DTensor.from_local(torch.ones(3), mesh, [Partial()])
    try:
        gc.grad_norm([part])
        raise AssertionError("a Partial gradient was taken")
    except NotImplementedError:
        pass
    dist.barrier()
    dist.destroy_process_group()
    out[rank] = 1


@pytest.mark.parametrize("world", [2])
def test_sharded_gradients(world):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    with ctx.Manager() as m:
        out = m.dict()
        mp.spawn(_rank, args=(world, port, out), nprocs=world, join=True)
        assert sorted(out.keys()) == list(range(world))


def test_host_tensors_and_norm_types_are_refused():
    from agent_factory_3_amd import grad_clip
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="GPU"):
        grad_clip.clip_grad_norm_([p], 1.0)
    with pytest.raises(NotImplementedError):
        grad_clip.clip_grad_norm_([p], 1.0, norm_type=3)
    with pytest.raises(ValueError):
        grad_clip.clip_grad_norm_([p], -1.0)
    assert float(grad_clip.clip_grad_norm_([], 1.0)) == 0.0


def test_c_entry_refuses_bad_arrays():
    """Argument errors come back before anything is launched (no GPU needed)."""
    import ctypes

    from agent_factory_3_amd import _capi
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    arr = lambda t, *v: (t * len(v))(*v)  # noqa: E731
    ptrs, f32 = arr(ctypes.c_uint64, 4096, 4160), arr(ctypes.c_uint8, 1, 1)
    call = lambda name, p, s, f, n, code, *rest: _capi.call(name, p, s, f, n, code, *rest)  # noqa: E731
    with pytest.raises(RuntimeError, match="share memory"):
        call("af3_grad_scale", ptrs, arr(ctypes.c_int64, 17, 4), f32, 2, 2, 8, 1, 1.0, None, None)
    for sizes, match in ((arr(ctypes.c_int64, 16, 0), "empty"), (arr(ctypes.c_int64, 16, -1), "empty")):
        with pytest.raises(RuntimeError, match=match):
            call("af3_grad_norm", ptrs, sizes, f32, 2, 2, 8, 100, None, None, None)
    with pytest.raises(RuntimeError, match="aligned"):
        call("af3_grad_norm", arr(ctypes.c_uint64, 4096, 4162), arr(ctypes.c_int64, 16, 1), f32, 2, 2, 8, 100, None, None, None)
    with pytest.raises(RuntimeError, match="norm_type"):
        call("af3_grad_norm", ptrs, arr(ctypes.c_int64, 16, 4), f32, 2, 3, 8, 100, None, None, None)
    with pytest.raises(RuntimeError, match="partials"):
        call("af3_grad_norm", ptrs, arr(ctypes.c_int64, 16, 20000), f32, 2, 2, 8, 2, None, None, None)
