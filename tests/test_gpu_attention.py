"""Sink attention on the GPU against the float64 oracle, with its derived element-wise bounds."""
import math

import pytest
import torch

from oracle import attention as oa

pytestmark = pytest.mark.gpu


def _make(dev, B, Hq, Hkv, Sq, Sk, D, seed=0, sinks=torch.bfloat16, layout="token"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(torch.bfloat16).to(dev)  # noqa: E731
    if layout == "token":   # [B, S, H, D] storage, as a projection leaves it
        q, k, v = r(B, Sq, Hq, D, std=2.0).transpose(1, 2), r(B, Sk, Hkv, D).transpose(1, 2), r(B, Sk, Hkv, D).transpose(1, 2)
    elif layout == "head":
        q, k, v = r(B, Hq, Sq, D, std=2.0), r(B, Hkv, Sk, D), r(B, Hkv, Sk, D)
    elif layout == "fused":  # views of one fused projection
        f = r(B, max(Sq, Sk), (Hq + 2 * Hkv) * D)
        h = f.view(B, max(Sq, Sk), Hq + 2 * Hkv, D).transpose(1, 2)
        q, k, v = h[:, :Hq, :Sq], h[:, Hq:Hq + Hkv, :Sk], h[:, Hq + Hkv:, :Sk]
    else:                    # odd address, odd strides: copied
        f = r(B, Hq + 2 * Hkv, max(Sq, Sk), D + 3)[..., 1:D + 1]
        q, k, v = f[:, :Hq, :Sq], f[:, Hq:Hq + Hkv, :Sk], f[:, Hq + Hkv:, :Sk]
    s = (torch.randn(Hq, generator=g) * 1.5).to(sinks).to(dev) if sinks is not None else None
    return q, k, v, s, r(B, Sq, Hq, D)


def _close(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - ref).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(),
                           float(((got - ref).abs() / tol)[bad].max()))


def _check(dev, B, Hq, Hkv, Sq, Sk, D, *, train=True, sinks=torch.bfloat16, layout="token", seed=0, **kw):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, B, Hq, Hkv, Sq, Sk, D, seed, sinks, layout)
    okw = dict(kw)
    if kw.get("cu_seqlens") is not None:
        kw["cu_seqlens"] = torch.tensor(kw["cu_seqlens"], dtype=torch.int32, device=dev)
    if kw.get("kv_range") is not None:
        kw["kv_range"] = torch.tensor(kw["kv_range"], dtype=torch.int32, device=dev)
    ref = oa.attention(q, k, v, s, dout=do if train else None, bounds=True, **okw)
    if not train:
        with torch.no_grad():
            out = sink_attention(q, k, v, s, **kw)
        _close(out, ref["out"], ref["out_tol"], "out")
        return
    leaves = [t.detach().requires_grad_() for t in (q, k, v, s) if t is not None]
    out = sink_attention(*(leaves if s is not None else leaves + [None]), **kw)
    _close(out, ref["out"], ref["out_tol"], "out")
    for n, g in zip(("dq", "dk", "dv", "dsinks"), torch.autograd.grad(out, leaves, do)):
        _close(g, ref[n], ref[n + "_tol"], n)


# one key tile, its edges, several row and key tiles; one token to some hundred
@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 300])
def test_lengths(dev, S):
    _check(dev, 1, 8, 1, S, S, 64, seed=S)


@pytest.mark.parametrize("window,first", [(1, 0), (2, 0), (31, 0), (64, 0), (65, 3), (128, 0), (128, 64), (128, 65),
                                          (10, 200), (299, 0), (300, 7), (1000, 1)])
def test_windows(dev, window, first):
    _check(dev, 1, 8, 2, 300, 300, 64, window=window, first=first, seed=window)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (2, 1), (10, 2), (7, 1), (16, 2), (64, 8), (64, 1), (128, 1), (100, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(dev, Hq, Hkv, D):
    _check(dev, 1, Hq, Hkv, 70, 70, D, window=40, seed=Hq)


@pytest.mark.parametrize("layout", ["token", "head", "fused", "odd"])
@pytest.mark.parametrize("D", [64, 128])
def test_storage(dev, layout, D):
    _check(dev, 2, 8, 2, 130, 130, D, layout=layout, window=50, first=2)


@pytest.mark.parametrize("sinks", [None, torch.float32, torch.bfloat16])
def test_sinks(dev, sinks):
    _check(dev, 2, 6, 3, 90, 90, 64, sinks=sinks)


@pytest.mark.parametrize("cu", [[0, 200], [0, 1, 2, 3, 200], [0, 0, 77, 77, 200, 200], [0, 64, 128, 192, 200],
                                [5, 60, 150], [0, 190], [200, 200], [0], [30, 31]])
@pytest.mark.parametrize("window,first", [(0, 0), (20, 0), (20, 9)])
def test_packed(dev, cu, window, first):
    _check(dev, 1, 8, 2, 200, 200, 64, cu_seqlens=cu, window=window, first=first)


def test_packed_many_short_sequences(dev):
    g = torch.Generator().manual_seed(5)
    cuts = sorted(torch.randint(0, 700, (90,), generator=g).tolist())
    _check(dev, 1, 4, 2, 700, 700, 64, cu_seqlens=[0] + cuts + [700])
    _check(dev, 1, 4, 4, 700, 700, 128, cu_seqlens=[0] + cuts + [700], window=30, first=2)


@pytest.mark.parametrize("rng", [[(0, 100), (0, 37), (0, 0)], [(0, 100), (63, 100), (100, 100)],
                                 [(10, 90), (64, 65), (-5, 400)]])
@pytest.mark.parametrize("window,first", [(0, 0), (24, 0), (24, 5)])
def test_padded_batches(dev, rng, window, first):
    _check(dev, 3, 8, 1, 100, 100, 64, kv_range=rng, window=window, first=first)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 50), (1, 257), (3, 1000), (9, 2100), (17, 300), (5, 2), (40, 0), (130, 700)])
@pytest.mark.parametrize("window,first", [(0, 0), (100, 0), (100, 70)])
def test_few_queries_over_a_cache(dev, Sq, Sk, window, first):
    _check(dev, 2, 16, 2, Sq, Sk, 64, train=False, window=window, first=first)
    if Sk <= 1000:
        _check(dev, 2, 16, 2, Sq, Sk, 64, window=window, first=first)


@pytest.mark.parametrize("D", [64, 128])
def test_one_token_over_long_caches(dev, D):
    _check(dev, 3, 8, 2, 1, 5000, D, train=False, kv_range=[(0, 5000), (4000, 5000), (4999, 5000)])
    _check(dev, 1, 64, 8, 1, 9001, D, train=False)
    _check(dev, 1, 64, 8, 2, 3001, D, window=2500, first=4, sinks=None)


def test_nothing_visible(dev):
    from agent_factory_3_amd.attention import sink_attention
    for sinks in (None, torch.bfloat16):
        q, k, v, s, do = _make(dev, 2, 4, 2, 20, 20, 64, sinks=sinks)
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = sink_attention(q, k, v, s, kv_range=torch.zeros(2, 2, dtype=torch.int64, device=dev))
        grads = torch.autograd.grad(out, (q, k, v), do)
        assert all((t == 0).all() for t in (out, *grads))
    # no tokens at all
    q, k, v, s, do = _make(dev, 2, 4, 2, 0, 0, 64)
    q, s = q.detach().requires_grad_(), s.requires_grad_()
    out = sink_attention(q, k, v, s)
    dq, ds = torch.autograd.grad(out, (q, s), do)
    assert out.shape == (2, 0, 4, 64) and dq.shape == q.shape and (ds == 0).all()


def test_garbage_outside_the_range_has_no_influence(dev):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 2, 8, 2, 100, 100, 64)
    rng = torch.tensor([[0, 61], [30, 100]], dtype=torch.int32, device=dev)
    res = []
    for bad in (0.0, math.nan, math.inf, float(torch.finfo(torch.bfloat16).min)):
        k2, v2 = k.clone(), v.clone()
        for b, (lo, hi) in enumerate(rng.tolist()):
            for t in (k2, v2):
                t[b, :, :lo] = bad
                t[b, :, hi:] = bad
        leaves = [t.detach().requires_grad_() for t in (q, k2, v2, s)]
        out = sink_attention(*leaves, window=20, kv_range=rng)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, do)])
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))
    assert all(torch.isfinite(t).all() for t in res[0])


def test_large_scores_and_lowest_values(dev):
    """Scores far beyond the exponential's range, and a sink of -inf or a very large one."""
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, 4, 2, 150, 150, 64)
    s = torch.tensor([-math.inf, 200.0, -1e30, 0.0], device=dev)
    q = (q.float() * 60).to(torch.bfloat16)
    ref = oa.attention(q, k, v, s, window=64, bounds=True)
    _close(sink_attention(q, k, v, s, window=64), ref["out"], ref["out_tol"], "out")


def test_same_bits_each_time_and_on_another_stream(dev):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, 16, 2, 333, 333, 64)

    def go():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
        out = sink_attention(*leaves, window=100, first=3)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    a = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed(dev):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, _ = _make(dev, 2, 16, 2, 1, 3000, 64)
    rng = torch.tensor([[0, 3000], [7, 3000]], dtype=torch.int32, device=dev)
    with torch.no_grad():
        want0 = sink_attention(q, k, v, s, kv_range=rng)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sink_attention(q, k, v, s, kv_range=rng)
        for n in range(3):
            if n:
                q.copy_(torch.randn(q.shape, device=dev))
                rng.copy_(torch.tensor([[n, 3000], [100 * n, 3000]], dtype=torch.int32))
            want = sink_attention(q, k, v, s, kv_range=rng)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert n or torch.equal(want, want0)


def test_expanded_gradient_and_broadcast_inputs(dev):
    """The gradient of a sum arrives with stride 0; keys shared by the batch are one tensor, their gradient a sum."""
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, _ = _make(dev, 3, 4, 2, 50, 50, 64)
    kl = k[:1].detach().requires_grad_()
    out = sink_attention(q, kl.expand(3, -1, -1, -1), v, s)
    (g,) = torch.autograd.grad(out.sum(), kl)
    ref = oa.attention(q, k[:1].expand(3, -1, -1, -1), v, s, dout=torch.ones_like(out), bounds=True)
    # torch sums the three batch rows' bf16 gradients
    tol = ref["dk_tol"].sum(0, keepdim=True) + 2 * oa.U * ref["dk"].abs().sum(0, keepdim=True)
    _close(g, ref["dk"].sum(0, keepdim=True), tol, "dk")


def test_refusals(dev):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, _ = _make(dev, 2, 4, 2, 8, 8, 64)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    rng = torch.tensor([[0, 8], [0, 8]], dtype=torch.int32, device=dev)
    for exc, args, kw in [
            (TypeError, (q.float(), k, v), {}), (TypeError, (q, k.half(), v), {}),
            (ValueError, (q[0], k, v), {}), (ValueError, (q, k[:1], v[:1]), {}), (ValueError, (q, k, v[:, :, :4]), {}),
            (ValueError, (q[:, :3], k, v), {}), (ValueError, (q[..., :32], k[..., :32], v[..., :32]), {}),
            (ValueError, (q, k[:, :0], v[:, :0]), {}),
            (ValueError, (q, k, v, s[:3]), {}), (ValueError, (q, k, v, s.half()), {}),
            (ValueError, (q, k, v, s.cpu()), {}), (RuntimeError, (q.cpu(), k, v), {}),
            (ValueError, (q, k, v), dict(window=-1)), (ValueError, (q, k, v), dict(first=-1)),
            (ValueError, (q, k, v), dict(scale=0.0)), (ValueError, (q, k, v), dict(scale=math.nan)),
            (ValueError, (q, k, v), dict(scale=-1.0)), (ValueError, (q, k, v), dict(cu_seqlens=cu)),
            (ValueError, (q[:1], k[:1], v[:1]), dict(cu_seqlens=cu, kv_range=rng[:1])),
            (ValueError, (q[:1, :, :3], k[:1], v[:1]), dict(cu_seqlens=cu)),
            (ValueError, (q[:1], k[:1], v[:1]), dict(cu_seqlens=cu.cpu())),
            (ValueError, (q[:1], k[:1], v[:1]), dict(cu_seqlens=cu.float())),
            (ValueError, (q, k, v), dict(kv_range=rng[:1])), (ValueError, (q, k, v), dict(kv_range=rng.float())),
            (ValueError, (q, k, v), dict(kv_range=rng.cpu()))]:
        with pytest.raises(exc):
            sink_attention(*args, **kw)


def test_unordered_lengths_stay_in_bounds(dev):
    """Cumulative lengths that decrease or leave the row give some finite answer and touch nothing else."""
    from agent_factory_3_amd.attention import sequence_starts, sink_attention
    q, k, v, s, do = _make(dev, 1, 4, 2, 200, 200, 64)
    t = torch.arange(200)
    for cu in ([150, 20, 90], [-40, 500], [0, 1000, -1000, 7]):
        cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        st = sequence_starts(cu, 200).cpu()
        assert (st >= 0).all() and (st <= t + 1).all()
        leaves = [x.detach().requires_grad_() for x in (q, k, v, s)]
        out = sink_attention(*leaves, cu_seqlens=cu, window=30, first=4)
        assert all(torch.isfinite(x).all() for x in (out, *torch.autograd.grad(out, leaves, do)))


@pytest.mark.parametrize("lens", [[1], [5, 3], [700, 1, 1, 324], [1500] * 3])
def test_starts_of_positions(dev, lens):
    from agent_factory_3_amd.attention import sequence_starts, sequence_starts_of_positions
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), device=dev)
    want = oa.starts_of(cu.tolist(), pos.numel()).to(torch.int32)
    assert torch.equal(sequence_starts_of_positions(pos[None]).cpu(), want)
    assert torch.equal(sequence_starts(cu, pos.numel()).cpu(), want)


@pytest.mark.parametrize("G", [1, 3, 8, 64])
@pytest.mark.parametrize("start", [1, 31, 32, 33, 40, 63, 64, 65])
def test_a_sequence_starts_inside_a_key_block(dev, G, start):
    """Keys of two sequences in one block of the key gradient, at every place of its waves; garbage in
    the later sequence's gradients must not reach the earlier one's keys."""
    _check(dev, 1, G, 1, 150, 150, 64, cu_seqlens=[0, start, 150], seed=start)
    _check(dev, 1, G, 1, 150, 150, 64, cu_seqlens=[0, start, start + 3, 150], window=20, first=2, seed=start)
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, G, 1, 150, 150, 64)
    cu = torch.tensor([0, start, 150], dtype=torch.int32, device=dev)
    res = []
    for bad in (0.0, math.nan):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        d2 = do.clone()
        d2[:, start:] += bad
        out = sink_attention(*leaves, s, cu_seqlens=cu)
        res.append([g[:, :, :start] for g in torch.autograd.grad(out, leaves, d2)])
    if start * G % 64 == 0:   # (else a tile of rows holds both sequences: the documented limit)
        assert all(torch.equal(a, b) for a, b in zip(*res))


def test_a_training_step_captured_and_replayed(dev):
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, 16, 2, 200, 200, 64)
    cu = torch.tensor([0, 77, 200], dtype=torch.int32, device=dev)

    def step(leaves):
        out = sink_attention(*leaves, window=50, first=1, cu_seqlens=cu)
        return [out, *torch.autograd.grad(out, leaves, do)]
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, s)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaves)
    for n in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, device=dev))
            cu.copy_(torch.tensor([0, 10 + 60 * n, 200], dtype=torch.int32))
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", ["q", "k", "v", "s"])
def test_gradients_of_one_input_alone(dev, which):
    from agent_factory_3_amd.attention import sink_attention
    t = dict(zip(("q", "k", "v", "s", "do"), _make(dev, 1, 4, 2, 60, 60, 64)))
    every = {n: t[n].detach().requires_grad_() for n in ("q", "k", "v", "s")}
    all_g = dict(zip(every, torch.autograd.grad(sink_attention(*every.values()), list(every.values()), t["do"])))
    one = {n: t[n].detach() for n in ("q", "k", "v", "s")}
    one[which].requires_grad_()
    (g,) = torch.autograd.grad(sink_attention(*one.values()), one[which], t["do"])
    assert torch.equal(g, all_g[which])
    with pytest.raises(RuntimeError):   # no second derivative
        (g,) = torch.autograd.grad(sink_attention(*every.values()), every[which], t["do"], create_graph=True)
        g.float().sum().backward()


def test_offsets_past_32_bits(dev):
    """Caches whose last rows lie past 2^31 elements, and a batch row that starts there."""
    from agent_factory_3_amd.attention import sink_attention
    S, H, D = 2_300_000, 8, 64     # 1.18e9 elements a batch row, 2.36e9 in all
    k = torch.zeros(2, S, H, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    for t in (k, v):
        t[:, :8].normal_()
        t[:, -700:].normal_()
    q = torch.randn(2, 3, 2 * H, D, device=dev).to(torch.bfloat16)
    s = torch.randn(2 * H, device=dev).to(torch.bfloat16)
    kw = dict(window=600, first=5)
    k2, v2 = (torch.cat([t[:, :5], t[:, -700:]], 1).transpose(1, 2) for t in (k, v))
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    with torch.no_grad():
        out = sink_attention(q, k, v, s, **kw)
    # the same keys without the gap: 705 of them, the first five kept
    ref = oa.attention(q, k2, v2, s, **kw, bounds=True)
    _close(out, ref["out"], ref["out_tol"], "out")
    # without a window the zeros between count too: 2.3 million of them, exp(0) each
    with torch.no_grad():
        out = sink_attention(q[:, :, -1:], k, v, s)
    z = torch.einsum("bhd,bhsd->bhs", q[:, :, -1].float().reshape(2, H, 2, D).reshape(2, 2 * H, D).cpu().double(),
                     torch.cat([k[:, :, :8], k[:, :, -700:]], 2).cpu().double().repeat_interleave(2, 1)) / 8
    e = torch.exp(z)
    den = e.sum(-1) + torch.exp(s.cpu().double()) + (S - 708)
    vv = torch.cat([v[:, :, :8], v[:, :, -700:]], 2).cpu().double().repeat_interleave(2, 1)
    want = torch.einsum("bhs,bhsd->bhd", e, vv) / den[..., None]
    mag = torch.einsum("bhs,bhsd->bhd", e, vv.abs()) / den[..., None]
    # p of the 708 keys rounded (2^-8), the count of zeros summed in fp32 (2^-24 per addition of 64 at a time: 2^-8 at most)
    assert ((out[:, 0].cpu().double() - want).abs() <= 2 ** -6 * mag).all()
    del k, v


def test_the_longest_packed_row(dev):
    """128000 tokens: the last sequences are what they are alone, forward and backward."""
    from agent_factory_3_amd.attention import sink_attention
    T, lens = 128000, [50000, 60000, 1, 17000, 999]
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v, do = (torch.randn(1, T, h, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2) for h in (8, 2, 2, 8))
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    for window in (0, 128):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = sink_attention(*leaves, window=window, cu_seqlens=cu)
        grads = torch.autograd.grad(out, leaves, do.transpose(1, 2))
        for a, n in ((110000, 1), (127001, 999)):
            r = oa.attention(*(t[:, :, a:a + n] for t in (q, k, v)), window=window, dout=do[:, :, a:a + n].transpose(1, 2),
                             bounds=True)
            _close(out[:, a:a + n], r["out"], r["out_tol"], "out")
            for name, t in zip(("dq", "dk", "dv"), grads):
                _close(t[:, :, a:a + n], r[name], r[name + "_tol"], name)


def test_saved_tensors_that_come_back_with_other_strides(dev):
    """Saved-tensor hooks may hand the backward equal tensors laid out differently (those that keep
    them on the host give dense ones for views with gaps): the same gradients."""
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 2, 8, 2, 90, 90, 64, layout="fused")
    leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]

    def grads():
        return torch.autograd.grad(sink_attention(*leaves, window=40, first=2), leaves, do)
    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def spread(t):    # every dimension's stride changed, gaps between all of them
        return torch.empty([2 * n for n in t.shape[::-1]], dtype=t.dtype, device=t.device).permute(
            *range(t.dim())[::-1])[tuple(slice(None, None, 2) for _ in t.shape)].copy_(t) if t.dtype == torch.bfloat16 else t
    with torch.autograd.graph.saved_tensors_hooks(spread, lambda t: t):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_largest_sinks(dev):
    """A sink of the type's largest value leaves nothing of any key; of its lowest value, it is no sink."""
    from agent_factory_3_amd.attention import sink_attention
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, s, do = _make(dev, 1, 4, 2, 90, 90, 64, sinks=dtype)
        s[0], s[1] = torch.finfo(dtype).max, torch.finfo(dtype).min
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
        out = sink_attention(*leaves, window=30)
        grads = torch.autograd.grad(out, leaves, do)
        assert not out[:, :, 0].any() and not grads[0][:, 0].any() and not grads[3][:2].any()
        assert all(torch.isfinite(t).all() for t in (out, *grads))
        # (the bits of a row go with its tile, whose rows move their running maximum together: the oracle's bounds)
        none = oa.attention(q[:, 1:2], k[:, :1], v[:, :1], window=30, bounds=True)
        _close(out[:, :, 1:2], none["out"], none["out_tol"], "out")


@pytest.mark.parametrize("window", [0, 20])
def test_gradients_of_rows_that_see_nothing_have_no_influence(dev, window):
    """Rows before a left-padded batch row's first key, and those whose window lies behind a
    right-padded one's last key, with garbage in their gradients."""
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 2, 8, 2, 150, 150, 64)
    rng = torch.tensor([[70, 150], [0, 61]], dtype=torch.int32, device=dev)
    none = 61 + window - 1 if window else 150
    res = []
    for bad in (0.0, math.nan, math.inf):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
        d = do.clone()
        d[0, :70] = bad
        d[1, none:] = bad
        res.append(torch.autograd.grad(sink_attention(*leaves, window=window, kv_range=rng), leaves, d))
        assert not res[-1][0][0, :, :70].any() and not res[-1][0][1, :, none:].any()
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


@pytest.mark.parametrize("cu", [[0, 190], [5, 200], [70, 75, 130], [3, 3, 64, 128], [64, 192], [199, 200], [0, 1], [200, 200]])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 4), (96, 2)])
@pytest.mark.parametrize("window,first", [(0, 0), (20, 0), (20, 9)])
def test_tokens_in_no_sequence_have_no_influence(dev, cu, Hq, Hkv, window, first):
    """Garbage in q, k, v and dout before a packed row's first sequence and behind its last: the same bits."""
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, Hq, Hkv, 200, 200, 64)
    dead = torch.ones(200, dtype=torch.bool, device=dev)
    dead[cu[0]:cu[-1]] = False
    c = torch.tensor(cu, dtype=torch.int32, device=dev)
    res = []
    for bad in (0.0, math.nan, math.inf):
        t = [x.clone() for x in (q, k, v)]
        for x in t:
            x[:, :, dead] = bad
        d = do.clone()
        d[:, dead] = bad
        leaves = [x.requires_grad_() for x in (*t, s.detach().clone())]
        out = sink_attention(*leaves, window=window, first=first, cu_seqlens=c)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, d)])
        assert not out[:, dead].any() and not any(g[:, :, dead].any() for g in res[-1][1:4])
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))
    assert all(torch.isfinite(t).all() for t in res[0])


def test_tokens_in_no_sequence_d128(dev):
    for cu, window, first in (([37, 100, 171], 0, 0), ([37, 100, 171], 50, 3)):
        _check(dev, 1, 6, 2, 200, 200, 128, cu_seqlens=cu, window=window, first=first)
        test_tokens_in_no_sequence_have_no_influence(dev, cu, 6, 2, window, first)


@pytest.mark.parametrize("G,D", [(1, 64), (8, 64), (3, 128)])
@pytest.mark.parametrize("window,first", [(0, 0), (20, 0), (20, 3)])
def test_a_batch_of_packed_rows(dev, G, D, window, first):
    """Starts of each batch row's own, forward and backward: every row as by itself, with the same bits."""
    from agent_factory_3_amd import attention
    S, cuts = 300, [[0, 70, 71, 300], [0, 150, 300], [0, 300], [0, 64, 128, 299, 300]]
    q, k, v, s, do = _make(dev, 4, 2 * G, 2, S, S, D)
    pos = torch.stack([torch.cat([torch.arange(b - a) for a, b in zip(c, c[1:])]) for c in cuts]).to(dev)
    starts = attention.sequence_starts_of_rows(pos)
    assert torch.equal(starts.cpu(), torch.stack([oa.starts_of(c, S) for c in cuts]).to(torch.int32))
    assert torch.equal(attention.sequence_starts_of_rows(pos[:1]), attention.sequence_starts_of_positions(pos[0])[None])
    leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
    out = attention._run(*leaves, D ** -0.5, window, first, None, starts, None)
    grads = torch.autograd.grad(out, leaves, do)
    if not first:
        import types
        for mask, ids in ((None, pos), (pos[..., None], None)):   # the layers' call, by either
            one, _ = attention.attention_forward(types.SimpleNamespace(is_causal=True), q, k, v, mask, position_ids=ids,
                                                 sliding_window=window, s_aux=s)
            assert torch.equal(one, out)
    dsinks = torch.zeros(2 * G, dtype=torch.float64)
    tol = torch.zeros(2 * G, dtype=torch.float64)
    for b, c in enumerate(cuts):
        one = [t[b:b + 1].detach().requires_grad_() for t in (q, k, v)]
        cu = torch.tensor(c, dtype=torch.int32, device=dev)
        o = attention.sink_attention(*one, s, window=window, first=first, cu_seqlens=cu)
        assert torch.equal(o, out[b:b + 1])
        for g, w in zip(torch.autograd.grad(o, one, do[b:b + 1]), grads):
            assert torch.equal(g, w[b:b + 1])
        ref = oa.attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], s, window=window, first=first, cu_seqlens=c,
                           dout=do[b:b + 1], bounds=True)
        dsinks += ref["dsinks"]
        tol += ref["dsinks_tol"]
    # (each row's bound holds a rounding of its own sum to bf16, together no less than the whole's one)
    _close(grads[3], dsinks, tol, "dsinks")


def _by_positions(q, k, v, s, pos, kv_range=None, window=0):
    """The layers' call: transformers' interface with position ids."""
    import types

    from agent_factory_3_amd import attention
    out, _ = attention.attention_forward(types.SimpleNamespace(is_causal=True), q, k, v, kv_range, position_ids=pos,
                                         sliding_window=window, s_aux=s)
    return out


@pytest.mark.parametrize("pad", [(0, 30), (30, 0), (7, 1), (64, 64), (0, 0)])
@pytest.mark.parametrize("window", [0, 20])
def test_a_padded_packed_row_keeps_its_sequences(dev, pad, window):
    """One row of sequences by position ids, with padding before or behind: each sequence sees itself alone."""
    lens = [50, 1, 40, 61]
    n, S = sum(lens), sum(lens) + sum(pad)
    q, k, v, s, do = _make(dev, 1, 8, 2, S, S, 64)
    pos = torch.cat([torch.ones(pad[0], dtype=torch.int64)] + [torch.arange(x) for x in lens] +
                    [torch.zeros(pad[1], dtype=torch.int64)])[None].to(dev)
    rng = torch.tensor([[pad[0], pad[0] + n]], dtype=torch.int32, device=dev)
    cu = [pad[0] + x for x in (0, 50, 51, 91, 152)]
    leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
    out = _by_positions(*leaves, pos, rng, window)
    ref = oa.attention(q, k, v, s, window=window, cu_seqlens=cu, dout=do, bounds=True)
    _close(out, ref["out"], ref["out_tol"], "out")
    for name, g in zip(("dq", "dk", "dv", "dsinks"), torch.autograd.grad(out, leaves, do)):
        _close(g, ref[name], ref[name + "_tol"], name)


def test_starts_of_rows_within_ranges(dev):
    from agent_factory_3_amd.attention import sequence_starts_of_rows
    pos = torch.tensor([[1, 1, 0, 1, 2, 0, 1, 0, 0], [0, 1, 2, 3, 4, 5, 0, 1, 0]], device=dev)
    for dtype in (torch.int32, torch.int64):
        rng = torch.tensor([[2, 7], [0, 8]], dtype=dtype, device=dev)
        assert sequence_starts_of_rows(pos, rng).tolist() == [[1, 2, 2, 2, 2, 5, 5, 8, 9], [0] * 6 + [6, 6, 9]]
    # a range inside a sequence starts it there; outside the row it is clamped
    t = torch.arange(2000)
    ends = [(-5, 3000), (700, 1500), (5, 5), (1500, 700), (2000, 2000)]
    got = sequence_starts_of_rows(t.to(dev).expand(5, -1), torch.tensor(ends, device=dev)).cpu()
    for row, (a, b) in zip(got, ends):
        assert torch.equal(row, torch.where((t >= a) & (t < b), max(a, 0), t + 1).to(torch.int32))
    for bad in (torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.zeros(2, 2, device=dev),
                torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            sequence_starts_of_rows(pos, bad)
    for bad, exc in ((pos[0], ValueError), (pos.float(), ValueError), (pos.cpu(), RuntimeError)):
        with pytest.raises(exc):
            sequence_starts_of_rows(bad)


def test_forward_mode_derivatives_are_refused(dev):
    import torch.autograd.forward_ad as fwd

    from agent_factory_3_amd import routing
    from agent_factory_3_amd.attention import sink_attention
    q, k, v, s, do = _make(dev, 1, 4, 2, 20, 20, 64)
    z = torch.randn(20, 8, device=dev).to(torch.bfloat16)
    kl, zl = k.detach().requires_grad_(), z.detach().requires_grad_()
    with fwd.dual_level():
        out, (loss, _) = sink_attention(q, kl, v, s), routing.balance_loss(zl, 2)
        dual = lambda t: fwd.make_dual(t.detach(), torch.ones_like(t))  # noqa: E731
        for keys in (k, kl):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                sink_attention(dual(q), keys, v, s)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            routing.balance_loss(dual(z), 2)
        # a tangent of the gradient that arrives
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, kl, dual(do))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(loss, zl, dual(torch.ones((), device=dev)))


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int64])
def test_integer_types_of_lengths_and_ranges(dev, dtype):
    from agent_factory_3_amd.attention import sequence_starts, sink_attention
    q, k, v, s, _ = _make(dev, 1, 4, 2, 300, 300, 64)
    cu, rng = torch.tensor([0, 20, 100], device=dev), torch.tensor([[10, 120]], device=dev)
    for n, t in (("cu_seqlens", cu), ("kv_range", rng)):
        assert torch.equal(sink_attention(q, k, v, s, **{n: t.to(dtype)}), sink_attention(q, k, v, s, **{n: t.int()}))
    assert torch.equal(sequence_starts(cu.to(dtype), 300), sequence_starts(cu.int(), 300))


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (6, 6, 128)])
@pytest.mark.parametrize("window", [0, 20])
def test_position_ids_are_the_cumulative_lengths(dev, Hq, Hkv, D, window):
    """transformers' interface with position ids that start again, forward and backward: the bits of
    the call with cumulative lengths, and the oracle's bounds."""
    from agent_factory_3_amd.attention import sink_attention
    lens = [50, 1, 40, 61]
    q, k, v, s, do = _make(dev, 1, Hq, Hkv, 152, 152, D)
    pos = torch.cat([torch.arange(x) for x in lens])[None].to(dev)
    cu = torch.tensor([0, 50, 51, 91, 152], dtype=torch.int32, device=dev)
    res = []
    for call in (lambda *t: _by_positions(*t, pos, None, window), lambda *t: sink_attention(*t, window=window, cu_seqlens=cu)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
        out = call(*leaves)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, do)])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    ref = oa.attention(q, k, v, s, window=window, cu_seqlens=cu.tolist(), dout=do, bounds=True)
    for name, t in zip(("out", "dq", "dk", "dv", "dsinks"), res[0]):
        _close(t, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("S", [1, 4095, 4096, 4097, 12288, 40001])
def test_starts_of_long_rows(dev, S):
    """Sequences that cross many blocks' tokens, one that fills its row, and starts at the blocks' edges."""
    from agent_factory_3_amd.attention import sequence_starts_of_positions, sequence_starts_of_rows
    g = torch.Generator().manual_seed(S)
    t = torch.arange(S)
    rows = [torch.zeros(S, dtype=torch.bool), torch.rand(S, generator=g) < 1e-3, torch.rand(S, generator=g) < 0.5,
            t % 4096 == 0, t % 4096 == 4095, t % 1024 == 1023, t % 64 == 63, t == 1, t == S - 1]
    want = torch.stack([torch.where(r, t, 0).cummax(0).values for r in rows])
    pos = (t - want + torch.randint(0, 1 << 40, (len(rows), 1), generator=g)).to(dev)
    assert torch.equal(sequence_starts_of_rows(pos).cpu(), want.to(torch.int32))
    for p, w in zip(pos, want):
        assert torch.equal(sequence_starts_of_positions(p).cpu(), w.to(torch.int32))
    a, b = S // 3, S - S // 4
    rng = torch.tensor([[a, b]] * len(rows), device=dev)
    inside = torch.where((t >= a) & (t < b), want.clamp(min=a), t + 1)
    assert torch.equal(sequence_starts_of_rows(pos, rng).cpu(), inside.to(torch.int32))


@pytest.mark.parametrize("window,first", [(0, 0), (600, 0), (600, 70)])
def test_packed_rows_whose_keys_are_split(dev, window, first):
    """Few enough tiles that each row's keys go over several blocks: sequences, tokens in none of them
    at both ends (garbage there too), and a batch of such rows."""
    from agent_factory_3_amd import attention
    S, cuts = 1100, [[30, 700, 1050], [0, 1, 1100], [0, 1040]]
    q, k, v, s, do = _make(dev, 3, 8, 1, S, S, 64)
    dead = torch.ones(3, S, dtype=torch.bool, device=dev)
    pos, rng = torch.zeros(3, S, dtype=torch.long), []
    for b, c in enumerate(cuts):
        dead[b, c[0]:c[-1]] = False
        pos[b, c[0]:c[-1]] = torch.cat([torch.arange(y - x) for x, y in zip(c, c[1:])])
        rng.append((c[0], c[-1]))
    for n, t in (("q", q), ("k", k), ("v", v)):
        t.transpose(1, 2)[dead] = math.nan
    do[dead] = math.inf
    starts = attention.sequence_starts_of_rows(pos.to(dev), torch.tensor(rng, device=dev))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention._run(*leaves, s, 0.125, window, first, None, starts, None)
    grads = torch.autograd.grad(out, leaves, do)
    for b, c in enumerate(cuts):
        one = [t[b:b + 1].detach().requires_grad_() for t in (q, k, v)]
        alone = attention.sink_attention(*one, s, window=window, first=first,
                                         cu_seqlens=torch.tensor(c, dtype=torch.int32, device=dev))
        alone_g = torch.autograd.grad(alone, one, do[b:b + 1])
        live = [x.clone() for x in (q[b:b + 1], k[b:b + 1], v[b:b + 1], do[b:b + 1])]
        for t in live[:3]:
            t.transpose(1, 2)[dead[b:b + 1]] = 0
        live[3][dead[b:b + 1]] = 0
        ref = oa.attention(*live[:3], s, window=window, first=first, cu_seqlens=c, dout=live[3], bounds=True)
        for o, g in ((out[b:b + 1], [x[b:b + 1] for x in grads]), (alone, alone_g)):
            _close(o, ref["out"], ref["out_tol"], "out")
            for name, x in zip(("dq", "dk", "dv"), g):
                _close(x, ref[name], ref[name + "_tol"], name)
