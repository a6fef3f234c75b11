"""Residual norms on the GPU against the float64 oracle."""
import pytest
import torch

from oracle import norms as on

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(rows, H, xt, rt, dev, *, post=False, gate=None, wt=None, seed=0, big=True):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": (rand(rows, H) * 1.5).to(xt), "weight": (rand(H) * 0.3 + 1).to(wt or xt), "residual": None, "post": None,
         "gate": None, "dr": None, "dh": rand(rows, H).to(xt)}
    if rt is not None:
        t["residual"] = (rand(rows, H) * 2 * (1 + 20 * (rand(H) > 2.0) * big)).to(rt)
        t["dr"] = rand(rows, H).to(rt)
    if post:
        t["post"] = (rand(H) * 0.3 + 1).to(wt or xt)
    if gate is not None:
        t["gate"] = (rand(*gate) * 0.7).to(wt or xt)
    return t, {n: None if v is None else v.to(dev) for n, v in t.items()}


def _call(d, scale=1.0, eps=1e-5, shape=None, grads=True):
    """Outputs and gradients of the public calls, as [rows, H]."""
    from agent_factory_3_amd import norms
    names = [n for n in ("x", "residual", "weight", "post", "gate") if d[n] is not None]
    d = dict(d)
    for n in names:
        if shape is not None and n in ("x", "residual"):
            d[n] = d[n].view(*shape, -1)
        d[n] = d[n].detach().requires_grad_(grads)
    if d["residual"] is None:
        h = norms.rms_norm(d["x"], d["weight"], eps)
        outs, ups, res = [h], [d["dh"].view(h.shape)], {"h": h}
    else:
        r, h = norms.residual_norm(d["x"], d["residual"], d["weight"], eps=eps, post_weight=d["post"], gate=d["gate"],
                                   scale=scale)
        res = {"r": r, "h": h}
        outs = [t for t in (r, h) if t is not None]
        ups = [d["dr"].view(r.shape)] + ([d["dh"].view(r.shape)] if h is not None else [])
    res = {n: t.detach() for n, t in res.items() if t is not None}
    if grads:
        key = {"post": "dpost_weight"}
        res.update((key.get(n, "d" + n), g) for n, g in zip(names, torch.autograd.grad(outs, [d[n] for n in names], ups)))
    return res


def _compare(got, want, rows):
    assert {n for n in want if not n.endswith("_tol")} == set(got)
    for n, t in got.items():
        t = t.detach().cpu().double().reshape(want[n].shape)
        err = (t - want[n]).abs()
        assert (err <= want[n + "_tol"]).all(), (n, float((err / want[n + "_tol"]).nan_to_num(nan=9e9).max()))


@pytest.mark.parametrize("H", [8, 9, 15, 64, 77, 513, 1000, 1024, 1025, 2047, 2880, 2881, 4096, 4100, 8192, 8193, 16383,
                               16384])
@pytest.mark.parametrize("xt,rt", [(BF, None), (BF, BF), (BF, F32), (F32, F32), (F32, None)])
def test_sizes_and_types(dev, H, xt, rt):
    rows = 5 if H > 100 else 33
    t, d = _inputs(rows, H, xt, rt, dev, seed=H)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], dr=t["dr"], dh=t["dh"])
    _compare(_call(d), want, rows)


@pytest.mark.parametrize("H", [64, 77, 2880, 5000, 16384])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token", "full", "one", "position"])
@pytest.mark.parametrize("post", [False, True])
def test_post_norm_gate_scale(dev, H, gate, post):
    B, S = 3, 7
    shape = {None: None, "channel": (H,), "sequence": (B, 1, H), "token": (B, S, 1), "full": (B, S, H), "one": (1,),
             "position": (1, S, H)}[gate]
    if gate is None and not post:
        pytest.skip("test_sizes_and_types")
    for xt, rt in ((BF, BF), (BF, F32), (F32, F32)):
        t, d = _inputs(B * S, H, xt, rt, dev, post=post, gate=shape, wt=F32 if rt is F32 else BF, seed=H)
        full = None if shape is None else t["gate"].expand(B, S, shape[-1]).reshape(B * S, shape[-1])
        want = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["post"], gate=full, scale=0.3, dr=t["dr"],
                                dh=t["dh"])
        if shape is not None:   # the gate's gradient, summed over what it is shared by
            for n in ("dgate", "dgate_tol"):
                v = want[n].view(B, S, shape[-1])
                want[n] = v.sum_to_size(shape) if len(shape) == 3 else v.sum((0, 1))
        _compare(_call(d, scale=0.3, shape=(B, S)), want, B * S)


@pytest.mark.parametrize("rows,H", [(1, 2880), (2047, 512), (2048, 512), (2049, 2880), (5003, 1024), (4111, 333), (9000, 64)])
@pytest.mark.parametrize("rt", [None, BF])
def test_row_counts(dev, rows, H, rt):
    t, d = _inputs(rows, H, BF, rt, dev, seed=rows)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], dr=t["dr"], dh=t["dh"])
    _compare(_call(d), want, rows)


def test_gate_groups_over_many_rows(dev):
    B, S, H = 5, 700, 264
    t, d = _inputs(B * S, H, BF, F32, dev, post=True, gate=(B, 1, H), seed=3)
    full = t["gate"].expand(B, S, H).reshape(B * S, H)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["post"], gate=full, dr=t["dr"], dh=t["dh"])
    want["dgate"], want["dgate_tol"] = (want[n].view(B, S, H).sum(1, keepdim=True) for n in ("dgate", "dgate_tol"))
    # (700 values of one type's rounding: the bound's last term is of the sum)
    _compare(_call(d, shape=(B, S)), want, B * S)


def test_only_some_outputs_and_gradients(dev):
    from agent_factory_3_amd import norms
    t, d = _inputs(40, 520, BF, BF, dev, post=True, gate=(520,))
    for names in (("x",), ("residual",), ("weight",), ("post",), ("gate",), ("x", "gate")):
        for used in ("r", "h", "both"):
            if names == ("weight",) and used == "r":
                continue
            dr, dh = (t["dr"] if used != "h" else None), (t["dh"] if used != "r" else None)
            want = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["post"], gate=t["gate"], dr=dr, dh=dh)
            leaf = {n: v.detach().requires_grad_(n in names) for n, v in d.items() if n not in ("dr", "dh")}
            r, h = norms.residual_norm(leaf["x"], leaf["residual"], leaf["weight"], post_weight=leaf["post"], gate=leaf["gate"])
            outs = [o for o, u in ((r, dr), (h, dh)) if u is not None]
            got = torch.autograd.grad(outs, [leaf[n] for n in names], [u.to(dev) for u in (dr, dh) if u is not None])
            _compare({{"post": "dpost_weight"}.get(n, "d" + n): g for n, g in zip(names, got)},
                     {k: v for k, v in want.items() if k.removesuffix("_tol") in
                      {{"post": "dpost_weight"}.get(n, "d" + n) for n in names}}, 40)
    # no norm after the sum
    want = on.residual_norm(t["x"], t["residual"], None, gate=t["gate"], scale=2.0, dr=t["dr"])
    _compare(_call({**d, "weight": None, "post": None}, scale=2.0), want, 40)
    want = on.residual_norm(t["x"], t["residual"], None, dr=t["dr"])
    _compare(_call({**d, "weight": None, "post": None, "gate": None}), want, 40)


@pytest.mark.parametrize("H", [96, 101])
def test_strides_and_alignment(dev, H):
    """Rows of wider tensors at any element, rows in another order, a broadcast row; weights that are views."""
    from agent_factory_3_amd import norms
    t, d = _inputs(60, H, BF, BF, dev, seed=1)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], dr=t["dr"], dh=t["dh"])
    for shift in (0, 1, 3, 8):
        e = dict(d)
        for n in ("x", "residual", "dr", "dh"):
            wide = torch.full((60, H + 13), float("nan"), dtype=BF, device=dev)
            wide[:, shift:shift + H] = d[n]
            e[n] = wide[:, shift:shift + H]
        two = torch.full((H, 2), float("nan"), dtype=BF, device=dev)
        two[:, 1] = d["weight"]
        e["weight"] = two[:, 1]
        leaf = {n: e[n].detach().requires_grad_() for n in ("x", "residual", "weight")}
        r, h = norms.residual_norm(leaf["x"], leaf["residual"], leaf["weight"])
        g = torch.autograd.grad([r, h], list(leaf.values()), [e["dr"], e["dh"]])
        _compare({"r": r, "h": h, "dx": g[0], "dresidual": g[1], "dweight": g[2]}, want, 60)
    # columns first, and one row for all
    col = d["x"].t().contiguous().t()
    assert torch.equal(norms.rms_norm(col, d["weight"]), norms.rms_norm(d["x"], d["weight"]))
    row = d["x"][:1].expand(60, H)
    assert torch.equal(norms.rms_norm(row, d["weight"]), norms.rms_norm(row.contiguous(), d["weight"]))
    leaf = d["x"].detach().requires_grad_()
    (g,) = torch.autograd.grad(norms.rms_norm(leaf, d["weight"]).float().sum(), leaf)   # an expanded gradient
    (g2,) = torch.autograd.grad(norms.rms_norm(leaf, d["weight"]), leaf, torch.ones_like(leaf))
    assert torch.equal(g, g2)


def test_rows_of_zeros_and_values_that_are_not_finite(dev):
    """A zero row gives zeros (eps holds the quotient); a NaN or infinity stays in its row."""
    from agent_factory_3_amd import norms
    t, d = _inputs(20, 2880, BF, BF, dev)
    d["x"][3] = 0
    d["residual"][3] = 0
    d["x"][5, 17], d["residual"][7, 2879] = float("nan"), float("inf")
    r, h = norms.residual_norm(d["x"], d["residual"], d["weight"])
    assert (h[3] == 0).all() and (r[3] == 0).all()
    assert h[5].isnan().all() and r[5].isnan().sum() == 1 and r[7, 2879].isinf() and h[7, 2879].isnan()
    ok = torch.tensor([i not in (5, 7) for i in range(20)], device=dev)
    assert h[ok].isfinite().all() and r[ok].isfinite().all()
    leaf = d["x"].detach().requires_grad_()
    r, h = norms.residual_norm(leaf, d["residual"], d["weight"])
    (g,) = torch.autograd.grad(h, leaf, d["dh"])
    assert g[ok].isfinite().all() and not g[5].isfinite().any()


def test_empty(dev):
    from agent_factory_3_amd import norms
    x = torch.empty(0, 5, 64, dtype=BF, device=dev, requires_grad=True)
    w = torch.ones(64, dtype=BF, device=dev, requires_grad=True)
    gate = torch.ones(64, dtype=BF, device=dev, requires_grad=True)
    r, h = norms.residual_norm(x, x, w, gate=gate)
    g = torch.autograd.grad([r, h], [x, w, gate], [r.detach(), h.detach()])
    assert r.shape == h.shape == g[0].shape == (0, 5, 64) and (g[1] == 0).all() and (g[2] == 0).all()


def test_same_bits_twice_and_on_another_stream(dev):
    t, d = _inputs(3000, 2880, BF, BF, dev, post=True, gate=(2880,))
    want = _call(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_captured(dev):
    from agent_factory_3_amd import norms
    t, d = _inputs(2500, 1024, BF, BF, dev)
    leaf = {n: d[n].clone().requires_grad_() for n in ("x", "residual", "weight")}

    def step():
        r, h = norms.residual_norm(leaf["x"], leaf["residual"], leaf["weight"])
        return (r.detach(), h.detach()) + torch.autograd.grad([r, h], list(leaf.values()), [d["dr"], d["dh"]])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        new = _inputs(2500, 1024, BF, BF, dev, seed=10 + n)[1]
        with torch.no_grad():
            for k in leaf:
                leaf[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        want = _call({**d, **{k: leaf[k].detach() for k in leaf}})
        for a, k in zip(held, ("r", "h", "dx", "dresidual", "dweight")):
            assert torch.equal(a, want[k]), k


def test_saved_tensors_that_come_back_with_other_strides(dev):
    t, d = _inputs(50, 200, BF, BF, dev, post=True, gate=(50, 1))
    want = _call(d)
    with torch.autograd.graph.save_on_cpu():
        got = _call(d)
    assert all(torch.equal(want[n], got[n]) for n in want)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.t().contiguous().t() if v.dim() == 2 else v, lambda v: v):
        got = _call(d)
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_rows_past_32_bit_offsets(dev):
    """A tensor of more than 2^31 elements: its last rows as alone."""
    from agent_factory_3_amd import norms
    H = 16384
    rows = (1 << 31) // H + 5
    x = torch.zeros(rows, H, dtype=BF, device=dev)
    w = torch.ones(H, dtype=BF, device=dev)
    x[-5:] = _inputs(5, H, BF, None, dev)[1]["x"]
    h = norms.rms_norm(x, w)
    assert torch.equal(h[-5:], norms.rms_norm(x[-5:].clone(), w)) and (h[0] == 0).all()


def test_refusals(dev):
    from agent_factory_3_amd import norms
    x = torch.zeros(4, 64, dtype=BF, device=dev)
    w = torch.zeros(64, dtype=BF, device=dev)
    for exc, args, kw in [(RuntimeError, (x.cpu(), x, w), {}), (TypeError, (x.half(), x.half(), w), {}),
                          (ValueError, (x[:, :7], x[:, :7], w[:7]), {}), (ValueError, (x, x[:3], w), {}),
                          (ValueError, (x, x, w[:63]), {}), (TypeError, (x.float(), x, w), {}),
                          (TypeError, (x, x, w.half()), {}), (RuntimeError, (x, x, w.cpu()), {}),
                          (ValueError, (x, x, w), dict(gate=w[:63])), (ValueError, (x, x, w), dict(gate=x.view(1, 4, 64))),
                          (ValueError, (x, x, w), dict(post_weight=w[:2])), (ValueError, (x, x, w), dict(eps=-1.0)),
                          (ValueError, (x, x, w), dict(scale=float("nan"))),
                          (RuntimeError, (x, x, w), dict(gate=w.cpu())), (TypeError, (x, x, w), dict(gate=w.int())),
                          (ValueError, (x.repeat(1, 257), x.repeat(1, 257), w.repeat(257)), {})]:
        with pytest.raises(exc):
            norms.residual_norm(*args, **kw)
    with pytest.raises(ValueError):
        norms.rms_norm(x[0, 0], w)


def test_one_tensor_in_several_places(dev):
    """x as the residual too, one weight for both norms: the gradients add up."""
    from agent_factory_3_amd import norms
    t, d = _inputs(30, 264, BF, BF, dev)
    x, w = (d[n].detach().requires_grad_() for n in ("x", "weight"))
    want = on.residual_norm(t["x"], t["x"], t["weight"], dr=t["dr"], dh=t["dh"])
    r, h = norms.residual_norm(x, x, w)
    (g,) = torch.autograd.grad([r, h], [x], [d["dr"], d["dh"]])
    both = want["dx"] + want["dresidual"]   # (each half rounded, and the sum)
    tol = want["dx_tol"] + want["dresidual_tol"] + 2.0 ** -8 * both.abs()
    assert ((g.cpu().double() - both).abs() <= tol).all()
    want = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["weight"], dr=t["dr"], dh=t["dh"])
    r, h = norms.residual_norm(x, d["residual"], w, post_weight=w)
    (g,) = torch.autograd.grad([r, h], [w], [d["dr"], d["dh"]])
    both = want["dweight"] + want["dpost_weight"]
    tol = want["dweight_tol"] + want["dpost_weight_tol"] + 2.0 ** -8 * both.abs()
    assert ((g.cpu().double() - both).abs() <= tol).all()


def test_gate_of_no_dimension_and_fp32_rows_at_any_element(dev):
    from agent_factory_3_amd import norms
    t, d = _inputs(20, 77, F32, F32, dev)
    wide = torch.full((20, 90), float("nan"), device=dev)
    wide[:, 5:82] = d["x"]
    gate = torch.tensor(0.5, device=dev, requires_grad=True)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], gate=torch.full((20, 1), 0.5), dr=t["dr"], dh=t["dh"])
    r, h = norms.residual_norm(wide[:, 5:82], d["residual"], d["weight"], gate=gate)
    (g,) = torch.autograd.grad([r, h], [gate], [d["dr"], d["dh"]])
    _compare({"r": r, "h": h}, {k: v for k, v in want.items() if k[0] in "rh"}, 20)
    # (20 rows' sums, each within its bound, added in fp32 and rounded to it)
    assert g.shape == () and abs(float(g) - float(want["dgate"].sum())) <= float(want["dgate_tol"].sum()) + 2.0 ** -20 * float(want["dgate"].abs().sum())


def test_frozen_weight_uses_the_stored_stream(dev):
    """Only x's and the residual's gradients (adapters trained elsewhere): within the bounds too, and
    where the weight is trained but its gradient not asked for."""
    from agent_factory_3_amd import norms
    t, d = _inputs(300, 1000, BF, BF, dev)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], dr=t["dr"], dh=t["dh"])
    for trained in (False, True):
        leaf = {n: d[n].detach().requires_grad_(n != "weight" or trained) for n in ("x", "residual", "weight")}
        r, h = norms.residual_norm(leaf["x"], leaf["residual"], leaf["weight"])
        g = torch.autograd.grad([r, h], [leaf["x"], leaf["residual"]], [d["dr"], d["dh"]])
        _compare({"dx": g[0], "dresidual": g[1]}, {k: want[k] for k in ("dx", "dx_tol", "dresidual", "dresidual_tol")}, 300)


@pytest.mark.parametrize("rows,H", [(1, 64), (511, 512), (512, 1016), (513, 333), (1023, 1032), (1024, 1025), (1025, 1030)])
@pytest.mark.parametrize("rt", [None, BF])
def test_row_counts_where_the_launch_changes(dev, rows, H, rt):
    t, d = _inputs(rows, H, BF, rt, dev, seed=rows)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], dr=t["dr"], dh=t["dh"])
    _compare(_call(d), want, rows)


@pytest.mark.parametrize("xt,rt", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("H,post,gate", [(9001, True, "sequence"), (8200, False, "token"), (12000, True, "channel"),
                                         (8193, True, "full"), (5003, True, "sequence")])
def test_long_rows_several_a_block(dev, xt, rt, H, post, gate):
    B, S = 2, 301
    shape = {"channel": (H,), "sequence": (B, 1, H), "token": (B, S, 1), "full": (B, S, H)}[gate]
    t, d = _inputs(B * S, H, xt, rt, dev, post=post, gate=shape, seed=H)
    full = t["gate"].expand(B, S, shape[-1]).reshape(B * S, shape[-1])
    for dh in (t["dh"], None):
        want = on.residual_norm(t["x"], t["residual"], t["weight"] if dh is not None else None, post=t["post"], gate=full,
                                scale=0.7, dr=t["dr"], dh=dh)
        for n in ("dgate", "dgate_tol"):
            v = want[n].view(B, S, shape[-1])
            want[n] = v.sum_to_size(shape) if len(shape) == 3 else v.sum((0, 1))
        got = _call({**d, "weight": d["weight"] if dh is not None else None}, scale=0.7, shape=(B, S))
        _compare(got, want, B * S)
        # each output of its own: the rows' gradients do not depend on which sums are wanted
        from agent_factory_3_amd import norms
        leaf = {n: d[n].view(B, S, H).detach().requires_grad_() for n in ("x", "residual")}
        r, h = norms.residual_norm(leaf["x"], leaf["residual"], d["weight"] if dh is not None else None,
                                   post_weight=d["post"], gate=d["gate"], scale=0.7)
        g = torch.autograd.grad([o for o in (r, h) if o is not None], list(leaf.values()),
                                [d["dr"].view(r.shape)] + ([d["dh"].view(r.shape)] if h is not None else []))
        keys = ("dx", "dresidual", "dx_tol", "dresidual_tol")
        _compare({"dx": g[0], "dresidual": g[1]}, {k: want[k] for k in keys}, B * S)


def test_tensors_without_memory_of_their_own_are_refused(dev):
    """A DTensor's address is 0: it must not pass for a tensor that is not given."""
    from agent_factory_3_amd import norms

    class Held(torch.Tensor):
        @classmethod
        def of(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} of a tensor without memory")

    x, w = torch.ones(2, 64, device=dev, dtype=BF), torch.ones(64, device=dev, dtype=BF)
    for name in ("x", "residual", "weight", "post_weight", "gate"):
        t = {"x": x, "residual": x, "weight": w, "post_weight": w, "gate": w}
        t[name] = Held.of(t[name])
        with pytest.raises(TypeError, match=name):
            norms.residual_norm(t["x"], t["residual"], t["weight"], post_weight=t["post_weight"], gate=t["gate"])
    with pytest.raises(TypeError, match="weight"):
        norms.rms_norm(x, Held.of(w))


@pytest.mark.parametrize("rows,H", [(1, 8), (300, 2880), (600, 512), (2048, 1000), (5, 9001)])
@pytest.mark.parametrize("xt,wt", [(BF, BF), (F32, F32), (BF, F32)])
def test_rms_norm_with_one_of_its_tensors_trained(dev, rows, H, xt, wt):
    """A trained weight behind a frozen x, and the other way round."""
    from agent_factory_3_amd import norms
    t, d = _inputs(rows, H, xt, None, dev, wt=wt, seed=H)
    want = on.residual_norm(t["x"], None, t["weight"], dh=t["dh"])
    for name in ("weight", "x"):
        leaf = {n: d[n].detach().requires_grad_(n == name) for n in ("x", "weight")}
        h = norms.rms_norm(leaf["x"], leaf["weight"])
        (g,) = torch.autograd.grad(h, leaf[name], d["dh"])
        _compare({"h": h, "d" + name: g}, {k: v for k, v in want.items() if k.removesuffix("_tol") in ("h", "d" + name)}, rows)


@pytest.mark.parametrize("H", [64, 2880, 8192, 9000, 16384])
@pytest.mark.parametrize("xt,rt", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_a_gated_branch_that_is_not_finite(dev, H, xt, rt, gate):
    """dx = scale gate dr whatever x holds, where only r's gradient arrives and x has no norm of its own; the
    gate's gradient is not finite where x is not."""
    from agent_factory_3_amd import norms
    rows = 9
    shape = {"channel": (H,), "token": (rows, 1), "full": (rows, H)}[gate]
    t, d = _inputs(rows, H, xt, rt, dev, gate=shape, seed=H)
    want = on.residual_norm(t["x"], t["residual"], None, gate=t["gate"], scale=0.5, dr=t["dr"])
    x = d["x"].clone()
    x[2, 5], x[4, H - 1], x[7, 0] = float("inf"), float("-inf"), float("nan")
    for used in (False, True):   # no weight; a weight whose output no loss reads
        leaf = {n: v.detach().requires_grad_() for n, v in (("x", x), ("residual", d["residual"]), ("gate", d["gate"]))}
        r, h = norms.residual_norm(leaf["x"], leaf["residual"], d["weight"] if used else None, gate=leaf["gate"], scale=0.5)
        dx, dres, dg = torch.autograd.grad(r, list(leaf.values()), d["dr"])
        _compare({"dx": dx, "dresidual": dres}, {k: v for k, v in want.items() if k.split("_")[0] in ("dx", "dresidual")}, rows)
        bad = ~x.isfinite()
        bad = bad.any(0) if gate == "channel" else bad.any(1, keepdim=True) if gate == "token" else bad
        assert torch.equal(dg.isfinite(), ~bad)


def test_more_rows_and_gates_than_a_launch_holds(dev):
    """Past 2^24 rows of four waves each, and 2^24 gate values shared by two rows (a launch holds less than 2^32
    threads).  Small whole numbers: every sum is exact."""
    from agent_factory_3_amd import norms
    G, H = (1 << 24) + 77, 8
    g = torch.Generator(dev).manual_seed(0)
    draw = lambda *s: torch.randint(-2, 3, s, generator=g, device=dev, dtype=torch.int8).to(BF)  # noqa: E731
    x, res, gate = draw(G, 2, H), draw(G, 2, H), draw(G, 1, 1).requires_grad_()
    r, _ = norms.residual_norm(x, res, gate=gate)
    assert torch.equal(r, res + gate.detach() * x)   # (at most 6)
    (dg,) = torch.autograd.grad(r, gate, res)
    assert torch.equal(dg, (res * x).sum((1, 2), dtype=F32)[:, None, None].to(BF))   # (at most 64)


@pytest.mark.parametrize("G,S,H,post,rt", [(257, 3, 264, True, BF), (3001, 3, 264, False, F32), (5000, 2, 77, True, BF),
                                           (700, 2, 5003, True, F32), (600, 2, 5003, False, BF), (300, 3, 9001, True, BF),
                                           (513, 2, 8200, False, F32)])
def test_gate_of_many_short_groups(dev, G, S, H, post, rt):
    """More groups than the backward has blocks: a gate [G, 1, H] shared by two or three rows."""
    t, d = _inputs(G * S, H, BF, rt, dev, post=post, gate=(G, 1, H), seed=H)
    full = t["gate"].expand(G, S, H).reshape(G * S, H)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["post"], gate=full, dr=t["dr"], dh=t["dh"])
    want["dgate"], want["dgate_tol"] = (want[n].view(G, S, H).sum(1, keepdim=True) for n in ("dgate", "dgate_tol"))
    _compare(_call(d, shape=(G, S)), want, G * S)
    # the gate's gradient alone, which no other sum is made beside
    from agent_factory_3_amd import norms
    gate = d["gate"].detach().requires_grad_()
    r, h = norms.residual_norm(d["x"].view(G, S, H), d["residual"].view(G, S, H), d["weight"], post_weight=d["post"], gate=gate)
    (g,) = torch.autograd.grad([r, h], gate, [d["dr"].view(r.shape), d["dh"].view(r.shape)])
    _compare({"dgate": g}, {k: want[k] for k in ("dgate", "dgate_tol")}, G * S)


def test_gate_of_heads_and_a_last_group_that_is_not_whole(dev):
    """[B, S, heads, D] with a gate [B, S, 1, D]; the C entry with 1001 rows in groups of two."""
    from agent_factory_3_amd import _capi
    B, S, N, D = 2, 301, 4, 64
    t, d = _inputs(B * S * N, D, BF, BF, dev, gate=(B, S, 1, D), seed=1)
    full = t["gate"].expand(B, S, N, D).reshape(-1, D)
    want = on.residual_norm(t["x"], t["residual"], t["weight"], gate=full, dr=t["dr"], dh=t["dh"])
    want["dgate"], want["dgate_tol"] = (want[n].view(B, S, N, D).sum(2, keepdim=True) for n in ("dgate", "dgate_tol"))
    _compare(_call(d, shape=(B, S, N)), want, B * S * N)
    for G, per in ((501, 2), (101, 10)):
        rows, H = G * per - 1, 72
        t, d = _inputs(rows, H, F32, F32, dev, gate=(G, H), seed=2)
        full = t["gate"].repeat_interleave(per, 0)[:rows]
        want = on.residual_norm(t["x"], t["residual"], None, gate=full, dr=t["dr"])
        for n in ("dgate", "dgate_tol"):
            want[n] = torch.cat([want[n], want[n].new_zeros(1, H)]).view(G, per, H).sum(1)
        want = {k: v for k, v in want.items() if k[0] == "d"}
        n = int(_capi.load().af3_residual_norm_bwd_workspace_bytes(rows, H, 1, H, per, 0, 0, 1))
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device=dev)
        dx, dres, dg = torch.empty_like(d["x"]), torch.empty_like(d["x"]), torch.full((G + 1, H), 7.0, device=dev)
        p = lambda v: v.data_ptr()  # noqa: E731
        _capi.call("af3_residual_norm_bwd", p(d["dr"]), H, None, 0, None, 1, 0, 0, p(d["x"]), 1, H, None, None, None, 0, None, 0,
                   p(d["gate"]), 1, H, per, 1.0, 1, rows, H, p(dx), p(dres), None, None, p(dg), p(ws), n,
                   torch.cuda.current_stream().cuda_stream)
        _compare({"dx": dx, "dresidual": dres, "dgate": dg[:G]}, want, rows)
        assert (dg[G] == 7).all()


def test_gate_of_more_groups_than_the_joining_launch_held(dev):
    """24000 groups of two rows of 2880.  Small whole numbers: every sum is exact."""
    from agent_factory_3_amd import norms
    G, S, H = 24000, 2, 2880
    g = torch.Generator(dev).manual_seed(0)
    draw = lambda *s: torch.randint(-2, 3, s, generator=g, device=dev, dtype=torch.int8).to(BF)  # noqa: E731
    x, res, gate = draw(G, S, H), draw(G, S, H), draw(G, 1, H).requires_grad_()
    r, _ = norms.residual_norm(x, res, gate=gate)
    (dg,) = torch.autograd.grad(r, gate, res)
    assert torch.equal(dg, (res * x).sum(1, keepdim=True))
