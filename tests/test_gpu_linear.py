"""Projections with an epilogue on the GPU against the float64 oracle."""
import pytest
import torch

from oracle import linear as ol

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(T, K, N, dev, *, bias=BF, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": rand(T, K).to(BF), "weight": (rand(N, K) * 1.5 * K ** -0.5).to(BF),
         "bias": rand(N).to(bias) if bias is not None else None,
         "residual": (rand(T, N) * 3).to(BF) if residual else None, "dy": rand(T, N).to(BF)}
    return t, {n: None if v is None else v.to(dev) for n, v in t.items()}


def _call(d, activation=None, grads=True):
    from agent_factory_3_amd.linear import linear
    names = [n for n in ("x", "weight", "bias", "residual") if d[n] is not None]
    leaf = {n: d[n].detach().requires_grad_(grads) for n in names}
    y = linear(leaf["x"], leaf["weight"], leaf.get("bias"), activation=activation, residual=leaf.get("residual"))
    out = {"y": y.detach()}
    if grads:
        out.update(("d" + n, g) for n, g in zip(names, torch.autograd.grad(y, list(leaf.values()), d["dy"].view(y.shape))))
    return out


def _compare(got, want):
    for n, t in got.items():
        err = (t.cpu().double().reshape(want[n].shape) - want[n]).abs()
        assert (err <= want[n + "_tol"]).all(), (n, float((err / want[n + "_tol"]).nan_to_num(nan=9e9).max()))


def _oracle(t, activation=None, grads=True):
    return ol.linear(t["x"], t["weight"], t["bias"], activation, t["residual"], t["dy"] if grads else None)


@pytest.mark.parametrize("T,K,N", [(1, 8, 8), (1, 1, 1), (3, 7, 5), (16, 64, 16), (17, 65, 31), (32, 200, 48), (33, 64, 64),
                                   (33, 63, 65), (64, 128, 72), (100, 1000, 513), (77, 2880, 512), (129, 72, 130),
                                   (257, 520, 256), (300, 96, 1030), (256, 256, 256), (513, 192, 385), (128, 4096, 136)])
def test_sizes(dev, T, K, N):
    t, d = _inputs(T, K, N, dev, seed=T)
    _compare(_call(d), _oracle(t))


@pytest.mark.parametrize("activation", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("T,K,N", [(5, 96, 40), (150, 88, 136), (70, 33, 51)])
@pytest.mark.parametrize("bias,residual", [(BF, False), (None, True), (F32, True)])
def test_activations(dev, activation, T, K, N, bias, residual):
    t, d = _inputs(T, K, N, dev, bias=bias, residual=residual)
    _compare(_call(d, activation), _oracle(t, activation))


@pytest.mark.parametrize("T,K,N", [(2048, 512, 2048), (1500, 1000, 1400), (4096, 64, 1920), (2050, 200, 1930), (6000, 256, 128)])
def test_every_tile_shape(dev, T, K, N):
    """Sizes whose three products take the large tiles, and sums split over blocks."""
    t, d = _inputs(T, K, N, dev, residual=False)
    _compare(_call(d), _oracle(t))


def test_exact_whole_numbers(dev):
    """Small whole numbers: every sum is exact, so a misplaced element of any tile shows."""
    from agent_factory_3_amd.linear import linear
    for T, K, N in ((40, 64, 48), (31, 72, 17), (520, 136, 400), (2048, 320, 2048), (1920, 192, 3840), (300, 2000, 264)):
        g = torch.Generator().manual_seed(T)
        x, w = (torch.randint(-2, 3, s, generator=g).float() for s in ((T, K), (N, K)))
        dy = torch.randint(-2, 3, (T, N), generator=g).float() * (torch.rand(T, N, generator=g) < 0.05)
        a, b = (v.to(dev, BF).requires_grad_() for v in (x, w))
        y = linear(a, b)
        dx, dw = torch.autograd.grad(y, [a, b], dy.to(dev, BF))
        for got, want in ((y, x @ w.t()), (dx, dy @ w), (dw, dy.t() @ x)):
            assert torch.equal(got.detach().cpu(), want.to(BF)), (T, K, N)   # (rounded once)


def test_strides_and_alignment(dev):
    """Views at any element of wider tensors (NaN beside them), transposed tensors, one row for all, 3 dimensions."""
    from agent_factory_3_amd.linear import linear
    for T, K, N in ((20, 72, 56), (200, 72, 56), (130, 77, 41)):
        t, d = _inputs(T, K, N, dev)
        want = _oracle(t)
        for shift in (0, 1, 8):
            e = {}
            for n in ("x", "weight", "residual", "dy"):
                rows, cols = d[n].shape
                wide = torch.full((rows, cols + 24), float("nan"), dtype=BF, device=dev)
                wide[:, shift:shift + cols] = d[n]
                e[n] = wide[:, shift:shift + cols]
            two = torch.full((N, 2), float("nan"), dtype=BF, device=dev)
            two[:, 0] = d["bias"]
            e["bias"] = two[:, 0]
            _compare(_call(e), want)
        e = {n: v.t().contiguous().t() if v.dim() == 2 else v for n, v in d.items()}
        _compare(_call(e), want)
        row = d["x"][:1].expand(T, K)
        assert torch.equal(linear(row, d["weight"]), linear(row.contiguous(), d["weight"]))
    t, d = _inputs(60, 40, 24, dev)
    three = {n: v.view(3, 20, -1) if n in ("x", "residual") else v for n, v in d.items()}
    a, b = _call(d), _call(three)
    assert b["y"].shape == (3, 20, 24) and all(torch.equal(a[n].view(-1), b[n].view(-1)) for n in a)


def test_only_some_gradients(dev):
    from agent_factory_3_amd.linear import linear
    t, d = _inputs(90, 64, 72, dev)
    want = _oracle(t, "silu")
    for names in (("x",), ("weight",), ("bias",), ("residual",), ("x", "bias")):
        leaf = {n: d[n].detach().requires_grad_(n in names) for n in ("x", "weight", "bias", "residual")}
        y = linear(leaf["x"], leaf["weight"], leaf["bias"], activation="silu", residual=leaf["residual"])
        g = torch.autograd.grad(y, [leaf[n] for n in names], d["dy"])
        _compare({"d" + n: v for n, v in zip(names, g)}, want)


@pytest.mark.parametrize("T", [20, 200])
def test_not_finite_stays_in_its_row(dev, T):
    """NaN in one row of x, infinity in one row of the weight: its outputs alone; padding adds nothing."""
    from agent_factory_3_amd.linear import linear
    t, d = _inputs(T, 75, 70, dev)
    clean = linear(d["x"], d["weight"], d["bias"])
    x, w = d["x"].clone(), d["weight"].clone()
    x[3, 74], w[69, 0] = float("nan"), float("inf")
    y = linear(x, w, d["bias"])
    assert y[3].isnan().all() and not y[:, 69].isfinite().any()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[3], keep[:, 69] = False, False
    assert torch.equal(y[keep], clean[keep])


def test_activations_at_large_arguments(dev):
    """Arguments of 100 and 1000 either way: 0 or the argument, slopes 0 or 1, never NaN.  (At -30 silu is
    -30 / (1 + e^30) = -2.8e-12 and its slope (1 - 30) e^-30 = -2.7e-12: 1e-11 and 40e-11 for 40 rows' sum.)"""
    from agent_factory_3_amd.linear import linear
    z = torch.tensor([-1000.0, -100.0, -30.0, 0.0, 30.0, 100.0, 1000.0], device=dev)
    for name in ("relu", "silu", "gelu", "gelu_tanh"):
        for T in (4, 40):
            x = torch.ones(T, 8, dtype=BF, device=dev, requires_grad=True)
            y = linear(x, torch.zeros(7, 8, dtype=BF, device=dev), z, activation=name)
            assert ((y[T - 1].float() - z.clamp(min=0).to(BF).float()).abs() <= 1e-11).all(), name
            b = z.clone().requires_grad_()
            (db,) = torch.autograd.grad(linear(x, torch.zeros(7, 8, dtype=BF, device=dev), b, activation=name).float().sum(), b)
            err = (db[[0, 1, 2, 4, 5, 6]] - torch.tensor([0.0, 0, 0, T, T, T], device=dev)).abs()
            assert (err <= 40e-11).all(), name


def test_empty(dev):
    from agent_factory_3_amd.linear import linear
    x = torch.empty(0, 3, 40, dtype=BF, device=dev, requires_grad=True)
    w = torch.ones(24, 40, dtype=BF, device=dev, requires_grad=True)
    b = torch.ones(24, dtype=BF, device=dev, requires_grad=True)
    y = linear(x, w, b, activation="gelu")
    g = torch.autograd.grad(y, [x, w, b], y.detach())
    assert y.shape == (0, 3, 24) and g[0].shape == x.shape and (g[1] == 0).all() and (g[2] == 0).all()


def test_streams_capture_and_same_bits(dev):
    T, K, N = 1500, 520, 264
    t, d = _inputs(T, K, N, dev)
    want = _call(d, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(d, "silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(want[n], got[n]) for n in want)
    held_in = {n: v.clone() for n, v in d.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _call(held_in, "silu")
    for n in range(3):
        new = _inputs(T, K, N, dev, seed=30 + n)[1]
        for k in held_in:
            held_in[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        want = _call(new, "silu")
        assert all(torch.equal(held[k], want[k]) for k in want)


def test_saved_tensors_that_come_back_with_other_strides(dev):
    t, d = _inputs(70, 50, 30, dev)
    want = _call(d, "gelu")
    with torch.autograd.graph.save_on_cpu():
        got = _call(d, "gelu")
    assert all(torch.equal(want[n], got[n]) for n in want)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.t().contiguous().t() if v.dim() == 2 else v, lambda v: v):
        got = _call(d, "gelu")
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_offsets_past_32_bits(dev):
    """x and y of more than 2^31 elements: the last rows as alone."""
    from agent_factory_3_amd.linear import linear
    K = N = 64
    T = (1 << 31) // K + 300
    x = torch.zeros(T, K, dtype=BF, device=dev)
    t, d = _inputs(300, K, N, dev, residual=False)
    x[-300:] = d["x"]
    y = linear(x, d["weight"])
    assert torch.equal(y[-300:], linear(d["x"], d["weight"])) and (y[:1000] == 0).all()
    del y
    # the sum over as many rows
    dy = torch.zeros(T, N, dtype=BF, device=dev)
    dy[-300:] = d["dy"]
    w = d["weight"].detach().requires_grad_()
    b = d["bias"].detach().requires_grad_()
    dw, db = torch.autograd.grad(linear(x, w, b), [w, b], dy)
    want = _oracle({**t, "residual": None})
    # (the same products in another grouping, with zeros between)
    assert ((dw.cpu().double() - want["dweight"]).abs() <= want["dweight_tol"]).all()
    assert ((db.cpu().double() - want["dbias"]).abs() <= want["dbias_tol"]).all()


def test_refusals(dev):
    from agent_factory_3_amd.linear import linear
    x = torch.zeros(4, 64, dtype=BF, device=dev)
    w = torch.zeros(32, 64, dtype=BF, device=dev)
    b = torch.zeros(32, dtype=BF, device=dev)
    for exc, args, kw in [(RuntimeError, (x.cpu(), w, b), {}), (RuntimeError, (x, w.cpu(), b), {}), (TypeError, (x.half(), w), {}),
                          (TypeError, (x.float(), w.float()), {}), (TypeError, (x, w, b.half()), {}), (ValueError, (x, w[:, :32]), {}),
                          (ValueError, (x, w, b[:31]), {}), (ValueError, (x, w[:0], None), {}), (ValueError, (x[:, :0], w[:, :0]), {}),
                          (ValueError, (x, w), dict(activation="tanh")), (ValueError, (x, w), dict(residual=x)),
                          (TypeError, (x, w), dict(residual=torch.zeros(4, 32, device=dev))), (ValueError, (x, w[0]), {})]:
        with pytest.raises(exc):
            linear(*args, **kw)


def test_second_derivatives_are_refused(dev):
    """A graph of the gradients can be asked for and gives the same bits, but is not differentiated: where dy
    has no gradient they have none either (torch's own error), else the error names the backward."""
    from agent_factory_3_amd import norms
    from agent_factory_3_amd.linear import linear
    t, d = _inputs(40, 64, 64, dev)
    x = d["x"].detach().requires_grad_()
    dy = d["dy"].detach().requires_grad_()
    for f in (lambda: linear(x, d["weight"], activation="silu"), lambda: norms.rms_norm(x, d["bias"])):
        (g,) = torch.autograd.grad(f(), x, d["dy"])
        for grad, message in ((d["dy"], "does not require grad"), (dy, "once_differentiable")):
            (g2,) = torch.autograd.grad(f(), x, grad, create_graph=True)
            assert torch.equal(g, g2)
            with pytest.raises(RuntimeError, match=message):
                g2.float().sum().backward()


def test_tensors_without_memory_of_their_own_are_refused(dev):
    """A DTensor's address is 0: it must not pass for a tensor that is not given."""
    from agent_factory_3_amd.linear import linear

    class Held(torch.Tensor):
        @classmethod
        def of(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} of a tensor without memory")

    x, w, b = (torch.ones(*s, device=dev, dtype=BF) for s in ((2, 64), (64, 64), (64,)))
    for name in ("x", "weight", "bias", "residual"):
        t = {"x": x, "weight": w, "bias": b, "residual": x}
        t[name] = Held.of(t[name])
        with pytest.raises(TypeError, match=name):
            linear(t["x"], t["weight"], t["bias"], residual=t["residual"])


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("T", [3, 40])
def test_activations_keep_their_digits_in_the_tail(dev, activation, T):
    """Arguments from -13 to 13 (the bias, exact, beside a product of 0): values within one rounding of their own
    size, however small; slopes within 2^-14 of their terms'."""
    from agent_factory_3_amd.linear import linear
    z = torch.linspace(-13, 13, 1041).to(BF).float()
    w, x = torch.zeros(z.numel(), 8, dtype=BF, device=dev), torch.ones(T, 8, dtype=BF, device=dev)
    b = z.to(dev).requires_grad_()
    y = linear(x, w, b, activation=activation)
    dy = torch.zeros_like(y)
    dy[T - 1] = 1
    (db,) = torch.autograd.grad(y, b, dy)
    zd = z.double()
    want, slope, _ = ol.act(zd, activation)
    if activation == "gelu":        # (1 + erf loses the tail's digits in 64 bits too, from -7 on)
        phi = 0.5 * torch.erfc(-zd / 2 ** 0.5)
        want, slope = zd * phi, phi + zd * torch.exp(-zd * zd / 2) / (2 * torch.pi) ** 0.5
    elif activation == "gelu_tanh":
        u = (2 / torch.pi) ** 0.5 * (zd + 0.044715 * zd ** 3)
        s = torch.sigmoid(2 * u)
        want = zd * s
        slope = s + zd * 2 * s * torch.sigmoid(-2 * u) * (2 / torch.pi) ** 0.5 * (1 + 0.134145 * zd * zd)
    # fp32's errors as in the oracle; bf16 and fp32 below 2^-118 are left alone (their exponentials vanish)
    err = (y.detach()[T - 1].cpu().double() - want).abs()
    assert (err <= (2.0 ** -8 + 2.0 ** -14) * want.abs() + 2.0 ** -118).all(), float(z[(err / want.abs()).nan_to_num().argmax()])
    terms = (want / zd).nan_to_num(nan=0.5).abs() + (slope - (want / zd).nan_to_num(nan=0.5)).abs()
    assert ((db.cpu().double() - slope).abs() <= 2.0 ** -14 * terms + 2.0 ** -118).all()


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("T", [3, 40])
def test_slope_of_nan_is_nan(dev, activation, T):
    """A NaN row of x: its gradient is NaN too, and no other row's."""
    from agent_factory_3_amd.linear import linear
    t, d = _inputs(T, 64, 24, dev, residual=False)
    x = d["x"].clone()
    x[1, 7] = float("nan")
    x.requires_grad_()
    (dx,) = torch.autograd.grad(linear(x, d["weight"], d["bias"], activation=activation), x, d["dy"])
    ok = torch.arange(T, device=dev) != 1
    assert dx[1].isnan().all() and dx[ok].isfinite().all()
