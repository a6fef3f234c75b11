"""Every tile shape of the projections' products in every operand layout, blocks that stay for several tiles, edge
tiles, sums split over blocks: on small whole numbers, whose sums are exact in any order, so that a misplaced or
missing element shows.  Each test asks the library which tiles it takes, so that it stays with the shape it is for."""
import ctypes

import pytest
import torch

from agent_factory_3_amd import _capi
from oracle import linear as ol

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _tile(M, N, K, p_trans=0, q_trans=0):
    """Rows, columns, stages of the tiles of a product, whether blocks share their k, and how many a block may make."""
    t = (ctypes.c_int * 4)()
    _capi.call("af3_linear_tile", M, N, K, p_trans, q_trans, t)
    items = -(-M // t[0]) * -(-N // t[1]) * t[3]
    return t[0], t[1], t[2], t[3] > 1, items > (512 if tuple(t[:3]) == (128, 128, 2) else 256)


def _ints(g, *shape, dev, to=2):
    return torch.randint(-to, to + 1, shape, generator=g, device=dev, dtype=torch.int8).to(BF)


# rows, columns and length of a product; tile rows, columns, stages; whether k is shared; whether blocks stay
PRODUCTS = [((2900, 4100, 330), (256, 256, 2, False, False)), ((6100, 4100, 330), (256, 256, 2, False, True)),
            ((2901, 4101, 331), (256, 256, 2, False, False)), ((6400, 4352, 320), (256, 256, 2, False, True)),
            ((4300, 1930, 200), (256, 192, 2, False, False)), ((4300, 4100, 520), (256, 192, 2, False, True)),
            ((4301, 4103, 523), (256, 192, 2, False, True)), ((4608, 3840, 576), (256, 192, 2, False, True)),
            ((2100, 1930, 5000), (256, 192, 2, True, False)),
            ((8001, 2881, 130), (128, 128, 2, False, True)), ((4358, 16, 5862), (128, 128, 2, True, False)),
            ((300, 270, 60), (128, 128, 4, False, False)), ((300, 270, 2000), (128, 128, 4, True, False))]


def test_products_take_the_tiles_they_are_here_for():
    for size, tile in PRODUCTS:
        for layout in ((0, 0), (0, 1), (1, 1)):
            assert _tile(*size, *layout) == tile, (size, layout, _tile(*size, *layout))


@pytest.mark.parametrize("size", [p[0] for p in PRODUCTS])
@pytest.mark.parametrize("bias,residual", [(None, False), (BF, False), (F32, True), (None, True)])
def test_forward(dev, size, bias, residual):
    from agent_factory_3_amd.linear import linear
    T, N, K = size
    g = torch.Generator(dev).manual_seed(T)
    x, w = _ints(g, T, K, dev=dev), _ints(g, N, K, dev=dev)
    b = _ints(g, N, dev=dev, to=100).to(bias) if bias is not None else None
    r = _ints(g, T, N, dev=dev, to=100) if residual else None
    want = x.float() @ w.float().t()
    for extra in (b, r):
        want = want if extra is None else want + extra.float()
    got = linear(x, w, b, residual=r)
    assert torch.equal(got, want.to(BF))   # (rounded once)
    # rows of wider tensors
    wide = torch.full((T, K + 8), float("nan"), dtype=BF, device=dev)
    wide[:, :K] = x
    assert torch.equal(linear(wide[:, :K], w, b, residual=r), got)


@pytest.mark.parametrize("size", [p[0] for p in PRODUCTS])
def test_input_gradient(dev, size):
    from agent_factory_3_amd.linear import linear
    T, K, N = size   # dx [T, K], a sum over N
    g = torch.Generator(dev).manual_seed(T)
    x, w, dy = _ints(g, T, K, dev=dev).requires_grad_(), _ints(g, N, K, dev=dev), _ints(g, T, N, dev=dev)
    (dx,) = torch.autograd.grad(linear(x, w), x, dy)
    assert torch.equal(dx, (dy.float() @ w.float()).to(BF))


@pytest.mark.parametrize("size", [p[0] for p in PRODUCTS])
def test_weight_gradient(dev, size):
    from agent_factory_3_amd.linear import linear
    N, K, T = size   # dw [N, K], a sum over T
    g = torch.Generator(dev).manual_seed(T)
    x, w, dy = _ints(g, T, K, dev=dev), _ints(g, N, K, dev=dev).requires_grad_(), _ints(g, T, N, dev=dev)
    b = torch.zeros(N, device=dev, requires_grad=True)
    dw, db = torch.autograd.grad(linear(x, w, b), [w, b], dy)
    assert torch.equal(dw, (dy.float().t() @ x.float()).to(BF)) and torch.equal(db, dy.float().sum(0))


@pytest.mark.parametrize("size", [p[0] for p in PRODUCTS])
@pytest.mark.parametrize("residual", [False, True])
def test_activations(dev, size, residual):
    """relu is exact, values and gradients (its slope from the kept sums); silu and gelu within their one rounding."""
    from agent_factory_3_amd.linear import linear
    T, N, K = size
    g = torch.Generator(dev).manual_seed(T)
    x, w = _ints(g, T, K, dev=dev), _ints(g, N, K, dev=dev)
    b = (_ints(g, N, dev=dev).float() / 4)
    r = _ints(g, T, N, dev=dev, to=100) if residual else None
    dy = _ints(g, T, N, dev=dev)
    z = x.float() @ w.float().t() + b
    leaf = x.detach().requires_grad_()
    y = linear(leaf, w, b, activation="relu", residual=r)
    res = r.float() if residual else 0.0
    assert torch.equal(y.detach(), (z.clamp(min=0) + res).to(BF))
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(dx, ((dy.float() * (z > 0)) @ w.float()).to(BF))
    # sums of a 64th the size, so that the slopes lie between 0 and 1; exact still
    small = (w.float() / 64).to(BF)
    zd = (x.double() @ small.double().t()) + b.double()
    for name in ("silu", "gelu"):
        leaf = x.detach().requires_grad_()
        bias = b.detach().requires_grad_()
        y = linear(leaf, small, bias, activation=name, residual=r)
        a, slope, curve = ol.act(zd, name)
        want = a + (r.double() if residual else 0.0)
        # (1 + erf's own error of 2^-53 at |z| = 20 is far below)
        assert ((y.detach().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * a.abs() + 2.0 ** -23 * want.abs() + 1e-12).all()
        (db,) = torch.autograd.grad(y, bias, dy)
        # the slope at z rounded to bf16, its own error, and the sum's: at most T / 8 + 1100 additions
        tol = (dy.double().abs() * (curve * 2.0 ** -8 * zd.abs() + 2.0 ** -14)).sum(0) + 2.0 ** -24 * (T / 8 + 1100) * (dy.double() * slope).abs().sum(0)
        assert ((db.double() - (dy.double() * slope).sum(0)).abs() <= tol).all()
