"""The float64 oracle of the residual norms against differences (CPU)."""
import pytest
import torch

from oracle import norms as on


@pytest.mark.parametrize("post,gate,residual,weight", [(False, None, False, True), (False, None, True, True),
                                                       (True, (1, 6), True, True), (True, (3, 1), True, True),
                                                       (True, (3, 6), True, False), (False, (1, 1), True, True)])
def test_gradients_match_differences(post, gate, residual, weight):
    g = torch.Generator().manual_seed(0)
    R, H = 3, 6
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = {"x": rand(R, H), "residual": rand(R, H) if residual else None, "weight": rand(H) if weight else None,
         "post": rand(H) if post else None, "gate": rand(*gate) if gate else None}
    dr, dh = rand(R, H) if residual else None, rand(R, H) if weight else None

    def loss(**kw):
        o = on.residual_norm(kw["x"], kw["residual"], kw["weight"], post=kw["post"], gate=kw["gate"], scale=0.7)
        return sum(((o[n] * d).sum() for n, d in (("r", dr), ("h", dh)) if d is not None), torch.zeros((), dtype=torch.float64))

    o = on.residual_norm(t["x"], t["residual"], t["weight"], post=t["post"], gate=t["gate"], scale=0.7, dr=dr, dh=dh)
    step = 1e-6
    for n, name in (("x", "dx"), ("residual", "dresidual"), ("weight", "dweight"), ("post", "dpost_weight"),
                    ("gate", "dgate")):
        if t[n] is None:
            continue
        for i in range(t[n].numel()):
            up, down = t[n].clone(), t[n].clone()
            up.view(-1)[i] += step
            down.view(-1)[i] -= step
            d = (loss(**{**t, n: up}) - loss(**{**t, n: down})) / (2 * step)
            # central differences: step^2 times third derivatives of order 10, and 1e-16 / step of the sums
            assert abs(float(d - o[name].reshape(-1)[i])) < 1e-8, (n, i)
