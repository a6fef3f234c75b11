"""The float64 oracle of the projection against differences (CPU)."""
import pytest
import torch

from oracle import linear as ol


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False)])
def test_gradients_match_differences(activation, bias, residual):
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = {"x": rand(3, 5), "weight": rand(4, 5), "bias": rand(4) if bias else None, "residual": rand(3, 4) if residual else None}
    dy = rand(3, 4)
    o = ol.linear(t["x"], t["weight"], t["bias"], activation, t["residual"], dy)
    step = 1e-6
    for n in t:
        if t[n] is None:
            continue
        for i in range(t[n].numel()):
            vals = []
            for d in (step, -step):
                v = t[n].clone()
                v.view(-1)[i] += d
                a = {**t, n: v}
                vals.append((ol.linear(a["x"], a["weight"], a["bias"], activation, a["residual"])["y"] * dy).sum())
            # central differences: step^2 times third derivatives of order 10 (100 with the products), and 1e-15 / step
            assert abs(float((vals[0] - vals[1]) / (2 * step) - o["d" + n].reshape(-1)[i])) < 1e-7, (n, i)
