"""The float64 oracles of sink attention and the balance loss against independent forms (CPU)."""
import math

import pytest
import torch

from oracle import attention as oa
from oracle import balance as ob


def _inputs(B, Hq, Hkv, Sq, Sk, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return r(B, Hq, Sq, D), r(B, Hkv, Sk, D), r(B, Hkv, Sk, D), r(Hq), r(B, Sq, Hq, D)


@pytest.mark.parametrize("window", [0, 3])
def test_matches_transformers_eager_attention(window):
    """transformers' gpt-oss eager attention under the mask that transformers makes for it."""
    from transformers.models.gpt_oss.modeling_gpt_oss import eager_attention_forward
    q, k, v, sinks, _ = _inputs(2, 4, 2, 9, 9, 16)
    mask = torch.zeros(9, 9, dtype=torch.float64).masked_fill_(~oa.visible(9, 9, window), torch.finfo(torch.float64).min)
    m = torch.nn.Module()
    m.num_key_value_groups, m.sinks = 2, sinks
    ref, _ = eager_attention_forward(m.eval(), q, k, v, mask[None, None], 0.25)
    got = oa.attention(q, k, v, sinks, scale=0.25, window=window)["out"]
    assert torch.allclose(got, ref, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("kw", [dict(), dict(window=2, first=1), dict(cu_seqlens=[0, 3, 3, 6]),
                                dict(kv_range=[(1, 5), (0, 0)])])
def test_gradients_match_autograd_and_differences(kw):
    B = 2 if "kv_range" in kw else 1
    q, k, v, sinks, do = _inputs(B, 4, 2, 7, 7, 8, seed=1)
    g = oa.attention(q, k, v, sinks, dout=do, **kw)

    def f(q, k, v, s):
        return (oa_out(q, k, v, s, kw) * do).sum()

    def oa_out(q, k, v, s, kw):  # a differentiable restatement
        outs = []
        starts = oa.starts_of(kw["cu_seqlens"], 7) if "cu_seqlens" in kw else None
        for b in range(B):
            ok = oa.visible(7, 7, kw.get("window", 0), kw.get("first", 0), starts,
                            kw["kv_range"][b] if "kv_range" in kw else None)
            z = (q[b] @ k[b].repeat_interleave(2, 0).transpose(1, 2)) / math.sqrt(8)
            z = torch.cat([z.masked_fill(~ok, -math.inf), s.view(-1, 1, 1).expand(-1, 7, 1)], -1)
            outs.append((torch.softmax(z, -1)[..., :-1] @ v[b].repeat_interleave(2, 0)).transpose(0, 1))
        return torch.stack(outs)

    leaves = [t.clone().requires_grad_() for t in (q, k, v, sinks)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for n, a in zip(("dq", "dk", "dv", "dsinks"), grads):
        assert torch.allclose(g[n], a, rtol=1e-10, atol=1e-12), n
    # a directional difference of the oracle itself
    gen = torch.Generator().manual_seed(2)
    d = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (q, k, v, sinks)]
    h = 1e-5
    val = lambda s: float((oa.attention(*(t + s * x for t, x in zip((q, k, v, sinks), d)), **kw)["out"] * do).sum())  # noqa: E731
    num = (val(h) - val(-h)) / (2 * h)
    ana = sum(float((g[n] * x).sum()) for n, x in zip(("dq", "dk", "dv", "dsinks"), d))
    assert abs(num - ana) < 1e-6 * max(1.0, abs(ana))


def test_empty_rows_and_masked_garbage():
    q, k, v, sinks, do = _inputs(1, 2, 1, 5, 5, 8)
    k[0, 0, 3:], v[0, 0, 3:] = math.nan, math.inf
    g = oa.attention(q, k, v, None, kv_range=[(2, 3)], dout=do)
    assert torch.isfinite(g["out"]).all() and (g["out"][0, :2] == 0).all()
    assert torch.equal(g["out"][0, 2:, 0], v[0, 0, 2].expand(3, 8))
    assert (g["dv"][0, 0, 3:] == 0).all() and (g["dq"][0, :, :2] == 0).all()


@pytest.mark.parametrize("masked", [False, True])
def test_balance_matches_transformers_and_autograd(masked):
    from transformers.models.gpt_oss.modeling_gpt_oss import load_balancing_loss_func
    g = torch.Generator().manual_seed(0)
    z = torch.randn(2 * 11, 8, generator=g, dtype=torch.float64)
    mask = (torch.rand(2, 11, generator=g) < 0.7).long() if masked else None
    leaf = z.clone().requires_grad_()
    ref = load_balancing_loss_func((leaf,), 8, 3, mask)
    (grad,) = torch.autograd.grad(ref, leaf)
    loss, counts, d = ob.balance_loss(z, 3, token_mask=mask)
    assert abs(float(loss) - float(ref.detach())) < 1e-6   # its masks are fp32
    assert torch.allclose(d, grad, rtol=1e-5, atol=1e-8)
    assert int(counts.sum()) == 3 * (22 if mask is None else int(mask.sum()))


def test_balance_top_k_ties_and_nan():
    z = torch.tensor([[1.0, 2.0, 2.0, float("nan"), -math.inf]])
    assert ob.top_k(z, 5).tolist() == [[1, 2, 0, 4, 3]]
    loss, counts, d = ob.balance_loss(torch.zeros(3, 4), 2, token_mask=torch.zeros(3))
    assert float(loss) == 0 and int(counts.sum()) == 0 and (d == 0).all()
