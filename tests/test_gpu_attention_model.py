"""gpt-oss trained with the operators together: sink attention, router, MXFP4 experts, balance loss.

A tiny GptOssModel with MXFP4 expert modules runs with attn_implementation="af3_sink".
Every attention call's output and gradients are held to the float64 oracle on the
tensors that the call saw (windows, sinks, padding and packing as the model passes
them); the model's output also to the same model with transformers' eager attention.
Gradients are not compared between the two models: eager rounds its scores to bf16,
which at scores of 20 (this model's largest) is off by up to 2^-8 20 = 0.08, so its
probabilities are 8% off and gradients through them likewise.
"""
import pytest
import torch

from agent_factory_3_amd import attention, quantizer_config, routing, routing_replay, workloads  # noqa: F401
from agent_factory_3_amd import quantization as Q
from oracle import attention as oa
from oracle import balance as ob

pytestmark = pytest.mark.gpu

E, H, I, K, HQ, HKV, W = 8, 128, 128, 2, 4, 2, 16


def _model(dev, impl):
    import types

    from transformers import GptOssConfig
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssModel
    cfg = GptOssConfig(num_hidden_layers=2, hidden_size=H, intermediate_size=I, num_local_experts=E,
                       num_experts_per_tok=K, num_attention_heads=HQ, num_key_value_heads=HKV, head_dim=64,
                       vocab_size=256, sliding_window=W, layer_types=["sliding_attention", "full_attention"],
                       initializer_range=0.2)
    cfg._attn_implementation = impl
    torch.manual_seed(0)
    model = GptOssModel(cfg)
    Q.replace_with_dequant_experts(model, quantization_config=types.SimpleNamespace(dequantize=False))
    g = torch.Generator().manual_seed(1)
    for layer in model.layers:
        ex = layer.mlp.experts
        for proj, rows, k in (("gate_up_proj", 2 * I, H), ("down_proj", H, I)):
            b, s = workloads.mxfp4_weight(g, (E, rows), k, 118, 121)
            Q._store_mxfp4_weights(b, s, ex, proj, dev)
        for n in ("gate_up_proj_bias", "down_proj_bias"):
            p = getattr(ex, n)
            setattr(ex, n, torch.nn.Parameter((torch.randn(p.shape, generator=g) * 0.1).to(dev), requires_grad=False))
    for n, p in list(model.named_parameters()):
        if "experts" not in n:
            mod = model.get_submodule(n.rpartition(".")[0])
            setattr(mod, n.rpartition(".")[2], torch.nn.Parameter(p.detach().to(dev, torch.bfloat16)))
    model.rotary_emb.to(dev)
    return model


def _grads(model, loss):
    ps = [(n, p) for n, p in model.named_parameters() if p.requires_grad and "embed" not in n]
    return {n: g for (n, _), g in zip(ps, torch.autograd.grad(loss, [p for _, p in ps], allow_unused=True))}


def _ids(B, S):
    return torch.randint(0, 256, (B, S), generator=torch.Generator().manual_seed(7))


def _replay(B, S):
    return torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(100 + i))[:K]
                        for i in range(B * S * 2)]).view(B, S, 2, K)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


class _Spy:
    """Records sink_attention's calls inside a model, with the gradients that arrive and leave."""

    def __init__(self, monkeypatch):
        self.calls = []
        orig = attention.sink_attention

        def call(q, k, v, s, **kw):
            out = orig(q, k, v, s, **kw)
            c = dict(q=q, k=k, v=v, s=s, kw=kw, out=out, g={})
            if out.requires_grad:
                for n, t in (("dout", out), ("dq", q), ("dk", k), ("dv", v)):
                    t.register_hook(lambda g, n=n: c["g"].__setitem__(n, g.detach().clone()))
            self.calls.append(c)
            return out
        monkeypatch.setattr(attention, "sink_attention", call)

    def check(self, dsinks=None):
        for i, c in enumerate(self.calls):
            kw, rng = c["kw"], c["kw"]["kv_range"]
            ref = oa.attention(c["q"], c["k"], c["v"], c["s"], scale=kw["scale"], window=kw["window"],
                               kv_range=None if rng is None else rng.tolist(), dout=c["g"].get("dout"), bounds=True)
            got = dict(out=c["out"], **{n: c["g"][n] for n in ("dq", "dk", "dv") if n in c["g"]})
            if dsinks is not None:
                got["dsinks"] = dsinks[i]
            for n, t in got.items():
                t = t.detach().cpu().double()
                assert ((t - ref[n]).abs() <= ref[n + "_tol"]).all(), (i, n)


@pytest.mark.parametrize("padded", [False, True])
def test_model_matches_oracle_and_eager_attention(dev, padded, monkeypatch):
    """Replayed experts, so that both models choose alike."""
    routing_replay.enable_routing_replay()
    ids, ri = _ids(2, 50).to(dev), _replay(2, 50).to(dev)
    mask = torch.ones(2, 50, dtype=torch.long, device=dev)
    if padded:
        mask[1, 37:] = 0
    w = torch.randn(2, 50, H, generator=torch.Generator().manual_seed(3)).to(dev) * mask[..., None]
    with torch.no_grad():
        want = _model(dev, "eager")(input_ids=ids, attention_mask=mask, routing_indices=ri,
                                    use_cache=False).last_hidden_state
    spy = _Spy(monkeypatch)
    model = _model(dev, "af3_sink")
    out = model(input_ids=ids, attention_mask=mask, routing_indices=ri, use_cache=False).last_hidden_state
    grads = _grads(model, (out.float() * w).sum())
    assert [c["kw"]["window"] for c in spy.calls] == [W, 0]
    spy.check([grads[f"layers.{l}.self_attn.sinks"] for l in range(2)])
    # Per layer about ten roundings to bf16 (2^-9 rms of the value each) meet on the residual stream, twice, and
    # eager rounds the scores besides: 2^-9 sqrt(2 * 10 * 2) = 1.3e-2 between two evaluations; allowed: three times that
    assert _rel(out.detach() * mask[..., None], want * mask[..., None]) < 4e-2


def test_packed_row_is_its_sequences_alone(dev):
    """A packed row, by position ids and by cumulative lengths, gives each sequence what it gets by itself."""
    model = _model(dev, "af3_sink")
    routing_replay.enable_routing_replay()
    lens = [13, 1, 40]
    ids, ri = _ids(1, sum(lens)).to(dev), _replay(1, sum(lens)).to(dev)
    pos = torch.cat([torch.arange(n) for n in lens])[None].to(dev)
    cu = torch.tensor([0, 13, 14, 54], dtype=torch.int32, device=dev)
    with torch.no_grad():
        by_pos = model(input_ids=ids, position_ids=pos, routing_indices=ri, use_cache=False).last_hidden_state
        by_cu = model(input_ids=ids, position_ids=pos, routing_indices=ri, use_cache=False, cu_seq_lens_q=cu,
                      cu_seq_lens_k=cu).last_hidden_state
        assert torch.equal(by_pos, by_cu)
        at = 0
        for n in lens:
            one = model(input_ids=ids[:, at:at + n], routing_indices=ri[:, at:at + n], use_cache=False).last_hidden_state
            # the same products in other tiles: sums in another order, roundings alike but for a few
            assert _rel(by_pos[:, at:at + n], one) < 2e-2
            at += n


def test_generation_with_a_cache_matches_the_whole_row(dev):
    model = _model(dev, "af3_sink")
    ids = _ids(2, 40).to(dev)
    mask = torch.ones(2, 40, dtype=torch.long, device=dev)
    mask[0, :9] = 0
    routing_replay.enable_routing_replay()
    ri = _replay(2, 40).to(dev)
    with torch.no_grad():
        pos = (mask.cumsum(1) - 1).clamp(min=0)
        whole = model(input_ids=ids, attention_mask=mask, position_ids=pos, routing_indices=ri,
                      use_cache=False).last_hidden_state
        out = model(input_ids=ids[:, :30], attention_mask=mask[:, :30], position_ids=pos[:, :30],
                    routing_indices=ri[:, :30], use_cache=True)
        got = []
        for t in range(30, 40):
            out = model(input_ids=ids[:, t:t + 1], attention_mask=mask[:, :t + 1], position_ids=pos[:, t:t + 1],
                        routing_indices=ri[:, t:t + 1], past_key_values=out.past_key_values, use_cache=True)
            got.append(out.last_hidden_state)
    assert _rel(torch.cat(got, 1), whole[:, 30:]) < 2e-2


def test_training_step_with_balance_loss(dev):
    """Policy gradient through attention and experts plus the balance loss, with activation checkpointing:
    the routers' gradients are those of the two parts, the balance part's own from the oracle."""
    model = _model(dev, "af3_sink")
    model.gradient_checkpointing_enable(dict(use_reentrant=False))
    model.train()
    ids = _ids(2, 60).to(dev)
    mask = torch.ones(2, 60, dtype=torch.long, device=dev)
    mask[1, 41:] = 0
    w = torch.randn(2, 60, H, generator=torch.Generator().manual_seed(3)).to(dev) * mask[..., None]

    def step(coef, keep=None):
        with routing.collect_balance(mask) as b:
            out = model(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
        if keep is not None:
            keep.update({layer: v[0] for layer, v in b._seen.items()}, losses=b.losses(), counts=b.counts())
        return _grads(model, (out.float() * w).sum() + coef * b.loss())
    keep = {}
    both, none = step(100.0, keep), step(0.0)
    for l, layer in enumerate(model.layers):
        logits = keep[layer.mlp].detach()
        loss, counts, dz = ob.balance_loss(logits, K, None, mask, 100.0 / 2)
        assert abs(float(keep["losses"][l].detach()) - float(loss)) < 1e-5
        assert torch.equal(keep["counts"][l].cpu().long(), counts) and int(counts.sum()) == K * 101
        # the bias gradient is the plain sum of the logits' gradient over tokens
        d = (both[f"layers.{l}.mlp.router.bias"].double() - none[f"layers.{l}.mlp.router.bias"].double()).cpu()
        if l == 1:  # (the first layer's router also moves what the second one sees)
            tol = 2 ** -8 * dz.abs().sum(0) + 2 ** -7 * (both[f"layers.{l}.mlp.router.bias"].double().abs().cpu() + dz.sum(0).abs())
            assert ((d - dz.sum(0)).abs() <= tol).all()
        assert both[f"layers.{l}.self_attn.sinks"].abs().max() > 0

def test_rejects_what_it_cannot_do(dev):
    model = _model(dev, "af3_sink")
    mask = torch.ones(1, 10, dtype=torch.long, device=dev)
    mask[0, 4] = 0
    with pytest.raises(ValueError, match="one run"):
        model(input_ids=_ids(1, 10).to(dev), attention_mask=mask)


def test_a_batch_of_packed_rows_in_the_model(dev):
    """Rows of a batch that hold several sequences each (by their position ids): every sequence as by itself,
    also with the cache that a forward makes by default."""
    routing_replay.enable_routing_replay()
    lens = [[13, 1, 40], [30, 20, 4]]
    ids, ri = _ids(2, 54).to(dev), _replay(2, 54).to(dev)
    pos = torch.stack([torch.cat([torch.arange(n) for n in row]) for row in lens]).to(dev)
    model = _model(dev, "af3_sink")
    with torch.no_grad():
        got = model(input_ids=ids, position_ids=pos, routing_indices=ri, use_cache=False).last_hidden_state
        assert torch.equal(got, model(input_ids=ids, position_ids=pos, routing_indices=ri).last_hidden_state)
        for b, row in enumerate(lens):
            at = 0
            for n in row:
                one = model(input_ids=ids[b:b + 1, at:at + n], routing_indices=ri[b:b + 1, at:at + n],
                            use_cache=False).last_hidden_state
                assert _rel(got[b:b + 1, at:at + n], one) < 2e-2   # (as for one packed row)
                at += n


@pytest.mark.parametrize("side", ["left", "right"])
def test_padded_rows_of_sequences(dev, side):
    """A packed row beside a padded one in a batch, and a padded packed row alone: each sequence as by itself."""
    routing_replay.enable_routing_replay()
    lens, S = [[13, 1, 40], [30, 7]], 54
    ids, ri = _ids(2, S).to(dev), _replay(2, S).to(dev)
    pos, mask, at0 = torch.zeros(2, S, dtype=torch.long), torch.zeros(2, S, dtype=torch.long), []
    for b, row in enumerate(lens):
        n = sum(row)
        a = S - n if side == "left" else 0
        pos[b, a:a + n], mask[b, a:a + n] = torch.cat([torch.arange(x) for x in row]), 1
        at0.append(a)
    pos, mask = pos.to(dev), mask.to(dev)
    model = _model(dev, "af3_sink")
    with torch.no_grad():
        both = model(input_ids=ids, attention_mask=mask, position_ids=pos, routing_indices=ri).last_hidden_state
        alone = model(input_ids=ids[1:], attention_mask=mask[1:], position_ids=pos[1:], routing_indices=ri[1:]).last_hidden_state
        for b, row in enumerate(lens):
            at = at0[b]
            for n in row:
                one = model(input_ids=ids[b:b + 1, at:at + n], routing_indices=ri[b:b + 1, at:at + n],
                            use_cache=False).last_hidden_state
                for got in (both[b:b + 1], alone) if b else (both[b:b + 1],):
                    assert _rel(got[:, at:at + n], one) < 2e-2   # (as for one packed row)
                at += n
