"""attn_implementation="af3_sink" and collect_balance in transformers' gpt-oss, without a GPU."""
import types

import pytest
import torch

from agent_factory_3_amd import attention, quantizer_config, routing  # noqa: F401  (registers)
from agent_factory_3_amd import quantization as Q


def test_registered_by_the_quantizer_module():
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    assert ALL_ATTENTION_FUNCTIONS["af3_sink"] is attention.attention_forward
    assert ALL_MASK_ATTENTION_FUNCTIONS["af3_sink"] is attention.attention_mask
    attention.register()


def _model(monkeypatch, seen, layers=2):
    from transformers import GptOssConfig
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssModel
    cfg = GptOssConfig(num_hidden_layers=layers, hidden_size=64, intermediate_size=64, num_local_experts=4,
                       num_experts_per_tok=2, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
                       vocab_size=128, sliding_window=8, layer_types=["sliding_attention", "full_attention"])
    cfg._attn_implementation = "af3_sink"
    torch.manual_seed(0)

    def stand_in(q, k, v, sinks, **kw):  # what the kernels would be called with
        seen.append(dict(q=q, k=k, v=v, sinks=sinks, **kw))
        return q.transpose(1, 2)
    monkeypatch.setattr(attention, "sink_attention", stand_in)
    return GptOssModel(cfg)


def test_layers_call_it_with_their_window_sinks_and_padding(monkeypatch):
    seen = []
    model = _model(monkeypatch, seen)
    ids = torch.randint(0, 128, (2, 12))
    mask = torch.ones(2, 12, dtype=torch.long)
    mask[0, :5] = 0                      # left padding
    mask[1, 9:] = 0                      # right padding
    with torch.no_grad():
        model(input_ids=ids, attention_mask=mask)
    assert [s["window"] for s in seen] == [8, 0]
    for s, layer in zip(seen, model.layers):
        assert s["sinks"] is layer.self_attn.sinks and s["scale"] == layer.self_attn.scaling
        assert s["kv_range"].tolist() == [[5, 12], [0, 9]] and s["kv_range"].dtype == torch.int32
    seen.clear()
    with torch.no_grad():
        model(input_ids=ids, attention_mask=torch.ones(2, 12))
    assert all(s["kv_range"] is None for s in seen)
    # a growing cache: keys and queries end together, the sliding layers' keys are cut
    seen.clear()
    with torch.no_grad():
        mask[1, 9:] = 1
        out = model(input_ids=ids, attention_mask=mask, use_cache=True)
        m2 = torch.cat([mask, torch.ones(2, 1, dtype=torch.long)], 1)
        model(input_ids=ids[:, :1], attention_mask=m2, past_key_values=out.past_key_values)
    dec = seen[2:]
    assert dec[1]["k"].shape[2] == 13 and dec[1]["q"].shape[2] == 1
    assert dec[0]["k"].shape[2] == 8      # window 8: seven kept and the new one
    assert dec[1]["kv_range"].tolist() == [[5, 13], [0, 13]] and dec[0]["kv_range"] is None


def test_mask_refusals():
    f = attention.attention_mask
    hole = torch.tensor([[True, False, True, True]])
    with pytest.raises(ValueError, match="one run"):
        f(1, 4, 4, attention_mask=hole)
    with pytest.raises(NotImplementedError):
        f(1, 4, 4, use_vmap=True)
    with pytest.raises(NotImplementedError):
        f(1, 1, 16, q_offset=torch.tensor(3))
    with pytest.raises(NotImplementedError):
        f(1, 1, 16, q_offset=3)           # a cache of fixed length
    with pytest.raises(ValueError):
        f(1, 4, 6, q_offset=2, attention_mask=torch.ones(1, 4, dtype=torch.bool))
    empty = torch.tensor([[False] * 4, [True] * 4])
    assert f(2, 4, 4, attention_mask=empty).tolist() == [[0, 0], [0, 4]]
    m = types.SimpleNamespace(is_causal=True)
    q = torch.zeros(1, 2, 4, 64)
    with pytest.raises(NotImplementedError):
        attention.attention_forward(m, q, q, q, None, dropout=0.1)
    with pytest.raises(NotImplementedError):
        attention.attention_forward(m, q, q, q, None, is_causal=False)
    with pytest.raises(ValueError):
        attention.attention_forward(m, q, q, q, torch.zeros(1, 1, 4, 4))
    with pytest.raises(ValueError):
        attention.attention_forward(m, q, q, q, None, cu_seq_lens_q=torch.zeros(2), cu_seq_lens_k=torch.zeros(3))


def test_refusals_before_any_launch():
    """Host tensors and bad arguments raise without touching a device."""
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        attention.sink_attention(q, q, q)
    with pytest.raises(RuntimeError, match="GPU"):
        routing.balance_loss(torch.zeros(4, 8), 2)


def test_c_entries_refuse_bad_arguments():
    """Argument errors come back as errors before any launch (no GPU needed)."""
    import ctypes

    from agent_factory_3_amd import _capi
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    st = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    ok = st(*[64] * 12)

    def fwd(strides=ok, starts=None, kv=None, B=1, Hq=2, Hkv=1, Sq=4, Sk=4, D=64, window=0, first=0, scale=0.1, q=64,
            cu=None, out=64, ws=None, n=0):
        _capi.call("af3_sink_attention_fwd", q, 64, 64, strides, None, 0, cu, 1 if cu else 0, starts, kv, B, Hq, Hkv,
                   Sq, Sk, D, window, first, scale, out, None, ws, n, None)
    for match, kw in (("share", dict(Hq=3, Hkv=2)), ("more than", dict(Hq=256)), ("dimension", dict(D=80)),
                      ("negative", dict(window=-1)), ("scale", dict(scale=0.0)), ("scale", dict(scale=float("nan"))),
                      ("length", dict(Sq=1 << 29)), ("multiples", dict(strides=st(*[64] * 8, 7))),
                      ("strides", dict(strides=st(64, 64, 1 << 23, *[64] * 6))),
                      ("strides", dict(strides=st(64, 64, -64, *[64] * 6))), ("packed", dict(starts=64, B=2)),
                      ("packed", dict(starts=64, Sk=5)), ("packed", dict(starts=64, kv=64)),
                      ("cu_seqlens", dict(cu=64)), ("null", dict(q=None)), ("null", dict(out=None)),
                      ("aligned", dict(q=72)), ("workspace", dict(Sk=4096)), ("null strides", dict(strides=None))):
        with pytest.raises(RuntimeError, match=match):
            fwd(**kw)
    lib = _capi.load()
    assert lib.af3_sink_attention_workspace_bytes(1, 8, 1, 1, 4096, 64, 0, 0, 0) > 0
    assert lib.af3_sink_attention_workspace_bytes(1, 8, 1, 0, 4096, 64, 0, 0, 1) == 0
    assert lib.af3_sink_attention_workspace_bytes(64, 64, 8, 128, 128, 64, 0, 0, 0) == 0
    bal = lambda *a: _capi.call("af3_balance_loss_fwd", *a)  # noqa: E731
    for a in ((64, 8, None, None, 4, 0, 1, 64, 64, 64, 64, 1 << 20, None), (64, 8, None, None, 4, 8, 9, 64, 64, 64, 64, 1 << 20, None),
              (64, 8, None, None, 4, 2000, 9, 64, 64, 64, 64, 1 << 20, None), (64, 4, None, None, 4, 8, 2, 64, 64, 64, 64, 1 << 20, None),
              (None, 8, None, None, 4, 8, 2, 64, 64, 64, 64, 1 << 20, None), (64, 8, None, None, 4, 8, 2, 64, 64, 64, 64, 4, None)):
        with pytest.raises(RuntimeError, match="balance_loss"):
            bal(*a)


def test_collect_balance_takes_each_layer_once(monkeypatch):
    """mlp_forward leaves its logits; the losses are made outside the layers (also
    under activation checkpointing, whose second run adds nothing)."""
    from transformers import GptOssConfig
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssModel
    cfg = GptOssConfig(num_hidden_layers=2, hidden_size=64, intermediate_size=64, num_local_experts=4,
                       num_experts_per_tok=2, num_attention_heads=2, num_key_value_heads=1, head_dim=32, vocab_size=128,
                       layer_types=["sliding_attention", "full_attention"])
    torch.manual_seed(0)
    model = GptOssModel(cfg)
    Q.replace_with_dequant_experts(model, quantization_config=types.SimpleNamespace(dequantize=False))
    monkeypatch.setattr(Q, "router_linear", torch.nn.functional.linear)
    monkeypatch.setattr(Q, "routing", lambda lg, k: (None, None, None))
    monkeypatch.setattr(Q, "on_device", lambda dev: __import__("contextlib").nullcontext())
    for layer in model.layers:
        layer.mlp.experts = torch.nn.Identity()
        layer.mlp.experts.forward = lambda x, *a, **k: x + torch.tanh(x)
    calls = []

    def loss(lg, k, ids, mask):
        calls.append((lg, k, ids, mask))
        return lg.float().pow(2).mean(), torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(routing, "balance_loss", loss)
    ids, mask = torch.randint(0, 128, (2, 5)), torch.ones(2, 5)
    grads = []
    for ckpt in (False, True):
        if ckpt:
            model.gradient_checkpointing_enable(dict(use_reentrant=False))
            model.train()
        model.zero_grad()
        calls.clear()
        with routing.collect_balance(mask) as b:
            out = model(input_ids=ids)
        total = out.last_hidden_state.float().pow(2).mean() + 0.5 * b.loss()
        assert len(calls) == 2 and all(c[0].shape == (10, 4) and c[1] == 2 and c[3].shape == (10,) for c in calls)
        total.backward()
        assert len(calls) == 2 and not routing._COLLECTORS
        assert b.counts().shape == (2, 4) and b.losses().shape == (2,)
        grads.append([layer.mlp.router.weight.grad.clone() for layer in model.layers])
    assert all(torch.allclose(a, c) and a.abs().sum() > 0 for a, c in zip(*grads))
    with routing.collect_balance() as b:
        pass
    with pytest.raises(RuntimeError, match="no MoE layer"):
        b.loss()


def test_c_entries_refuse_what_a_launch_or_32_bits_cannot_hold():
    import ctypes

    from agent_factory_3_amd import _capi
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    strides = (ctypes.c_int64 * 12)(*[64] * 12)
    for match, B, Sq, Sk, scale in (("rows", 1 << 21, 1, 1, 0.1), ("rows", 1 << 17, 1, 1 << 20, 0.1),
                                    ("scale", 1, 4, 4, 3e38)):
        with pytest.raises(RuntimeError, match=match):
            _capi.call("af3_sink_attention_fwd", 64, 64, 64, strides, None, 0, None, 0, None, None, B, 8, 8, Sq, Sk, 64,
                       0, 0, scale, 64, None, None, 0, None)
        with pytest.raises(RuntimeError, match=match):
            _capi.call("af3_sink_attention_bwd", 64, 64, 64, 64, strides, None, 0, None, None, B, 8, 8, Sq, Sk, 64, 0, 0,
                       scale, 64, 64, 64, 64, 64, None, 64, 0, None)


def test_sequence_starts_refuse_host_tensors():
    with pytest.raises(RuntimeError, match="GPU"):
        attention.sequence_starts(torch.tensor([0, 4]), 4)
    with pytest.raises(RuntimeError, match="GPU"):
        attention.sequence_starts_of_positions(torch.arange(4))
    with pytest.raises(ValueError):
        attention.sequence_starts(torch.tensor([0.0, 4.0]), 4)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor's tangent must not be dropped silently (checked before anything else of the tensors)."""
    import torch.autograd.forward_ad as fwd
    q, z = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16), torch.zeros(4, 8)
    with fwd.dual_level():
        for i in range(3):
            t = [q, q, q]
            t[i] = fwd.make_dual(q, torch.ones_like(q))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                attention.sink_attention(*t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.sink_attention(q, q, q, fwd.make_dual(torch.zeros(2), torch.ones(2)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            routing.balance_loss(fwd.make_dual(z, torch.ones_like(z)), 2)
        with pytest.raises(RuntimeError, match="GPU"):   # no tangent: as outside
            attention.sink_attention(q, q, q)


def test_another_threads_forward_is_not_collected():
    """Scoring in another thread beside training leaves the collecting thread's logits alone."""
    import threading
    logits = {n: torch.full((3, 4), float(i)) for i, n in enumerate(("here", "there"))}
    seen, other = [], threading.Barrier(2, timeout=20)

    def scoring():
        other.wait()
        seen.append(bool(routing._COLLECTORS))
        if routing._COLLECTORS:
            routing._COLLECTORS[-1].add("layer", logits["there"], 2)
        with routing.collect_balance() as mine:
            routing._COLLECTORS[-1].add("layer", logits["there"], 2)
            other.wait()
            other.wait()
        seen.append(mine)
    t = threading.Thread(target=scoring)
    t.start()
    with routing.collect_balance() as b:
        routing._COLLECTORS[-1].add("layer", logits["here"], 2)
        other.wait()
        other.wait()      # (the other thread's own collector is open)
        assert routing._COLLECTORS[-1] is b
        other.wait()
        t.join(20)
    assert not routing._COLLECTORS
    assert seen[0] is False and b._seen["layer"][0] is logits["here"]
    assert seen[1]._seen["layer"][0] is logits["there"]
    # nested: the innermost gets the layers
    with routing.collect_balance() as b:
        with routing.collect_balance() as inner:
            assert routing._COLLECTORS[-1] is inner
        assert routing._COLLECTORS[-1] is b
    assert not routing._COLLECTORS


def test_score_capping_is_refused():
    """Models with capped scores pass softcap: it must not be ignored."""
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    m = types.SimpleNamespace(is_causal=True)
    with pytest.raises(NotImplementedError, match="softcap"):
        attention.attention_forward(m, q, q, q, None, softcap=30.0)
    with pytest.raises(RuntimeError, match="GPU"):
        attention.attention_forward(m, q, q, q, None, softcap=None)


def test_c_entries_of_starts_refuse_bad_arguments():
    import ctypes

    from agent_factory_3_amd import _capi
    if not _capi.lib_path().exists():
        pytest.skip("library not built")
    for a in ((64, 8, -1, 8, None, 64, None), (64, 8, 1, -8, None, 64, None), (64, 7, 1, 8, None, 64, None),
              (64, 1 << 29, 1, 1 << 29, None, 64, None), (64, 8, 1 << 22, 8, None, 64, None),
              (64, 8192, 1 << 21, 8192, None, 64, None), (None, 8, 1, 8, None, 64, None), (64, 8, 1, 8, None, None, None)):
        with pytest.raises(RuntimeError, match="seq_starts_rows"):
            _capi.call("af3_seq_starts_rows", *a)
    _capi.call("af3_seq_starts_rows", None, 0, 0, 8, None, None, None)   # nothing to do
    _capi.call("af3_seq_starts_rows", None, 0, 8, 0, None, None, None)
    # a batch of packed rows says how many rows of starts there are
    st = (ctypes.c_int64 * 9)(*[64] * 9)
    for n_seqs, cu in ((0, None), (1, None), (3, None), (2, 64)):
        with pytest.raises(RuntimeError, match="packed"):
            _capi.call("af3_sink_attention_fwd", 64, 64, 64, st, None, 0, cu, n_seqs, 64, None, 2, 2, 1, 4, 4, 64, 0, 0,
                       0.1, 64, None, None, 0, None)
