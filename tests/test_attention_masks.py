"""What af3_sink's mask function makes of the mask functions that transformers hands it (CPU)."""
import pytest
import torch

from agent_factory_3_amd import attention, quantizer_config  # noqa: F401  (registers)


def _model(layers=2):
    from transformers import GptOssConfig
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssModel
    cfg = GptOssConfig(num_hidden_layers=layers, hidden_size=64, intermediate_size=64, num_local_experts=4,
                       num_experts_per_tok=2, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
                       vocab_size=128, sliding_window=8, layer_types=["sliding_attention", "full_attention"])
    cfg._attn_implementation = "af3_sink"
    torch.manual_seed(0)
    return GptOssModel(cfg)


POS = [[0, 1, 2, 0, 1, 2], [0, 1, 0, 1, 2, 3]]
STARTS = [[0, 0, 0, 3, 3, 3], [0, 0, 2, 2, 2, 2]]


def _starts(pos, kv_range=None):
    at = torch.arange(pos.shape[1])
    new = torch.ones_like(pos, dtype=torch.bool)
    new[:, 1:] = pos[:, 1:] != pos[:, :-1] + 1
    return torch.where(new, at, 0).cummax(1).values.to(torch.int32)


def _stand_in(monkeypatch):
    """What the kernels would be called with."""
    import contextlib
    seen = []

    def run(q, k, v, sinks, scale, window, first, cu_seqlens, starts, kv_range):
        assert cu_seqlens is None and kv_range is None and scale == 0.125
        seen.append((q.shape, window, starts))
        return q.transpose(1, 2)
    monkeypatch.setattr(attention, "_run", run)
    monkeypatch.setattr(attention, "_check", lambda *a: None)
    monkeypatch.setattr(attention, "_device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(attention, "sink_attention", lambda q, *a, **kw: seen.append((q.shape, kw)) or q.transpose(1, 2))
    return seen


def test_layers_read_a_batch_of_packed_rows_from_its_position_ids(monkeypatch):
    """gpt-oss gives its mask functions no position ids: its layers read them, of every row."""
    seen, asked = _stand_in(monkeypatch), []
    monkeypatch.setattr(attention, "sequence_starts_of_rows",
                        lambda pos, rng=None: asked.append((pos.tolist(), rng)) or torch.tensor(STARTS, dtype=torch.int32))
    with torch.no_grad():
        _model()(input_ids=torch.randint(0, 128, (2, 6)), position_ids=torch.tensor(POS))
    assert asked == [(POS, None)] * 2 and [s[1] for s in seen] == [8, 0]
    assert all(s[0] == (2, 2, 6, 64) and s[2].tolist() == STARTS for s in seen)


@pytest.mark.parametrize("pos,starts", [(POS, STARTS), (POS[:1], [STARTS[0]] * 2)])
@pytest.mark.parametrize("window", [0, 8])
def test_the_packing_that_transformers_finds(pos, starts, window, monkeypatch):
    """Models that give their mask functions position ids (one row of them may stand for all): the packing
    is in the mask function, and every layer gets the places in their sequences that were made of it."""
    from transformers.masking_utils import create_causal_mask, create_sliding_window_causal_mask
    make = create_sliding_window_causal_mask if window else create_causal_mask
    cfg = _model(layers=2).config
    mask = make(config=cfg, inputs_embeds=torch.zeros(2, 6, 64), attention_mask=None, past_key_values=None,
                position_ids=torch.tensor(pos))
    assert mask.shape == (2, 6, 1) and (torch.arange(6) - mask[..., 0]).tolist() == starts
    seen = _stand_in(monkeypatch)
    monkeypatch.setattr(attention, "sequence_starts_of_rows", _starts)
    q = torch.zeros(2, 2, 6, 64)
    out, _ = attention.attention_forward(None, q, q, q, mask, scaling=0.125, sliding_window=window, is_causal=True)
    assert out.shape == (2, 6, 2, 64) and seen[0][1] == window and seen[0][2].tolist() == starts
    same = make(config=cfg, inputs_embeds=torch.zeros(2, 6, 64), attention_mask=None, past_key_values=None,
                position_ids=torch.arange(6).expand(2, 6))
    assert same is None
    with pytest.raises(ValueError, match="mask"):   # another batch's
        attention.attention_forward(None, q[:1], q[:1], q[:1], mask, is_causal=True)


def test_mask_functions_that_it_cannot_honour_are_refused():
    from transformers import masking_utils as mu
    f = attention.attention_mask
    win = mu.sliding_window_causal_mask_function(3)
    assert f(1, 6, 6, mask_function=mu.causal_mask_function) is None and f(1, 6, 6, mask_function=win) is None
    assert f(1, 1, 6, q_offset=5, mask_function=mu.and_masks(win, mu.causal_mask_function)) is None
    chunks = mu.chunked_causal_mask_function(4, torch.tensor([0]))
    assert f(1, 4, 4, mask_function=chunks) is None   # one chunk: causal
    packed = mu.packed_sequence_mask_function(torch.tensor([[0, 0, 1, 1]]))
    for kw in (dict(q_length=6, kv_length=6, mask_function=chunks),
               dict(q_length=1, kv_length=6, q_offset=5, mask_function=chunks),
               dict(q_length=4, kv_length=4, mask_function=mu.and_masks(mu.causal_mask_function, lambda b, h, q, k: k > 0)),
               dict(q_length=4, kv_length=4, mask_function=mu.or_masks(mu.causal_mask_function, packed)),
               dict(q_length=4, kv_length=4, mask_function=mu.bidirectional_mask_function),
               dict(q_length=4, kv_length=6, q_offset=2, mask_function=mu.and_masks(mu.causal_mask_function, packed)),
               dict(q_length=4, kv_length=4, mask_function=mu.and_masks(mu.causal_mask_function, packed),
                    attention_mask=torch.tensor([[1, 1, 1, 0]]))):
        with pytest.raises(NotImplementedError, match="af3_sink"):
            f(1, **kw)
