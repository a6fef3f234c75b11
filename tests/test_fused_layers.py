"""The fused layers' wiring on the CPU: host tensors run as before, routing replay reaches the experts
whichever of the two is enabled first (each order in a process of its own: both patch a class)."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CODE = r'''
import sys, types
import torch
sys.path.insert(0, "agent-factory-3_amd")
from transformers import GptOssConfig
from transformers.models.gpt_oss.modeling_gpt_oss import GptOssModel, GptOssMLP
from agent_factory_3_amd import routing_replay
from agent_factory_3_amd.fused_layers import enable_fused_layers

seen = []
orig = GptOssMLP.forward
def mlp(self, hidden_states, *a, **k):
    seen.append(routing_replay.current_router_indices(self))
    return orig(self, hidden_states, *a, **k)
GptOssMLP.forward = mlp
cfg = GptOssConfig(num_hidden_layers=2, hidden_size=64, intermediate_size=64, num_local_experts=4, num_experts_per_tok=2,
                   num_attention_heads=2, num_key_value_heads=1, head_dim=32, vocab_size=128, sliding_window=8,
                   layer_types=["sliding_attention", "full_attention"])
cfg._attn_implementation = "eager"
torch.manual_seed(0)
model, other = GptOssModel(cfg), GptOssModel(cfg)
ids = torch.arange(12)[None] % 7
with torch.no_grad():
    want = model(ids, use_cache=False).last_hidden_state
    for step in sys.argv[1].split(","):
        if step == "replay":
            routing_replay.enable_routing_replay(model)
        else:
            assert enable_fused_layers(model) == 2 and enable_fused_layers(model) == 2
    ri = torch.arange(12 * 2 * 2).view(1, 12, 2, 2)
    seen.clear()
    got = model(ids, use_cache=False, **({"routing_indices": ri} if "replay" in sys.argv[1] else {})).last_hidden_state
    assert torch.equal(got, want)          # host tensors: transformers' own path
    if "replay" in sys.argv[1]:
        assert torch.equal(seen[0], ri[:, :, 0]) and torch.equal(seen[1], ri[:, :, 1])
        assert all(routing_replay.current_router_indices(l.mlp) is None for l in model.layers)
    seen.clear()
    assert torch.equal(model(ids, use_cache=False).last_hidden_state, want) and seen == [None, None]
    other(ids, use_cache=False)            # a model that was not enabled
assert not hasattr(other.layers[0], "_af3_fused")
try:
    enable_fused_layers(torch.nn.Linear(2, 2))
    raise SystemExit("a model without layers was taken")
except ValueError:
    print("ok")
'''


@pytest.mark.parametrize("order", ["fused", "replay,fused", "fused,replay"])
def test_orders(order):
    r = subprocess.run([sys.executable, "-c", CODE, order], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
