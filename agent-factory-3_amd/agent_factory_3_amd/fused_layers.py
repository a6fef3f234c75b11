"""gpt-oss's decoder layers on the MI355X norms and projections.

``enable_fused_layers(model)`` runs a loaded model's norms, the residual add before
the experts and the attention projections on ``norms`` and ``linear``: transformers'
GptOssDecoderLayer adds and normalises in five elementwise passes each way, and its
projections' bias gradients in passes of their own.  Weights, module names and state
dicts stay as they are; PEFT may wrap the projections before or after (its adapters
run as before around the base layers).  Layers whose tensors the kernels do not take
(another type, on the host, sharded weights outside a gather) run as they did.
"""
from __future__ import annotations

import logging
import types

import torch

from . import norms, routing_replay
from .linear import linear

logger = logging.getLogger(__name__)

_ATTR = "_af3_fused"


def _plain(t) -> bool:
    return t is None or not hasattr(t, "device_mesh")   # (a sharded weight is a DTensor)


def _norm_takes(norm, x) -> bool:
    w = getattr(norm, "weight", None)
    return (x.is_cuda and x.dtype in norms._TYPES and w is not None and w.dtype in norms._TYPES and w.device == x.device
            and hasattr(norm, "variance_epsilon") and _plain(w)
            and w.shape == x.shape[-1:]   # (else a placeholder: the weight comes with the module's call)
            and norms.MIN_HIDDEN <= x.shape[-1] <= norms.MAX_HIDDEN)


def _norm_forward(self, hidden_states):
    if not _norm_takes(self, hidden_states):
        return type(self).forward(self, hidden_states)
    return norms.rms_norm(hidden_states, self.weight, self.variance_epsilon)


def _linear_forward(self, input):
    ts = [t for t in (input, self.weight, self.bias) if t is not None]
    if not all(t.is_cuda and t.dtype == torch.bfloat16 and t.device == input.device and _plain(t) for t in ts):
        return type(self).forward(self, input)
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != torch.bfloat16:   # (its product's type)
        return type(self).forward(self, input)
    return linear(input, self.weight, self.bias)


# (a bound method is pickled by its name: a model saved whole loads with its classes' own forwards)
_norm_forward.__name__ = _linear_forward.__name__ = "forward"


def _layer_forward(self, hidden_states, attention_mask=None, position_ids=None, past_key_values=None, use_cache=False,
                   position_embeddings=None, **kwargs):
    """GptOssDecoderLayer.forward with the add and the norm between attention and experts as one."""
    h, _ = self.self_attn(hidden_states=self.input_layernorm(hidden_states), attention_mask=attention_mask,
                          position_ids=position_ids, past_key_values=past_key_values, use_cache=use_cache,
                          position_embeddings=position_embeddings, **kwargs)
    norm = self.post_attention_layernorm
    if _norm_takes(norm, h) and h.dtype == hidden_states.dtype and h.shape == hidden_states.shape:
        residual, h = norms.residual_norm(h, hidden_states, norm.weight, eps=norm.variance_epsilon)
    else:
        residual = hidden_states + h
        h = norm(residual)
    h, _ = self.mlp(h)
    return residual + h


def _bind(module, forward):
    """Make ``forward`` the module's, under a hook of accelerate's where it has one."""
    setattr(module, "_old_forward" if hasattr(module, "_hf_hook") else "forward", types.MethodType(forward, module))


def _patch_layer_class():
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssDecoderLayer
    if getattr(GptOssDecoderLayer, "_af3_fused_layers", False):
        return
    orig_forward = GptOssDecoderLayer.forward

    def forward(self, hidden_states, *args, **kwargs):
        if not getattr(self, _ATTR, False):
            return orig_forward(self, hidden_states, *args, **kwargs)
        # (routing replay, enabled before, lies in the forward that this one stands in for)
        with routing_replay.layer_indices(self, kwargs):
            return _layer_forward(self, hidden_states, *args, **kwargs)

    GptOssDecoderLayer.forward = forward
    GptOssDecoderLayer._af3_fused_layers = True


def enable_fused_layers(model, projections: bool = True) -> int:
    """Run ``model``'s GptOssDecoderLayers on the fused kernels; returns how many.

    Every GptOssRMSNorm runs on ``norms.rms_norm``, the add and norm between attention
    and experts on ``norms.residual_norm`` (whose module's forward, and hooks on it, are
    then not called), and with ``projections`` q, k, v and o (the layers inside PEFT's
    wrappers too) on ``linear.linear``: a few percent slower than the library's products
    forward, faster backward, and deterministic.  Results differ from transformers' by
    roundings.  Again is harmless; a copy of the model is fused too, one saved and loaded whole
    needs the call again.
    """
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssDecoderLayer, GptOssRMSNorm
    layers = [m for m in model.modules() if isinstance(m, GptOssDecoderLayer)]
    if not layers:
        raise ValueError("enable_fused_layers: the model has no GptOssDecoderLayer")
    _patch_layer_class()
    for m in model.modules():
        if type(m) is GptOssRMSNorm:
            _bind(m, _norm_forward)
    for layer in layers:
        setattr(layer, _ATTR, True)
        if hasattr(layer, "_hf_hook"):   # (it holds the class's forward of before)
            _bind(layer, GptOssDecoderLayer.forward)
        if projections:
            for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
                m = getattr(layer.self_attn, name)
                m = getattr(m, "base_layer", m)
                if type(m) is torch.nn.Linear:
                    _bind(m, _linear_forward)
    logger.info("fused norms%s enabled for %d layers", " and projections" if projections else "", len(layers))
    return len(layers)
