"""A transformers backbone's attention and norms on the framework's kernels.

    use_in_backbone(model, rms_norm=False, feed_forward=False, embedding=False)

switches a transformers model in place: its attention to `sparton_amd.attention` (through the
library's own registry of attention implementations, under the name "sparton"), its LayerNorms to
`SpartonLayerNorm`, and the output blocks of BERT, RoBERTa and XLM-RoBERTa layers to the norm with
the residual sum inside. Parameters, their names and the state_dict stay as they are. The families are
the reference's (training/model.py:14-40): bert, distilbert, roberta, xlm-roberta; decoder-only
backbones whose attention goes through the same registry run causal. Asked for, the rest of such a backbone's
layer is switched too: root-mean-square norms to `SpartonRMSNorm` (and layers that add their attention's output
and norm the sum to the norm that does both), gated feed-forward blocks to `gated_linear`, embeddings to
`SpartonEmbedding`. Whether a module computes what the kernels do is found by running a small copy of it on
the CPU; one that does not keeps its own forward.

What the kernels do not compute is refused when it is asked for, never approximated: dropout on the
attention probabilities, sliding windows, position biases, masks that are not one value per key.
"""
from __future__ import annotations

import copy
import functools
import inspect
from typing import Dict, Optional

import torch
from torch import Tensor, nn

from . import feed_forward as _ff
from ._look import PLAIN, computes
from .attention import KEY_MASK_DTYPES, attention
from .embedding import SpartonEmbedding
from .norm import SpartonLayerNorm, SpartonRMSNorm, computes_rms_norm

NAME = "sparton"
# dense -> dropout -> LayerNorm(. + input): the output blocks of an encoder layer.
_RESIDUAL_BLOCKS = ("BertSelfOutput", "BertOutput", "RobertaSelfOutput", "RobertaOutput", "XLMRobertaSelfOutput",
                    "XLMRobertaOutput")
_REQUIRED = inspect.Parameter.empty  # the default of a parameter that has none
_UNSUPPORTED = ("sliding_window", "softcap", "s_aux", "position_bias", "head_mask")


def attention_forward(module: nn.Module, query: Tensor, key: Tensor, value: Tensor, attention_mask: Optional[Tensor],
                      scaling: Optional[float] = None, dropout: float = 0.0, is_causal: Optional[bool] = None, **kwargs):
    """The registry's signature: query [B,Hq,Sq,D], key and value [B,Hk,Sk,D], and the mask that
    `key_mask` below returned. Gives ([B,Sq,Hq,D], None)."""
    if dropout:
        raise ValueError("sparton attention has no dropout on its probabilities: set the model's attention dropout "
                         f"to 0 (got {dropout})")
    for name in _UNSUPPORTED:
        if kwargs.get(name) is not None:
            raise ValueError(f"sparton attention does not support {name}")
    if kwargs.get("output_attentions"):
        raise ValueError("sparton attention forms no matrix of probabilities to return (output_attentions)")
    if attention_mask is not None and attention_mask.dim() != 2:
        raise ValueError(f"sparton attention takes one mask value per key [B,Sk], got {tuple(attention_mask.shape)}")
    causal = bool(getattr(module, "is_causal", False) if is_causal is None else is_causal)
    out = attention(query, key, value, attention_mask, causal=causal, scale=scaling)
    return out.transpose(1, 2), None


def key_mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None, attention_mask=None, **kwargs):
    """The registry's mask: the tokenizer's values of the keys, [B, kv_length], or None. Its column j is
    position j, and the keys are the positions from kv_offset on; a position past its last column takes no
    part. What is causal is known to the attention itself, whose rows are the last ones of the keys: behind
    several rows there may be no room in a cache allocated ahead; behind one row the room is masked, from the
    cache's length on the device, if that is where the cache keeps it."""
    from transformers.masking_utils import bidirectional_mask_function, causal_mask_function
    if mask_function not in (None, bidirectional_mask_function, causal_mask_function):
        raise ValueError("sparton attention supports plain bidirectional and causal attention over padded batches; "
                         "this model asks for another pattern (windows, packed sequences)")
    one = mask_function is causal_mask_function and q_length == 1 and isinstance(q_offset, Tensor)
    if mask_function is causal_mask_function and not one and int(q_offset) + q_length != kv_offset + kv_length:
        raise ValueError("sparton attention's causal rows are the last ones of the keys; this cache has room behind them")
    if attention_mask is not None and attention_mask.dtype not in KEY_MASK_DTYPES:
        attention_mask = attention_mask != 0  # true or false to transformers too, whatever the type
    if attention_mask is not None and (kv_offset != 0 or attention_mask.shape[-1] != kv_length):
        attention_mask = attention_mask[:, kv_offset:kv_offset + kv_length]
        attention_mask = nn.functional.pad(attention_mask, (0, kv_length - attention_mask.shape[-1]))
    if one:
        at = torch.arange(kv_offset, kv_offset + kv_length, device=kwargs.get("device") or q_offset.device)
        seen = (at <= q_offset).expand(batch_size, -1)
        attention_mask = seen if attention_mask is None else seen & (attention_mask != 0)
    return attention_mask


def register() -> None:
    """Make attn_implementation="sparton" known to transformers: once per process, before a switched model
    that was pickled elsewhere, or saved with its config, runs there."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface
    AttentionInterface.register(NAME, attention_forward)
    AttentionMaskInterface.register(NAME, key_mask)


def _residual_norm(self, hidden_states: Tensor, input_tensor: Tensor) -> Tensor:
    norm, hidden_states = self.LayerNorm, self.dropout(self.dense(hidden_states))
    if isinstance(norm, SpartonLayerNorm) and _ff.untouched(norm):
        return norm(hidden_states, input_tensor)
    return norm(hidden_states + input_tensor)  # a hook sees the norm's one input; another forward takes no residual


class _BlockForward(functools.partial):
    """A block's forward bound to it. A method of a function that its class does not have could not be pickled."""

    @property
    def __self__(self):
        return self.args[0]


def _gated_block(self, *args, **kwargs) -> Tensor:
    gate, up = self.gate_proj, self.up_proj
    activation = _ff.plain_activation(self.act_fn)
    # an adapter or a hook came since, or the input goes by its name
    if activation is None or not _ff.plain_linears(gate, up) or kwargs or len(args) != 1:
        return type(self).forward(self, *args, **kwargs)
    (x,) = args
    h = _ff.gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, activation)
    return self.down_proj(h)


def _pre_norm_layer(self, params, more, *args, **kwargs) -> Tensor:
    """params: the names and defaults of what the layer's own forward takes; more: whether it takes other names too. All
    but the hidden states go to the attention by their names, as they do there."""
    given = dict(zip((name for name, _ in params), args))
    call = {**dict(params), **given, **kwargs}
    if (len(args) > len(params) or given.keys() & kwargs.keys() or any(v is _REQUIRED for v in call.values())
            or not more and len(call) > len(params)):
        return type(self).forward(self, *args, **kwargs)  # which refuses the call
    hidden_states = call.pop(params[0][0])
    attended = self.self_attn(hidden_states=self.input_layernorm(hidden_states), **call)[0]
    norm = self.post_attention_layernorm
    if isinstance(norm, SpartonRMSNorm) and _ff.untouched(norm):
        hidden_states, residual = norm(attended, hidden_states)
    else:  # a hook sees a norm's one input and output, and another module or forward takes no residual
        residual = hidden_states + attended
        hidden_states = norm(residual)
    return residual + self.mlp(hidden_states)


# ---- what a module computes: a small copy of it, on the CPU, against the formula -------------

class _Times(nn.Module):
    """Stands for a submodule: what goes through it is seen in the result."""

    def __init__(self, factor: float):
        super().__init__()
        self.factor = factor

    def forward(self, x):
        return x * self.factor


class _Attended(nn.Module):
    """Stands for the attention; takes the hidden states by their name, and beside them what `others` says alone."""

    def __init__(self, others):
        super().__init__()
        self.others = others

    def forward(self, *, hidden_states, **kwargs):
        if kwargs.keys() != self.others.keys() or any(kwargs[n] is not v for n, v in self.others.items()):
            raise ValueError("another call of the attention")
        return hidden_states * 3.0, None


def _is_rms_norm(m: nn.Module) -> bool:
    return (not isinstance(m, SpartonRMSNorm) and type(m).__name__.endswith("RMSNorm")
            and list(m._parameters) == ["weight"] and computes_rms_norm(m))


def _is_gated_block(m: nn.Module) -> bool:
    """down_proj(act_fn(gate_proj(x)) * up_proj(x)) of plain linears, and nothing else in it."""
    return (_ff.computes_gated_block(m) and all(type(t) is nn.Linear for t in (m.gate_proj, m.up_proj, m.down_proj))
            and m.gate_proj.weight.shape == m.up_proj.weight.shape)


def _params(m: nn.Module) -> Optional[tuple]:
    """((name, default or _REQUIRED), ...) of what m's class's forward takes, and whether it takes other names too; None
    if names alone do not say it."""
    ps = list(inspect.signature(type(m).forward).parameters.values())[1:]
    more = bool(ps) and ps[-1].kind is ps[-1].VAR_KEYWORD
    if more:
        ps.pop()
    if not ps or any(p.kind is not p.POSITIONAL_OR_KEYWORD for p in ps):
        return None
    return tuple((p.name, p.default) for p in ps), more


def _is_pre_norm_layer(m: nn.Module) -> bool:
    """h = x + self_attn(input_layernorm(x)); h + mlp(post_attention_layernorm(h)), what it takes besides x going to
    the attention."""
    names = ("input_layernorm", "self_attn", "post_attention_layernorm", "mlp")
    if set(m._modules) != set(names) or m._parameters or m._buffers:
        return False
    found = _params(m)
    if found is None:
        return False
    params, more = found
    # flags keep their defaults; what may be None is something here, to be seen again in the attention
    others = {n: object() if default is None or default is _REQUIRED else default for n, default in params[1:]}
    if more:
        others["another_name"] = object()
    x = torch.linspace(-1, 1, 12, **PLAIN).view(1, 3, 4)
    children = dict(zip(names, (_Times(2.0), _Attended(others), _Times(5.0), _Times(7.0))))
    return computes(m, children, x, lambda: 36.0 * (x * 7.0), **others)  # x + 3 * 2 x, and 1 + 5 * 7 times that


def use_in_backbone(model: nn.Module, *, rms_norm: bool = False, feed_forward: bool = False,
                    embedding: bool = False) -> nn.Module:
    """Switch a transformers model (or a masked LM with its head) in place; returns it. A model that
    cannot be switched, or that has nothing of a kind that is asked for, raises and stays as it was."""
    norms = [(module, name, SpartonLayerNorm.of(child)) for module in model.modules()
             for name, child in module.named_children()
             if type(child) is nn.LayerNorm and len(child.normalized_shape) == 1 and child.weight is not None
             and "forward" not in child.__dict__]
    modules = list(model.modules())
    children = [(module, name, child) for module in modules for name, child in module.named_children()]
    made: Dict[int, nn.Module] = {}  # a module in several places becomes one

    def replaced(child: nn.Module, make) -> nn.Module:
        if id(child) not in made:
            made[id(child)] = make(child)
        return made[id(child)]

    forwards = []
    if rms_norm:
        found = [(m, n, replaced(c, SpartonRMSNorm.of)) for m, n, c in children if _is_rms_norm(c)]
        if not found and not any(isinstance(m, SpartonRMSNorm) for m in modules):
            raise ValueError(f"{type(model).__name__} has no root-mean-square norm that the kernels compute")
        norms += found
        ours = {id(c) for _, _, c in children if isinstance(c, SpartonRMSNorm) or id(c) in made}
        forwards += [(m, _pre_norm_layer, *_params(m)) for m in modules if "forward" not in m.__dict__ and _is_pre_norm_layer(m)
                     and id(m.post_attention_layernorm) in ours]
    if feed_forward:
        blocks = [m for m in modules if _is_gated_block(m)]
        if not blocks:
            raise ValueError(f"{type(model).__name__} has no gated feed-forward block that the kernels compute")
        forwards += [(m, _gated_block) for m in blocks if "forward" not in m.__dict__]
    if embedding:
        found = [(m, n, replaced(c, SpartonEmbedding.of)) for m, n, c in children
                 if type(c) is nn.Embedding and "forward" not in c.__dict__]
        if not found and not any(isinstance(m, SpartonEmbedding) for m in modules):
            raise ValueError(f"{type(model).__name__} has no nn.Embedding")
        norms += found
    register()
    before = model.config._attn_implementation
    model.set_attn_implementation(NAME)
    if model.config._attn_implementation != NAME:
        model.set_attn_implementation(before)
        raise ValueError(f"{type(model).__name__} does not take its attention from transformers' registry")
    for module, name, child in norms:
        setattr(module, name, child)
    for module, forward, *more in forwards:
        module.forward = _BlockForward(forward, module, *more)
    for module in model.modules():
        if type(module).__name__ in _RESIDUAL_BLOCKS and isinstance(module.LayerNorm, SpartonLayerNorm):
            module.forward = _BlockForward(_residual_norm, module)
    return model
