"""A transformers backbone's attention and norms on the framework's kernels.

    use_in_backbone(model)

switches a transformers model in place: its attention to `sparton_amd.attention` (through the
library's own registry of attention implementations, under the name "sparton"), its LayerNorms to
`SpartonLayerNorm`, and the output blocks of BERT, RoBERTa and XLM-RoBERTa layers to the norm with
the residual sum inside. Parameters, their names and the state_dict stay as they are. The families are
the reference's (training/model.py:14-40): bert, distilbert, roberta, xlm-roberta; decoder-only
backbones whose attention goes through the same registry run causal.

What the kernels do not compute is refused when it is asked for, never approximated: dropout on the
attention probabilities, sliding windows, position biases, masks that are not one value per key.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch import Tensor, nn

from .attention import KEY_MASK_DTYPES, attention
from .norm import SpartonLayerNorm

NAME = "sparton"
# dense -> dropout -> LayerNorm(. + input): the output blocks of an encoder layer.
_RESIDUAL_BLOCKS = ("BertSelfOutput", "BertOutput", "RobertaSelfOutput", "RobertaOutput", "XLMRobertaSelfOutput",
                    "XLMRobertaOutput")
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
    return self.LayerNorm(self.dropout(self.dense(hidden_states)), input_tensor)


class _BlockForward(functools.partial):
    """A block's forward bound to it. A method of a function that its class does not have could not be pickled."""

    @property
    def __self__(self):
        return self.args[0]


def use_in_backbone(model: nn.Module) -> nn.Module:
    """Switch a transformers model (or a masked LM with its head) in place; returns it. A model that
    cannot be switched raises and stays as it was."""
    norms = [(module, name, SpartonLayerNorm.of(child)) for module in model.modules()
             for name, child in module.named_children()
             if type(child) is nn.LayerNorm and len(child.normalized_shape) == 1 and child.weight is not None]
    register()
    before = model.config._attn_implementation
    model.set_attn_implementation(NAME)
    if model.config._attn_implementation != NAME:
        model.set_attn_implementation(before)
        raise ValueError(f"{type(model).__name__} does not take its attention from transformers' registry")
    for module, name, norm in norms:
        setattr(module, name, norm)
    for module in model.modules():
        if type(module).__name__ in _RESIDUAL_BLOCKS and isinstance(module.LayerNorm, SpartonLayerNorm):
            module.forward = _BlockForward(_residual_norm, module)
    return model
