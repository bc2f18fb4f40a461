"""Embedding lookup with scaling, and its gradient by sorted tokens, on hand-written HIP kernels.

    out[..., :] = scale * weight[ids[...], :]
    d_weight[v] = scale * sum of d_out over the places where ids == v, in their order

The first operator of a backbone (the reference runs torch's, training/model.py:88-139). The gradient
sorts the tokens and adds each one's rows in order, so it is bitwise reproducible; a token that half of
the batch has (a padding or separator token) is summed in chunks by many waves, and the chunks by few.

    sparton::embedding_fwd(ids, weight, scale) -> out
    sparton::embedding_bwd(d_out, ids, rows, scale, padding) -> d_weight [rows, D]

An id outside the table reads nothing: its row is NaN and it has no gradient (checking ids on the host
would wait for the device). Device tensors only, like the head.
"""
from __future__ import annotations

import copy
from typing import Optional

import torch
from torch import Tensor, nn

from . import _eager, _lib

MAX_WIDTH = 1 << 20
MAX_SCALE = torch.finfo(torch.float32).max
ID_DTYPES = (torch.int64, torch.int32)
_FLOAT_DTYPES = tuple(_lib.DTYPE_CODE)


def _check(ids: Tensor, table: Tensor, rows: int, scale: float, op: str) -> None:
    """table: the weight, or the gradient of the rows; its last dimension is the width."""
    if ids.dtype not in ID_DTYPES:
        raise TypeError(f"{op}: ids must be int64 or int32, got {ids.dtype}")
    if table.dtype not in _FLOAT_DTYPES:
        raise TypeError(f"{op}: the table must be float32, bfloat16 or float16, got {table.dtype}")
    if not 1 <= table.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{op}: row width {table.shape[-1]} must be between 1 and {MAX_WIDTH}")
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"{op}: scale must be finite in float32, got {scale}")
    if rows >= 2 ** 31 - 1 or ids.numel() > 2 ** 31 - 1025:
        raise ValueError(f"{op}: {ids.numel()} ids of {rows} rows are too many")
    if ids.device != table.device:
        raise ValueError(f"{op}: ids and the table must be on one device, got {ids.device} and {table.device}")
    if not table.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {table.device})")


def _check_table(ids: Tensor, weight: Tensor, scale: float, op: str) -> None:
    if weight.dim() != 2:
        raise ValueError(f"{op}: weight must be [V, D], got {tuple(weight.shape)}")
    _check(ids, weight, weight.shape[0], scale, op)


@torch.library.custom_op("sparton::embedding_fwd", mutates_args=())
def embedding_fwd(ids: Tensor, weight: Tensor, scale: float, padding: int) -> Tensor:
    """scale * weight[ids]; `padding` (-1: none) is the row that gets no gradient."""
    _eager.refuse_forward_mode("sparton::embedding_fwd", weight)
    _check_table(ids, weight, scale, "sparton::embedding_fwd")
    return _eager.load().embedding(ids, weight, scale, padding)


@embedding_fwd.register_fake
def _(ids, weight, scale, padding):
    return weight.new_empty((*ids.shape, weight.shape[1]))


@torch.library.custom_op("sparton::embedding_bwd", mutates_args=())
def embedding_bwd(d_out: Tensor, ids: Tensor, rows: int, scale: float, padding: int) -> Tensor:
    """The gradient [rows, D] of the table, in d_out's dtype: fp32 sums, rounded once."""
    op = "sparton::embedding_bwd"
    if tuple(d_out.shape[:-1]) != tuple(ids.shape) or d_out.dim() == 0:
        raise ValueError(f"{op}: d_out must be {tuple(ids.shape)} rows, got {tuple(d_out.shape)}")
    if rows < 0:
        raise ValueError(f"{op}: rows must not be negative, got {rows}")
    _check(ids, d_out, rows, scale, op)
    return _eager.load().embedding_bwd(d_out, ids, rows, scale, padding)


@embedding_bwd.register_fake
def _(d_out, ids, rows, scale, padding):
    return d_out.new_empty((rows, d_out.shape[-1]))


def _setup_context(ctx, inputs, output):
    ids, weight, scale, padding = inputs
    ctx.save_for_backward(ids)
    ctx.rows, ctx.scale, ctx.padding = weight.shape[0], scale, padding


def _backward(ctx, d_out):
    (ids,) = ctx.saved_tensors
    return None, torch.ops.sparton.embedding_bwd(d_out, ids, ctx.rows, ctx.scale, ctx.padding), None, None


embedding_fwd.register_autograd(_backward, setup_context=_setup_context)


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[ids]: [*ids.shape, D] in weight's dtype, from ids (int64 or int32, any shape) and weight
    [V, D]. The row padding_idx (negative: from the end, as torch counts) gets no gradient. An id outside
    [0, V) gives a row of NaN and has no gradient."""
    scale = float(scale)
    padding = -1
    if padding_idx is not None:
        rows = weight.shape[0] if weight.dim() > 0 else 0
        if not -rows <= padding_idx < rows:
            raise ValueError(f"embedding: padding_idx {padding_idx} is not one of {rows} rows")
        padding = int(padding_idx) % rows
    if torch.compiler.is_compiling() or not weight.is_cuda:  # the registered op: fake + autograd
        return torch.ops.sparton.embedding_fwd(ids, weight, scale, padding)
    _check_table(ids, weight, scale, "embedding")
    return _eager.load().embedding(ids, weight, scale, padding)


class SpartonEmbedding(nn.Embedding):
    """An nn.Embedding on the kernels above, with an optional factor: module.scale * weight[ids].
    `SpartonEmbedding.of(embedding)` shares an existing module's parameter (name and state_dict unchanged)
    and keeps its hooks; of a SpartonEmbedding, its factor too, times this one. Renormed, sparse and frequency-scaled
    embeddings are refused, and modules with another forward than nn.Embedding's."""

    scale: float = 1.0

    def __init__(self, *args, scale: float = 1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self._check_module(self)
        self.scale = float(scale)

    @staticmethod
    def _check_module(m: nn.Embedding) -> None:
        if m.max_norm is not None or m.sparse or m.scale_grad_by_freq:
            raise ValueError(f"SpartonEmbedding has no max_norm, sparse or scale_grad_by_freq, got {m}")
        if not 1 <= m.embedding_dim <= MAX_WIDTH:
            raise ValueError(f"SpartonEmbedding takes rows up to {MAX_WIDTH}, got {m.embedding_dim}")

    @classmethod
    def of(cls, module: nn.Embedding, scale: float = 1.0) -> "SpartonEmbedding":
        cls._check_module(module)
        if type(module).forward not in (nn.Embedding.forward, cls.forward) or "forward" in module.__dict__:
            raise ValueError(f"SpartonEmbedding computes nn.Embedding's rows times a factor; {module} has another forward")
        m = copy.copy(module)  # the same hooks and mode
        m.__class__ = cls
        m._parameters = dict(m._parameters)  # and parameters, until either module is given another one
        m.scale = float(scale) * (module.scale if isinstance(module, SpartonEmbedding) else 1.0)
        return m

    def forward(self, input: Tensor) -> Tensor:
        return embedding(input, self.weight, self.scale, self.padding_idx)
