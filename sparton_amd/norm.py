"""LayerNorm of a backbone's rows, with the residual sum in front of it, on hand-written HIP kernels.

    y = LayerNorm(x + residual) * weight + bias        per row over the last dimension D

Every encoder layer of a BERT-like backbone has it twice (the reference runs torch's,
training/model.py:88-139); the transform before the head has the same norm behind its gelu
(transform.py). One pass reads x and residual and writes y; the backward reads dy, x and residual and
writes one gradient, which serves both, and the column sums for weight and bias, deterministically.
The residual sum is formed in fp32 and not rounded, so nothing of it is stored.

    sparton::layer_norm_fwd(x, residual?, weight, bias?, eps) -> (y, mean, rstd)
    sparton::layer_norm_bwd(dy, x, residual?, weight, has_bias, mean, rstd) -> (dx, d_weight, d_bias)

Device tensors only, like the head.
"""
from __future__ import annotations

import copy
import math
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _eager, _lib

MAX_WIDTH = 16384
_FLOAT_DTYPES = tuple(_lib.DTYPE_CODE)


def _check(x: Tensor, residual: Optional[Tensor], weight: Tensor, bias: Optional[Tensor], eps: float, op: str) -> int:
    if x.dim() < 1 or x.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"{op}: x must be a float tensor [..., D], got {x.dtype} {tuple(x.shape)}")
    D = x.shape[-1]
    if not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"{op}: row width {D} must be between 1 and {MAX_WIDTH}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{op}: residual must be {x.dtype} {tuple(x.shape)}, got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    for t in (weight, bias):
        if t is not None and (tuple(t.shape) != (D,) or t.dtype not in (torch.float32, x.dtype)
                              or t.dtype != weight.dtype):
            raise ValueError(f"{op}: weight and bias must be [{D}], both float32 or both {x.dtype}, got "
                             f"{t.dtype} {tuple(t.shape)}")
    for t in (residual, weight, bias):
        if t is not None and t.device != x.device:
            raise ValueError(f"{op}: all tensors must be on {x.device}, got {t.device}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"{op}: eps must be finite and not negative, got {eps}")
    if not x.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {x.device})")
    return D


@torch.library.custom_op("sparton::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Tensor, bias: Optional[Tensor],
                   eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(y in x's dtype, mean, rstd), the last two per row in fp32 for the backward."""
    _check(x, residual, weight, bias, eps, "sparton::layer_norm_fwd")
    return _eager.load().layer_norm_fwd(x, residual, weight, bias, eps)


@layer_norm_fwd.register_fake
def _(x, residual, weight, bias, eps):
    D = x.shape[-1]
    row = x.new_empty((x.numel() // D if D else 0,), dtype=torch.float32)
    return x.new_empty(x.shape), row, row.clone()


@torch.library.custom_op("sparton::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy: Tensor, x: Tensor, residual: Optional[Tensor], weight: Tensor, has_bias: bool, mean: Tensor,
                   rstd: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """(dx in x's dtype, which is the residual's gradient too; d_weight and d_bias in the weight's)."""
    op = "sparton::layer_norm_bwd"
    D = _check(x, residual, weight, None, 0.0, op)
    M = x.numel() // D
    if dy.shape != x.shape or dy.device != x.device:
        raise ValueError(f"{op}: dy must be {tuple(x.shape)} on {x.device}, got {tuple(dy.shape)} on {dy.device}")
    for t in (mean, rstd):
        if tuple(t.shape) != (M,) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{op}: mean and rstd must be contiguous float32 [{M}] on {x.device}")
    return _eager.load().layer_norm_bwd(dy, x, residual, weight, has_bias, mean, rstd)


@layer_norm_bwd.register_fake
def _(dy, x, residual, weight, has_bias, mean, rstd):
    return x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty((x.shape[-1] if has_bias else 0,))


def _setup_context(ctx, inputs, output):
    x, residual, weight, bias, _eps = inputs
    _y, mean, rstd = output
    ctx.mark_non_differentiable(mean, rstd)  # kept for the backward only
    ctx.set_materialize_grads(False)
    ctx.has_bias = bias is not None
    ctx.save_for_backward(x, residual, weight, mean, rstd)


def _backward(ctx, dy, _dmean, _drstd):
    x, residual, weight, mean, rstd = ctx.saved_tensors
    if dy is None:  # y did not reach the loss
        return None, None, None, None, None
    dx, dw, db = torch.ops.sparton.layer_norm_bwd(dy, x, residual, weight, ctx.has_bias, mean, rstd)
    return dx, (dx if residual is not None else None), dw, (db if ctx.has_bias else None), None


layer_norm_fwd.register_autograd(_backward, setup_context=_setup_context)


def layer_norm(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, eps: float = 1e-5,
               residual: Optional[Tensor] = None) -> Tensor:
    """LayerNorm(x + residual) * weight + bias over the last dimension (up to 16384), in x's dtype;
    weight and bias are float32 (masters) or of x's dtype, and get their gradients in it."""
    eps = float(eps)
    if torch.compiler.is_compiling() or not x.is_cuda:  # the registered op: fake + autograd
        return torch.ops.sparton.layer_norm_fwd(x, residual, weight, bias, eps)[0]
    _check(x, residual, weight, bias, eps, "layer_norm")
    return _eager.load().layer_norm(x, residual, weight, bias, eps)


class SpartonLayerNorm(nn.LayerNorm):
    """An affine nn.LayerNorm over the last dimension on the kernels above, with an optional residual:
    norm(x, residual) is LayerNorm(x + residual). `SpartonLayerNorm.of(layer_norm)` shares an existing
    module's parameters (names and state_dict unchanged) and keeps its hooks.

    Under autocast the inputs are cast to float32 and so is the output, as torch's layer_norm does;
    inputs of two dtypes are summed in the wider one, as torch's sum would be."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self._check_module(self)

    @staticmethod
    def _check_module(layer_norm: nn.LayerNorm) -> None:
        if len(layer_norm.normalized_shape) != 1 or layer_norm.weight is None:
            raise ValueError(f"SpartonLayerNorm needs an affine LayerNorm over one dimension, got {layer_norm}")
        if layer_norm.normalized_shape[0] > MAX_WIDTH:
            raise ValueError(f"SpartonLayerNorm takes rows up to {MAX_WIDTH}, got {layer_norm.normalized_shape[0]}")

    @classmethod
    def of(cls, layer_norm: nn.LayerNorm) -> "SpartonLayerNorm":
        cls._check_module(layer_norm)
        m = copy.copy(layer_norm)  # the same hooks and mode
        m.__class__ = cls
        m._parameters = dict(m._parameters)  # and parameters, until either module is given another one
        return m

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        dev = x.device.type
        if dev in ("cuda", "cpu") and torch.is_autocast_enabled(dev):
            x = x.float()
            residual = residual.float() if residual is not None else None
        if residual is not None and residual.dtype != x.dtype:
            dt = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(dt), residual.to(dt)
        weight, bias = self.weight, self.bias
        if weight.dtype not in (torch.float32, x.dtype):
            weight, bias = weight.to(x.dtype), bias.to(x.dtype) if bias is not None else None
        return layer_norm(x, weight, bias, self.eps, residual)
