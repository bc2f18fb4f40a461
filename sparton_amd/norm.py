"""LayerNorm and root-mean-square norm of a backbone's rows, with the residual sum in front, on hand-written HIP
kernels.

    y = LayerNorm(x + residual) * weight + bias        per row over the last dimension D

Every encoder layer of a BERT-like backbone has it twice (the reference runs torch's,
training/model.py:88-139); the transform before the head has the same norm behind its gelu
(transform.py). One pass reads x and residual and writes y; the backward reads dy, x and residual and
writes one gradient, which serves both, and the column sums for weight and bias, deterministically.
The residual sum is formed in fp32 and not rounded, so nothing of it is stored.

    sparton::layer_norm_fwd(x, residual?, weight, bias?, eps) -> (y, mean, rstd)
    sparton::layer_norm_bwd(dy, x, residual?, weight, has_bias, mean, rstd) -> (dx, d_weight, d_bias)

The root-mean-square norm of decoder backbones has the sum as an output too (the next layer's residual), and
its rows in e4m3 with a scale each where a product in 8 bits reads them:

    h = x + residual;   y = h / sqrt(mean(h^2) + eps) * weight

    sparton::rms_norm_fwd(x, residual?, weight, eps) -> (y, h, rstd)      h is empty without a residual
    sparton::rms_norm_bwd(dy, dh?, h, weight, rstd) -> (dx, d_weight)
    sparton::rms_norm_8bit(x, residual?, weight, eps) -> (y in e4m3, scale, h)

Device tensors only, like the head.
"""
from __future__ import annotations

import copy
import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor, nn

from . import _eager, _lib
from ._look import PLAIN, computes, holds_only

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


# ---- the root-mean-square norm ----------------------------------------------------------------

@torch.library.custom_op("sparton::rms_norm_fwd", mutates_args=())
def rms_norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(y and the rounded sum h in x's dtype, rstd per row in fp32 for the backward); h is empty without a residual."""
    _eager.refuse_forward_mode("sparton::rms_norm_fwd", x, residual, weight)
    _check(x, residual, weight, None, eps, "sparton::rms_norm_fwd")
    return _eager.load().rms_norm_fwd(x, residual, weight, eps)


@rms_norm_fwd.register_fake
def _(x, residual, weight, eps):
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    return x.new_empty(x.shape), x.new_empty(x.shape if residual is not None else (0,)), x.new_empty(
        (rows,), dtype=torch.float32)


@torch.library.custom_op("sparton::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(dy: Tensor, dh: Optional[Tensor], h: Tensor, weight: Tensor, rstd: Tensor) -> Tuple[Tensor, Tensor]:
    """(the gradient of x and of the residual alike, in h's dtype; d_weight in the weight's). h: the forward's, or x
    where there was no residual; dh: its gradient."""
    op = "sparton::rms_norm_bwd"
    D = _check(h, None, weight, None, 0.0, op)
    for t in (dy, dh):
        if t is not None and (t.shape != h.shape or t.device != h.device):
            raise ValueError(f"{op}: dy and dh must be {tuple(h.shape)} on {h.device}, got {tuple(t.shape)} on {t.device}")
    if tuple(rstd.shape) != (h.numel() // D,) or rstd.dtype != torch.float32 or rstd.device != h.device \
            or not rstd.is_contiguous():
        raise ValueError(f"{op}: rstd must be contiguous float32 [{h.numel() // D}] on {h.device}")
    return _eager.load().rms_norm_bwd(dy, dh.to(h.dtype) if dh is not None else None, h, weight, rstd)


@rms_norm_bwd.register_fake
def _(dy, dh, h, weight, rstd):
    return h.new_empty(h.shape), weight.new_empty(weight.shape)


def _rms_setup_context(ctx, inputs, output):
    x, residual, weight, _eps = inputs
    _y, h, rstd = output
    ctx.mark_non_differentiable(rstd)
    ctx.set_materialize_grads(False)
    ctx.has_residual = residual is not None
    ctx.save_for_backward(h if residual is not None else x, weight, rstd)


def _rms_backward(ctx, dy, dh, _drstd):
    h, weight, rstd = ctx.saved_tensors
    dh = dh if ctx.has_residual else None
    if dy is None:  # y did not reach the loss
        return dh, dh, None, None
    dx, dw = torch.ops.sparton.rms_norm_bwd(dy, dh, h, weight, rstd)
    return dx, (dx if ctx.has_residual else None), dw, None


rms_norm_fwd.register_autograd(_rms_backward, setup_context=_rms_setup_context)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6,
             residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (up to 16384), in x's dtype; weight is float32 (a
    master) or of x's dtype, and gets its gradient in it. With a residual: (the norm of h = x + residual, h); the norm
    reads the sum before it is rounded."""
    eps = float(eps)
    if torch.compiler.is_compiling() or not x.is_cuda:  # the registered op: fake + autograd
        y, h, _ = torch.ops.sparton.rms_norm_fwd(x, residual, weight, eps)
        return y if residual is None else (y, h)
    _check(x, residual, weight, None, eps, "rms_norm")
    if residual is None:
        return _eager.load().rms_norm(x, weight, eps)
    return _eager.load().rms_norm_add(x, residual, weight, eps)


@torch.library.custom_op("sparton::rms_norm_8bit", mutates_args=())
def _rms_norm_8bit(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(y in e4m3, a scale a row, h), without a gradient; h is empty without a residual."""
    _eager.refuse_forward_mode("sparton::rms_norm_8bit", x, residual, weight)
    _check(x, residual, weight, None, eps, "sparton::rms_norm_8bit")
    return _eager.load().rms_norm_8bit(x, residual, weight, eps)


@_rms_norm_8bit.register_fake
def _(x, residual, weight, eps):
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(x.shape[:-1], dtype=torch.float32),
            x.new_empty(x.shape if residual is not None else (0,)))


def rms_norm_8bit(x: Tensor, weight: Tensor, eps: float = 1e-6, residual: Optional[Tensor] = None):
    """(y8, scale), with a residual (y8, scale, h): the rows of rms_norm in e4m3, y ~ y8 * scale[..., None], as
    feed_forward.gated_linear_8bit reads them. scale (fp32) puts a row's largest magnitude at 448. For inference:
    inputs that ask for a gradient are refused."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm_8bit has no gradient: call it under torch.no_grad()")
    eps = float(eps)
    if torch.compiler.is_compiling() or not x.is_cuda:
        y, scale, h = torch.ops.sparton.rms_norm_8bit(x, residual, weight, eps)
    else:
        _check(x, residual, weight, None, eps, "rms_norm_8bit")
        y, scale, h = _eager.load().rms_norm_8bit(x, residual, weight, eps)
    return (y, scale) if residual is None else (y, scale, h)


def _weight_and_eps(m: nn.Module) -> Optional[Tuple[Tensor, float]]:
    weight, eps = getattr(m, "weight", None), getattr(m, "variance_epsilon", getattr(m, "eps", None))
    return (weight, eps) if isinstance(weight, Tensor) and weight.dim() == 1 and isinstance(eps, float) else None


def computes_rms_norm(m: nn.Module) -> bool:
    """weight * x / sqrt(mean(x^2) + eps), seen on a copy with another weight."""
    found = _weight_and_eps(m)
    if found is None or "forward" in m.__dict__:
        return False
    (weight, eps), g = found, torch.Generator("cpu").manual_seed(0)
    n = weight.shape[0]
    x, w = torch.randn(3, n, generator=g, **PLAIN), torch.rand(n, generator=g, **PLAIN) + 0.5
    probe = copy.copy(m)
    probe._parameters = {"weight": nn.Parameter(w)}
    return computes(probe, {}, x, lambda: w * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps))


class SpartonRMSNorm(nn.Module):
    """A root-mean-square norm over the last dimension on the kernels above: norm(x), or norm(x, residual) for
    (norm of the sum, sum). `SpartonRMSNorm.of(module)` shares an existing module's weight (name and state_dict
    unchanged) and keeps its hooks; a module that computes something else (seen on a small copy, on the CPU) is refused.

    A weight wider than x (float32 masters) stays as it is and the result is x's dtype; under autocast too, as the
    inputs are rows of the autocast dtype there."""

    def __init__(self, width: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        if not 1 <= width <= MAX_WIDTH:
            raise ValueError(f"SpartonRMSNorm takes rows up to {MAX_WIDTH}, got {width}")
        self.weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.eps = float(eps)

    @classmethod
    def of(cls, module: nn.Module) -> "SpartonRMSNorm":
        found = _weight_and_eps(module)
        if found is None:
            raise ValueError(f"SpartonRMSNorm needs a weight over one dimension and an epsilon, got {module}")
        weight, eps = found
        ours = type(module).forward is cls.forward and "forward" not in module.__dict__
        if not ours and not holds_only(module) and not computes_rms_norm(module):
            raise ValueError(f"SpartonRMSNorm computes weight * x / sqrt(mean(x^2) + eps), which {module} does not")
        if not 1 <= weight.shape[0] <= MAX_WIDTH:
            raise ValueError(f"SpartonRMSNorm takes rows up to {MAX_WIDTH}, got {weight.shape[0]}")
        m = copy.copy(module)  # the same hooks and mode
        m.__class__ = cls
        m._parameters = dict(m._parameters)  # and parameters, until either module is given another one
        m.eps = float(eps)
        return m

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}"

    def forward(self, x: Tensor, residual: Optional[Tensor] = None):
        weight = self.weight
        if residual is not None and residual.dtype != x.dtype:
            dt = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(dt), residual.to(dt)
        if weight.dtype not in (torch.float32, x.dtype):
            weight = weight.to(x.dtype)
        return rms_norm(x, weight, self.eps, residual)
