"""Gated feed-forward product of a backbone layer, forward and backward, on hand-written HIP kernels.

    g = x Wg' + bg;   u = x Wu' + bu;   h = act(g) u

the first half of a gated block, whose second is a plain product. (The reference's backbones run
torch's, training/model.py:88-139.) Both projections, the activation and the product are one kernel:
g and u meet in registers. The backward has one product for x and one for both weights, and keeps g and u
in fp32 in between. A few rows (new tokens) take a kernel that streams the weights once; rows and weights
in e4m3 with a scale a row take the matrix cores' 8-bit rate.

    sparton::gated_infer(x, w_gate, w_up, b_gate?, b_up?, activation) -> h
    sparton::gated_fwd(x, w_gate, w_up, b_gate?, b_up?, activation) -> (h, gate, up)
    sparton::gated_bwd(dh, x, w_gate, w_up, gate, up, activation, has_b_gate, has_b_up, need_x=True, need_w=True)
        -> (dx, d_w_gate, d_w_up, d_b_gate, d_b_up)
    sparton::gated_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, activation, out_dtype) -> h

Device tensors only, like the head.
"""
from __future__ import annotations

import copy
from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import _eager, _lib
from ._look import PLAIN, computes, holds_only

ACTIVATIONS = tuple(_lib.ACTIVATION_CODE)
MAX_WIDTH = 1 << 20
E4M3_MAX = 448.0
_FLOAT_DTYPES = tuple(_lib.DTYPE_CODE)
_E4M3 = torch.float8_e4m3fn


def _code(activation: str, op: str) -> int:
    if activation not in _lib.ACTIVATION_CODE:
        raise ValueError(f"{op}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    return _lib.ACTIVATION_CODE[activation]


def _check_shapes(x: Tensor, w_gate: Tensor, w_up: Tensor, op: str) -> Tuple[int, int]:
    D = x.shape[-1] if x.dim() > 0 else 0
    if not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"{op}: x must be [..., D] with D between 1 and {MAX_WIDTH}, got {tuple(x.shape)}")
    for w in (w_gate, w_up):
        if w.dim() != 2 or w.shape[1] != D or w.shape != w_gate.shape or w.shape[0] > MAX_WIDTH:
            raise ValueError(f"{op}: w_gate and w_up must both be [F, {D}] with F up to {MAX_WIDTH}, got "
                             f"{tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    if x.numel() // D >= 2 ** 31:
        raise ValueError(f"{op}: {x.numel() // D} rows are too many")
    return D, w_gate.shape[0]


def _require_device(x: Tensor, others, op: str) -> None:
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"{op}: all tensors must be on {x.device}, got {t.device}")
    if not x.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {x.device})")


def _check(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor], b_up: Optional[Tensor], op: str) -> None:
    _D, width = _check_shapes(x, w_gate, w_up, op)
    for t in (w_gate, w_up, b_gate, b_up):
        if t is not None and (x.dtype not in _FLOAT_DTYPES or t.dtype != x.dtype):
            raise TypeError(f"{op}: x, weights and biases must share one float dtype, got {x.dtype} and {t.dtype}")
    for b in (b_gate, b_up):
        if b is not None and tuple(b.shape) != (width,):
            raise ValueError(f"{op}: biases must be [{width}], got {tuple(b.shape)}")
    _require_device(x, (w_gate, w_up, b_gate, b_up), op)


@torch.library.custom_op("sparton::gated_fwd", mutates_args=())
def gated_fwd(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor], b_up: Optional[Tensor],
              activation: str) -> Tuple[Tensor, Tensor, Tensor]:
    """(h in x's dtype; g and u, fp32 [rows, F], for the backward)."""
    op = "sparton::gated_fwd"
    code = _code(activation, op)
    _eager.refuse_forward_mode(op, x, w_gate, w_up, b_gate, b_up)
    _check(x, w_gate, w_up, b_gate, b_up, op)
    return _eager.load().gated_fwd(x, w_gate, w_up, b_gate, b_up, code)


@gated_fwd.register_fake
def _(x, w_gate, w_up, b_gate, b_up, activation):
    width = w_gate.shape[0]
    saved = x.new_empty((x.numel() // x.shape[-1], width), dtype=torch.float32)
    return x.new_empty((*x.shape[:-1], width)), saved, torch.empty_like(saved)


@torch.library.custom_op("sparton::gated_infer", mutates_args=())
def gated_infer(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor], b_up: Optional[Tensor],
                activation: str) -> Tensor:
    """h alone, without a gradient: g and u are not written."""
    op = "sparton::gated_infer"
    code = _code(activation, op)
    _eager.refuse_forward_mode(op, x, w_gate, w_up, b_gate, b_up)
    _check(x, w_gate, w_up, b_gate, b_up, op)
    return _eager.load().gated(x, w_gate, w_up, b_gate, b_up, code)


@gated_infer.register_fake
def _(x, w_gate, w_up, b_gate, b_up, activation):
    return x.new_empty((*x.shape[:-1], w_gate.shape[0]))


@torch.library.custom_op("sparton::gated_bwd", mutates_args=())
def gated_bwd(dh: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, gate: Tensor, up: Tensor, activation: str,
              has_b_gate: bool, has_b_up: bool, need_x: bool = True,
              need_w: bool = True) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(dx, d_w_gate, d_w_up, d_b_gate, d_b_up) in x's dtype; those that are not asked for are empty, as the biases' are
    where there are none."""
    op = "sparton::gated_bwd"
    code = _code(activation, op)
    _check(x, w_gate, w_up, None, None, op)
    D, width = x.shape[-1], w_gate.shape[0]
    if tuple(dh.shape) != (*x.shape[:-1], width):
        raise ValueError(f"{op}: dh must be {(*x.shape[:-1], width)}, got {tuple(dh.shape)}")
    for t in (gate, up):
        if tuple(t.shape) != (x.numel() // D, width) or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{op}: gate and up must be contiguous float32 [{x.numel() // D}, {width}]")
    _require_device(x, (dh, gate, up), op)
    return _eager.load().gated_bwd(dh, x, w_gate, w_up, gate, up, code, has_b_gate, has_b_up, need_x, need_w)


@gated_bwd.register_fake
def _(dh, x, w_gate, w_up, gate, up, activation, has_b_gate, has_b_up, need_x=True, need_w=True):
    width = w_gate.shape[0]
    return (x.new_empty(x.shape if need_x else (0,)), *(w.new_empty(w.shape if need_w else (0,)) for w in (w_gate, w_up)),
            x.new_empty((width if has_b_gate else 0,)), x.new_empty((width if has_b_up else 0,)))


def _setup_context(ctx, inputs, output):
    x, w_gate, w_up, b_gate, b_up, activation = inputs
    _h, gate, up = output
    ctx.mark_non_differentiable(gate, up)  # kept for the backward only
    ctx.set_materialize_grads(False)
    ctx.activation, ctx.has_b_gate, ctx.has_b_up = activation, b_gate is not None, b_up is not None
    ctx.save_for_backward(x, w_gate, w_up, gate, up)


def _backward(ctx, dh, _d_gate, _d_up):
    if dh is None:  # h did not reach the loss
        return (None,) * 6
    x, wg, wu, bg, bu = ctx.needs_input_grad[:5]
    bg, bu = bg and ctx.has_b_gate, bu and ctx.has_b_up
    grads = torch.ops.sparton.gated_bwd(dh, *ctx.saved_tensors, ctx.activation, bg, bu, x, wg or wu)
    return (*(g if need else None for g, need in zip(grads, (x, wg, wu, bg, bu))), None)


gated_fwd.register_autograd(_backward, setup_context=_setup_context)


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor] = None, b_up: Optional[Tensor] = None,
                 activation: str = "silu") -> Tensor:
    """act(x w_gate' + b_gate) * (x w_up' + b_up): [..., F] from x [..., D] and weights [F, D] (as nn.Linear has
    them), one float dtype. activation: "silu", "gelu" (erf), "gelu_tanh" or "relu". A width that is not a multiple
    of 16 bytes costs padded copies of x and the weights. Under autocast the inputs are cast to its dtype, as
    torch's linear does."""
    code = _code(activation, "gated_linear")
    dev = x.device.type
    if dev in ("cuda", "cpu") and torch.is_autocast_enabled(dev):
        dt = torch.get_autocast_dtype(dev)
        x, w_gate, w_up = x.to(dt), w_gate.to(dt), w_up.to(dt)
        b_gate, b_up = (b.to(dt) if b is not None else None for b in (b_gate, b_up))
    if torch.compiler.is_compiling() or not x.is_cuda:  # the registered op: fake + autograd
        _check_shapes(x, w_gate, w_up, "gated_linear")
        if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, b_gate, b_up))):
            return torch.ops.sparton.gated_infer(x, w_gate, w_up, b_gate, b_up, activation)
        return torch.ops.sparton.gated_fwd(x, w_gate, w_up, b_gate, b_up, activation)[0]
    _check(x, w_gate, w_up, b_gate, b_up, "gated_linear")
    return _eager.load().gated(x, w_gate, w_up, b_gate, b_up, code)


def _check_8bit(x: Tensor, x_scale: Tensor, w_gate: Tensor, gate_scale: Tensor, w_up: Tensor, up_scale: Tensor,
                out_dtype: torch.dtype, op: str) -> None:
    _D, width = _check_shapes(x, w_gate, w_up, op)
    for t in (x, w_gate, w_up):
        if t.dtype != _E4M3:
            raise TypeError(f"{op}: x and weights must be float8_e4m3fn, got {t.dtype}")
    if out_dtype not in _FLOAT_DTYPES:
        raise TypeError(f"{op}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    for t, shape in ((x_scale, tuple(x.shape[:-1])), (gate_scale, (width,)), (up_scale, (width,))):
        if tuple(t.shape) != shape or t.dtype != torch.float32:
            raise ValueError(f"{op}: a scale a row is float32 {shape}, got {t.dtype} {tuple(t.shape)}")
    _require_device(x, (x_scale, w_gate, gate_scale, w_up, up_scale), op)


@torch.library.custom_op("sparton::gated_8bit", mutates_args=())
def gated_8bit(x: Tensor, x_scale: Tensor, w_gate: Tensor, gate_scale: Tensor, w_up: Tensor, up_scale: Tensor,
               activation: str, out_dtype: torch.dtype) -> Tensor:
    """gated_linear_8bit, without a gradient."""
    op = "sparton::gated_8bit"
    code = _code(activation, op)
    _eager.refuse_forward_mode(op, x, x_scale, w_gate, gate_scale, w_up, up_scale)
    _check_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, out_dtype, op)
    return _eager.load().gated_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, code, out_dtype)


@gated_8bit.register_fake
def _(x, x_scale, w_gate, gate_scale, w_up, up_scale, activation, out_dtype):
    return x.new_empty((*x.shape[:-1], w_gate.shape[0]), dtype=out_dtype)


def gated_linear_8bit(x: Tensor, x_scale: Tensor, w_gate: Tensor, gate_scale: Tensor, w_up: Tensor, up_scale: Tensor,
                      activation: str = "silu", out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """act(g) * u of e4m3 rows: g = (x w_gate') x_scale gate_scale, u likewise, summed in fp32. x [..., D] and x_scale
    [...] as rms_norm_8bit gives them, weights [F, D] and scales [F] as quantize_rows does. For inference: inputs that
    ask for a gradient are refused."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, x_scale, w_gate, gate_scale, w_up, up_scale)):
        raise ValueError("gated_linear_8bit has no gradient: call it under torch.no_grad()")
    if torch.compiler.is_compiling() or not x.is_cuda:
        return torch.ops.sparton.gated_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, activation, out_dtype)
    code = _code(activation, "gated_linear_8bit")
    _check_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, out_dtype, "gated_linear_8bit")
    return _eager.load().gated_8bit(x, x_scale, w_gate, gate_scale, w_up, up_scale, code, out_dtype)


def quantize_rows(t: Tensor) -> Tuple[Tensor, Tensor]:
    """(e4m3 rows, fp32 scale of each): t ~ rows * scale[..., None], the largest magnitude of a row at 448. To lay out
    a model's weights once; plain torch operations."""
    t = t.detach().float()
    scale = (t.abs().amax(-1) / E4M3_MAX).clamp_min(2.0 ** -126)
    return (t / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(_E4M3), scale


def activation_name(fn) -> Optional[str]:
    """The kernels' name of a module's activation, or None if they do not compute it. A subclass may compute anything."""
    cls = type(fn)
    theirs = cls.__name__ if cls.__module__ == "transformers.activations" else None
    if cls is nn.SiLU or fn is F.silu or theirs == "SiLUActivation":
        return "silu"
    if cls is nn.GELU:
        return "gelu_tanh" if fn.approximate == "tanh" else "gelu"
    if fn is F.gelu or theirs == "GELUActivation":
        return "gelu"
    if theirs == "GELUTanh":
        return "gelu_tanh"
    if cls is nn.ReLU or fn is F.relu:
        return "relu"
    return None


def hooked(m: nn.Module) -> bool:
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


def untouched(m: nn.Module) -> bool:
    """Whether a call of m is its class's forward and nothing else."""
    return "forward" not in m.__dict__ and not hooked(m)


def plain_linears(*modules: nn.Module) -> bool:
    """Whether these do no more than their weights and biases say, which is all that the kernel reads of them: not so
    for an adapter around one, another forward, or hooks."""
    return all(type(m) is nn.Linear and untouched(m) for m in modules)


def plain_activation(fn) -> Optional[str]:
    """activation_name of what the kernel may compute in fn's place: None for a module with hooks or a forward of its
    own, which it would pass by."""
    return activation_name(fn) if not isinstance(fn, nn.Module) or untouched(fn) else None


_ACTIVATE = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}


class _Bare(nn.Module):
    """What an activation's class computes: its hooks are not called for a look at the block."""

    def __init__(self, fn):
        super().__init__()
        self.fn = [fn]  # not a submodule

    def forward(self, x):
        fn = self.fn[0]
        return type(fn).forward(fn, x) if isinstance(fn, nn.Module) else fn(x)


def computes_gated_block(m: nn.Module) -> bool:
    """down_proj(act_fn(gate_proj(x)) * up_proj(x)) with an activation of the kernels, and nothing else in it; the
    projections may be anything."""
    if set(m._modules) != {"gate_proj", "up_proj", "down_proj", "act_fn"} or m._parameters or m._buffers:
        return False
    name = activation_name(m.act_fn)
    if name is None:
        return False
    with torch.random.fork_rng(devices=[]):  # their first weights are not the caller's random numbers
        small = [nn.Linear(*n, **PLAIN) for n in ((4, 6), (4, 6), (6, 4))]
    x = torch.linspace(-2, 2, 12, **PLAIN).view(3, 4)
    return computes(m, dict(zip(("gate_proj", "up_proj", "down_proj"), small), act_fn=_Bare(m.act_fn)), x,
                    lambda: small[2](_ACTIVATE[name](small[0](x)) * small[1](x)))


class SpartonGatedMLP(nn.Module):
    """A gated block, down_proj(act(gate_proj(x)) * up_proj(x)), its first half on the kernels above.
    `SpartonGatedMLP.of(block)` shares the three nn.Linear of an existing block (names and state_dict unchanged) and
    keeps its hooks; a block that computes something else (seen on a small copy, on the CPU) is refused.
    Projections that are more than plain nn.Linear (adapters, hooks) run as they are, then the activation."""

    def __init__(self, gate_proj: nn.Linear, up_proj: nn.Linear, down_proj: nn.Linear, activation: str = "silu"):
        super().__init__()
        _code(activation, "SpartonGatedMLP")
        self._check_shapes(gate_proj, up_proj, down_proj)
        self.gate_proj, self.up_proj, self.down_proj, self.activation = gate_proj, up_proj, down_proj, activation

    @staticmethod
    def _check_shapes(gate_proj: nn.Module, up_proj: nn.Module, down_proj: nn.Module) -> None:
        if gate_proj.weight.shape != up_proj.weight.shape or down_proj.in_features != gate_proj.out_features:
            raise ValueError("SpartonGatedMLP needs gate_proj and up_proj of one shape and down_proj behind them, got "
                             f"{gate_proj}, {up_proj} and {down_proj}")

    @classmethod
    def of(cls, block: nn.Module) -> "SpartonGatedMLP":
        name = plain_activation(getattr(block, "act_fn", None))
        if name is None:
            raise ValueError(f"SpartonGatedMLP computes {', '.join(ACTIVATIONS)}, without hooks; this block's activation "
                             f"is {getattr(block, 'act_fn', None)!r}")
        if "forward" in block.__dict__ or not (holds_only(block) or computes_gated_block(block)):
            raise ValueError("SpartonGatedMLP computes down_proj(act_fn(gate_proj(x)) * up_proj(x)), which "
                             f"{block} does not")
        cls._check_shapes(block.gate_proj, block.up_proj, block.down_proj)
        m = copy.copy(block)  # the same hooks and mode
        m.__class__ = cls
        m._modules = {n: c for n, c in block._modules.items() if n in ("gate_proj", "up_proj", "down_proj")}
        m.activation = name
        return m

    def forward(self, x: Tensor) -> Tensor:
        gate, up = self.gate_proj, self.up_proj
        if not plain_linears(gate, up):
            return self.down_proj(_ACTIVATE[self.activation](gate(x)) * up(x))
        return self.down_proj(gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, self.activation))
