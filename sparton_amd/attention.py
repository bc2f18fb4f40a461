"""Attention of a backbone layer, forward and backward, on hand-written HIP kernels.

    s_ij = scale q_i . k_j;  p_i = softmax of s_i over the keys that row i may look at;  o_i = sum_j p_ij v_j

The reference leaves its backbones' attention to torch (training/model.py:88-139). Here one MFMA
kernel runs the forward with running row statistics (no [Sq, Sk] matrix in memory), and two the
backward, which recomputes the probabilities: one for dq, one for dk and dv, without atomics, so
every result is bitwise reproducible. A padded batch costs what its keys cost: 64 keys without a set
mask value are skipped. A few query rows against many keys (one new token, a long cache) are split
over the keys and joined.

    sparton::attention_fwd(q, k, v, key_mask?, causal, scale) -> (out, lse [B, Hq, Sq] fp32)
    sparton::attention_bwd(d_out, q, k, v, key_mask?, out, lse, causal, scale) -> (dq, dk, dv)

Device tensors only, like the head.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _eager, _lib

MAX_HEAD_DIM = 128
_FLOAT_DTYPES = tuple(_lib.DTYPE_CODE)
# A float mask is refused: added to the scores (0 keeps a key) and multiplied into them (0 drops it)
# are both in use, and mean the opposite of each other.
KEY_MASK_DTYPES = (torch.bool, torch.uint8, torch.int32, torch.int64)


def _check(q: Tensor, k: Tensor, v: Tensor, key_mask: Optional[Tensor], scale: float, op: str) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{op}: q must be [B,Hq,Sq,D] and k, v [B,Hk,Sk,D], got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, Hq, _Sq, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"{op}: k and v must both be [{B},Hk,Sk,{D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    Hk, Sk = k.shape[1], k.shape[2]
    if Hk == 0 and Hq > 0 or Hk > 0 and Hq % Hk != 0:
        raise ValueError(f"{op}: {Hq} query heads cannot share {Hk} key heads evenly")
    if not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"{op}: head size {D} must be between 1 and {MAX_HEAD_DIM}")
    if q.dtype not in _FLOAT_DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{op}: q, k and v must share one float dtype, got {q.dtype}/{k.dtype}/{v.dtype}")
    if key_mask is not None:
        if tuple(key_mask.shape) != (B, Sk):
            raise ValueError(f"{op}: key_mask must be [B,Sk]=[{B},{Sk}], got {tuple(key_mask.shape)}")
        if key_mask.dtype not in KEY_MASK_DTYPES:
            raise TypeError(f"{op}: key_mask must be bool or integer (nonzero: the key takes part), got "
                            f"{key_mask.dtype}")
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"{op}: scale must be positive and finite, got {scale}")
    for t in (k, v, key_mask):
        if t is not None and t.device != q.device:
            raise ValueError(f"{op}: all tensors must be on {q.device}, got {t.device}")


def _require_device(t: Tensor, op: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {t.device})")


@torch.library.custom_op("sparton::attention_fwd", mutates_args=())
def attention_fwd(q: Tensor, k: Tensor, v: Tensor, key_mask: Optional[Tensor], causal: bool,
                  scale: float) -> Tuple[Tensor, Tensor]:
    """(out [B,Hq,Sq,D], laid out [B,Sq,Hq,D]; lse [B,Hq,Sq] fp32, base-2 log of each row's sum of
    exponentials, which the backward uses)."""
    op = "sparton::attention_fwd"
    _check(q, k, v, key_mask, scale, op)
    _require_device(q, op)
    out, lse = _eager.load().attention_fwd(q, k, v, key_mask, causal, scale)
    return (out if out.shape[3] * out.element_size() % 16 == 0 else out.clone()), lse


def _like(t: Tensor) -> Tensor:
    B, H, S, D = t.shape
    return t.new_empty((B, S, H, D)).transpose(1, 2)


@attention_fwd.register_fake
def _(q, k, v, key_mask, causal, scale):
    return _like(q), q.new_empty(q.shape[:3], dtype=torch.float32)


@torch.library.custom_op("sparton::attention_bwd", mutates_args=())
def attention_bwd(d_out: Tensor, q: Tensor, k: Tensor, v: Tensor, key_mask: Optional[Tensor], out: Tensor,
                  lse: Tensor, causal: bool, scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) in the inputs' dtype, each rounded once from its fp32 sum."""
    op = "sparton::attention_bwd"
    _check(q, k, v, key_mask, scale, op)
    _require_device(q, op)
    if d_out.shape != q.shape or out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"{op}: d_out and out must be {tuple(q.shape)}, out in {q.dtype}, got "
                         f"{tuple(d_out.shape)} and {tuple(out.shape)} {out.dtype}")
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError(f"{op}: lse must be contiguous float32 {tuple(q.shape[:3])}, got {lse.dtype} "
                         f"{tuple(lse.shape)}")
    for t in (d_out, out, lse):
        if t.device != q.device:
            raise ValueError(f"{op}: all tensors must be on {q.device}, got {t.device}")
    grads = _eager.load().attention_bwd(d_out, q, k, v, key_mask, out, lse, causal, scale)
    return tuple(g if g.shape[3] * g.element_size() % 16 == 0 else g.clone() for g in grads)


@attention_bwd.register_fake
def _(d_out, q, k, v, key_mask, out, lse, causal, scale):
    return _like(q), _like(k), _like(v)


def _setup_context(ctx, inputs, output):
    q, k, v, key_mask, causal, scale = inputs
    out, lse = output
    ctx.mark_non_differentiable(lse)  # kept for the backward only
    ctx.set_materialize_grads(False)
    ctx.causal, ctx.scale = causal, scale
    ctx.save_for_backward(q, k, v, key_mask, out, lse)


def _backward(ctx, d_out, _d_lse):
    q, k, v, key_mask, out, lse = ctx.saved_tensors
    if d_out is None:  # out did not reach the loss
        return None, None, None, None, None, None
    dq, dk, dv = torch.ops.sparton.attention_bwd(d_out, q, k, v, key_mask, out, lse, ctx.causal, ctx.scale)
    return dq, dk, dv, None, None, None


attention_fwd.register_autograd(_backward, setup_context=_setup_context)


def attention(q: Tensor, k: Tensor, v: Tensor, key_mask: Optional[Tensor] = None, *, causal: bool = False,
              scale: Optional[float] = None) -> Tensor:
    """softmax(scale q k^T) v over the keys that take part.

    q [B,Hq,Sq,D], k and v [B,Hk,Sk,D] with Hq a multiple of Hk (query head h reads key head
    h / (Hq / Hk)), D <= 128, one float dtype; strided views are read as they are where rows start on
    16 bytes. key_mask [B,Sk], bool or integer as a tokenizer gives it: nonzero takes part. causal: row
    i sees the keys j <= i + Sk - Sq. scale defaults to D ** -0.5. Returns [B,Hq,Sq,D], laid out
    [B,Sq,Hq,D] in memory. A row that sees no key gives zeros, and gives and takes no gradient. Keys whose
    mask is zero may hold anything; what causal alone hides is multiplied by 0, so NaN and infinities
    there can reach the rows before it, as in torch's products.
    Under autocast the inputs are cast to its dtype, as torch's attention does."""
    dev = q.device.type
    if dev in ("cuda", "cpu") and torch.is_autocast_enabled(dev):
        dt = torch.get_autocast_dtype(dev)
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if scale is None:  # of a shape that is refused below, any
        scale = float(q.shape[-1]) ** -0.5 if q.dim() > 0 and q.shape[-1] > 0 else 1.0
    scale = float(scale)
    if torch.compiler.is_compiling() or not q.is_cuda:  # the registered op: fake + autograd
        return torch.ops.sparton.attention_fwd(q, k, v, key_mask, causal, scale)[0]
    _check(q, k, v, key_mask, scale, "attention")
    return _eager.load().attention(q, k, v, key_mask, causal, scale)
