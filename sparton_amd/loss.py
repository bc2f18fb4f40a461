"""The SPLADE training loss on SpartonHead's reps, fused on the GPU.

Reference: training/train.py -- info_nce_loss (:73-77), l1_regularization (:80-82),
flops_regularization (:85-87), get_reg_weight (:90-94) and their combination in
compute_loss (:164-197):

    total = CE(q, d, T) + w_l1 (L1(q) + L1(d)) + w_flops (FL(q) + FL(d))

The reference evaluates these as a dozen small torch ops over the [B, V] reps (the score
GEMM, softmax/cross entropy, abs, two sums per regulariser, squares, means). Here one HIP
pass reads q and d once and produces the partial scores and sums per 64-column vocabulary
slice, a fixed-order reduction and a one-workgroup finish give the six scalars, and one HIP
pass writes both gradients. Everything accumulates in fp32 (the reference's score GEMM
runs in the reps dtype), deterministically. Device tensors only, like the head.

    sparton::splade_loss_fwd(q, d?, temperature, w_ce, w_l1, w_flops)
        -> (out[6] fp32 = (total, CE, L1 q, L1 d, FLOPS q, FLOPS d), probs [Bq, Bd] fp32)
    sparton::splade_loss_bwd(grad_out[6], q, d?, probs, w_ce, w_l1, w_flops) -> (dq, dd)

Batches of up to 64 rows on each side take the slice-staged kernels above. Larger batches
take GEMM-shaped HIP kernels on the matrix cores (the bf16/fp16 MFMA: products of 16-bit
reps are exact in fp32, fp32 values are sums of bf16 parts that hold all their bits; P against bf16 reps, whose
gradients are rounded to bf16, takes two parts, within 2^-17 of it): a
split-vocabulary score GEMM with a fixed-order sum of its partials, per-slice row and column
statistics, a row softmax, and a backward that recomputes each vocabulary slice's column sums
and forms both gradients tile by tile (sparton_loss.hip). Limits: 1 <= Bq <= Bd when documents are given (the labels
arange(Bq) index d's rows); the C ABI reports sizes past its int offsets as unsupported.

preference_loss is the objective of a second training stage, on pairs that a frozen reference model
scores too (the reference has none; its losses above see only positives and in-batch negatives):

    sparton::preference_fwd(q, pos, neg, ref_margin?, temperature, beta, smoothing)
        -> (loss, margin [B] fp32, coef [B] fp32)
    sparton::preference_bwd(grad, q, pos, neg, coef) -> (dq, dpos, dneg)
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import _eager, _lib

SMALL_MAX_ROWS = 64    # rows per side taken by the slice-staged kernels (the library's own rule); larger batches take the GEMM kernels
_FLOAT_DTYPES = tuple(_lib.DTYPE_CODE)


class SpladeLossOutput(NamedTuple):
    """The scalars compute_loss (train.py:178-197) forms and logs: total is what it
    back-propagates, the others are the terms it adds up (each differentiable too)."""
    total: Tensor
    contrastive: Tensor
    l1_q: Tensor
    l1_d: Tensor
    flops_q: Tensor
    flops_d: Tensor


def _check(q: Tensor, d: Optional[Tensor], op: str) -> Tuple[int, int, int]:
    if not q.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {q.device})")
    if q.dim() != 2 or q.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"{op}: query reps must be a 2-D float tensor [B, V], got {q.dtype} {tuple(q.shape)}")
    Bq, V = q.shape
    Bd = 0
    if d is not None:
        if d.dim() != 2 or d.dtype != q.dtype or d.shape[1] != V or d.device != q.device:
            raise ValueError(f"{op}: document reps must be [B, {V}] {q.dtype} on {q.device}, got "
                             f"{d.dtype} {tuple(d.shape)} on {d.device}")
        Bd = d.shape[0]
        if Bq > Bd:
            raise ValueError(f"{op}: {Bq} queries but {Bd} documents; the labels arange(Bq) "
                             "index the documents, so Bq <= Bd")
    if Bq < 1 or V < 1:
        raise ValueError(f"{op}: needs at least one query row and V >= 1, got Bq={Bq} V={V}")
    return Bq, Bd, V


def _fwd_impl(q: Tensor, d: Optional[Tensor], temperature: float, w_ce: float, w_l1: float,
              w_flops: float) -> Tuple[Tensor, Tensor]:
    op = "sparton::splade_loss_fwd"
    Bq, Bd, V = _check(q, d, op)
    if d is not None and not temperature > 0.0:
        raise ValueError(f"{op}: temperature must be > 0, got {temperature}")
    q = q.contiguous()
    d = d.contiguous() if d is not None else None
    out = torch.empty((6,), dtype=torch.float32, device=q.device)
    probs = torch.empty((Bq, Bd), dtype=torch.float32, device=q.device)
    L = _lib.load()
    nbytes = int(L.sparton_loss_workspace_bytes(Bq, Bd, V))
    ws = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        rc = L.sparton_loss_fwd(q.data_ptr(), d.data_ptr() if d is not None else None, Bq, Bd, V,
                                float(temperature), float(w_ce), float(w_l1), float(w_flops),
                                out.data_ptr(), probs.data_ptr() if Bd else None, ws.data_ptr(),
                                nbytes, _lib.DTYPE_CODE[q.dtype],
                                torch.cuda.current_stream(q.device).cuda_stream)
    _lib.check(rc, op)
    return out, probs


def _bwd_impl(grad_out: Tensor, q: Tensor, d: Optional[Tensor], probs: Tensor, w_ce: float,
              w_l1: float, w_flops: float) -> Tuple[Tensor, Tensor]:
    op = "sparton::splade_loss_bwd"
    Bq, Bd, V = _check(q, d, op)
    q = q.contiguous()
    d = d.contiguous() if d is not None else None
    g = grad_out.to(device=q.device, dtype=torch.float32).contiguous()
    dq = torch.empty_like(q)
    dd = torch.empty_like(d) if d is not None else q.new_empty((0, V))
    L = _lib.load()
    with torch.cuda.device(q.device):
        rc = L.sparton_loss_bwd(q.data_ptr(), d.data_ptr() if d is not None else None,
                                probs.data_ptr() if Bd else None, g.data_ptr(), Bq, Bd, V,
                                float(w_ce), float(w_l1), float(w_flops), dq.data_ptr(),
                                dd.data_ptr() if d is not None else None, _lib.DTYPE_CODE[q.dtype],
                                torch.cuda.current_stream(q.device).cuda_stream)
    _lib.check(rc, op)
    return dq, dd


@torch.library.custom_op("sparton::splade_loss_fwd", mutates_args=())
def splade_loss_fwd(q: Tensor, d: Optional[Tensor], temperature: float, w_ce: float, w_l1: float,
                    w_flops: float) -> Tuple[Tensor, Tensor]:
    """(out[6], probs): out = (total, CE, L1 q, L1 d, FLOPS q, FLOPS d) in fp32; probs =
    (softmax(S) - I) / (Bq T), which the backward uses."""
    return _fwd_impl(q, d, temperature, w_ce, w_l1, w_flops)


@splade_loss_fwd.register_fake
def _(q, d, temperature, w_ce, w_l1, w_flops):
    Bd = d.shape[0] if d is not None else 0
    return q.new_empty((6,), dtype=torch.float32), q.new_empty((q.shape[0], Bd), dtype=torch.float32)


@torch.library.custom_op("sparton::splade_loss_bwd", mutates_args=())
def splade_loss_bwd(grad_out: Tensor, q: Tensor, d: Optional[Tensor], probs: Tensor, w_ce: float,
                    w_l1: float, w_flops: float) -> Tuple[Tensor, Tensor]:
    """(dq, dd) in the reps dtype; dd is [0, V] when d is None."""
    return _bwd_impl(grad_out, q, d, probs, w_ce, w_l1, w_flops)


@splade_loss_bwd.register_fake
def _(grad_out, q, d, probs, w_ce, w_l1, w_flops):
    return torch.empty_like(q), (torch.empty_like(d) if d is not None else q.new_empty((0, q.shape[1])))


def _setup_context(ctx, inputs, output):
    q, d, temperature, w_ce, w_l1, w_flops = inputs
    _out, probs = output
    ctx.has_d = d is not None
    ctx.w = (w_ce, w_l1, w_flops)
    ctx.mark_non_differentiable(probs)  # kept for the backward only
    ctx.save_for_backward(q, d if d is not None else q.new_empty(0), probs)


def _backward(ctx, g_out, _g_probs):
    q, d, probs = ctx.saved_tensors
    if g_out is None:  # out did not reach the loss
        return None, None, None, None, None, None
    dq, dd = torch.ops.sparton.splade_loss_bwd(g_out, q, d if ctx.has_d else None, probs, *ctx.w)
    return dq, (dd if ctx.has_d else None), None, None, None, None


splade_loss_fwd.register_autograd(_backward, setup_context=_setup_context)


def _run(q: Tensor, d: Optional[Tensor], temperature: float, w_ce: float, w_l1: float,
         w_flops: float) -> Tuple[Tensor, ...]:
    """The six terms (total, CE, L1(q), L1(d), FL(q), FL(d)) as separate scalars."""
    if torch.compiler.is_compiling() or not q.is_cuda:
        out, _ = torch.ops.sparton.splade_loss_fwd(q, d, temperature, w_ce, w_l1, w_flops)
        return out.unbind(0)
    # eager: the C++ op (autograd in C++), the same implementation as the custom ops; its six
    # outputs are separate, so backpropagating one term materialises no gradients of the
    # others
    _check(q, d, "splade_loss")
    if d is not None and not temperature > 0.0:
        raise ValueError(f"splade_loss: temperature must be > 0, got {temperature}")
    return _eager.load().splade_loss(q, d, float(temperature), float(w_ce), float(w_l1), float(w_flops))


def splade_loss(query_reps: Tensor, doc_reps: Optional[Tensor], temperature: float = 1.0,
                lambda_l1: float = 0.0, lambda_flops: float = 0.0) -> SpladeLossOutput:
    """InfoNCE + weighted L1 and FLOPS regularisers of both sides in one fused pass
    (train.py:178-197 with the weights already warmed up, see get_reg_weight)."""
    return SpladeLossOutput(*_run(query_reps, doc_reps, temperature, 1.0, lambda_l1, lambda_flops))


def info_nce_loss(query_reps: Tensor, doc_reps: Tensor, temperature: float = 1.0) -> Tensor:
    """In-batch negatives contrastive loss (train.py:73-77)."""
    return _run(query_reps, doc_reps, temperature, 1.0, 0.0, 0.0)[0]


def l1_regularization(reps: Tensor) -> Tensor:
    """mean_b sum_v |reps| (train.py:80-82)."""
    return _run(reps, None, 1.0, 0.0, 1.0, 0.0)[0]


def flops_regularization(reps: Tensor) -> Tensor:
    """mean_v (sum_b reps)^2 (train.py:85-87)."""
    return _run(reps, None, 1.0, 0.0, 0.0, 1.0)[0]


def get_reg_weight(current_step: int, warmup_steps: int, target_lambda: float) -> float:
    """Linear warm-up from 0 to target_lambda (train.py:90-94)."""
    if warmup_steps <= 0:
        return target_lambda
    return target_lambda * min(1.0, current_step / warmup_steps)


def splade_training_loss(query_reps: Tensor, doc_reps: Tensor, step: int, temperature: float = 1.0,
                         lambda_l1: float = 1e-4, lambda_flops: float = 1e-4,
                         reg_warmup_steps: int = 10000) -> SpladeLossOutput:
    """compute_loss's loss (train.py:164-197) at a training step: the warmed-up weights, then
    splade_loss. Defaults are LSRTrainingArguments' (train.py:50-66)."""
    return splade_loss(query_reps, doc_reps, temperature,
                       get_reg_weight(step, reg_warmup_steps, lambda_l1),
                       get_reg_weight(step, reg_warmup_steps, lambda_flops))


class PreferenceLossOutput(NamedTuple):
    """loss is back-propagated; margin [B] (fp32, not differentiable) is each pair's log ratio, for
    logging, or as another model's ref_margin."""
    loss: Tensor
    margin: Tensor


def _check_pairs(q: Tensor, pos: Tensor, neg: Tensor, ref: Optional[Tensor], temperature: float, beta: float,
                 smoothing: float, op: str) -> None:
    if q.dim() != 2 or q.dtype not in _FLOAT_DTYPES or q.shape[0] < 1 or q.shape[1] < 1:
        raise ValueError(f"{op}: query reps must be a 2-D float tensor [B, V], B and V at least 1, got {q.dtype} "
                         f"{tuple(q.shape)}")
    for t, name in ((pos, "preferred"), (neg, "rejected")):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{op}: {name} document reps must be {tuple(q.shape)} {q.dtype} on {q.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if ref is not None:
        if tuple(ref.shape) != (q.shape[0],) or ref.dtype != torch.float32 or ref.device != q.device:
            raise ValueError(f"{op}: ref_margin must be float32 [{q.shape[0]}] on {q.device}, got {ref.dtype} "
                             f"{tuple(ref.shape)} on {ref.device}")
        if ref.requires_grad:
            raise ValueError(f"{op}: ref_margin is the frozen reference model's and gets no gradient; detach it")
    for v, name in ((temperature, "temperature"), (beta, "beta")):
        if not (v > 0.0 and math.isfinite(v)):
            raise ValueError(f"{op}: {name} must be positive and finite, got {v}")
    if not 0.0 <= smoothing <= 0.5:
        raise ValueError(f"{op}: label_smoothing must lie in [0, 0.5], got {smoothing}")
    if not q.is_cuda:
        raise RuntimeError(f"{op} only supports ROCm/HIP device tensors (got device {q.device})")


@torch.library.custom_op("sparton::preference_fwd", mutates_args=())
def preference_fwd(q: Tensor, pos: Tensor, neg: Tensor, ref_margin: Optional[Tensor], temperature: float, beta: float,
                   smoothing: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(loss, margin [B], coef [B]) in fp32; coef = d loss / d(q.pos) of each row, which the backward uses."""
    _check_pairs(q, pos, neg, ref_margin, temperature, beta, smoothing, "sparton::preference_fwd")
    return _eager.load().preference_fwd(q, pos, neg, ref_margin, temperature, beta, smoothing)


@preference_fwd.register_fake
def _(q, pos, neg, ref_margin, temperature, beta, smoothing):
    row = q.new_empty((q.shape[0],), dtype=torch.float32)
    return q.new_empty((), dtype=torch.float32), row, row.clone()


@torch.library.custom_op("sparton::preference_bwd", mutates_args=())
def preference_bwd(grad: Tensor, q: Tensor, pos: Tensor, neg: Tensor, coef: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dpos, dneg) in the reps dtype, from the loss's upstream gradient (a scalar)."""
    op = "sparton::preference_bwd"
    _check_pairs(q, pos, neg, None, 1.0, 1.0, 0.0, op)
    if grad.numel() != 1 or tuple(coef.shape) != (q.shape[0],) or coef.dtype != torch.float32 or not coef.is_contiguous():
        raise ValueError(f"{op}: grad must be a scalar and coef contiguous float32 [{q.shape[0]}], got "
                         f"{tuple(grad.shape)} and {coef.dtype} {tuple(coef.shape)}")
    for t in (grad, coef):
        if t.device != q.device:
            raise ValueError(f"{op}: all tensors must be on {q.device}, got {t.device}")
    return _eager.load().preference_bwd(grad, q, pos, neg, coef)


@preference_bwd.register_fake
def _(grad, q, pos, neg, coef):
    return q.new_empty(q.shape), q.new_empty(q.shape), q.new_empty(q.shape)


def _preference_setup(ctx, inputs, output):
    q, pos, neg = inputs[:3]
    _loss, margin, coef = output
    ctx.mark_non_differentiable(margin, coef)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(q, pos, neg, coef)


def _preference_backward(ctx, g_loss, _g_margin, _g_coef):
    q, pos, neg, coef = ctx.saved_tensors
    if g_loss is None:  # the loss did not reach what is differentiated
        return None, None, None, None, None, None, None
    return (*torch.ops.sparton.preference_bwd(g_loss, q, pos, neg, coef), None, None, None, None)


preference_fwd.register_autograd(_preference_backward, setup_context=_preference_setup)


def preference_loss(query_reps: Tensor, pos_reps: Tensor, neg_reps: Tensor, ref_margin: Optional[Tensor] = None, *,
                    beta: float = 1.0, temperature: float = 1.0, label_smoothing: float = 0.0) -> PreferenceLossOutput:
    """Preference loss on pairs: row i of the reps [B, V] is a query, the document preferred for it and
    one rejected. A retriever gives documents the probabilities softmax(q.d / temperature), so a pair's
    log ratio log P(pos) - log P(neg) is its score margin m = (q.pos - q.neg) / temperature, and with
    the reference model's margins r (preference_margin of its reps; default zeros)

        loss = mean of -(1 - label_smoothing) log sigma(z) - label_smoothing log sigma(-z),  z = beta (m - r)

    Scores and sums are fp32 whatever the reps dtype, over the difference pos - neg, so that close
    scores do not cancel."""
    args = (query_reps, pos_reps, neg_reps, ref_margin, float(temperature), float(beta), float(label_smoothing))
    if torch.compiler.is_compiling() or not query_reps.is_cuda:  # the registered op: fake + autograd
        loss, margin, _ = torch.ops.sparton.preference_fwd(*args)
        return PreferenceLossOutput(loss, margin)
    _check_pairs(*args, "preference_loss")
    return PreferenceLossOutput(*_eager.load().preference_loss(*args))


@torch.no_grad()
def preference_margin(query_reps: Tensor, pos_reps: Tensor, neg_reps: Tensor, temperature: float = 1.0) -> Tensor:
    """The margins [B] (fp32) of a reference model's reps, for preference_loss's ref_margin."""
    if torch.compiler.is_compiling():  # the registered op, which has a fake
        return torch.ops.sparton.preference_fwd(query_reps, pos_reps, neg_reps, None, float(temperature), 1.0, 0.0)[1]
    _check_pairs(query_reps, pos_reps, neg_reps, None, float(temperature), 1.0, 0.0, "preference_margin")
    return _eager.load().preference_margin(query_reps, pos_reps, neg_reps, float(temperature))
