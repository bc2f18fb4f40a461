"""Attention in 64 bits from its definition, and how far the kernels may be from it.

u is half a step of the type, torch.finfo(t).eps / 2, relative to the value. The kernels' roundings:
  scores      fp32 sums of D products: |ds_ij| <= (D + 2) 2^-24 scale sum_d |q k|, and the exponential's
              own error and its argument's rounding, 2^-22 (1 + |s| + |L|): ep_ij, relative, of p_ij
  p, ds       rounded to the type for the next product: u each (fp16: 2^-25 absolute where p lies below
              the normal range; ds is scaled by column, so 2^-34 of the column's largest)
  sums        over n terms in fp32: n 2^-24 of the sum of magnitudes
  outputs     rounded once: u
Each bound adds these up over the terms; no term is fitted.
"""
import math

import torch

U32 = 2.0 ** -24


def allowed_pairs(B, Sq, Sk, mask, causal, device):
    a = torch.ones(B, 1, Sq, Sk, dtype=torch.bool, device=device)
    if causal:
        a = a.tril(Sk - Sq)
    if mask is not None:
        a = a & (mask != 0)[:, None, None, :]
    return a


def reference(q, k, v, mask, causal, scale, do):
    """{name: (value, tolerance)} for out, dq, dk, dv, all in 64 bits on q's device. q, k, v and do are
    the rounded inputs; masked keys are taken as zeros, so they may hold anything."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    B, Hq, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    G = Hq // Hk if Hk else 1
    on = allowed_pairs(B, Sq, Sk, mask, causal, q.device)
    if mask is not None:
        keep = (mask != 0)[:, None, :, None]
        k, v = torch.where(keep, k, 0.0), torch.where(keep, v, 0.0)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    kt, vt = k.transpose(-1, -2).contiguous(), v.transpose(-1, -2).contiguous()
    s = torch.where(on, scale * (q @ kt), -math.inf)
    some = on.any(-1, keepdim=True)
    top = torch.where(some, s.amax(-1, keepdim=True) if Sk else 0.0, 0.0)
    e = torch.where(on, torch.exp(s - top), 0.0)
    total = torch.where(some, e.sum(-1, keepdim=True), 1.0)
    p = e / total
    L = top + torch.log(total)
    ep = torch.where(on, (D + 2) * U32 * scale * (q.abs() @ kt.abs())
                     + 2.0 ** -22 * (1 + torch.where(on, s, 0.0).abs() + L.abs()), 0.0)
    # a row's sum carries its terms' errors: p is off by its own and by the largest of its row
    ep = ep + (p * ep).sum(-1, keepdim=True) + (Sk + 4) * U32
    n_k, n_q = Sk + 4, G * Sq + 4
    out = p @ v
    tol_o = u * out.abs() + (p * (u + ep + n_k * U32) + tiny * on) @ v.abs()
    pt, dot = p.transpose(-1, -2).contiguous(), do
    dv = pt @ dot
    tol_dv = ((p * (u + ep + n_q * U32) + tiny * on).transpose(-1, -2).contiguous()) @ dot.abs()
    dp, delta = do @ vt, (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = (D + 2) * U32 * (do.abs() @ vt.abs())
    e_delta = (do.abs() * (tol_o + (D + 2) * U32 * out.abs())).sum(-1, keepdim=True)
    e_ds = (u + ep + 4 * U32) * ds.abs() + p * (e_dp + e_delta)
    if tiny and Sk and Sq:
        e_ds = e_ds + 2.0 ** -34 * torch.maximum(ds.abs().amax(-1, keepdim=True), ds.abs().amax(-2, keepdim=True)) * on
    dq = scale * (ds @ k)
    tol_dq = u * dq.abs() + scale * ((e_ds + n_k * U32 * ds.abs()) @ k.abs())
    dst = ds.transpose(-1, -2).contiguous()
    dk = scale * (dst @ q)
    tol_dk = scale * ((e_ds + n_q * U32 * ds.abs()).transpose(-1, -2).contiguous() @ q.abs())

    def shared(t):  # the sum over the query heads of a key head
        return t.reshape(B, Hk, G, Sk, D).sum(2)

    dk, dv = shared(dk), shared(dv)
    sub = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126  # an output's own smallest step
    return dict(out=(out, tol_o + sub), dq=(dq, tol_dq + sub), dk=(dk, u * dk.abs() + shared(tol_dk) + sub),
                dv=(dv, u * dv.abs() + shared(tol_dv) + sub))


def close(got, want, what):
    value, tol = want
    assert got.shape == value.shape, f"{what}: {tuple(got.shape)} for {tuple(value.shape)}"
    if got.numel() == 0:
        return 0.0
    err = (got.detach().double() - value).abs()
    assert bool(torch.isfinite(err).all()), f"{what}: not finite"
    worst = float((err / tol).max())
    assert worst <= 1.0, f"{what}: {worst:.2f} times the tolerance (largest error {float(err.max()):.3e})"
    return worst
