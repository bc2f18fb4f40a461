"""Performance cases of the operators around the head: attention, LayerNorm and the preference loss.

A case is a dict of plain values. `listed()` gives the named ones, `draw(rng)` one more of the same
ranges, `prepare(case, seed)` what a program holds before the call, `run(state)` one pass, `work(case)`
the bytes and operations such a pass cannot do without, `exact(case, seed)` the same outputs in 64
bits. With `own` false, `run` computes each operator from elementary torch operations in 32 bits and
rounds once at the end; with `own` true it calls the framework's operator.

Kinds:
  attention   attention(q, k, v, key_mask): the output, and with `train` the gradients of q, k, v
  norm        layer_norm(x, weight, bias, residual): the output, and with `train` every gradient
  preference  preference_loss(q, pos, neg, ref_margin): loss, margins and the gradients of the reps
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    att = dict(kind="attention", causal=False, train=True, mask="int64", holes=False, empty=False, layout="bshd")
    norm = dict(kind="norm", eps=1e-12, residual=True, bias=True, vec="same", train=True)
    pref = dict(kind="preference", beta=1.0, smoothing=0.0)
    return [
        # One short query through an encoder layer: the smallest serving call, all latency.
        dict(att, name="att-query", B=1, Hq=12, Hk=12, Sq=16, Sk=16, Dh=64, dtype="bf16", len_lo=16, len_hi=16, train=False),
        # An encoder layer of the headline training workload (batch 32, 256 positions, width 768), right-padded.
        dict(att, name="att-bert", B=32, Hq=12, Hk=12, Sq=256, Sk=256, Dh=64, dtype="bf16", len_lo=32, len_hi=256),
        # Long documents in fp16.
        dict(att, name="att-longdoc", B=8, Hq=12, Hk=12, Sq=512, Sk=512, Dh=64, dtype="fp16", len_lo=288, len_hi=512),
        # fp32 training at an odd batch and length.
        dict(att, name="att-fp32", B=7, Hq=12, Hk=12, Sq=181, Sk=181, Dh=64, dtype="fp32", len_lo=24, len_hi=181, mask="bool"),
        # A decoder-only backbone of width 4096 with shared key heads: causal, and the documents padded.
        dict(att, name="att-llm", B=16, Hq=32, Hk=8, Sq=512, Sk=512, Dh=128, dtype="bf16", len_lo=128, len_hi=512, causal=True),
        # One very long document: the largest call.
        dict(att, name="att-long", B=1, Hq=12, Hk=12, Sq=8192, Sk=8192, Dh=64, dtype="bf16", len_lo=8192, len_hi=8192, mask="none"),
        # One new token per sequence against a long cache of keys and values.
        dict(att, name="att-token", B=4, Hq=32, Hk=8, Sq=1, Sk=20001, Dh=128, dtype="bf16", len_lo=9000, len_hi=20001, train=False, layout="bhsd"),
        # The norm of one short query, fp32 as models are loaded: latency again.
        dict(norm, name="norm-query", M=16, D=768, dtype="fp32", train=False),
        # The headline workload's rows with the residual sum, as every encoder layer has it twice.
        dict(norm, name="norm-bert", M=8192, D=768, dtype="bf16"),
        # Rows of the wide model, the norm's vectors as fp32 masters.
        dict(norm, name="norm-wide", M=16385, D=4096, dtype="bf16", residual=False, vec="fp32", eps=1e-5),
        # Pairs at the headline workload's batch and vocabulary.
        dict(pref, name="pref-bert", B=32, V=30522, dtype="bf16"),
        # A large batch of pairs over the multilingual vocabulary.
        dict(pref, name="pref-xlmr", B=500, V=250002, dtype="bf16", smoothing=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "norm", "norm", "preference"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        D = rng.choice([384, 768, 768, 1000, 1024, 1023, 4096, _log(rng, 8, 8192)])
        M = min(_log(rng, 1, 65536), max(1, int(6.0e7 / D)))
        return dict(kind=kind, M=M, D=D, dtype=dtype, eps=rng.choice([1e-12, 1e-5]), residual=rng.random() < 0.5,
                    bias=rng.random() < 0.8, vec=rng.choice(["same", "fp32"]), train=rng.random() < 0.7)
    if kind == "preference":
        V = rng.choice([30522, 30522, 50265, _log(rng, 3000, 250002)])
        B = min(_log(rng, 1, 2000), max(1, int((1.2e8 if dtype != "fp32" else 6.0e7) / V)))
        return dict(kind=kind, B=B, V=V, dtype=dtype, beta=rng.choice([0.5, 1.0]), smoothing=rng.choice([0.0, 0.1]))
    Hk = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 4])
    Dh = rng.choice([32, 64, 64, 64, 80, 128])
    form = rng.choice(["self", "self", "self", "few"])
    causal = rng.random() < 0.3
    if form == "self":
        Sq = Sk = _log(rng, 1, 4096)
        train = rng.random() < 0.7 and Sk >= 4  # rows that see one key have no gradient but rounding's
    else:  # one or a few new tokens against a cache
        Sq, Sk, train = rng.choice([1, 1, 2, 5, 17]), _log(rng, 64, 40000), False
    budget = 4.0e9 / Dh / (1 if dtype != "fp32" else 8)  # pairs, well under the largest listed case's cost
    B = max(1, min(_log(rng, 1, 64), int(budget / (Hk * group * Sq * Sk)), int(1.5e8 / (Hk * group * max(Sq, Sk) * Dh))))
    return dict(kind=kind, B=B, Hq=Hk * group, Hk=Hk, Sq=Sq, Sk=Sk, Dh=Dh, dtype=dtype, causal=causal, train=train,
                mask=rng.choice(["int64", "int64", "bool", "none"]), holes=rng.random() < 0.2 and Sk >= 32, empty=rng.random() < 0.15 and B > 1,
                layout=rng.choice(["bshd", "bhsd", "fused"]), len_lo=max(1, Sk // 8), len_hi=Sk)


# ---- inputs -------------------------------------------------------------------------

def _rand(g, *n):
    return torch.randn(*n, generator=g, device="cuda")


def _lengths(case):
    """Lengths spread evenly from len_lo to len_hi, the longest among them."""
    B = case["B"]
    lo, hi = case["len_lo"], case["len_hi"]
    return [hi - (hi - lo) * i // max(1, B - 1) for i in range(B)]


def _attention_inputs(case, seed):
    """(q, k, v, key mask or None, gradient of the output), q [B, Hq, Sq, Dh] and so on."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, Hq, Hk, Sq, Sk, Dh = (case[n] for n in ("B", "Hq", "Hk", "Sq", "Sk", "Dh"))
    dt = DTYPES[case["dtype"]]
    if case["layout"] == "fused" and Sq == Sk:    # views of one projection's output
        qkv = _rand(g, B, Sq, Hq + 2 * Hk, Dh).to(dt)
        q, k, v = (t.transpose(1, 2) for t in qkv.split([Hq, Hk, Hk], dim=2))
    elif case["layout"] == "bhsd":                # a cache, laid out by head
        q, k, v = _rand(g, B, Hq, Sq, Dh).to(dt), _rand(g, B, Hk, Sk, Dh).to(dt), _rand(g, B, Hk, Sk, Dh).to(dt)
    else:                                         # three projections
        q, k, v = (_rand(g, B, S, H, Dh).to(dt).transpose(1, 2) for S, H in ((Sq, Hq), (Sk, Hk), (Sk, Hk)))
    do = _rand(g, B, Sq, Hq, Dh).mul_(0.02).to(dt).transpose(1, 2)
    mask = None
    if case["mask"] != "none":
        lengths = torch.tensor(_lengths(case), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
        mask = torch.arange(Sk, device="cuda")[None, :] < lengths[:, None]
        if case["holes"]:
            mask &= torch.rand(B, Sk, generator=g, device="cuda") < 0.7
        if case["empty"]:
            mask[B // 2] = False
        mask = mask if case["mask"] == "bool" else mask.to(torch.int64)
    return q, k, v, mask, do


def _norm_inputs(case, seed):
    """(x, residual or None, weight, bias or None, gradient of y)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, D, dt = case["M"], case["D"], DTYPES[case["dtype"]]
    vt = torch.float32 if case["vec"] == "fp32" else dt
    x, dy = _rand(g, M, D).add_(0.1).to(dt), _rand(g, M, D).mul_(0.02).to(dt)
    r = _rand(g, M, D).to(dt) if case["residual"] else None
    w = (1.0 + 0.1 * _rand(g, D)).to(vt)
    b = (0.1 * _rand(g, D)).to(vt) if case["bias"] else None
    return x, r, w, b, dy


def _preference_inputs(case, seed):
    """(q, pos, neg, the reference model's margins): reps as the head gives them early in training, about 30% active."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, V, dt = case["B"], case["V"], DTYPES[case["dtype"]]
    q, p, n = (torch.log1p(torch.relu(_rand(g, B, V).sub_(0.5))).to(dt) for _ in range(3))
    return q, p, n, 0.5 * _rand(g, B)


def _temperature(case):
    """Scores of dense reps grow with the vocabulary; this keeps the margins near one."""
    return math.sqrt(case["V"]) / 4.0


def prepare(case, seed):
    if case["kind"] == "norm":
        x, r, w, b, dy = _norm_inputs(case, seed)
        leaves = [t for t in (x, r, w, b) if t is not None]
        state = dict(case=case, x=x, r=r, w=w, b=b, dy=dy)
    elif case["kind"] == "preference":
        q, p, n, ref = _preference_inputs(case, seed)
        leaves = [q, p, n]
        state = dict(case=case, q=q, p=p, n=n, ref=ref)
    else:
        q, k, v, mask, do = _attention_inputs(case, seed)
        leaves = [q, k, v]
        state = dict(case=case, q=q, k=k, v=v, mask=mask, do=do)
    if case.get("train", True):
        for t in leaves:
            t.requires_grad_()
    state["leaves"] = leaves
    return state


# ---- one pass -----------------------------------------------------------------------

def _own_attention(state):
    from sparton_amd.attention import attention
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return attention(state["q"], state["k"], state["v"], state["mask"], causal=case["causal"])
    out = attention(state["q"], state["k"], state["v"], state["mask"], causal=case["causal"])
    return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["do"])]


def _own_norm(state):
    from sparton_amd.norm import layer_norm
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return layer_norm(state["x"], state["w"], state["b"], eps=case["eps"], residual=state["r"])
    y = layer_norm(state["x"], state["w"], state["b"], eps=case["eps"], residual=state["r"])
    return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])]


def _own_preference(state):
    from sparton_amd.loss import preference_loss
    case = state["case"]
    res = preference_loss(state["q"], state["p"], state["n"], state["ref"], beta=case["beta"],
                          temperature=_temperature(case), label_smoothing=case["smoothing"])
    return [res.loss.detach(), res.margin, *torch.autograd.grad(res.loss, state["leaves"])]


def _plain_attention(state):
    case, dt = state["case"], state["q"].dtype
    B, Hq, Hk, Sq, Sk, Dh = (case[n] for n in ("B", "Hq", "Hk", "Sq", "Sk", "Dh"))
    G, scale = Hq // Hk, Dh ** -0.5
    q = state["q"].float().reshape(B, Hk, G, Sq, Dh)   # query heads by the key head that they share
    k, v = state["k"].float()[:, :, None], state["v"].float()[:, :, None]
    allowed = torch.ones(1, 1, 1, Sq, Sk, dtype=torch.bool, device=q.device)
    if case["causal"]:
        allowed = allowed.tril(Sk - Sq)
    if state["mask"] is not None:
        keys = state["mask"] != 0
        allowed = allowed & keys[:, None, None, None, :]
        k, v = (torch.where(keys[:, None, None, :, None], t, 0.0) for t in (k, v))
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    s = torch.where(allowed, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0.0, 1.0, total))
    o = torch.matmul(p, v)
    out = o.reshape(B, Hq, Sq, Dh).to(dt)
    if not case["train"]:
        return out
    do = state["do"].float().reshape(B, Hk, G, Sq, Dh)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k).mul_(scale).reshape(B, Hq, Sq, Dh)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2).mul_(scale)
    return [out, dq.to(dt), dk.to(dt), dv.to(dt)]


def _plain_norm(state):
    case, dt = state["case"], state["x"].dtype
    w = state["w"].float()
    h = state["x"].float() if state["r"] is None else state["x"].float() + state["r"].float()
    c = h - h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + case["eps"])
    xhat = c * rstd
    y = xhat * w
    if state["b"] is not None:
        y = y + state["b"].float()
    y = y.to(dt)
    if not case["train"]:
        return y
    dy = state["dy"].float()
    g = dy * w
    dx = (rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))).to(dt)
    grads = [dx] if state["r"] is None else [dx, dx]
    grads.append((dy * xhat).sum(0).to(state["w"].dtype))
    if state["b"] is not None:
        grads.append(dy.sum(0).to(state["b"].dtype))
    return [y, *grads]


def _plain_preference(state):
    case, dt = state["case"], state["q"].dtype
    beta, eps, T, B = case["beta"], case["smoothing"], _temperature(case), case["B"]
    q, p, n = state["q"].detach().float(), state["p"].detach().float(), state["n"].detach().float()
    diff = p - n
    margin = (q * diff).sum(1) / T
    z = beta * (margin - state["ref"])
    # -log sigma(z) = max(-z, 0) + log(1 + exp(-|z|))
    tail = torch.log1p(torch.exp(-z.abs()))
    loss = ((1.0 - eps) * (torch.clamp_min(-z, 0.0) + tail) + eps * (torch.clamp_min(z, 0.0) + tail)).mean()
    c = (torch.where(z > 0, 1.0, torch.exp(-z.abs())) / (1.0 + torch.exp(-z.abs())) - (1.0 - eps)) * (beta / (B * T))
    dp = c[:, None] * q
    return [loss, margin, (c[:, None] * diff).to(dt), dp.to(dt), (-dp).to(dt)]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": _own_attention, "norm": _own_norm, "preference": _own_preference}[kind](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "preference": _plain_preference}[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    """Each input read once and each output written once; multiply-adds count two."""
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        M, D, n = case["M"], case["D"], 1 + bool(case["residual"])
        ve = 4 if case["vec"] == "fp32" else e
        rows, vecs = n + 1, 1 + bool(case["bias"])  # x (and the residual) in, y out
        flops = 8.0 * M * D
        if case["train"]:                           # dy in and one gradient out, which serves x and the residual
            rows, vecs, flops = rows + 2, 2 * vecs, flops + 14.0 * M * D
        return dict(bytes=float(rows * M * D * e + vecs * D * ve), flops=flops)
    if case["kind"] == "preference":
        B, V = case["B"], case["V"]
        return dict(bytes=6.0 * B * V * e + 12.0 * B, flops=7.0 * B * V)
    B, Hq, Hk, Sq, Sk, Dh = (case[n] for n in ("B", "Hq", "Hk", "Sq", "Sk", "Dh"))
    lengths = [Sk] * B if case["mask"] == "none" else _lengths(case)
    if case["mask"] != "none" and case["empty"]:
        lengths = lengths[: B - 1]
    share = 0.7 if case["mask"] != "none" and case["holes"] else 1.0

    def pairs(n):
        """Pairs of a query row and one of the first n keys that the row may look at."""
        if not case["causal"]:
            return Sq * n
        first = min(n, max(0, Sk - Sq + 1))                 # keys of the first row
        grow = min(Sq, n - first + 1) if n > first else 1   # rows until all n are seen
        return first * grow + grow * (grow - 1) // 2 + (Sq - grow) * n

    total = share * Hq * sum(pairs(n) for n in lengths)
    keys = share * Hk * Dh * sum(lengths)                   # masked keys need not be read
    rows = float(B * Hq * Sq * Dh)
    bytes_ = (2.0 * keys + 2.0 * rows) * e + (0 if case["mask"] == "none" else B * Sk * (1 if case["mask"] == "bool" else 8))
    flops = 4.0 * Dh * total
    if case["train"]:  # the output's gradient in; three gradients out
        bytes_ += (2.0 * rows + 2.0 * B * Hk * Sk * Dh) * e
        flops += 10.0 * Dh * total
    return dict(bytes=bytes_, flops=flops)


# ---- the same in 64 bits ------------------------------------------------------------------

def _exact_attention(case, seed):
    q, k, v, mask, do = _attention_inputs(case, seed)
    B, Hq, Hk, Sq, Sk, Dh = (case[n] for n in ("B", "Hq", "Hk", "Sq", "Sk", "Dh"))
    if 14.0 * B * Hq * Sq * Sk * Dh > 4.0e12:
        return None
    f64 = torch.float64
    outs = [torch.zeros(t.shape, dtype=f64, device="cuda") for t in (q, q, k, v)]
    rows, cols = torch.arange(Sq, device="cuda"), torch.arange(Sk, device="cuda")
    for b in range(B):
        keys = torch.ones(Sk, dtype=torch.bool, device="cuda") if mask is None else mask[b] != 0
        at = cols[keys]                                     # the keys that take part, and no others
        if at.numel() == 0:
            continue
        hidden = at[None, :] > rows[:, None] + (Sk - Sq) if case["causal"] else None
        step = max(1, int(1.0e9 / (Sq * at.numel())))
        for h0 in range(0, Hq, step):
            hs = torch.arange(h0, min(Hq, h0 + step), device="cuda")
            kv = hs // (Hq // Hk)
            qq = q[b, hs].to(f64).requires_grad_()
            kk, vv = (t[b, kv][:, at].to(f64).requires_grad_() for t in (k, v))
            with torch.enable_grad():
                s = (qq @ kk.transpose(1, 2)) / math.sqrt(Dh)
                if hidden is not None:
                    s = s.masked_fill(hidden, -math.inf)
                p = torch.softmax(s, -1)
                if hidden is not None:
                    p = torch.where(hidden.all(-1)[:, None], torch.zeros_like(p), p)
                o = p @ vv
            outs[0][b, hs] = o.detach()
            if case["train"]:
                gq, gk, gv = torch.autograd.grad(o, (qq, kk, vv), do[b, hs].to(f64))
                outs[1][b, hs] = torch.nan_to_num(gq) if hidden is not None and bool(hidden.all(-1).any()) else gq
                place = (kv[:, None], at[None, :])
                outs[2][b].index_put_(place, gk, accumulate=True)
                outs[3][b].index_put_(place, gv, accumulate=True)
            del s, p, o
    return outs if case["train"] else outs[0]


def _exact_norm(case, seed):
    x, r, w, b, dy = _norm_inputs(case, seed)
    leaves = [t.double().requires_grad_() for t in (x, r, w, b) if t is not None]
    named = iter(leaves)
    x, r, w, b = (next(named) if t is not None else None for t in (x, r, w, b))
    with torch.enable_grad():
        h = x if r is None else x + r
        y = torch.nn.functional.layer_norm(h, (case["D"],), w, b, case["eps"])
    if not case["train"]:
        return y.detach()
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.double())]


def _exact_preference(case, seed):
    q, p, n, ref = _preference_inputs(case, seed)
    q, p, n = (t.double().requires_grad_() for t in (q, p, n))
    eps = case["smoothing"]
    with torch.enable_grad():
        margin = ((q * p).sum(1) - (q * n).sum(1)) / _temperature(case)
        z = case["beta"] * (margin - ref.double())
        good, bad = torch.nn.functional.logsigmoid(z), torch.nn.functional.logsigmoid(-z)
        loss = -((1.0 - eps) * good + eps * bad).mean()
    return [loss.detach(), margin.detach(), *torch.autograd.grad(loss, (q, p, n))]


def exact(case, seed):
    return {"attention": _exact_attention, "norm": _exact_norm, "preference": _exact_preference}[case["kind"]](case, seed)
