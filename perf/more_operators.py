"""Performance cases of a gated backbone's other operators: the embedding, the root-mean-square norm and
the gated feed-forward product.

A case is a dict of plain values. `listed()` gives the named ones, `draw(rng)` one more of the same
ranges, `prepare(case, seed)` what a program holds before the call, `run(state)` one pass, `work(case)`
the bytes and operations such a pass cannot do without, `exact(case, seed)` the same outputs in 64
bits. With `own` false, `run` computes each operator from elementary torch operations in 32 bits and
rounds once at the end; with `own` true it calls the framework's operator.

Kinds:
  embedding  embedding(ids, weight, scale, padding_idx): the rows, and with `train` the table's gradient
  rms        rms_norm(x, weight, eps, residual): the rows (and the sum), and with `train` every gradient
  rms8       rms_norm_8bit(...): rows in e4m3, their scales (and the sum)
  gated      gated_linear(x, w_gate, w_up, b_gate, b_up, activation): act(x Wg' + bg) (x Wu' + bu), and
             with `train` every gradient
  gated8     gated_linear_8bit(...): the same on rows and weights in e4m3 with a scale a row
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126  # of a row without a nonzero value: its reciprocal is finite


def listed():
    emb = dict(kind="embedding", scale=1.0, ids="tokens", pad=0.35, train=True)
    rms = dict(kind="rms", eps=1e-6, residual=True, vec="same", train=True)
    gated = dict(kind="gated", act="silu", bias=False, train=True)
    return [
        # The tokens of one short query: the smallest serving call, all latency.
        dict(emb, name="emb-query", N=16, V=30522, D=768, dtype="bf16", pad=0.0, train=False),
        # The headline training workload's tokens (32 x 256, right-padded) and its vocabulary.
        dict(emb, name="emb-bert", N=8192, V=30522, D=768, dtype="bf16"),
        # The multilingual vocabulary, rows scaled by the root of their width, an odd number of tokens.
        dict(emb, name="emb-xlmr", N=16391, V=250002, D=768, dtype="fp16", scale=27.712812921102035, pad=0.2),
        # The norm of four new tokens of the wide model: latency again.
        dict(rms, name="rms-token", M=4, D=4096, dtype="bf16", train=False),
        # The wide model's rows with the residual's addition, as every layer has it twice.
        dict(rms, name="rms-llm", M=8192, D=4096, dtype="bf16"),
        # fp32 rows of an odd width and number.
        dict(rms, name="rms-odd", M=7001, D=1023, dtype="fp32", residual=False),
        # The wide model's rows on their way to products in 8 bits.
        dict(rms, name="rms-8bit", kind="rms8", M=8192, D=4096, dtype="bf16", train=False),
        # The feed-forward block of four new tokens: the weights are read for four rows.
        dict(gated, name="gated-token", M=4, D=4096, F=11264, dtype="bf16", train=False),
        # A gated encoder layer of the headline workload's rows and width.
        dict(gated, name="gated-bert", M=8192, D=768, F=2048, dtype="bf16", act="gelu"),
        # The wide model in training: the largest call.
        dict(gated, name="gated-llm", M=8192, D=4096, F=11264, dtype="bf16"),
        # fp32 training at odd sizes, with biases.
        dict(gated, name="gated-fp32", M=1000, D=768, F=2051, dtype="fp32", act="gelu_tanh", bias=True),
        # The wide model's prompts in 8 bits.
        dict(gated, name="gated-8bit", kind="gated8", M=8192, D=4096, F=11264, dtype="bf16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embedding", "embedding", "embedding", "rms", "rms", "rms8", "gated", "gated", "gated", "gated", "gated8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "embedding":
        D = rng.choice([384, 768, 768, 1000, 1024, 1023, 4096, _log(rng, 8, 4096)])
        ids = rng.choice(["tokens", "tokens", "tokens", "positions"])
        V = _log(rng, 16, 8192) if ids == "positions" else min(rng.choice([30522, 30522, 50265, 250002, _log(rng, 100, 250002)]), int(1.9e8 / D))
        N = min(_log(rng, 1, 65536), max(1, int(2.0e7 / D)))
        return dict(kind=kind, N=N, V=V, D=D, dtype=dtype, scale=rng.choice([1.0, math.sqrt(D)]), ids=ids,
                    pad=rng.choice([0.0, 0.1, 0.5]) if ids == "tokens" else 0.0, train=rng.random() < 0.75)
    if kind in ("rms", "rms8"):
        D = rng.choice([384, 768, 1000, 1024, 1023, 4096, 4096, 8192, _log(rng, 8, 8192)])
        M = min(_log(rng, 1, 65536), max(1, int(3.3e7 / D)))
        return dict(kind=kind, M=M, D=D, dtype=dtype, eps=rng.choice([1e-6, 1e-5]), residual=rng.random() < 0.6,
                    vec=rng.choice(["same", "fp32"]), train=kind == "rms" and rng.random() < 0.7)
    D = rng.choice([384, 768, 768, 1000, 1024, 2048, 4096, _log(rng, 64, 4096)])
    F = rng.choice([1024, 2048, 2051, 4096, 8192, 11264, _log(rng, 64, 11264)])
    M = min(rng.choice([_log(rng, 1, 64), _log(rng, 64, 16384), _log(rng, 64, 16384)]), int(3.7e11 / D / F))
    case = dict(kind=kind, M=M, D=D, F=F, dtype=dtype, act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]))
    if kind == "gated8":
        return dict(case, dtype=rng.choice(["bf16", "bf16", "fp16"]), bias=False, train=False)
    return dict(case, bias=rng.random() < 0.25, train=M >= 4 and rng.random() < 0.65)


# ---- inputs -------------------------------------------------------------------------

def _rand(g, *n):
    return torch.randn(*n, generator=g, device="cuda")


def _embedding_inputs(case, seed):
    """(ids, table, gradient of the rows). A token's rank is spread over its logarithm, as words are;
    token 0 pads. Positions count up, again for every sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, V, D, dt = case["N"], case["V"], case["D"], DTYPES[case["dtype"]]
    if case["ids"] == "positions":
        ids = torch.arange(N, device="cuda") % V
    else:
        ids = torch.rand(N, generator=g, device="cuda", dtype=torch.float64).mul_(math.log(V)).exp_().long().clamp_(1, V - 1)
        ids[torch.rand(N, generator=g, device="cuda") < case["pad"]] = 0
    return ids, _rand(g, V, D).mul_(0.02).to(dt), _rand(g, N, D).mul_(0.02).to(dt)


def _rms_inputs(case, seed):
    """(x, residual or None, weight, gradient of y, gradient of the sum)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, D, dt = case["M"], case["D"], DTYPES[case["dtype"]]
    x, dy, dh = _rand(g, M, D).to(dt), _rand(g, M, D).mul_(0.02).to(dt), _rand(g, M, D).mul_(0.02).to(dt)
    r = _rand(g, M, D).mul_(2.0).to(dt) if case["residual"] else None
    w = (1.0 + 0.1 * _rand(g, D)).to(torch.float32 if case["vec"] == "fp32" else dt)
    return x, r, w, dy, dh


def _gated_inputs(case, seed):
    """(x, w_gate, w_up, b_gate or None, b_up or None, gradient of the output): normed rows, and weights
    that keep the projections near one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, D, F, dt = case["M"], case["D"], case["F"], DTYPES[case["dtype"]]
    x = _rand(g, M, D).to(dt)
    wg, wu = (_rand(g, F, D).mul_(D ** -0.5).to(dt) for _ in range(2))
    bg, bu = ((0.2 * _rand(g, F)).to(dt) for _ in range(2)) if case["bias"] else (None, None)
    return x, wg, wu, bg, bu, _rand(g, M, F).mul_(0.02).to(dt)


def _to_e4m3(t):
    """Rows in e4m3 with a scale each."""
    scale = (t.abs().amax(-1) / E4M3_MAX).clamp_min(LEAST_SCALE)
    return (t / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), scale


def _gated8_inputs(case, seed):
    """(x, its scales, w_gate, its scales, w_up, its scales): what the norm in 8 bits gives, and a model's
    weights as a serving program keeps them."""
    x, wg, wu = _gated_inputs(case, seed)[:3]
    return [t for part in (x, wg, wu) for t in _to_e4m3(part.float())]


def prepare(case, seed):
    kind = case["kind"]
    if kind == "embedding":
        ids, w, dy = _embedding_inputs(case, seed)
        leaves, state = [w], dict(ids=ids, w=w, dy=dy)
    elif kind in ("rms", "rms8"):
        x, r, w, dy, dh = _rms_inputs(case, seed)
        leaves, state = [t for t in (x, r, w) if t is not None], dict(x=x, r=r, w=w, dy=dy, dh=dh)
    elif kind == "gated":
        x, wg, wu, bg, bu, dh = _gated_inputs(case, seed)
        leaves, state = [t for t in (x, wg, wu, bg, bu) if t is not None], dict(x=x, wg=wg, wu=wu, bg=bg, bu=bu, dh=dh)
    else:
        leaves, state = [], dict(zip(("x", "sx", "wg", "sg", "wu", "su"), _gated8_inputs(case, seed)))
    if case["train"]:
        for t in leaves:
            t.requires_grad_()
    return dict(state, case=case, leaves=leaves)


# ---- one pass -----------------------------------------------------------------------

def _padding(case):
    return 0 if case["pad"] > 0 else None


def _own_embedding(state):
    from sparton_amd.embedding import embedding
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return embedding(state["ids"], state["w"], scale=case["scale"], padding_idx=_padding(case))
    out = embedding(state["ids"], state["w"], scale=case["scale"], padding_idx=_padding(case))
    return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["dy"])]


def _own_rms(state):
    from sparton_amd.norm import rms_norm
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return rms_norm(state["x"], state["w"], eps=case["eps"], residual=state["r"])
    out = rms_norm(state["x"], state["w"], eps=case["eps"], residual=state["r"])
    if state["r"] is None:
        return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["dy"])]
    return [*(t.detach() for t in out), *torch.autograd.grad(out, state["leaves"], (state["dy"], state["dh"]))]


def _own_rms8(state):
    from sparton_amd.norm import rms_norm_8bit
    with torch.no_grad():
        return rms_norm_8bit(state["x"], state["w"], eps=state["case"]["eps"], residual=state["r"])


def _own_gated(state):
    from sparton_amd.feed_forward import gated_linear
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return gated_linear(state["x"], state["wg"], state["wu"], state["bg"], state["bu"], activation=case["act"])
    out = gated_linear(state["x"], state["wg"], state["wu"], state["bg"], state["bu"], activation=case["act"])
    return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["dh"])]


def _own_gated8(state):
    from sparton_amd.feed_forward import gated_linear_8bit
    case = state["case"]
    with torch.no_grad():
        return gated_linear_8bit(state["x"], state["sx"], state["wg"], state["sg"], state["wu"], state["su"],
                                 activation=case["act"], out_dtype=DTYPES[case["dtype"]])


def _plain_embedding(state):
    case, w, ids = state["case"], state["w"], state["ids"]
    out = (w[ids].float() * case["scale"]).to(w.dtype)
    if not case["train"]:
        return out
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids, state["dy"].float() * case["scale"])
    if _padding(case) is not None:
        dw[_padding(case)] = 0.0
    return [out, dw.to(w.dtype)]


def _plain_sum(state):
    return state["x"].float() if state["r"] is None else state["x"].float() + state["r"].float()


def _plain_rms(state):
    case, dt, w = state["case"], state["x"].dtype, state["w"].float()
    h = _plain_sum(state)
    q = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + case["eps"])
    xhat = h * q
    outs = [(xhat * w).to(dt)] if state["r"] is None else [(xhat * w).to(dt), h.to(dt)]
    if not case["train"]:
        return outs if state["r"] is not None else outs[0]
    dy = state["dy"].float()
    g = dy * w
    dx = q * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if state["r"] is None:
        grads = [dx.to(dt)]
    else:
        grads = [(dx + state["dh"].float()).to(dt)] * 2
    return [*outs, *grads, (dy * xhat).sum(0).to(state["w"].dtype)]


def _plain_rms8(state):
    case, dt = state["case"], state["x"].dtype
    h = _plain_sum(state)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + case["eps"]) * state["w"].float()
    outs = list(_to_e4m3(y))
    return outs if state["r"] is None else [*outs, h.to(dt)]


def _act(g, name):
    """(act(g), its derivative)."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    a, b = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * a * (1.0 + 3.0 * b * g * g)


def _plain_gated(state):
    case, dt = state["case"], state["x"].dtype
    x, wg, wu = state["x"].float(), state["wg"].float(), state["wu"].float()
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    if case["bias"]:
        g, u = g + state["bg"].float(), u + state["bu"].float()
    a, da = _act(g, case["act"])
    out = (a * u).to(dt)
    if not case["train"]:
        return out
    dh = state["dh"].float()
    dg, du = dh * u * da, dh * a
    grads = [torch.matmul(dg, wg) + torch.matmul(du, wu), torch.matmul(dg.t(), x), torch.matmul(du.t(), x)]
    if case["bias"]:
        grads += [dg.sum(0), du.sum(0)]
    return [out, *(t.to(dt) for t in grads)]


def _plain_gated8(state):
    x, sx = state["x"].float(), state["sx"][:, None]
    g = torch.matmul(x, state["wg"].float().t()) * sx * state["sg"]
    u = torch.matmul(x, state["wu"].float().t()) * sx * state["su"]
    return (_act(g, state["case"]["act"])[0] * u).to(DTYPES[state["case"]["dtype"]])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"embedding": _own_embedding, "rms": _own_rms, "rms8": _own_rms8, "gated": _own_gated,
                "gated8": _own_gated8}[kind](state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "rms": _plain_rms, "rms8": _plain_rms8, "gated": _plain_gated,
                "gated8": _plain_gated8}[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------

def _distinct(case):
    """How many rows of the table the ids name, on average."""
    N, V = case["N"], case["V"]
    if case["ids"] == "positions":
        return min(N, V)
    k = torch.arange(1, V, dtype=torch.float64)
    share = torch.log1p(1.0 / k) / math.log(V)
    return float(-torch.expm1(N * (1.0 - case["pad"]) * torch.log1p(-share)).sum()) + (1.0 if case["pad"] > 0 else 0.0)


def work(case):
    """Each input read once and each output written once; multiply-adds count two."""
    e, train = 4 if case["dtype"] == "fp32" else 2, case["train"]
    if case["kind"] == "embedding":
        N, V, D = case["N"], case["V"], case["D"]
        rows = _distinct(case) + N + (N + V if train else 0)
        return dict(bytes=8.0 * N + rows * D * e, flops=float(N * D * (2 if train else 1)))
    if case["kind"] in ("rms", "rms8"):
        M, D, res = case["M"], case["D"], case["residual"]
        ve = 4 if case["vec"] == "fp32" else e
        if case["kind"] == "rms8":
            return dict(bytes=float(M * D * ((3 if res else 1) * e + 1) + 4 * M + D * ve), flops=7.0 * M * D)
        rows, vecs, flops = 4 if res else 2, 1, 5.0 * M * D
        if train:  # the gradients of y and of the sum in, one out, which serves x and the residual
            rows, vecs, flops = rows + (3 if res else 2), 2, flops + 9.0 * M * D
        return dict(bytes=float(rows * M * D * e + vecs * D * ve), flops=flops)
    M, D, F = case["M"], case["D"], case["F"]
    if case["kind"] == "gated8":
        return dict(bytes=float(M * D + 2 * F * D + 4 * M + 8 * F + 2 * M * F), flops=4.0 * M * D * F)
    vecs = 2 * F if case["bias"] else 0
    n = M * D + 2 * F * D + vecs + M * F
    if train:
        n += M * F + M * D + 2 * F * D + vecs
    return dict(bytes=float(n * e), flops=(12.0 if train else 4.0) * M * D * F)


# ---- the same in 64 bits ------------------------------------------------------------------

def _exact_embedding(case, seed):
    ids, w, dy = _embedding_inputs(case, seed)
    out = w.index_select(0, ids).double() * case["scale"]
    if not case["train"]:
        return out
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    real = ids != _padding(case) if _padding(case) is not None else torch.ones_like(ids, dtype=torch.bool)
    dw.index_put_((ids[real],), dy[real].double(), accumulate=True)
    return [out, dw * case["scale"]]


def _exact_rms(case, seed):
    x, r, w, dy, dh = _rms_inputs(case, seed)
    leaves = [t.double().requires_grad_() for t in (x, r, w) if t is not None]
    with torch.enable_grad():
        h = leaves[0] if r is None else leaves[0] + leaves[1]
        y = torch.nn.functional.rms_norm(h, (case["D"],), leaves[-1], case["eps"])
    if case["kind"] == "rms8":
        scale = y.detach().abs().amax(-1) / E4M3_MAX
        outs = [y.detach() / scale[:, None], scale]
        return outs if r is None else [*outs, h.detach()]
    outs, ups = ([y], [dy]) if r is None else ([y, h], [dy, dh])
    plain = [t.detach() for t in outs]
    if not case["train"]:
        return plain if r is not None else plain[0]
    return [*plain, *torch.autograd.grad(outs, leaves, [t.double() for t in ups])]


def _exact_act(g, name):
    if name == "silu":
        return torch.nn.functional.silu(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if name == "gelu_tanh" else "none")


def _exact_gated(case, seed):
    x, wg, wu, bg, bu, dh = _gated_inputs(case, seed)
    leaves = [t.double().requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    biases = leaves[3:] if case["bias"] else (None, None)
    with torch.enable_grad():
        linear = torch.nn.functional.linear
        out = _exact_act(linear(leaves[0], leaves[1], biases[0]), case["act"]) * linear(leaves[0], leaves[2], biases[1])
    if not case["train"]:
        return out.detach()
    return [out.detach(), *torch.autograd.grad(out, leaves, dh.double())]


def _exact_gated8(case, seed):
    x, sx, wg, sg, wu, su = _gated8_inputs(case, seed)
    x, wg, wu = (t.float().double() * s.double()[:, None] for t, s in ((x, sx), (wg, sg), (wu, su)))
    return _exact_act(x @ wg.t(), case["act"]) * (x @ wu.t())


def exact(case, seed):
    return {"embedding": _exact_embedding, "rms": _exact_rms, "rms8": _exact_rms, "gated": _exact_gated,
            "gated8": _exact_gated8}[case["kind"]](case, seed)
