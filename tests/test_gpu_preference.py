"""GPU parity of the preference loss against its formulas in 64 bits.

Tolerances, with u = eps / 2 of the reps dtype: a margin is an fp32 sum of V products of q and a rounded
difference, |margin error| <= (V + 3) 2^-24 sum |q| (|pos| + |neg|) / T =: em (and one rounding of the
result). z's error is beta em + 2^-23 (|beta m| + |beta r|) =: ez; the loss and sigma change by at most ez
(their slopes are at most 1 and 1/4) plus 2^-21 of the loss's terms (exponential, logarithm). A
coefficient c = (sigma(z) - (1 - eps)) beta / (B T) is then within ec = (ez / 4 + 2^-21) beta / (B T),
and gradients within ec |factor| + (u + 3 2^-24) |gradient|. At large |z| sigma(-z) is small: its slope
is sigma(-z) itself, so the bound takes min(1/4, the sum of sigma(-z) over the two ends of z +- ez).
"""
import math

import pytest
import torch

from _parity import say
from sparton_amd.loss import preference_loss, preference_margin

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def make(B, V, dt, device, seed=0, scale=1.0, density=0.3):
    g = torch.Generator().manual_seed(seed + B + 3 * V)
    reps = lambda: (torch.log1p(torch.relu(torch.randn(B, V, generator=g) * 2 - 1)) * scale
                    * (torch.rand(B, V, generator=g) < density + 0.3)).to(DT[dt]).to(device)
    return reps(), reps(), reps(), torch.randn(B, generator=g).to(device)


def reference(q, p, n, ref, beta, T, eps, up=1.0):
    u = torch.finfo(q.dtype).eps / 2
    q, p, n = (t.detach().double() for t in (q, p, n))
    B, V = q.shape
    r = torch.zeros(B, dtype=torch.float64, device=q.device) if ref is None else ref.double()
    m = (q * (p - n)).sum(1) / T
    z = beta * (m - r)
    ls = torch.nn.functional.logsigmoid
    terms = -(1 - eps) * ls(z) - eps * ls(-z)
    c = (torch.sigmoid(z) - (1 - eps)) * beta / (B * T) * up
    em = (V + 3) * E * (q.abs() * (p.abs() + n.abs())).sum(1) / T + 2 * E * m.abs()
    ez = beta * em + 2 * E * beta * (m.abs() + r.abs())
    slope = torch.minimum(torch.full_like(z, 0.25), torch.sigmoid(-(z.abs() - ez)))
    ec = (ez * slope + 2.0 ** -21 * (torch.sigmoid(-z.abs()) + eps)) * beta / (B * T) * abs(up)
    grads = (c[:, None] * (p - n), c[:, None] * q, -c[:, None] * q)
    tols = [ec[:, None] * f.abs() + (u + 3 * E) * g.abs() for f, g in zip(((p - n), q, q), grads)]
    tols[0] = tols[0] + 2 * E * c.abs()[:, None] * (p.abs() + n.abs())
    sub = 2.0 ** -25 if u == 2.0 ** -11 else 2.0 ** -126
    return dict(loss=(terms.mean(), (ez + 2.0 ** -21 * (terms + z.abs())).mean() + (B + 2) * E * terms.mean()),
                margin=(m, em), dq=(grads[0], tols[0] + sub), dp=(grads[1], tols[1] + sub), dn=(grads[2], tols[2] + sub))


def run(q, p, n, ref, beta, T, eps, up=1.0):
    leaves = [t.detach().requires_grad_() for t in (q, p, n)]
    res = preference_loss(*leaves, ref, beta=beta, temperature=T, label_smoothing=eps)
    assert not res.margin.requires_grad and res.loss.dim() == 0
    grads = torch.autograd.grad(res.loss * up, leaves)
    with torch.no_grad():
        again = preference_loss(q, p, n, ref, beta=beta, temperature=T, label_smoothing=eps)
    assert torch.equal(again.loss.nan_to_num(), res.loss.nan_to_num())
    assert torch.equal(again.margin.nan_to_num(), res.margin.nan_to_num())
    torch.cuda.synchronize()
    return dict(loss=res.loss.detach(), margin=res.margin, dq=grads[0], dp=grads[1], dn=grads[2])


def check(args, beta=1.0, T=1.0, eps=0.0, up=1.0):
    got, want = run(*args, beta, T, eps, up), reference(*args, beta, T, eps, up)
    worst = []
    for n in want:
        value, tol = want[n]
        ratio = float(((got[n].double() - value).abs() / (tol + 1e-300)).max())
        assert ratio <= 1.0, f"{n}: {ratio:.2f} times the tolerance"
        worst.append(f"{n} {ratio:.2f}")
    say("   of the tolerance: " + ", ".join(worst))
    return got


CASES = [  # B, V, dtype, with reference, beta, T, smoothing, upstream gradient
    (1, 1, "fp32", True, 1.0, 1.0, 0.0, 1.0),
    (3, 5, "bf16", False, 0.5, 2.0, 0.1, 1.0),      # below one vector
    (2, 8, "fp16", True, 1.0, 1.0, 0.0, 1.0),
    (5, 9, "bf16", True, 1.0, 1.0, 0.2, -2.0),      # one vector and a moved one
    (1, 30522, "bf16", True, 1.0, 40.0, 0.0, 1.0),  # one row, split over many workgroups
    (32, 30522, "bf16", True, 1.0, 40.0, 0.0, 1.0),
    (7, 30523, "fp16", True, 2.0, 40.0, 0.1, 1024.0),
    (33, 4099, "fp32", False, 0.1, 10.0, 0.5, 0.5),
    (2049, 301, "bf16", True, 1.0, 3.0, 0.0, 1.0),  # more rows than workgroups, one chunk each
    (1500, 64, "fp32", True, 1.0, 3.0, 0.05, 1.0),
    (3, 250002, "bf16", True, 1.0, 120.0, 0.0, 1.0),
]


@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_preference_matches_64_bits(case, device):
    B, V, dt, with_ref, beta, T, eps, up = case
    say(f"preference loss {case}")
    q, p, n, ref = make(B, V, dt, device)
    check((q, p, n, ref if with_ref else None), beta, T, eps, up)


def test_preference_extreme_margins(device):
    """Margins of hundreds either way: no overflow, a vanishing gradient on the right side and slope one on
    the wrong one."""
    say("extreme margins")
    q, p, n, ref = make(4, 500, "fp32", device, scale=3.0)
    p[0] += 1.0
    n[1] += 1.0
    got = check((q, p, n, ref), T=0.5)
    assert bool(torch.isfinite(got["loss"]))
    check((q, p, n, ref), T=0.5, eps=0.25)


def test_preference_equal_documents(device):
    """pos == neg: margin 0, loss log 2, dq = 0 and opposite document gradients."""
    say("equal documents")
    q, p, _, _ = make(6, 1000, "bf16", device)
    got = run(q, p, p, None, 1.0, 1.0, 0.0)
    assert float(got["loss"]) == pytest.approx(math.log(2.0), rel=2.0 ** -21)
    assert torch.count_nonzero(got["margin"]) == 0 and torch.count_nonzero(got["dq"]) == 0
    assert torch.equal(got["dp"], -got["dn"]) and torch.count_nonzero(got["dp"]) > 0


def test_preference_margin_is_the_losses(device):
    say("margins")
    q, p, n, ref = make(9, 5000, "fp16", device)
    m = preference_margin(q.requires_grad_(), p, n, 3.0)
    assert not m.requires_grad and torch.equal(m, run(q.detach(), p, n, None, 1.0, 3.0, 0.0)["margin"])
    got = run(q.detach(), p, n, m, 1.0, 3.0, 0.0)  # a model against itself: z = 0
    assert float(got["loss"]) == pytest.approx(math.log(2.0), rel=2.0 ** -21)


def test_preference_nan_stays_in_its_row(device):
    say("NaN in one row")
    q, p, n, ref = make(8, 3000, "bf16", device)
    want = run(q, p, n, ref, 1.0, 20.0, 0.0)
    q2 = q.clone()
    q2[3, 17] = float("nan")
    got = run(q2, p, n, ref, 1.0, 20.0, 0.0)
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert bool(got["loss"].isnan()) and bool(got["margin"][3].isnan())
    for name in ("margin", "dq", "dp", "dn"):
        assert torch.equal(got[name][keep], want[name][keep])


def test_preference_shared_and_strided(device):
    """One query for every pair (stride 0), slices of a wider buffer, the same reps as query and document."""
    say("shared, strided")
    q, p, n, ref = make(5, 777, "fp32", device)
    q1 = q[:1].clone().requires_grad_()
    res = preference_loss(q1.expand(5, -1), p, n, ref, temperature=5.0)
    (d,) = torch.autograd.grad(res.loss, q1)
    whole = run(q[:1].expand(5, -1).contiguous(), p, n, ref, 1.0, 5.0, 0.0)
    tol = 5 * E * whole["dq"].abs().sum(0)
    assert torch.equal(res.loss, whole["loss"]) and bool(((d[0] - whole["dq"].double().sum(0)).abs() <= tol).all())
    buf = torch.empty(5, 3 * 777, device=device)
    views = [buf[:, i * 777:(i + 1) * 777].copy_(t) for i, t in enumerate((q, p, n))]
    got, want = run(*views, ref, 1.0, 5.0, 0.0), run(q, p, n, ref, 1.0, 5.0, 0.0)
    assert all(torch.equal(got[k], want[k]) for k in want)
    x = q.clone().requires_grad_()
    (dx,) = torch.autograd.grad(preference_loss(x, x, n, ref, temperature=5.0).loss, x)
    parts = run(q, q, n, ref, 1.0, 5.0, 0.0)
    assert torch.equal(dx, parts["dq"] + parts["dp"])


def test_preference_gradients_against_differences(device):
    say("differences")
    q, p, n, ref = make(6, 400, "fp32", device)
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g).to(device) * 0.2 for t in (q, p, n)]
    got, want = run(q, p, n, ref, 1.0, 10.0, 0.1), reference(q, p, n, ref, 1.0, 10.0, 0.1)
    names = ("dq", "dp", "dn")
    along = sum(float((got[k].double() * d.double()).sum()) for k, d in zip(names, dirs))
    exact = sum(float((want[k][0] * d.double()).sum()) for k, d in zip(names, dirs))
    tol = sum(float((want[k][1] * d.double().abs()).sum()) for k, d in zip(names, dirs))
    h, v, v64 = 2.0 ** -6, [], []
    for s in (1, -1):
        moved = [t + s * h * d for t, d in zip((q, p, n), dirs)]
        value, t = reference(*moved, ref, 1.0, 10.0, 0.1)["loss"]
        v.append(float(preference_loss(*moved, ref, temperature=10.0, label_smoothing=0.1).loss))
        v64.append(float(value))
        tol += (float(t) + E * abs(float(value))) / (2 * h)
    tol += abs((v64[0] - v64[1]) / (2 * h) - exact)
    assert abs(along - (v[0] - v[1]) / (2 * h)) <= tol


def test_preference_deterministic_op_and_compile(device):
    say("deterministic, opcheck, compile")
    q, p, n, ref = make(40, 30522, "bf16", device)
    a, b = run(q, p, n, ref, 1.0, 40.0, 0.0), run(q, p, n, ref, 1.0, 40.0, 0.0)
    loss, margin, coef = torch.ops.sparton.preference_fwd(q, p, n, ref, 40.0, 1.0, 0.0)
    grads = torch.ops.sparton.preference_bwd(torch.ones((), device=device), q, p, n, coef)
    for k, t in zip(("loss", "margin", "dq", "dp", "dn"), (loss, margin, *grads)):
        assert torch.equal(a[k], b[k]) and torch.equal(a[k], t), k
    q, p, n, ref = make(4, 200, "fp32", device)
    ql = q.clone().requires_grad_()
    torch.library.opcheck(torch.ops.sparton.preference_fwd, (ql, p, n, ref, 5.0, 1.0, 0.1),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = lambda x: preference_loss(x, p, n, ref, temperature=5.0).loss * 2
    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    assert torch.equal(torch.autograd.grad(cf(ql), ql)[0], torch.autograd.grad(f(ql), ql)[0])


def test_preference_graph_replays(device):
    say("graph")
    sets = [make(16, 30522, "bf16", device, seed=s) for s in range(3)]
    held = [t.clone() for t in sets[0]]
    up = torch.ones((), device=device)

    def step():
        loss, margin, coef = torch.ops.sparton.preference_fwd(*held, 40.0, 1.0, 0.0)
        return (loss, margin, *torch.ops.sparton.preference_bwd(up, *held[:3], coef))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for s in (1, 2, 0):
        for t, new in zip(held, sets[s]):
            t.copy_(new)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_preference_margin_compiles(device):
    say("margin, compile")
    q, p, n, _ = make(5, 300, "bf16", device)
    f = lambda a, b, c: preference_margin(a, b, c, 3.0) * 2
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(q.requires_grad_(), p, n)
    assert not got.requires_grad and torch.equal(got, f(q, p, n))
