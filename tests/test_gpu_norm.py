"""GPU parity of LayerNorm with the residual sum against its formulas in 64 bits.

Tolerances, with u = eps / 2 of a type (half a step, relative): mean and variance are fp32 sums of D
terms, so with h = x + r (one fp32 rounding), c = h - mean and s2 = var + eps
    |mean error|  <= (D + 2) 2^-24 mean|h|                          =: em
    |c error|     <= em + 2^-24 (|h| + |c|)                          =: ec
    rstd, relative: half of var's error, (D + 4) 2^-24 + 2 mean(|c| ec) / s2, and 2^-22 for the root =: er
    |xhat error|  <= rstd ec + |xhat| er                             =: ex
    y:  |w| ex + (2^-23) (|xhat w| + |b|) + u |y|
    g = dy w, c1 = mean g, c2 = mean(g xhat), t = g - c1 - xhat c2:
        c1: (D + 2) 2^-24 mean|g| =: e1;  c2: mean(|g| ex) + (D + 2) 2^-24 mean|g xhat| =: e2
        dx: rstd (e1 + |xhat| e2 + ex |c2| + 4 2^-24 (|g| + |c1| + |xhat c2|)) + |dx| (er + u)
    dw: sum |dy| ex + (M + 4) 2^-24 sum |dy xhat| + u |dw|;  db: (M + 4) 2^-24 sum |dy| + u |db|
"""
import pytest
import torch

from _parity import say
from sparton_amd.norm import SpartonLayerNorm, layer_norm

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def make(shape, dt, vec, device, residual=True, bias=True, seed=0, offset=0.0):
    g = torch.Generator().manual_seed(seed + shape[-1])
    rand = lambda *n: torch.randn(*n, generator=g)
    D, t = shape[-1], DT[dt]
    vt = torch.float32 if vec == "fp32" else t
    x, dy = (rand(*shape) + offset).to(t), (rand(*shape) * 0.05).to(t)
    r = rand(*shape).to(t) if residual else None
    w, b = (1 + 0.1 * rand(D)).to(vt), (0.1 * rand(D)).to(vt) if bias else None
    return [None if a is None else a.to(device) for a in (x, r, w, b, dy)]


def reference(x, r, w, b, dy, eps):
    t, vt, D = x.dtype, w.dtype, x.shape[-1]
    u, uv = torch.finfo(t).eps / 2, torch.finfo(vt).eps / 2
    f = lambda a: None if a is None else a.detach().double().reshape(-1, D) if a.dim() > 1 else a.detach().double()
    X, R, DY = (None if a is None else a.detach().double().reshape(-1, D) for a in (x, r, dy))
    W, Bv = w.detach().double(), None if b is None else b.detach().double()
    M = X.shape[0]
    h = X if R is None else X + R
    mean = h.mean(-1, keepdim=True)
    c = h - mean
    s2 = (c * c).mean(-1, keepdim=True) + eps
    rstd = s2 ** -0.5
    xh = c * rstd
    em = (D + 2) * E * h.abs().mean(-1, keepdim=True)
    ec = em + E * (h.abs() + c.abs())
    er = 0.5 * ((D + 4) * E + 2 * (c.abs() * ec).mean(-1, keepdim=True) / s2) + 2.0 ** -22
    ex = rstd * ec + xh.abs() * er
    y = xh * W + (0 if Bv is None else Bv)
    tol = {"y": W.abs() * ex + 2 * E * ((xh * W).abs() + (0 if Bv is None else Bv.abs())) + u * y.abs()}
    g = DY * W
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    e1 = (D + 2) * E * g.abs().mean(-1, keepdim=True)
    e2 = (g.abs() * ex).mean(-1, keepdim=True) + (D + 2) * E * (g * xh).abs().mean(-1, keepdim=True)
    tol["dx"] = (rstd * (e1 + xh.abs() * e2 + ex * c2.abs() + 4 * E * (g.abs() + c1.abs() + (xh * c2).abs()))
                 + dx.abs() * (er + u))
    dw, db = (DY * xh).sum(0), DY.sum(0)
    tol["dw"] = (DY.abs() * ex).sum(0) + (M + 4) * E * (DY * xh).abs().sum(0) + uv * dw.abs()
    tol["db"] = (M + 4) * E * DY.abs().sum(0) + uv * db.abs()
    sub = 2.0 ** -25 if t == torch.float16 else 2.0 ** -126
    return {n: (a, tol[n] + sub) for n, a in (("y", y), ("dx", dx), ("dw", dw), ("db", db))}


def run(x, r, w, b, dy, eps):
    leaves = [a.detach().requires_grad_() for a in (x, r, w, b) if a is not None]
    it = iter(leaves)
    xl, rl, wl, bl = (next(it) if a is not None else None for a in (x, r, w, b))
    y = layer_norm(xl, wl, bl, eps, rl)
    grads = dict(zip([n for n, a in zip(("dx", "dr", "dw", "db"), (x, r, w, b)) if a is not None],
                     torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps, r), y)
    torch.cuda.synchronize()
    return dict(y=y.detach(), **grads)


def check(args, eps=1e-5):
    x, r, w, b, dy = args
    got, want = run(*args, eps), reference(*args, eps)
    worst = []
    for n in got:
        value, tol = want["dx" if n == "dr" else n]
        a = got[n].double().reshape(value.shape)
        assert got[n].dtype == (x.dtype if n in ("y", "dx", "dr") else w.dtype)
        ratio = float(((a - value).abs() / tol).max()) if a.numel() else 0.0
        assert ratio <= 1.0, f"{n}: {ratio:.2f} times the tolerance"
        worst.append(f"{n} {ratio:.2f}")
    if r is not None:
        assert torch.equal(got["dx"], got["dr"])
    say("   of the tolerance: " + ", ".join(worst))
    return got


CASES = [  # shape, dtype, vectors, residual, bias
    ((1, 1), "fp32", "same", False, True),           # one element: xhat = 0
    ((3, 2), "bf16", "same", True, True),            # rows below one vector
    ((5, 7), "fp16", "fp32", True, False),
    ((4, 3), "fp32", "same", True, True),
    ((1, 8), "bf16", "fp32", False, True),
    ((9, 9), "bf16", "same", True, True),            # one vector and a moved one
    ((33, 100), "fp32", "same", False, False),
    ((2, 17, 768), "bf16", "same", True, True),
    ((4, 50, 768), "fp16", "fp32", True, True),
    ((300, 768), "fp32", "same", True, True),
    ((70, 1000), "bf16", "same", False, True),
    ((70, 1023), "bf16", "fp32", True, True),        # odd rows: no vector is aligned
    ((41, 1025), "fp16", "same", True, True),        # four waves a row
    ((5, 2047), "fp32", "same", False, True),
    ((6, 2049), "bf16", "same", True, True),         # eight waves a row
    ((130, 4096), "bf16", "fp32", False, True),
    ((3, 6304), "fp16", "same", True, True),
    ((3, 8195), "fp32", "same", False, True),
    ((2, 16384), "bf16", "same", True, True),        # the widest
    ((2, 16383), "fp32", "same", True, True),
    ((5000, 384), "bf16", "fp32", True, True),       # more rows than waves
    ((20001, 64), "fp16", "same", True, True),
]


@pytest.mark.parametrize("shape,dt,vec,res,bias", CASES, ids=["-".join(map(str, (*c[0], *c[1:]))) for c in CASES])
def test_norm_matches_64_bits(shape, dt, vec, res, bias, device):
    say(f"layer_norm {shape} {dt} {vec} residual={res} bias={bias}")
    check(make(shape, dt, vec, device, res, bias))


def test_norm_of_offset_and_constant_rows(device):
    """A mean far larger than the deviations, eps that decides, and constant rows."""
    say("offset rows")
    check(make((20, 768), "fp32", "same", device, residual=False, offset=300.0))
    check(make((20, 768), "bf16", "same", device, offset=-50.0), eps=1e-12)
    x, r, w, b, dy = make((6, 768), "fp32", "same", device, residual=False)
    got = run(torch.full_like(x, 2.5), None, w, b, dy, 1e-5)
    assert torch.equal(got["y"], b.expand_as(x))


def test_norm_empty(device):
    say("no rows")
    got = run(*make((0, 64), "bf16", "same", device), 1e-5)
    assert got["y"].shape == (0, 64) and torch.count_nonzero(got["dw"]) == 0 and torch.count_nonzero(got["db"]) == 0


def test_norm_strided_and_unaligned(device):
    """Views (a slice of columns, a transposed batch, rows that start anywhere): the contiguous result's bits."""
    say("strided")
    x, r, w, b, dy = make((12, 30, 96), "bf16", "same", device)
    want = run(x, r, w, b, dy, 1e-5)
    wide = torch.empty(12, 30, 200, dtype=x.dtype, device=device)[..., 3:99].copy_(x)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=device)[1:].view(x.shape).copy_(x)
    wo = torch.empty(97, dtype=w.dtype, device=device)[1:].copy_(w)
    for t in (wide, swapped, odd):
        got = run(t, r, wo, b, dy, 1e-5)
        assert all(torch.equal(got[n], want[n]) for n in want)
    got = run(x, r, w, b, dy.transpose(0, 1).contiguous().transpose(0, 1), 1e-5)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_norm_broadcast_weight_and_shared_input(device):
    """x as its own residual gets both gradients; a weight used twice gets their sum."""
    say("shared inputs")
    x, _, w, b, dy = make((10, 64), "fp32", "same", device, residual=False)
    one = run(x, x, w, b, dy, 1e-5)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(layer_norm(xl, wl, b, 1e-5, xl), (xl, wl), dy)
    assert torch.equal(dx, 2 * one["dx"]) and torch.equal(dw, one["dw"])
    y = layer_norm(xl, wl, b, 1e-5, xl) + layer_norm(xl, wl, b, 1e-5, xl)
    assert torch.equal(torch.autograd.grad(y, wl, dy)[0], 2 * one["dw"])


def test_norm_gradients_against_differences(device):
    """Directional derivative against central differences of the fp32 forward; the tolerance is the
    differences' own error in 64 bits, the forward's over h, and the gradients' along the direction."""
    say("differences")
    x, r, w, b, up = make((9, 70), "fp32", "same", device)
    g = torch.Generator().manual_seed(3)
    args, names = [x, r, w, b], ("dx", "dr", "dw", "db")
    dirs = [torch.randn(t.shape, generator=g).to(device) for t in args]
    got, want = run(x, r, w, b, up, 1e-5), reference(x, r, w, b, up, 1e-5)
    want["dr"] = want["dx"]
    h = 2.0 ** -7
    along = sum(float((got[n].double() * d.double()).sum()) for n, d in zip(names, dirs))
    exact = sum(float((want[n][0] * d.double()).sum()) for n, d in zip(names, dirs))
    tol = sum(float((want[n][1] * d.double().abs()).sum()) for n, d in zip(names, dirs))
    v, v64 = [], []
    for s in (1, -1):
        mx, mr, mw, mb = (t + s * h * d for t, d in zip(args, dirs))
        y, ty = reference(mx, mr, mw, mb, up, 1e-5)["y"]
        with torch.no_grad():
            v.append(float((up.double() * layer_norm(mx, mw, mb, 1e-5, mr).double()).sum()))
        v64.append(float((up.double() * y).sum()))
        tol += float((up.double().abs() * ty).sum()) / (2 * h)
    tol += abs((v64[0] - v64[1]) / (2 * h) - exact)
    assert abs(along - (v[0] - v[1]) / (2 * h)) <= tol


def test_norm_nan_stays_in_its_row(device):
    say("NaN in one row")
    x, r, w, b, dy = make((40, 768), "bf16", "same", device)
    want = run(x, r, w, b, dy, 1e-5)
    x2 = x.clone()
    x2[7, 5], x2[9, 700] = float("nan"), float("inf")
    with torch.no_grad():
        y = layer_norm(x2, w, b, 1e-5, r)
    rows = torch.ones(40, dtype=torch.bool)
    rows[7] = rows[9] = False
    assert torch.equal(y[rows.to(device)], want["y"][rows.to(device)])
    assert bool(y[7].isnan().all()) and bool(y[9].isnan().any())


def test_norm_deterministic_and_op_equals_function(device):
    say("deterministic")
    x, r, w, b, dy = make((3001, 768), "bf16", "fp32", device)
    a, c = run(x, r, w, b, dy, 1e-12), run(x, r, w, b, dy, 1e-12)
    y, mean, rstd = torch.ops.sparton.layer_norm_fwd(x, r, w, b, 1e-12)
    dx, dw, db = torch.ops.sparton.layer_norm_bwd(dy, x, r, w, True, mean, rstd)
    for n, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert torch.equal(a[n], c[n]) and torch.equal(a[n], t), n


def test_norm_module(device):
    """SpartonLayerNorm.of shares the module's parameters; autocast and two dtypes as torch has them."""
    say("module")
    ln = torch.nn.LayerNorm(256, eps=1e-12).to(device)
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5)
        ln.bias.uniform_(-1, 1)
    m = SpartonLayerNorm.of(ln)
    assert m.weight is ln.weight and list(m.state_dict()) == ["weight", "bias"] and isinstance(m, torch.nn.LayerNorm)
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(10, 256, generator=g).to(device) for _ in range(2))
    for y, h in ((m(x), x), (m(x, r), x + r)):
        v, tol = reference(h, None, ln.weight, ln.bias, h, 1e-12)["y"]
        assert bool(((y.double() - v).abs() <= 2 * tol).all())  # twice: h itself was rounded once more for the reference
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m(x.bfloat16(), r).dtype == torch.float32
        assert torch.equal(m(x.bfloat16(), r), m(x.bfloat16().float(), r))
    assert torch.equal(m(x.bfloat16(), r), m(x.bfloat16().float(), r))  # bf16 + fp32 is fp32
    mixed = m(x.bfloat16(), r.bfloat16())
    assert mixed.dtype == torch.bfloat16
    mixed.float().sum().backward()
    assert ln.weight.grad.dtype == torch.float32 and torch.isfinite(ln.weight.grad).all()
    half = SpartonLayerNorm.of(torch.nn.LayerNorm(256).to(device, torch.float16))
    assert half(x).dtype == torch.float32 and half(x.half()).dtype == torch.float16


def test_norm_opcheck_and_compile(device):
    say("opcheck, compile")
    x, r, w, b, dy = make((6, 5, 64), "fp32", "same", device)
    xl = x.clone().requires_grad_()
    torch.library.opcheck(torch.ops.sparton.layer_norm_fwd, (xl, r, w, b, 1e-5),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = lambda a, c: layer_norm(a, c, b, 1e-5, r) * 2
    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    wl = w.clone().requires_grad_()
    for p, q in zip(torch.autograd.grad(cf(xl, wl), (xl, wl), dy), torch.autograd.grad(f(xl, wl), (xl, wl), dy)):
        assert torch.equal(p, q)


def test_norm_graph_replays(device):
    say("graph")
    sets = [make((100, 768), "bf16", "same", device, seed=s) for s in range(3)]
    held = [t.clone() for t in sets[0]]

    def step():
        x, r, w, b, dy = held
        y, mean, rstd = torch.ops.sparton.layer_norm_fwd(x, r, w, b, 1e-5)
        return (y, *torch.ops.sparton.layer_norm_bwd(dy, x, r, w, True, mean, rstd))

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
        assert all(torch.equal(a, c) for a, c in zip(outs, want))


@pytest.mark.parametrize("D", [5, 301, 907, 1501, 3001, 6007, 12001])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_norm_with_more_rows_than_workgroups(dt, D, device):
    """Each width's kernels for each type, where a workgroup takes several rows (the forward's at 4096 rows of one
    wave, 1024 of four, 512 of eight; the backward's at 2048, 512 and 256)."""
    M = 4500 if D <= 1024 else 1100
    say(f"layer_norm {M} x {D} {dt}")
    check(make((M, D), dt, "fp32" if D % 3 else "same", device))
