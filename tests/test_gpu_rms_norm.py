"""GPU parity of the root-mean-square norm against its formulas in 64 bits.

Tolerances, with u = eps / 2 of a type (half a step, relative) and E = 2^-24: h = x + r is one fp32 rounding, the
mean of squares an fp32 sum of D positive terms, so with s2 = mean(h^2) + eps
    rstd, relative: (D + 6) E / 2 + 2^-22 for the root =: er
    y:  |y| (er + 4 E + u);   h: |h| (E + u)
    xhat = h rstd, of the stored h (rounded to u where there is a residual): |xhat| ex, ex = er + 2 E (+ u)
    g = dy w, c = mean(g xhat): ec = mean|g xhat| (ex + (D + 4) E)
    dx: rstd (|xhat| ec + |xhat c| ex + ...), in full in the test; dw: sum |dy xhat| (ex + (M + 4) E) + u |dw|
    8 bits: a value is off by half a step, 2^-4 of it, or 2^-10 scale below e4m3's normal range (2^-6 scale);
            scale: (er + 6 E) of it"""
import pytest
import torch

from _parity import say
from sparton_amd.norm import SpartonRMSNorm, rms_norm, rms_norm_8bit

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def make(shape, dt, vec, device, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed + shape[-1])
    rand = lambda *n: torch.randn(*n, generator=g)
    D, t = shape[-1], DT[dt]
    x, dy, dh = rand(*shape).to(t), (rand(*shape) * 0.05).to(t), (rand(*shape) * 0.05).to(t)
    r = rand(*shape).to(t) if residual else None
    w = (1 + 0.1 * rand(D)).to(torch.float32 if vec == "fp32" else t)
    return [None if a is None else a.to(device) for a in (x, r, w, dy, dh)]


def reference(x, r, w, dy, dh, eps):
    t, D = x.dtype, x.shape[-1]
    u, uv = torch.finfo(t).eps / 2, torch.finfo(w.dtype).eps / 2
    X, R, DY, DH = (None if a is None else a.detach().double().reshape(-1, D) for a in (x, r, dy, dh))
    W, M = w.detach().double(), X.shape[0]
    h = X if R is None else X + R
    q = ((h * h).mean(-1, keepdim=True) + eps) ** -0.5
    xh = h * q
    er = (D + 6) * E / 2 + 2.0 ** -22
    ex = er + 2 * E + (u if R is not None else 0.0)
    y = xh * W
    g = DY * W
    c = (g * xh).mean(-1, keepdim=True)
    ec = (g * xh).abs().mean(-1, keepdim=True) * (ex + (D + 4) * E)
    dx = q * (g - xh * c)
    tdx = q * (xh.abs() * ec * (1 + ex) + (xh * c).abs() * ex + 4 * E * (g.abs() + (xh * c).abs())) + dx.abs() * er
    if R is not None:
        dx = dx + DH
        tdx = tdx + E * (dx.abs() + DH.abs())
    tdx = tdx + u * (dx.abs() + tdx)
    dw = (DY * xh).sum(0)
    tdw = (DY * xh).abs().sum(0) * (ex + (M + 4) * E) + uv * dw.abs()
    sub = 2.0 ** -25 if t == torch.float16 else 2.0 ** -126
    out = {"y": (y, y.abs() * (er + 4 * E + u)), "h": (h, h.abs() * (E + u)), "dx": (dx, tdx), "dw": (dw, tdw)}
    return {n: (a, b + sub) for n, (a, b) in out.items()}


def run(x, r, w, dy, dh, eps):
    leaves = [a.detach().requires_grad_() for a in (x, r, w) if a is not None]
    out = rms_norm(leaves[0], leaves[-1], eps, leaves[1] if r is not None else None)
    outs, ups = ([out], [dy]) if r is None else (list(out), [dy, dh])
    grads = torch.autograd.grad(outs, leaves, ups)
    with torch.no_grad():
        again = rms_norm(x, w, eps, r)
    for a, b in zip(outs, [again] if r is None else again):
        assert torch.equal(a.detach().nan_to_num(), b.nan_to_num())
    torch.cuda.synchronize()
    got = dict(zip(["y", "h"], (o.detach() for o in outs)))
    got.update(zip(["dx", "dr", "dw"] if r is not None else ["dx", "dw"], grads))
    return got


def check(args, eps=1e-6):
    x, r, w, dy, dh = args
    got, want = run(*args, eps), reference(*args, eps)
    worst = []
    for n in got:
        value, tol = want["dx" if n == "dr" else n]
        assert got[n].dtype == (w.dtype if n == "dw" else x.dtype) and got[n].shape == (w.shape if n == "dw" else x.shape)
        a = got[n].double().reshape(value.shape)
        ratio = float(((a - value).abs() / tol).max()) if a.numel() else 0.0
        assert ratio <= 1.0, f"{n}: {ratio:.2f} times the tolerance"
        worst.append(f"{n} {ratio:.2f}")
    if r is not None:
        assert torch.equal(got["dx"], got["dr"])
    say("   of the tolerance: " + ", ".join(worst))
    return got


CASES = [  # shape, dtype, weight, residual
    ((1, 1), "fp32", "same", False), ((3, 2), "bf16", "same", True), ((5, 7), "fp16", "fp32", True),
    ((4, 3), "fp32", "same", True), ((1, 8), "bf16", "fp32", False), ((9, 9), "bf16", "same", True),
    ((33, 100), "fp32", "same", False), ((2, 17, 768), "bf16", "same", True), ((4, 50, 768), "fp16", "fp32", True),
    ((300, 768), "fp32", "same", True), ((70, 1023), "bf16", "fp32", True), ((41, 1025), "fp16", "same", True),
    ((5, 2047), "fp32", "same", False), ((6, 2049), "bf16", "same", True), ((130, 4096), "bf16", "fp32", False),
    ((3, 6304), "fp16", "same", True), ((3, 8195), "fp32", "same", True), ((2, 16384), "bf16", "same", True),
    ((2, 16383), "fp32", "same", True), ((20001, 64), "fp16", "same", True),
]


@pytest.mark.parametrize("shape,dt,vec,res", CASES, ids=["-".join(map(str, (*c[0], *c[1:]))) for c in CASES])
def test_rms_norm_matches_64_bits(shape, dt, vec, res, device):
    say(f"rms_norm {shape} {dt} {vec} residual={res}")
    check(make(shape, dt, vec, device, res))


@pytest.mark.parametrize("D", [5, 301, 907, 1501, 3001, 6007, 12001])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_rms_norm_with_more_rows_than_workgroups(dt, D, device):
    M = 4500 if D <= 1024 else 1100
    say(f"rms_norm {M} x {D} {dt}")
    check(make((M, D), dt, "fp32" if D % 3 else "same", device))


def test_rms_norm_of_large_small_and_zero_rows(device):
    say("large, small, zero")
    x, r, w, dy, dh = make((20, 768), "fp32", "same", device)
    check([1e10 * x, 1e10 * r, w, dy, dh])
    check([1e-10 * x, 1e-10 * r, w, dy, dh], eps=1e-5)
    got = run(0 * x, 0 * r, w, dy, dh, 1e-6)
    assert torch.count_nonzero(got["y"]) == 0 and torch.count_nonzero(got["dw"]) == 0
    torch.testing.assert_close(got["dx"], dh + dy * w * 1e3, rtol=1e-5, atol=0)


def test_rms_norm_of_one_output(device):
    """A loss that reads only the rows, or only the sum."""
    say("one output")
    x, r, w, dy, dh = make((30, 200), "bf16", "same", device)
    both = run(x, r, w, dy, torch.zeros_like(dh), 1e-6)
    leaves = [a.detach().requires_grad_() for a in (x, r, w)]
    y, h = rms_norm(leaves[0], leaves[2], 1e-6, leaves[1])
    dx, dr, dw = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert torch.equal(dx, both["dx"]) and torch.equal(dr, dx) and torch.equal(dw, both["dw"])
    dx, dr, dw = torch.autograd.grad(h, leaves, dh, allow_unused=True)
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and dw is None


def test_rms_norm_empty(device):
    say("no rows")
    got = run(*make((0, 64), "bf16", "same", device), 1e-6)
    assert got["y"].shape == (0, 64) and torch.count_nonzero(got["dw"]) == 0
    y, scale, h = rms_norm_8bit(*(make((0, 64), "bf16", "same", device)[i] for i in (0, 2)), 1e-6,
                                make((0, 64), "bf16", "same", device)[1])
    assert y.shape == (0, 64) and scale.shape == (0,) and h.shape == (0, 64)


def test_rms_norm_strided_and_unaligned(device):
    say("strided")
    x, r, w, dy, dh = make((12, 30, 96), "bf16", "same", device)
    want = run(x, r, w, dy, dh, 1e-6)
    wide = torch.empty(12, 30, 200, dtype=x.dtype, device=device)[..., 3:99].copy_(x)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=device)[1:].view(x.shape).copy_(x)
    wo = torch.empty(97, dtype=w.dtype, device=device)[1:].copy_(w)
    back = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    for t in (wide, swapped, odd):
        got = run(t, back(r), wo, back(dy), back(dh), 1e-6)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_rms_norm_of_one_tensor_twice(device):
    say("x as its own residual")
    x, _, w, dy, dh = make((10, 64), "fp32", "same", device, residual=False)
    one = run(x, x, w, dy, dh, 1e-6)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(rms_norm(xl, wl, 1e-6, xl), (xl, wl), (dy, dh))
    assert torch.equal(dx, 2 * one["dx"]) and torch.equal(dw, one["dw"])


def test_rms_norm_against_differences(device):
    say("differences")
    x, r, w, up, uph = make((9, 70), "fp32", "same", device)
    g = torch.Generator().manual_seed(3)
    args, names = [x, r, w], ("dx", "dr", "dw")
    dirs = [torch.randn(t.shape, generator=g).to(device) for t in args]
    got, want = run(x, r, w, up, uph, 1e-6), reference(x, r, w, up, uph, 1e-6)
    want["dr"] = want["dx"]
    step = 2.0 ** -7
    along = sum(float((got[n].double() * d.double()).sum()) for n, d in zip(names, dirs))
    exact = sum(float((want[n][0] * d.double()).sum()) for n, d in zip(names, dirs))
    tol = sum(float((want[n][1] * d.double().abs()).sum()) for n, d in zip(names, dirs))
    v, v64 = [], []
    for s in (1, -1):
        mx, mr, mw = (t + s * step * d for t, d in zip(args, dirs))
        ref = reference(mx, mr, mw, up, uph, 1e-6)
        with torch.no_grad():
            y, h = rms_norm(mx, mw, 1e-6, mr)
        v.append(float((up.double() * y.double() + uph.double() * h.double()).sum()))
        v64.append(float((up.double() * ref["y"][0] + uph.double() * ref["h"][0]).sum()))
        tol += float((up.double().abs() * ref["y"][1] + uph.double().abs() * ref["h"][1]).sum()) / (2 * step)
    tol += abs((v64[0] - v64[1]) / (2 * step) - exact)
    assert abs(along - (v[0] - v[1]) / (2 * step)) <= tol


def test_rms_norm_nan_stays_in_its_row(device):
    say("NaN in one row")
    x, r, w, dy, dh = make((40, 768), "bf16", "same", device)
    want = run(x, r, w, dy, dh, 1e-6)
    want8 = [t.float() for t in rms_norm_8bit(x, w, 1e-6, r)]
    x2 = x.clone()
    x2[7, 5], x2[9, 700] = float("nan"), float("inf")
    rows = torch.ones(40, dtype=torch.bool)
    rows[7] = rows[9] = False
    rows = rows.to(device)
    with torch.no_grad():
        y, h = rms_norm(x2, w, 1e-6, r)
        y8, scale, _ = rms_norm_8bit(x2, w, 1e-6, r)
    assert torch.equal(y[rows], want["y"][rows]) and torch.equal(h[rows], want["h"][rows])
    assert bool(y[7].isnan().all()) and bool(y[9, 700].isnan())
    assert torch.equal(y8.float()[rows], want8[0][rows]) and torch.equal(scale[rows], want8[1][rows])
    assert bool(y8.float()[7].isnan().all()) and bool(y8.float()[9, 700].isnan())


def test_rms_norm_deterministic_and_op_equals_function(device):
    say("deterministic")
    x, r, w, dy, dh = make((3001, 768), "bf16", "fp32", device)
    a, c = run(x, r, w, dy, dh, 1e-6), run(x, r, w, dy, dh, 1e-6)
    y, h, q = torch.ops.sparton.rms_norm_fwd(x, r, w, 1e-6)
    dx, dw = torch.ops.sparton.rms_norm_bwd(dy, dh, h, w, q)
    for n, t in (("y", y), ("h", h), ("dx", dx), ("dw", dw)):
        assert torch.equal(a[n], c[n]) and torch.equal(a[n], t), n


@pytest.mark.parametrize("shape,dt,vec,res", CASES, ids=["-".join(map(str, (*c[0], *c[1:]))) for c in CASES])
def test_rms_norm_8bit_matches_64_bits(shape, dt, vec, res, device):
    say(f"rms_norm_8bit {shape} {dt} {vec} residual={res}")
    x, r, w, dy, dh = make(shape, dt, vec, device, res)
    out = rms_norm_8bit(x, w, 1e-6, r)
    D = shape[-1]
    er = (D + 6) * E / 2 + 2.0 ** -22 + 6 * E
    want, _ = reference(x, r, w, dy, dh, 1e-6)["y"]
    y8, scale = out[0], out[1]
    assert y8.dtype == torch.float8_e4m3fn and y8.shape == x.shape and scale.shape == x.shape[:-1]
    s64 = want.abs().amax(-1) / 448.0
    assert bool(((scale.reshape(-1).double() - s64).abs() <= er * s64).all())
    got = y8.float().double().reshape(want.shape) * scale.double().reshape(-1, 1)
    tol = torch.maximum(want.abs() * 2.0 ** -4, 2.0 ** -10 * s64[:, None]) * (1 + 4 * er) + want.abs() * 4 * er
    assert bool(((got - want).abs() <= tol).all())
    assert bool((y8.float().abs().amax(-1) == 448.0).all())
    if res:
        assert torch.equal(out[2], run(x, r, w, dy, dh, 1e-6)["h"])


def test_rms_norm_8bit_of_zero_and_tiny_rows(device):
    say("8 bits: zero, tiny")
    x, _, w, _, _ = make((6, 100), "fp32", "same", device, residual=False)
    x[1] = 0.0
    x[2] *= 1e-42
    y8, scale = rms_norm_8bit(x, w, 1e-6)
    assert torch.count_nonzero(y8.float()[1]) == 0 and float(scale[1]) == 2.0 ** -126
    assert bool(y8.float().isfinite().all()) and bool((scale >= 2.0 ** -126).all())
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm_8bit(x.requires_grad_(), w, 1e-6)


def test_rms_norm_module(device):
    say("module")
    class Theirs(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.weight = torch.nn.Parameter(torch.rand(256) + 0.5)
            self.variance_epsilon = 1e-5
    theirs = Theirs().to(device)
    m = SpartonRMSNorm.of(theirs)
    assert m.weight is theirs.weight and list(m.state_dict()) == ["weight"] and m.eps == 1e-5
    x, r, _, dy, dh = make((10, 256), "fp32", "same", device)
    y, h = m(x, r)
    assert torch.equal(h, x + r) and torch.equal(y, rms_norm(x, theirs.weight, 1e-5, r)[0])
    y, h = m(x.bfloat16(), r)
    assert y.dtype == h.dtype == torch.float32
    m(x.bfloat16()).float().sum().backward()
    assert theirs.weight.grad.dtype == torch.float32
    assert SpartonRMSNorm(16, device=device, dtype=torch.float16)(x[:, :16]).dtype == torch.float32


def test_rms_norm_opcheck_and_compile(device):
    say("opcheck, compile")
    x, r, w, dy, dh = make((6, 5, 64), "fp32", "same", device)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    for res in (r, None):
        torch.library.opcheck(torch.ops.sparton.rms_norm_fwd, (xl, res, w, 1e-6),
                              test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    torch.library.opcheck(torch.ops.sparton.rms_norm_8bit, (x, r, w, 1e-6), test_utils=("test_schema", "test_faketensor"))

    def f(a, c):
        y, h = rms_norm(a, c, 1e-6, r)
        return (y * 2 + h).sin() + rms_norm(a, c)
    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    for p, q in zip(torch.autograd.grad(cf(xl, wl), (xl, wl), dy), torch.autograd.grad(f(xl, wl), (xl, wl), dy)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("through", ["y", "h", "both"])
def test_rms_norm_leaves_do_not_share_a_gradient(through, device):
    """x and the residual have equal gradients, in memory of their own: scaling one (clipping) leaves the other."""
    say(f"two leaves {through}")
    x, r = (torch.randn(40, 96, device=device, requires_grad=True) for _ in range(2))
    w = torch.ones(96, device=device, requires_grad=True)
    y, h = rms_norm(x, w, 1e-6, r)
    ((y.square().sum() if through != "h" else 0) + (h.square().sum() if through != "y" else 0)).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    before = r.grad.clone()
    x.grad.mul_(2.0)
    assert torch.equal(r.grad, before)


@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_changed_before_its_backward(residual, device):
    """The backward reads h, or x where there is no residual: changed in place in between, autograd raises."""
    say(f"changed in place, residual={residual}")
    x, r = (torch.randn(4, 96, device=device, requires_grad=True) for _ in range(2))
    w = torch.ones(96, device=device, requires_grad=True)
    a = x * 1.0
    y, h = rms_norm(a, w, 1e-6, r) if residual else (rms_norm(a, w), a)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
