"""GPU parity of the gated feed-forward product against its formulas in 64 bits.

Small integers first: x, weights and dh in {-1, 0, 1} with relu make g, u, dg and du integers that every type holds,
and all sums exact in fp32, so every result has to be the exact one rounded once.

Tolerances otherwise, with u = eps / 2 of the type (half a step, relative) and E = 2^-24: a product is an fp32 sum,
    eg = (D + 2) E (|x| |Wg|' + |bg|), eu likewise
    8 bits: + 4 E |g| for the scales; and the matrix instructions align the products of eight neighbours to the
    largest one's power of two 2^e and drop what is below 2^(e - 13) of the seven others (measured: beside a product
    of 2^16 one of 2^3 counts and one of 2^2 does not; eight places further all do), so at most
    7 * 2^-13 sum over the eights of max |x| max |w|, before the scales
    the activations are evaluated to rho = (16 + 8 g^2 + |g|^3) E of themselves (arguments rounded once: erfc and exp
    of -t change by about t^2 and t times that), and have slopes up to 1.15 and curvatures up to 1:
    ea = 1.15 eg + rho |a|,  ed = eg + rho (1 + |a'|)
    h:  |u| ea + |a| eu + ea eu + (E + u) |h|
    du: |dh| ea + E |du| =: fu;  dg: |dh| (|u| ed + |a'| eu + ed eu) + 2 E |dg| =: fg
    dx: (fg + u |dg|) |Wg| + (fu + u |du|) |Wu| + (2 F + 8) E (|dg| |Wg| + |du| |Wu|) + u |dx|
    dW: (fg + u |dg|)' |x| + (M + 8) E |dg|' |x| + u |dW|;  db: sum fg + (M + 8) E sum |dg| + u |db|
These are worst cases. Roundings are as often up as down, so in the 2-norm the error of each result is also held to
3 u (dg or du, the result) of it, and in fp32 to 2^-18."""
import pytest
import torch

from _parity import say
from sparton_amd.feed_forward import SpartonGatedMLP, gated_linear, gated_linear_8bit, quantize_rows

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24
NAMES = ("dx", "dwg", "dwu", "dbg", "dbu")


def make(M, D, F, dt, device, bias=False, seed=0, whole=False):
    g = torch.Generator().manual_seed(seed + 7 * M + D + F)
    if whole:
        rand = lambda *n: torch.randint(-1, 2, n, generator=g).float()
        x, wg, wu, dh, bg, bu = rand(M, D), rand(F, D), rand(F, D), rand(M, F), rand(F), rand(F)
    else:
        rand = lambda *n: torch.randn(*n, generator=g)
        x, wg, wu, dh = rand(M, D), rand(F, D) * D ** -0.5, rand(F, D) * D ** -0.5, rand(M, F) * 0.1
        bg, bu = rand(F) * 0.3, rand(F) * 0.3
    both = (bg, bu) if bias else (None, None)
    return [None if t is None else t.to(DT[dt]).to(device) for t in (x, wg, wu, *both, dh)]


def act(g, name):
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[name]
    leaf = g.detach().requires_grad_()
    with torch.enable_grad():
        a = f(leaf)
        (d,) = torch.autograd.grad(a.sum(), leaf)
    return a.detach(), d


def reference(x, wg, wu, bg, bu, dh, name, scales=None, out=None):
    """name -> (value, tolerance); scales (x's, w_gate's, w_up's) of e4m3 rows, whose result is of type `out`."""
    u = torch.finfo(out or x.dtype).eps / 2
    sub = 2.0 ** -25 if (out or x.dtype) == torch.float16 else 2.0 ** -126
    X, WG, WU, DH = (None if t is None else t.float().double() for t in (x, wg, wu, dh))
    M, D, F = X.shape[0], X.shape[1], WG.shape[0]
    if scales is not None:
        X, WG, WU = (t * s.double()[:, None] for t, s in zip((X, WG, WU), scales))
    g, v = X @ WG.t().contiguous(), X @ WU.t().contiguous()
    eg, ev = (D + 2) * E * (X.abs() @ WG.abs().t().contiguous()), (D + 2) * E * (X.abs() @ WU.abs().t().contiguous())
    if bg is not None:
        g, eg = g + bg.double(), eg + (D + 2) * E * bg.double().abs()
    if bu is not None:
        v, ev = v + bu.double(), ev + (D + 2) * E * bu.double().abs()
    if scales is not None:
        top = lambda t: torch.nn.functional.pad(t.abs(), (0, -D % 8)).view(t.shape[0], -1, 8).amax(-1)
        eg = eg + 4 * E * g.abs() + 7 * 2.0 ** -13 * (top(X) @ top(WG).t().contiguous())
        ev = ev + 4 * E * v.abs() + 7 * 2.0 ** -13 * (top(X) @ top(WU).t().contiguous())
    a, d = act(g, name)
    rho = (16 + 8 * g * g + g.abs() ** 3) * E
    ea, ed = 1.15 * eg + rho * a.abs(), eg + rho * (1 + d.abs())
    if name == "relu":  # the slope jumps where g's sign may be the other one
        ed = ed + (g.abs() <= eg).double()
    h = a * v
    res = {"h": (h, v.abs() * ea + a.abs() * ev + ea * ev + (E + u) * h.abs() + sub)}
    if DH is None:
        return res
    du, dg = DH * a, DH * v * d
    fu = DH.abs() * ea + E * du.abs() + sub
    fg = DH.abs() * (v.abs() * ed + d.abs() * ev + ed * ev) + 2 * E * dg.abs() + sub
    ru, rg = fu + u * du.abs(), fg + u * dg.abs()
    dx = dg @ WG + du @ WU
    res["dx"] = dx, rg @ WG.abs() + ru @ WU.abs() + (2 * F + 8) * E * (dg.abs() @ WG.abs() + du.abs() @ WU.abs()) + u * dx.abs() + sub
    for n, t, r, f in (("g", dg, rg, fg), ("u", du, ru, fu)):
        dw = t.t().contiguous() @ X
        res["dw" + n] = dw, r.t().contiguous() @ X.abs() + (M + 8) * E * (t.abs().t().contiguous() @ X.abs()) + u * dw.abs() + sub
        res["db" + n] = t.sum(0), f.sum(0) + (M + 8) * E * t.abs().sum(0) + u * t.sum(0).abs() + sub
    return res


def run(x, wg, wu, bg, bu, dh, name):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = gated_linear(*leaves, activation=name)
    have = [(n, t) for n, t in zip(NAMES, leaves) if t is not None]
    grads = torch.autograd.grad(h, [t for _, t in have], dh)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, wg, wu, bg, bu, activation=name).nan_to_num(), h.nan_to_num())
    torch.cuda.synchronize()
    return dict(h=h.detach(), **{n: t for (n, _), t in zip(have, grads)})


def check(args, name):
    x, wg = args[:2]
    got, want = run(*args, name), reference(*args, name)
    worst = []
    most = 2.0 ** -18 if x.dtype == torch.float32 else 3 * torch.finfo(x.dtype).eps / 2
    for n, t in got.items():
        value, tol = want[n]
        assert t.dtype == x.dtype and t.shape == value.shape
        if not t.numel():
            continue
        ratio = float(((t.double() - value).abs() / tol).max())
        off = float((t.double() - value).norm() / value.norm().clamp_min(1e-30))
        assert ratio <= 1.0, f"{n}: {ratio:.2f} times the tolerance"
        assert off <= most or name == "relu", f"{n}: off by {off:.2e} in the 2-norm"
        worst.append(f"{n} {ratio:.2f} ({off:.1e})")
    say("   of the tolerance: " + ", ".join(worst))
    return got


SIZES = [  # M, D, F: few rows, both tile sizes, every edge within and at a tile, split inner dimensions
    (1, 8, 1), (1, 64, 32), (3, 72, 33), (16, 768, 100), (32, 8, 64), (33, 200, 65), (64, 1000, 31), (65, 64, 64), (65, 8, 1),
    (100, 136, 127), (128, 128, 128), (129, 72, 129), (200, 1024, 257), (257, 768, 300), (300, 520, 1000), (1000, 64, 2048),
    (512, 256, 4000), (2049, 264, 1500), (4096, 128, 3000), (1500, 2048, 1100), (405, 280, 13097), (11459, 672, 97),
    (68, 536, 9814), (2984, 1424, 920), (6642, 1864, 65), (2505, 1544, 2664), (5442, 1616, 1175),
    (6181, 1760, 5774), (11978, 1728, 3322), (8373, 136, 9767), (13143, 520, 745),
]


@pytest.mark.parametrize("M,D,F", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
@pytest.mark.parametrize("dt", list(DT))
def test_gated_of_small_integers_is_exact(dt, M, D, F, device):
    """Every product's layout: one element out of place shows."""
    say(f"gated integers {M} {D} {F} {dt}")
    args = make(M, D, F, dt, device, bias=M % 2 == 1, whole=True)
    got, want = run(*args, "relu"), reference(*args, "relu")
    assert float(want["h"][0].abs().max()) < 2 ** 24
    for n, t in got.items():
        assert torch.equal(t, want[n][0].to(t.dtype)), n


CASES = [  # M, D, F, dtype, activation, biases
    (1, 64, 40, "bf16", "silu", True), (5, 768, 100, "fp16", "gelu", False), (17, 1000, 257, "fp32", "gelu_tanh", True),
    (50, 72, 96, "bf16", "gelu", True), (64, 768, 2051, "bf16", "silu", False), (65, 768, 130, "fp16", "silu", True),
    (181, 384, 300, "fp32", "silu", False), (300, 768, 1000, "bf16", "gelu_tanh", False), (1000, 768, 2051, "fp32", "gelu_tanh", True),
    (2000, 264, 1100, "bf16", "silu", True), (2100, 512, 2048, "fp16", "gelu", True), (700, 1001, 515, "bf16", "silu", True),
    (90, 33, 70, "fp32", "gelu", True), (4100, 1024, 1030, "bf16", "gelu", False), (260, 2048, 5000, "fp16", "relu", False),
]


@pytest.mark.parametrize("M,D,F,dt,name,bias", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_gated_matches_64_bits(M, D, F, dt, name, bias, device):
    say(f"gated {M} {D} {F} {dt} {name} bias={bias}")
    check(make(M, D, F, dt, device, bias), name)


E4M3_SIZES = [(1, 16, 1), (5, 64, 33), (32, 768, 100), (33, 144, 65), (64, 1000, 96), (65, 128, 64), (100, 272, 127),
              (129, 4096, 129), (300, 768, 1000), (3000, 256, 2100), (200, 33, 70), (679, 72, 5466)]


@pytest.mark.parametrize("M,D,F", E4M3_SIZES, ids=["-".join(map(str, s)) for s in E4M3_SIZES])
@pytest.mark.parametrize("out", list(DT))
def test_gated_8bit(out, M, D, F, device):
    say(f"gated 8 bits {M} {D} {F} -> {out}")
    x, wg, wu, *_ = make(M, D, F, "fp32", device, whole=True)
    to = torch.float8_e4m3fn
    ones = [torch.ones(n, device=device) for n in (M, F, F)]
    h = gated_linear_8bit(x.to(to), ones[0], wg.to(to), ones[1], wu.to(to), ones[2], "relu", DT[out])
    assert torch.equal(h, reference(x, wg, wu, None, None, None, "relu")["h"][0].to(DT[out]))
    x, wg, wu, *_ = make(M, D, F, "fp32", device)
    parts = [quantize_rows(t) for t in (x, wg, wu)]
    h = gated_linear_8bit(*(t for p in parts for t in p), "silu", DT[out])
    value, tol = reference(*(p[0] for p in parts), None, None, None, "silu", [p[1] for p in parts], DT[out])["h"]
    assert h.dtype == DT[out] and h.shape == (M, F)
    ratio = float(((h.double() - value).abs() / tol).max())
    assert ratio <= 1.0, f"{ratio:.2f} times the tolerance"


def test_gated_shapes_strides_and_alignment(device):
    say("shapes")
    x, wg, wu, bg, bu, dh = make(60, 96, 72, "bf16", device, bias=True)
    want = run(x, wg, wu, bg, bu, dh, "silu")
    h = gated_linear(x.view(3, 4, 5, 96), wg, wu, bg, bu)
    assert h.shape == (3, 4, 5, 72) and torch.equal(h.view(60, 72), want["h"])
    both = torch.cat([wg, wu])
    wide = torch.empty(60, 200, dtype=x.dtype, device=device)[:, 3:99].copy_(x)
    odd = torch.empty(60 * 96 + 1, dtype=x.dtype, device=device)[1:].view(60, 96).copy_(x)
    across = dh.t().contiguous().t()
    for xx in (wide, odd, x.t().contiguous().t()):
        got = run(xx, both[:72], both[72:], torch.cat([bu, bg])[72:], bu, across, "silu")
        assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("M", [0, 1, 70])
def test_gated_empty(M, device):
    say(f"empty {M}")
    x, wg, wu, bg, bu, dh = make(M, 64, 40, "bf16", device, bias=True)
    if M == 0:
        got = run(x, wg, wu, bg, bu, dh, "silu")
        assert got["h"].shape == (0, 40) and got["dx"].shape == (0, 64)
        assert all(torch.count_nonzero(got[n]) == 0 for n in NAMES[1:])
    got = run(x, wg[:0], wu[:0], bg[:0], bu[:0], dh[:, :0], "silu")
    assert got["h"].shape == (M, 0) and torch.count_nonzero(got["dx"]) == 0 and got["dwg"].shape == (0, 64)


def test_gated_nan_stays_in_its_rows_and_columns(device):
    say("NaN")
    for M in (40, 300):
        x, wg, wu, _, _, dh = make(M, 96, 200, "bf16", device)
        want = gated_linear(x, wg, wu)
        x[7, 5], wu[11, 3], wg[190, 95] = float("nan"), float("inf"), float("nan")
        got = gated_linear(x, wg, wu)
        rows, cols = torch.arange(M, device=device) != 7, torch.ones(200, dtype=torch.bool, device=device)
        cols[11] = cols[190] = False
        assert torch.equal(got[rows][:, cols], want[rows][:, cols])
        assert bool(got[7].isnan().all()) and bool(got[:, 190].isnan().all())


def test_gated_what_is_needed(device):
    """Gradients of some inputs only, and a step with none."""
    say("some gradients")
    x, wg, wu, bg, bu, dh = make(100, 64, 48, "bf16", device, bias=True)
    want = run(x, wg, wu, bg, bu, dh, "silu")
    for ask in ("dx", "dwg", "dwu", "dbg", "dbu"):
        leaves = [t.detach().requires_grad_(n == ask) for n, t in zip(NAMES, (x, wg, wu, bg, bu))]
        h = gated_linear(*leaves)
        (g,) = torch.autograd.grad(h, [t for t in leaves if t.requires_grad], dh)
        assert torch.equal(g, want[ask]), ask
    assert not gated_linear(x, wg, wu, bg, bu).requires_grad
    w = wg.detach().requires_grad_()  # one tensor as both weights: the sum
    (g,) = torch.autograd.grad(gated_linear(x, w, w), w, dh)
    each = run(x, wg, wg, None, None, dh, "silu")
    torch.testing.assert_close(g, each["dwg"] + each["dwu"], rtol=0, atol=0)


def test_gated_deterministic_and_op_equals_function(device):
    say("deterministic")
    for M, D, F, dt in ((700, 768, 515, "bf16"), (200, 64, 100, "fp32")):
        x, wg, wu, bg, bu, dh = make(M, D, F, dt, device, bias=True)
        a, b = run(x, wg, wu, bg, bu, dh, "gelu"), run(x, wg, wu, bg, bu, dh, "gelu")
        h, g, u = torch.ops.sparton.gated_fwd(x, wg, wu, bg, bu, "gelu")
        grads = torch.ops.sparton.gated_bwd(dh, x, wg, wu, g, u, "gelu", True, True)
        for n, t in zip(("h", *NAMES), (h, *grads)):
            assert torch.equal(a[n], b[n]) and torch.equal(a[n], t), n


def test_gated_against_differences(device):
    say("differences")
    args = make(9, 40, 30, "fp32", device, bias=True)
    dh, name = args[-1], "gelu"
    g = torch.Generator().manual_seed(3)
    dirs = [torch.randn(t.shape, generator=g).to(device) for t in args[:5]]
    got, want = run(*args, name), reference(*args, name)
    step = 2.0 ** -9
    along = sum(float((got[n].double() * d.double()).sum()) for n, d in zip(NAMES, dirs))
    exact = sum(float((want[n][0] * d.double()).sum()) for n, d in zip(NAMES, dirs))
    tol = sum(float((want[n][1] * d.double().abs()).sum()) for n, d in zip(NAMES, dirs))
    v, v64 = [], []
    for s in (1, -1):
        moved = [t + s * step * d for t, d in zip(args[:5], dirs)]
        value, t = reference(*moved, None, name)["h"]
        with torch.no_grad():
            v.append(float((dh.double() * gated_linear(*moved, activation=name).double()).sum()))
        v64.append(float((dh.double() * value).sum()))
        tol += float((dh.double().abs() * t).sum()) / (2 * step)
    tol += abs((v64[0] - v64[1]) / (2 * step) - exact)
    assert abs(along - (v[0] - v[1]) / (2 * step)) <= tol


def test_gated_autocast_and_module(device):
    say("module")
    class Block(torch.nn.Module):
        def __init__(self, act_fn):
            super().__init__()
            self.gate_proj, self.up_proj = (torch.nn.Linear(64, 96, bias=b) for b in (True, False))
            self.down_proj, self.act_fn = torch.nn.Linear(96, 64), act_fn
        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))
    for act_fn in (torch.nn.SiLU(), torch.nn.GELU(), torch.nn.GELU(approximate="tanh"), torch.nn.ReLU()):
        block = Block(act_fn).to(device)
        ours = SpartonGatedMLP.of(block)
        assert list(ours.state_dict()) == list(block.state_dict()) and ours.up_proj.weight is block.up_proj.weight
        x = torch.randn(3, 50, 64, device=device)
        torch.testing.assert_close(ours(x), block(x), rtol=1e-4, atol=1e-5)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert ours(x).dtype == torch.bfloat16
        ours(x).sum().backward()
        assert block.gate_proj.weight.grad.dtype == torch.float32
    with pytest.raises(ValueError, match="activation"):
        SpartonGatedMLP.of(Block(torch.nn.Tanh()))


def test_gated_opcheck_and_compile(device):
    say("opcheck, compile")
    x, wg, wu, bg, bu, dh = make(20, 64, 48, "fp32", device, bias=True)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    torch.library.opcheck(torch.ops.sparton.gated_fwd, (*leaves, bg, None, "silu"),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = lambda *t: gated_linear(*t, bg, bu) * 2
    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    for p, q in zip(torch.autograd.grad(cf(*leaves), leaves, dh), torch.autograd.grad(f(*leaves), leaves, dh)):
        assert torch.equal(p, q)
