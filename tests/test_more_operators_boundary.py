"""CPU checks of the RMS norm, embedding and gated product's entry points: what the C ABI refuses (before any HIP
call, with addresses that are never read), what the Python functions refuse, and their fakes."""
import pytest
import torch
from torch import nn

import sparton_amd
from sparton_amd import _lib
from sparton_amd.embedding import SpartonEmbedding, embedding
from sparton_amd.feed_forward import (SpartonGatedMLP, activation_name, gated_linear, gated_linear_8bit, quantize_rows)
from sparton_amd.norm import SpartonRMSNorm, rms_norm, rms_norm_8bit

P = 0x10000  # 16- and 256-byte aligned address that is never read


# ---- the RMS norm -------------------------------------------------------------------------

def rfwd(**kw):
    a = dict(x=P, r=P, w=P, vec=0, eps=1e-6, y=P, h=P, q=P, M=4, D=64, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_rms_norm_fwd(*a.values())


def rquant(**kw):
    a = dict(x=P, r=P, w=P, vec=0, eps=1e-6, y=P, scale=P, h=P, M=4, D=64, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_rms_norm_fwd_quantized(*a.values())


def rbwd(**kw):
    a = dict(dy=P, dh=P, h=P, w=P, vec=0, q=P, dx=P, dw=P, ws=P, ws_bytes=1 << 30, M=4, D=64, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_rms_norm_bwd(*a.values())


BOTH = [
    (dict(M=-1), -1), (dict(D=0), -1), (dict(dtype=3), -1), (dict(vec=2), -1), (dict(x=None), -1), (dict(w=None), -1),
    (dict(y=None), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1),
    (dict(D=16385), -3), (dict(M=1 << 60), -3), (dict(x=P + 1), -2), (dict(w=P + 2), -2), (dict(h=P + 1), -2),
    (dict(M=0), 0), (dict(vec=1, w=P + 1), -2),
]


@pytest.mark.parametrize("kw,code", BOTH)
def test_rms_norm_fwd_checks(kw, code):
    assert rfwd(**kw) == code and rquant(**kw) == code


def test_rms_norm_fwd_checks_of_one():
    assert rfwd(q=P + 2) == -2 and rfwd(y=P + 1) == -2
    assert rquant(scale=None) == -1 and rquant(scale=P + 2) == -2
    assert rquant(y=P + 1, x=P + 1) == -2 and rquant(y=P + 1, M=0) == 0  # bytes lie anywhere


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(dtype=-1), -1), (dict(vec=2), -1), (dict(dy=None), -1), (dict(h=None), -1), (dict(dx=None), -1),
    (dict(q=None), -1), (dict(D=20000), -3), (dict(ws=None), -4), (dict(ws_bytes=8), -4), (dict(ws=P + 16), -2),
    (dict(dy=P + 1), -2), (dict(dh=P + 1), -2), (dict(dw=P + 2), -2), (dict(M=0, dw=None), 0),
])
def test_rms_norm_bwd_checks(kw, code):
    assert rbwd(**kw) == code


def test_rms_norm_workspace():
    size = _lib.load().sparton_rms_norm_workspace_bytes
    assert size(0, 64) == 0 and size(5, 0) == 0 and size(5, 20000) == 0
    assert size(1, 768) == 768 * 4
    assert size(10 ** 9, 4096) <= 512 * 4096 * 4


@pytest.mark.parametrize("f", [rms_norm, rms_norm_8bit])
@pytest.mark.parametrize("args,kw,error", [
    ((torch.zeros(3, 8).double(), torch.ones(8).double()), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(9)), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8).half()), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), dict(residual=torch.zeros(8)), ValueError),  # no broadcast
    ((torch.zeros(3, 8), torch.ones(8)), dict(residual=torch.zeros(3, 8).half()), ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), dict(eps=-1e-5), ValueError),
    ((torch.zeros(3, 0), torch.ones(0)), {}, ValueError),
    ((torch.zeros(3, 16385), torch.ones(16385)), {}, ValueError),
    ((torch.zeros(()), torch.ones(1)), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), {}, RuntimeError),
    ((torch.zeros(3, 8), torch.ones(8)), dict(residual=torch.zeros(3, 8)), RuntimeError),
])
def test_rms_norm_refusals(f, args, kw, error):
    with pytest.raises(error):
        f(*args, **kw)


def test_rms_norm_module_surface():
    class Theirs(nn.Module):
        def __init__(self, shape=(32,), **kw):
            super().__init__()
            self.weight = nn.Parameter(torch.ones(shape))
            for k, v in kw.items():
                setattr(self, k, v)
    theirs = Theirs(variance_epsilon=1e-5)
    m = SpartonRMSNorm.of(theirs)
    assert m.weight is theirs.weight and m.eps == 1e-5 and list(m.state_dict()) == ["weight"]
    assert SpartonRMSNorm.of(nn.RMSNorm(16, eps=1e-3)).eps == 1e-3 and sparton_amd.SpartonRMSNorm is SpartonRMSNorm
    for bad in (Theirs((4, 8), eps=1e-5), Theirs(), Theirs(eps=None), nn.Identity(), Theirs(16400, eps=1e-5)):
        with pytest.raises(ValueError):
            SpartonRMSNorm.of(bad)
    with pytest.raises(ValueError):
        SpartonRMSNorm(16385)
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        m(torch.zeros(2, 32))


# ---- the embedding ------------------------------------------------------------------------

def efwd(**kw):
    a = dict(ids=P, ids_dtype=0, table=P, scale=1.0, out=P, N=8, V=100, D=64, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_embedding_fwd(*a.values())


def ebwd(**kw):
    a = dict(ids=P, ids_dtype=0, dy=P, scale=1.0, pad=-1, dw=P, ws=P, ws_bytes=1 << 40, N=8, V=100, D=64, dtype=1,
             stream=None)
    a.update(kw)
    return _lib.load().sparton_embedding_bwd(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(N=-1), -1), (dict(V=-1), -1), (dict(D=0), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(ids_dtype=2), -1),
    (dict(ids_dtype=3), -1), (dict(ids=None), -1), (dict(ids=P + 4), -2), (dict(ids=P + 2, ids_dtype=1), -2),
    (dict(V=2 ** 31 - 1), -3), (dict(N=2 ** 31), -3), (dict(D=(1 << 20) + 1), -3), (dict(N=1 << 30, D=1 << 20), -3),
    (dict(V=2 ** 31 - 2, D=1 << 20), -3),  # a wave a row of the table
])
def test_embedding_checks(kw, code):
    assert efwd(**kw) == code and ebwd(**kw) == code


def test_embedding_checks_of_one():
    assert efwd(table=None) == -1 and efwd(out=None) == -1 and efwd(out=P + 1) == -2 and efwd(table=P + 1) == -2
    assert efwd(N=0, ids=None) == 0
    assert ebwd(dy=None) == -1 and ebwd(dw=None) == -1 and ebwd(dw=P + 1) == -2 and ebwd(dy=P + 1) == -2
    assert ebwd(ws=None) == -4 and ebwd(ws_bytes=64) == -4 and ebwd(ws=P + 16) == -2 and ebwd(V=0, dw=None) == 0


def test_embedding_forward_has_its_own_limits():
    """The join's workgroups, 256 threads for each 32 ids, bound the backward: 2^37 / 256 ids of narrow rows."""
    N = 2 ** 29
    assert ebwd(N=N, dy=None) == -3 and efwd(N=N, out=None) == -1  # accepted as far as the missing address
    assert ebwd(N=N - 32, dy=None) == -1
    size = _lib.load().sparton_embedding_workspace_bytes
    assert size(N, 100, 64, 1) == 0 and size(N - 32, 100, 64, 1) > 0
    assert efwd(N=2 ** 31 - 1025, D=64, out=None) == -1 and efwd(N=2 ** 31 - 1025, D=72, out=None) == -3


def test_embedding_workspace():
    size = _lib.load().sparton_embedding_workspace_bytes
    assert size(0, 100, 64, 1) == 0 and size(8, 100, 0, 1) == 0 and size(8, 100, 64, 7) == 0
    assert size(8, 100, 64, 1) == 4 * 256 + 2 * 64 * 4
    assert size(65536, 30522, 768, 1) == 4 * 65536 * 4 + 2048 * 2 * 768 * 4


IDS, TABLE = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)


@pytest.mark.parametrize("args,kw,error", [
    ((IDS.to(torch.int16), TABLE), {}, TypeError),
    ((IDS.float(), TABLE), {}, TypeError),
    ((IDS, TABLE.double()), {}, TypeError),
    ((IDS, TABLE[0]), {}, ValueError),
    ((IDS, TABLE[:, :0]), {}, ValueError),
    ((IDS, TABLE), dict(scale=float("inf")), ValueError),
    ((IDS, TABLE), dict(scale=float("nan")), ValueError),
    ((IDS, TABLE), dict(padding_idx=5), ValueError),
    ((IDS, TABLE), dict(padding_idx=-6), ValueError),
    ((IDS, TABLE), {}, RuntimeError),
    ((IDS, TABLE), dict(padding_idx=-1), RuntimeError),
])
def test_embedding_refusals(args, kw, error):
    with pytest.raises(error):
        embedding(*args, **kw)


@pytest.mark.parametrize("scale", [1e39, -1e39, 1e308])
def test_an_embeddings_scale_past_fp32_is_refused(scale):
    """The kernel's factor is fp32: it would be infinite."""
    with pytest.raises(ValueError, match="finite"):
        embedding(IDS, TABLE, scale=scale)
    with pytest.raises(ValueError, match="finite"):
        torch.ops.sparton.embedding_bwd(TABLE[:3], IDS, 5, scale, -1)


def test_embedding_module_surface():
    m = nn.Embedding(10, 8, padding_idx=2)
    ours = SpartonEmbedding.of(m)
    assert ours.weight is m.weight and ours.padding_idx == 2 and ours.scale == 1.0 and isinstance(ours, nn.Embedding)
    assert list(ours.state_dict()) == ["weight"] and sparton_amd.SpartonEmbedding is SpartonEmbedding
    assert SpartonEmbedding(10, 8, scale=3).scale == 3.0
    for kw in (dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        with pytest.raises(ValueError, match="SpartonEmbedding"):
            SpartonEmbedding.of(nn.Embedding(10, 8, **kw))
        with pytest.raises(ValueError, match="SpartonEmbedding"):
            SpartonEmbedding(10, 8, **kw)
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        ours(IDS)


# ---- the gated product --------------------------------------------------------------------

def gfwd(**kw):
    a = dict(x=P, wg=P, wu=P, bg=P, bu=P, act=0, h=P, g=P, u=P, M=4, D=64, F=32, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_gated_fwd(*a.values())


def gquant(**kw):
    a = dict(x=P, sx=P, wg=P, sg=P, wu=P, su=P, act=0, h=P, M=4, D=64, F=32, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_gated_fwd_quantized(*a.values())


def gbwd(**kw):
    a = dict(dh=P, x=P, wg=P, wu=P, g=P, u=P, act=0, dx=P, dwg=P, dwu=P, dbg=P, dbu=P, ws=P, ws_bytes=1 << 40, M=4, D=64,
             F=32, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_gated_bwd(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(D=0), -1), (dict(F=-1), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(act=4), -1),
    (dict(act=-1), -1), (dict(D=60), -1), (dict(x=None), -1), (dict(wg=None), -1), (dict(wu=None), -1),
    (dict(x=P + 8), -2), (dict(wg=P + 8), -2), (dict(wu=P + 4), -2), (dict(D=1 << 21), -3), (dict(F=1 << 21), -3),
    (dict(M=1 << 31), -3), (dict(M=1 << 30, F=1 << 20), -3), (dict(D=1 << 20, F=1 << 20), -3),
])
def test_gated_checks(kw, code):
    assert gfwd(**kw) == code and gbwd(**kw) == code
    assert gquant(**kw) == code


def test_gated_checks_of_one():
    assert gfwd(g=None) == -1 and gfwd(h=None) == -1 and gfwd(h=P + 1) == -2 and gfwd(bg=P + 1) == -2 and gfwd(u=P + 2) == -2
    assert gfwd(M=0, x=None) == 0 and gfwd(F=0, wg=None) == 0 and gfwd(D=62, dtype=0) == -1
    assert gquant(sx=None) == -1 and gquant(su=P + 2) == -2 and gquant(D=72) == -1 and gquant(M=0) == 0
    assert gbwd(dh=None) == -1 and gbwd(g=None) == -1 and gbwd(dwg=None) == -1 and gbwd(dx=P + 1) == -2
    assert gbwd(ws=None) == -4 and gbwd(ws_bytes=16) == -4 and gbwd(ws=P + 16) == -2
    assert gbwd(F=0) == -3 and gbwd(F=0, dx=None, dwg=None, dwu=None) == 0


def test_gated_workspace():
    size = _lib.load().sparton_gated_workspace_bytes
    assert size(0, 64, 32, 0, 1) == 0 and size(4, 60, 32, 0, 1) == 0 and size(4, 64, 0, 0, 1) == 0
    # dg and du; of dW's 1408 tiles the 128 that do not fill the CUs once more are split in two
    assert size(8192, 4096, 11264, 0, 1) == 2 * 8192 * 11264 * 2 + 128 * 2 * 256 * 256 * 4
    assert size(8192, 4096, 8192, 0, 1) == 2 * 8192 * 8192 * 2       # whole rounds: no partial sums
    assert size(4, 64, 33, 0, 1) == 2 * 4 * 40 * 2 + -(2 * 4 * 40 * 2) % 256  # rows padded to 16 bytes
    assert size(4, 64, 33, 1, 1) > size(4, 64, 33, 0, 1)
    assert size(8192, 768, 2048, 0, 1) == 2 * 8192 * 2048 * 2
    assert size(300, 768, 2048, 0, 1) > 2 * 300 * 2048 * 2           # few tiles: dx splits its inner dimension


def split_of(rows, cols, turns, slabs, es, may_split):
    """(128 x 128 tiles, splits, tiles that are split): the rule of sparton_gated.hip once more."""
    cdiv, best = lambda a, b: -(-a // b), None
    for small in (0, 1):
        b, slots = (128, 512) if small else (256, 256)
        tiles = cdiv(rows, b) * cdiv(cols, b) * turns
        rest, around = tiles % slots, 6.0 if small else 10.0
        every = (3.6 if small else 7.3) if es == 4 else (0.9 if small else 1.45)
        some = (1.95 if small else 7.3) if es == 4 else (0.5 if small else 1.3)
        for n in range(1, 17):
            per, groups = cdiv(slabs, n), rest * n
            if n > 1 and (not may_split or rest == 0 or slabs < 4 * n or cdiv(slabs, per) != n or groups > 2 * slots):
                continue
            time = tiles // slots * (slabs * every + around)
            if rest:
                time += cdiv(groups, slots) * (per * (some if groups < 256 or (small and groups == 256) else every) + around)
            if n > 1:
                time += 3.0 + 0.03 * time + rest * b * b * (8.0 * n + 2.0) / 6e6
            if best is None or time < best[0]:
                best = (time, small == 1, n, rest if n > 1 else 0)
    return best[1:]


def few(M):
    """Blocks of 16 rows of the kernel for few of them."""
    return 1 if M <= 16 else 2 if M <= 32 else 4


def gated_kernels(M, D, F, dt):
    """The kernels that a training step of these sizes launches: (product, type, 128 x 128 tiles, which of them are
    split: none, all or the last)."""
    cdiv, es = lambda a, b: -(-a // b), 4 if dt == "fp32" else 2
    D += -D % (16 // es)
    fwd = ("few", dt, few(M), None) if M <= (32 if F * D > 1 << 23 else 64) else ("fwd", dt, split_of(M, 2 * F, 1, cdiv(D * es, 128), es, False)[0], None)
    dx, dw = split_of(M, D, 1, 2 * cdiv(F * es, 128), es, True), split_of(F, D, 2, cdiv(M * es, 128), es, True)
    b = {True: 128, False: 256}
    which = lambda s, rows, turns: None if s[1] == 1 else "all" if s[2] == cdiv(rows, b[s[0]]) * cdiv(D, b[s[0]]) * turns else "last"
    return {fwd, ("dx", dt, dx[0], which(dx, M, 1)), ("dw", dt, dw[0], which(dw, F, 2))}


def test_the_gated_cases_reach_every_kernel():
    from test_gpu_gated import E4M3_SIZES, SIZES
    every = {(p, dt, small, split) for p in ("dx", "dw") for dt in ("fp32", "bf16", "fp16") for small in (True, False)
             for split in (None, "all", "last")}
    every |= {("fwd", dt, small, None) for dt in ("fp32", "bf16", "fp16") for small in (True, False)}
    every |= {("few", dt, blocks, None) for dt in ("fp32", "bf16", "fp16") for blocks in (1, 2, 4)}
    got = set().union(*(gated_kernels(*s, dt) for s in SIZES for dt in ("fp32", "bf16", "fp16")))
    assert got == every, every ^ got
    bits8 = {("few", few(M)) if M <= 64 else ("fwd", split_of(M, 2 * F, 1, -(-(D + -D % 16) // 128), 1, False)[0])
             for M, D, F in E4M3_SIZES}
    assert bits8 == {("fwd", True), ("fwd", False), ("few", 1), ("few", 2), ("few", 4)}


def test_the_rule_above_is_the_librarys():
    """The workspace tells how the inner dimensions are split."""
    from test_gpu_gated import CASES, SIZES
    cdiv, up = lambda a, b: -(-a // b), lambda n: n + -n % 256
    for M, D, F, dt in [*((*s, dt) for s in SIZES for dt in ("fp32", "bf16")), *(c[:4] for c in CASES),
                        (8192, 768, 2048, "bf16"), (512, 4096, 11264, "bf16"), (2048, 768, 1152, "fp16")]:
        es = 4 if dt == "fp32" else 2
        D, Fp = D + -D % (16 // es), F + -F % (16 // es)
        both = split_of(M, D, 1, 2 * cdiv(F * es, 128), es, True), split_of(F, D, 2, cdiv(M * es, 128), es, True)
        part = max(shared * n * (128 if small else 256) ** 2 * 4 for small, n, shared in both)
        got = _lib.load().sparton_gated_workspace_bytes(M, D, F, 0, ("fp32", "bf16", "fp16").index(dt))
        assert got == up(2 * M * Fp * es) + part, (M, D, F, dt)


X, W = torch.zeros(3, 8), torch.zeros(6, 8)


@pytest.mark.parametrize("args,kw,error", [
    ((X, W, W), dict(activation="tanh"), ValueError),
    ((X, W, W[:5]), {}, ValueError),
    ((X, W[:, :7], W[:, :7]), {}, ValueError),
    ((X, W[0], W[0]), {}, ValueError),
    ((torch.zeros(()), W, W), {}, ValueError),
    ((X[:, :0], W[:, :0], W[:, :0]), {}, ValueError),
    ((X, W.half(), W.half()), {}, TypeError),
    ((X.double(), W.double(), W.double()), {}, TypeError),
    ((X, W, W, torch.zeros(6).half()), {}, TypeError),
    ((X, W, W, torch.zeros(5)), {}, ValueError),
    ((X, W, W, None, torch.zeros(6, 1)), {}, ValueError),
    ((X, W, W), {}, RuntimeError),
    ((X, W, W, torch.zeros(6), torch.zeros(6)), dict(activation="gelu"), RuntimeError),
])
def test_gated_refusals(args, kw, error):
    with pytest.raises(error):
        gated_linear(*args, **kw)


def test_gated_8bit_refusals():
    x, sx = quantize_rows(torch.randn(3, 16))
    w, sw = quantize_rows(torch.randn(6, 16))
    good = [x, sx, w, sw, w, sw]
    for i, bad, error in ((0, torch.zeros(3, 16), TypeError), (2, w.view(torch.uint8), TypeError), (1, sx[:2], ValueError),
                          (3, sw.half(), ValueError), (5, sw[:, None], ValueError), (4, w[:5], ValueError)):
        with pytest.raises(error):
            gated_linear_8bit(*good[:i], bad, *good[i + 1:])
    with pytest.raises(TypeError):
        gated_linear_8bit(*good, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        gated_linear_8bit(*good)


def test_quantize_rows():
    t = torch.randn(7, 40) * torch.logspace(-3, 3, 7)[:, None]
    t[2] = 0.0
    rows, scale = quantize_rows(t)
    assert rows.dtype == torch.float8_e4m3fn and scale.shape == (7,) and torch.count_nonzero(rows[2].float()) == 0
    back = rows.float() * scale[:, None]
    assert bool(((back - t).abs() <= t.abs() * 2.0 ** -4 * 1.0001 + scale[:, None] * 2.0 ** -10 * 1.0001).all())
    assert torch.equal(rows[0].float().abs().amax(), torch.tensor(448.0))


def test_gated_module_surface():
    gate, up, down = nn.Linear(8, 6), nn.Linear(8, 6, bias=False), nn.Linear(6, 8)
    m = SpartonGatedMLP(gate, up, down, "gelu_tanh")
    assert list(m.state_dict()) == ["gate_proj.weight", "gate_proj.bias", "up_proj.weight", "down_proj.weight", "down_proj.bias"]
    assert sparton_amd.SpartonGatedMLP is SpartonGatedMLP
    for bad in ((gate, nn.Linear(8, 5), down), (gate, up, nn.Linear(5, 8))):
        with pytest.raises(ValueError):
            SpartonGatedMLP(*bad)
    with pytest.raises(ValueError, match="activation"):
        SpartonGatedMLP(gate, up, down, "tanh")
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        m(X)


def test_activation_names():
    f = nn.functional
    for fn, name in ((nn.SiLU(), "silu"), (f.silu, "silu"), (nn.GELU(), "gelu"), (nn.GELU(approximate="tanh"), "gelu_tanh"),
                     (f.gelu, "gelu"), (nn.ReLU(), "relu"), (nn.Tanh(), None), (None, None)):
        assert activation_name(fn) == name
    from transformers.activations import ACT2FN
    x = torch.linspace(-4, 4, 101)
    ours = {"silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "relu": f.relu}
    named = 0
    for fn in ("silu", "gelu", "gelu_pytorch_tanh", "gelu_new", "relu", "quick_gelu", "relu2", "mish"):
        name = activation_name(ACT2FN[fn])
        if name is not None:  # what is taken computes the same
            torch.testing.assert_close(ACT2FN[fn](x), ours[name](x), rtol=1e-5, atol=1e-6)
            named += 1
    assert named >= 4 and activation_name(ACT2FN["quick_gelu"]) is None and activation_name(ACT2FN["relu2"]) is None


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.sparton
    with FakeTensorMode():
        x, w = torch.empty(3, 5, 32, dtype=torch.bfloat16), torch.empty(32)
        y, h, q = ops.rms_norm_fwd(x, x, w, 1e-6)
        assert y.shape == x.shape == h.shape and y.dtype == h.dtype == x.dtype and q.shape == (15,) and q.dtype == torch.float32
        assert ops.rms_norm_fwd(x, None, w, 1e-6)[1].shape == (0,)
        dx, dw = ops.rms_norm_bwd(y, None, h, w, q)
        assert dx.shape == x.shape and dw.shape == (32,) and dw.dtype == torch.float32
        y, scale, h = ops.rms_norm_8bit(x, x, w, 1e-6)
        assert y.dtype == torch.float8_e4m3fn and scale.shape == (3, 5) and h.shape == x.shape
        ids, table = torch.empty(3, 5, dtype=torch.int64), torch.empty(70, 32, dtype=torch.float16)
        out = ops.embedding_fwd(ids, table, 1.0, -1)
        assert out.shape == (3, 5, 32) and out.dtype == torch.float16
        assert ops.embedding_bwd(out, ids, 70, 1.0, -1).shape == (70, 32)
        wg = torch.empty(48, 32, dtype=torch.bfloat16)
        h, g, u = ops.gated_fwd(x, wg, wg, None, None, "silu")
        assert h.shape == (3, 5, 48) and h.dtype == x.dtype and g.shape == u.shape == (15, 48) and g.dtype == torch.float32
        dx, dwg, dwu, dbg, dbu = ops.gated_bwd(h, x, wg, wg, g, u, "silu", True, False)
        assert dx.shape == x.shape and dwg.shape == dwu.shape == wg.shape and dbg.shape == (48,) and dbu.shape == (0,)
        x8, w8 = (torch.empty(n, 32, dtype=torch.float8_e4m3fn) for n in (5, 48))
        s5, s48 = torch.empty(5), torch.empty(48)
        assert ops.gated_8bit(x8, s5, w8, s48, w8, s48, "silu", torch.float16).shape == (5, 48)
