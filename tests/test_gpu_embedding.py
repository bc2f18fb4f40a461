"""GPU parity of the embedding and of its gradient against their formulas in 64 bits.

Tolerances, with u = eps / 2 of the table's type (half a step, relative) and E = 2^-24: the factor is one
fp32 rounding from the caller's number and the product another,
    out:      (u + 2 E) |out|, exact for a factor of 1
    d_weight: a token of n places is an fp32 sum of n terms, then the factor:
              (n + 4) E |scale| sum |d_out| + (u + 2 E) |d_weight|"""
import pytest
import torch

from _parity import say
from sparton_amd.embedding import SpartonEmbedding, embedding

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def make(N, V, D, dt, device, seed=0, ids="tokens", id_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + N + V + D)
    if ids == "tokens":      # ranks spread over their logarithm: a few tokens have many places
        t = (torch.rand(N, generator=g) * torch.log(torch.tensor(float(V)))).exp().long().clamp_(0, V - 1)
    elif ids == "one":
        t = torch.full((N,), V - 1)
    elif ids == "halves":    # two tokens, whose runs cross every chunk
        t = (torch.rand(N, generator=g) < 0.5).long() * (V - 1)
    elif ids == "up":
        t = torch.arange(N) % V
    else:                    # down
        t = (V - 1 - torch.arange(N) % V)
    w = torch.randn(V, D, generator=g).to(DT[dt])
    dy = torch.randn(N, D, generator=g).to(DT[dt])
    return t.to(id_dtype).to(device), w.to(device), dy.to(device)


def reference(ids, w, dy, scale, padding):
    """(out, its tolerance, d_weight, its tolerance); ids outside the table are NaN rows without a gradient."""
    u, V = torch.finfo(w.dtype).eps / 2, w.shape[0]
    sub = 2.0 ** -25 if w.dtype == torch.float16 else 2.0 ** -126
    ids, dy = ids.reshape(-1).long(), dy.reshape(-1, w.shape[1]).double()
    real = (ids >= 0) & (ids < V)
    out = torch.full((ids.numel(), w.shape[1]), float("nan"), dtype=torch.float64, device=w.device)
    out[real] = w.double()[ids[real]] * scale
    some = real & (ids != padding) if padding is not None else real
    zeros = lambda *n: torch.zeros(*n, dtype=torch.float64, device=w.device)
    dw = zeros(V, w.shape[1]).index_put_((ids[some],), dy[some], accumulate=True) * scale
    size = zeros(V, w.shape[1]).index_put_((ids[some],), dy[some].abs(), accumulate=True) * abs(scale)
    n = torch.bincount(ids[some], minlength=V)[:, None].double()
    return (out, (0.0 if scale == 1.0 else (u + 2 * E) * out.abs() + sub), dw,
            (n + 4) * E * size + (u + 2 * E) * dw.abs() + sub)


def run(ids, w, dy, scale=1.0, padding=None):
    leaf = w.detach().requires_grad_()
    out = embedding(ids, leaf, scale, padding)
    (dw,) = torch.autograd.grad(out, leaf, dy.reshape(out.shape))
    with torch.no_grad():
        assert torch.equal(embedding(ids, w, scale, padding).nan_to_num(7.0), out.nan_to_num(7.0))
    torch.cuda.synchronize()
    return out.detach(), dw


def check(ids, w, dy, scale=1.0, padding=None):
    out, dw = run(ids, w, dy, scale, padding)
    want, tol, wdw, tdw = reference(ids, w, dy, scale, padding)
    got = out.reshape(want.shape).double()
    assert out.dtype == w.dtype == dw.dtype and out.shape == (*ids.shape, w.shape[1]) and dw.shape == w.shape
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(((got - want).nan_to_num(0.0).abs() <= (tol if isinstance(tol, float) else tol.nan_to_num(0.0))).all())
    assert bool(((dw.double() - wdw).abs() <= tdw).all())
    assert torch.count_nonzero(dw[(tdw == tdw.min()).all(-1) & (wdw == 0).all(-1)]) == 0
    return out, dw


CASES = [  # N, V, D, dtype, ids
    (1, 1, 1, "fp32", "up"), (1, 5, 8, "bf16", "up"), (3, 7, 3, "bf16", "up"), (31, 100, 7, "fp16", "tokens"),
    (32, 100, 8, "fp32", "one"), (33, 100, 9, "bf16", "one"), (64, 3, 64, "bf16", "halves"), (65, 1000, 100, "fp16", "down"),
    (1000, 50, 33, "fp32", "tokens"), (1023, 2000, 768, "bf16", "tokens"), (1024, 2000, 768, "bf16", "up"),
    (1025, 2000, 768, "fp16", "down"), (2048, 30522, 384, "fp32", "tokens"), (5000, 30522, 768, "bf16", "tokens"),
    (4097, 512, 1023, "bf16", "up"), (3000, 10, 257, "fp32", "tokens"), (3001, 4000, 512, "fp16", "one"),
    (16384, 40, 72, "bf16", "halves"), (16385, 30522, 64, "bf16", "tokens"), (40000, 250002, 16, "fp16", "tokens"),
    (32768, 500, 16, "fp32", "down"), (32769, 500, 16, "bf16", "tokens"), (70001, 33, 5, "fp32", "tokens"), (262145, 1000, 8, "bf16", "tokens"), (40, 300, 20000, "bf16", "tokens"),
]


@pytest.mark.parametrize("N,V,D,dt,ids", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_embedding_matches_64_bits(N, V, D, dt, ids, device):
    say(f"embedding {N} of {V} x {D} {dt} {ids}")
    check(*make(N, V, D, dt, device, ids=ids))


@pytest.mark.parametrize("scale,padding", [(27.7, None), (-0.3, 0), (1.0, -1), (0.0, 5), (2.0, 39)])
def test_embedding_scale_and_padding(scale, padding, device):
    say(f"embedding scale {scale} padding {padding}")
    for dt in DT:
        ids, w, dy = make(3000, 40, 96, dt, device, id_dtype=torch.int32)
        out, dw = run(ids, w, dy, scale, padding)
        check(ids, w, dy, scale, None if padding is None else padding % 40)
        assert padding is None or torch.count_nonzero(dw[padding]) == 0


def test_embedding_shapes(device):
    say("shapes")
    _, w, _ = make(8, 50, 24, "bf16", device)
    ids = torch.randint(0, 50, (4, 3, 5), device=device)
    dy = torch.randn(4, 3, 5, 24, device=device).bfloat16()
    want = check(ids, w, dy)
    # expanded and transposed ids, a table that is a view, a gradient that is one
    row = ids[:1].expand(4, 3, 5)
    check(row, w, dy)
    out, dw = run(ids.transpose(0, 2), w, dy.transpose(0, 2).contiguous())
    assert torch.equal(out.transpose(0, 2), want[0])
    wide = torch.empty(50, 31, dtype=w.dtype, device=device)[:, 5:29].copy_(w)
    odd = torch.empty(50 * 24 + 1, dtype=w.dtype, device=device)[1:].view(50, 24).copy_(w)
    for table in (wide, odd):
        got = run(ids, table, dy.transpose(0, 1).contiguous().transpose(0, 1))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert embedding(torch.tensor(3, device=device), w).shape == (24,)


def test_embedding_empty(device):
    say("no ids, no rows")
    ids, w, dy = make(4, 50, 24, "bf16", device)
    out, dw = run(ids[:0].reshape(0, 3), w, dy[:0])
    assert out.shape == (0, 3, 24) and dw.shape == (50, 24) and torch.count_nonzero(dw) == 0
    out, dw = run(ids, w[:0], dy)
    assert bool(out.isnan().all()) and dw.shape == (0, 24)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_embedding_ids_outside_the_table(dtype, device):
    say("outside")
    ids, w, dy = make(2000, 60, 40, "bf16", device, id_dtype=dtype)
    bad = torch.tensor([60, -1, 2 ** 31 - 1, -2 ** 31, 61, -100], dtype=dtype)
    if dtype == torch.int64:
        bad = torch.cat([bad, torch.tensor([2 ** 32, 2 ** 32 + 5, -2 ** 63, 2 ** 63 - 1])])
    ids[100:100 + bad.numel()] = bad.to(device)
    ids[-1] = 60
    out, dw = check(ids, w, dy)
    assert bool(out[100:100 + bad.numel()].isnan().all()) and bool(dw.isfinite().all())


def test_embedding_nan_stays_in_its_rows(device):
    say("NaN")
    ids, w, dy = make(2000, 60, 40, "fp32", device)
    want = run(ids, w, dy)
    w2, dy2 = w.clone(), dy.clone()
    w2[7], dy2[ids == 9] = float("nan"), float("inf")
    out, dw = run(ids, w2, dy2)
    keep, rows = ids != 7, torch.arange(60, device=device) != 9
    assert torch.equal(out[keep], want[0][keep]) and torch.equal(dw[rows], want[1][rows])
    assert bool(out[~keep].isnan().all())


def test_embedding_deterministic_and_op_equals_function(device):
    say("deterministic")
    ids, w, dy = make(20000, 3000, 256, "bf16", device)
    a, b = run(ids, w, dy, 3.0, 7), run(ids, w, dy, 3.0, 7)
    out = torch.ops.sparton.embedding_fwd(ids, w, 3.0, 7)
    dw = torch.ops.sparton.embedding_bwd(dy, ids, 3000, 3.0, 7)
    for got in (b, (out, dw)):
        assert torch.equal(a[0], got[0]) and torch.equal(a[1], got[1])


def test_embedding_against_differences(device):
    """Directional derivative; the operator is linear in the table, so one difference of any size has no error of
    its own but the forward's."""
    say("differences")
    ids, w, dy = make(900, 70, 30, "fp32", device)
    g = torch.Generator().manual_seed(1)
    d = torch.randn(w.shape, generator=g).to(device)
    _, dw = run(ids, w, dy, 1.5)
    tdw = reference(ids, w, dy, 1.5, None)[3]
    with torch.no_grad():
        a, b = embedding(ids, w + d, 1.5), embedding(ids, w - d, 1.5)
    diff = float((dy.double() * (a.double() - b.double())).sum()) / 2
    both = torch.cat([w + d, w - d]).double()
    moved = float(((w + d).double() - (w - d).double() - 2 * d.double()).abs().max()) / 2
    tol = float((tdw * d.double().abs()).sum()) + float(dy.double().abs().sum()) * 1.5 * (
        2 * E * float(both.abs().max()) + moved)
    assert abs(diff - float((dw.double() * d.double()).sum())) <= tol


def test_embedding_module(device):
    say("module")
    m = torch.nn.Embedding(100, 32, padding_idx=3).to(device)
    ours = SpartonEmbedding.of(m, scale=2.0)
    assert ours.weight is m.weight and list(ours.state_dict()) == ["weight"] and isinstance(ours, torch.nn.Embedding)
    ids = torch.randint(0, 100, (6, 9), device=device)
    ids[0, 0] = 3
    assert torch.equal(ours(ids), 2 * m(ids))
    dy = torch.randn(6, 9, 32, device=device)
    (want,) = torch.autograd.grad(m(ids), m.weight, 2 * dy)
    (got,) = torch.autograd.grad(ours(ids), m.weight, dy)
    assert torch.count_nonzero(got[3]) == 0
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


def test_embedding_opcheck_and_compile(device):
    say("opcheck, compile")
    ids, w, dy = make(60, 50, 24, "fp32", device)
    leaf = w.clone().requires_grad_()
    torch.library.opcheck(torch.ops.sparton.embedding_fwd, (ids, leaf, 2.0, 1),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = lambda t: embedding(ids, t, 2.0, 1) * 2
    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    a, b = (torch.autograd.grad(c(leaf), leaf, dy)[0] for c in (cf, f))
    assert torch.equal(a, b)


def test_embedding_of_more_ids_than_a_gradient_takes(device):
    """2^29 narrow rows: looked up, and refused before the lookup where a gradient is asked for."""
    say("2^29 ids")
    N, D = 2 ** 29, 8
    ids = torch.zeros(N, dtype=torch.int32, device=device)
    places = torch.tensor([0, 1, 7, N // 2, N - 2, N - 1], device=device)
    ids[places] = torch.tensor([3, 1, 2, 3, 1, 2], dtype=torch.int32, device=device)
    w = torch.randn(4, D, device=device).bfloat16()
    out = embedding(ids, w)
    assert torch.equal(out[places], w[ids[places].long()]) and torch.equal(out[N // 3], w[0])
    with pytest.raises(RuntimeError, match="too many for a gradient"):
        embedding(ids, w.requires_grad_())
