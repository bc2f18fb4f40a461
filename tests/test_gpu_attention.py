"""GPU parity of the attention kernels against 64 bits (tests/_attention_ref.py derives the tolerances)."""
import math

import pytest
import torch

from _attention_ref import U32, allowed_pairs, close, reference
from _parity import say
from sparton_amd.attention import attention

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def make(B, Hq, Hk, Sq, Sk, D, dt, mask, device, seed=0, scale_do=0.05):
    """q, k, v as projections give them ([B,S,H,D] in memory), the key mask and an upstream gradient."""
    g = torch.Generator().manual_seed(seed + 1000 * Sq + Sk)
    rand = lambda *n: torch.randn(*n, generator=g).to(DT[dt]).to(device)
    q, k, v = (rand(B, S, H, D).transpose(1, 2) for S, H in ((Sq, Hq), (Sk, Hk), (Sk, Hk)))
    do = (torch.randn(B, Sq, Hq, D, generator=g) * scale_do).to(DT[dt]).to(device).transpose(1, 2)
    m = None
    if mask != "none":
        lens = torch.randint(max(1, Sk // 3), Sk + 1, (B,), generator=g)
        m = torch.arange(Sk)[None, :] < lens[:, None]
        if "holes" in mask:
            m &= torch.rand(B, Sk, generator=g) < 0.5
        if "left" in mask:
            m = m.flip(1)
        if "empty" in mask:
            m[B // 2] = False
        kind = torch.bool if "bool" in mask else torch.int32 if "int32" in mask else torch.uint8 if "uint8" in mask else torch.int64
        m = m.to(kind).to(device)
    return q, k, v, m, do


def run(q, k, v, m, do, causal, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, m, causal=causal, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    with torch.no_grad():
        assert torch.equal(attention(q, k, v, m, causal=causal, scale=scale).nan_to_num(), out.detach().nan_to_num())
    torch.cuda.synchronize()
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)))


def check(q, k, v, m, do, causal, scale=None):
    got = run(q, k, v, m, do, causal, scale)
    want = reference(q, k, v, m, causal, q.shape[-1] ** -0.5 if scale is None else scale, do)
    say("   of the tolerance: " + ", ".join(f"{n} {close(got[n], want[n], n):.2f}" for n in want))
    return got


CASES = [  # B, Hq, Hk, Sq, Sk, D, dtype, mask, causal
    (1, 1, 1, 1, 1, 64, "bf16", "none", False),           # one token sees itself
    (1, 2, 2, 1, 1, 64, "fp32", "none", True),
    (2, 2, 2, 16, 16, 64, "bf16", "int64", False),        # fewer than one MFMA block
    (2, 3, 3, 33, 33, 64, "fp16", "bool holes", False),
    (2, 2, 2, 64, 64, 64, "bf16", "none", True),          # whole tiles
    (2, 4, 2, 65, 65, 64, "bf16", "int64", True),         # one past them, shared heads
    (1, 2, 2, 127, 129, 64, "fp32", "int64 left", False),
    (3, 2, 1, 40, 70, 32, "bf16", "uint8 holes empty", False),
    (3, 2, 2, 130, 131, 128, "bf16", "int32 empty", True),
    (1, 8, 2, 181, 181, 128, "fp16", "int64", True),
    (2, 2, 2, 181, 181, 64, "fp32", "int64 holes", True),
    (1, 2, 1, 100, 260, 128, "fp32", "int64 empty", False),
    (1, 2, 2, 300, 50, 64, "bf16", "none", True),         # more rows than keys: the first see none
    (2, 2, 2, 70, 40, 64, "fp32", "int64 holes", True),
    (1, 2, 2, 50, 60, 80, "bf16", "int64", False),        # head sizes between the kernels' own
    (2, 2, 2, 45, 45, 24, "fp32", "int64", True),
    (1, 2, 2, 30, 37, 20, "bf16", "none", False),         # rows of 40 bytes: padded
    (1, 1, 1, 20, 21, 5, "fp32", "none", False),
    (1, 1, 1, 9, 12, 1, "fp16", "none", False),
    (4, 12, 12, 256, 256, 64, "bf16", "int64", False),
    (2, 4, 4, 512, 512, 64, "fp16", "int64", False),
    (1, 2, 2, 1100, 1100, 64, "bf16", "int64 holes", True),
    (1, 1, 1, 700, 4300, 64, "bf16", "int64 holes", False),  # the mask's words pass one 2048-key chunk
    (64, 12, 12, 260, 260, 64, "bf16", "int64 empty", False),  # many workgroups: two row blocks a wave
]


@pytest.mark.parametrize("case", CASES, ids=["-".join(str(x).replace(" ", "_") for x in c) for c in CASES])
def test_attention_matches_64_bits(case, device):
    B, Hq, Hk, Sq, Sk, D, dt, mask, causal = case
    say(f"attention {case}")
    check(*make(B, Hq, Hk, Sq, Sk, D, dt, mask, device), causal)


FEW = [  # rows of a key head at most 32: waves share the keys, and long keys are split over workgroups
    (1, 1, 1, 1, 100, 64, "bf16", "none", False),
    (2, 8, 2, 1, 5001, 128, "bf16", "int64", False),
    (1, 4, 4, 1, 4097, 64, "fp32", "int64 holes", False),
    (3, 2, 2, 17, 3000, 64, "fp16", "int64 empty", True),
    (1, 8, 1, 4, 2500, 32, "bf16", "bool left", True),
    (1, 4, 1, 8, 9000, 128, "fp32", "int64 holes", False),
    (1, 2, 2, 40, 9001, 64, "bf16", "int64 holes", True),   # more rows than that, and a split all the same
    (2, 1, 1, 5, 700, 96, "bf16", "int64 empty", False),
]


@pytest.mark.parametrize("case", FEW, ids=["-".join(str(x).replace(" ", "_") for x in c) for c in FEW])
def test_attention_few_rows_many_keys(case, device):
    B, Hq, Hk, Sq, Sk, D, dt, mask, causal = case
    say(f"attention, few rows {case}")
    check(*make(B, Hq, Hk, Sq, Sk, D, dt, mask, device), causal)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Sq,Sk,causal", [(150, 150, False), (150, 150, True), (1, 3000, False)])
def test_masked_keys_may_hold_anything(dt, Sq, Sk, causal, device):
    """NaN, infinities and the type's lowest value in masked keys and values: no output or gradient of
    a key that takes part changes by a bit, and theirs are zeros."""
    say(f"masked keys {dt} {Sq} {Sk} {causal}")
    q, k, v, m, do = make(2, 2, 2, Sq, Sk, 64, dt, "int64 holes", device)
    off = (m == 0)[:, None, :, None].expand(k.shape)
    clean = run(q, torch.where(off, 0.0, k), torch.where(off, 0.0, v), m, do, causal)
    for bad in (float("nan"), float("inf"), torch.finfo(DT[dt]).min):
        got = run(q, torch.where(off, bad, k), torch.where(off, -bad, v), m, do, causal)
        for n in clean:
            assert torch.equal(got[n], clean[n]), (n, bad)
    assert torch.count_nonzero(clean["dk"][off]) == 0 and torch.count_nonzero(clean["dv"][off]) == 0


def test_rows_without_keys_are_zero(device):
    say("rows without keys")
    for dt in DT:
        q, k, v, m, do = make(3, 2, 2, 70, 90, 64, dt, "int64", device)
        m[1] = 0
        got = run(q, k, v, m, do, False)
        for n in got:
            assert torch.count_nonzero(got[n][1]) == 0 and torch.count_nonzero(got[n][0]) > 0, n
        got = run(q[:, :, :50], k[:, :, :20], v[:, :, :20], None, do[:, :, :50], True)  # 30 rows see nothing
        assert torch.count_nonzero(got["out"][:, :, :30]) == 0 and torch.count_nonzero(got["dq"][:, :, :30]) == 0
        assert torch.count_nonzero(got["out"][:, :, 30:]) > 0


def test_empty_sizes(device):
    say("empty sizes")
    z = lambda *n: torch.randn(*n, device=device, dtype=torch.bfloat16)
    got = run(z(2, 2, 5, 64), z(2, 2, 0, 64), z(2, 2, 0, 64), None, z(2, 2, 5, 64), False)
    assert torch.count_nonzero(got["out"]) == 0 and torch.count_nonzero(got["dq"]) == 0 and got["dk"].numel() == 0
    got = run(z(2, 2, 0, 64), z(2, 2, 7, 64), z(2, 2, 7, 64), None, z(2, 2, 0, 64), False)
    assert got["out"].shape == (2, 2, 0, 64) and torch.count_nonzero(got["dk"]) == 0 and torch.count_nonzero(got["dv"]) == 0
    got = run(z(0, 2, 5, 64), z(0, 2, 7, 64), z(0, 2, 7, 64), None, z(0, 2, 5, 64), True)
    assert got["out"].shape == (0, 2, 5, 64)


def test_layouts_give_the_same_bits(device):
    """One fused projection's views, head-major tensors, a batch shared by stride 0, rows that start off
    16 bytes, a last dimension that is not the innermost: the same values, the same bits."""
    say("layouts")
    q, k, v, m, do = make(2, 4, 4, 75, 75, 64, "bf16", "int64", device)
    want = run(*(t.contiguous() for t in (q, k, v)), m, do.contiguous(), False)
    fused = torch.cat([t.transpose(1, 2) for t in (q, k, v)], dim=2)
    views = [t.transpose(1, 2) for t in fused.split(4, dim=2)]
    odd = [torch.empty(t.numel() + 3, dtype=t.dtype, device=device)[3:].view(t.shape).copy_(t) for t in (q, k, v)]
    inner = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    for name, ts in (("fused", views), ("projections", (q, k, v)), ("unaligned", odd), ("transposed", inner)):
        got = run(*ts, m, do, False)
        for n in want:
            assert torch.equal(got[n], want[n]), (name, n)
    k1, v1, m1 = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), m[:1].expand(2, -1)
    a, b = run(q, k1, v1, m1, do, False), run(q, k1.contiguous(), v1.contiguous(), m1.contiguous(), do, False)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    wide = torch.empty(2, 3 * 75, dtype=m.dtype, device=device)[:, ::3]  # a mask with an inner stride
    wide.copy_(m)
    got = run(q, k, v, wide, do, False)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_expanded_inputs_get_summed_gradients(device):
    """A key shared by every batch row: autograd sums the rows' gradients."""
    say("expanded inputs")
    q, k, v, m, do = make(3, 2, 2, 40, 50, 64, "fp32", "int64", device)
    k1, v1 = k[:1].detach().requires_grad_(), v[:1].detach().requires_grad_()
    out = attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), m)
    dk, dv = torch.autograd.grad(out, (k1, v1), do)
    want = reference(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), m, False, 64 ** -0.5, do)
    for got, n in ((dk, "dk"), (dv, "dv")):
        value, tol = (t.sum(0, keepdim=True) for t in want[n])
        close(got, (value, tol + 2 * 2.0 ** -24 * want[n][0].abs().sum(0, keepdim=True)), n)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_large_and_small_magnitudes(dt, device):
    """Peaked rows (scores up to hundreds), all-negative scores, and gradients near the bottom of fp16."""
    say(f"magnitudes {dt}")
    q, k, v, m, do = make(1, 2, 2, 90, 140, 64, dt, "int64", device)
    check(q * 8, k * 4, v, m, do, False)
    check(q, k, v, m, do, False, scale=3.0)
    check(q.abs() * 4, -k.abs() * 4, v, m, do, True)
    check(q, k, v, m, do * 0.002, False)
    check(q * 0, k, v, m, do * 40, False, scale=1e-3)


def test_deterministic_and_op_equals_function(device):
    say("deterministic; the custom op and the C++ path agree")
    q, k, v, m, do = make(3, 8, 4, 300, 300, 64, "bf16", "int64 holes", device)
    a, b = run(q, k, v, m, do, True), run(q, k, v, m, do, True)
    out, lse = torch.ops.sparton.attention_fwd(q, k, v, m, True, 64 ** -0.5)
    grads = torch.ops.sparton.attention_bwd(do, q, k, v, m, out, lse, True, 64 ** -0.5)
    for n, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert torch.equal(a[n], b[n]) and torch.equal(a[n], t), n


def test_split_equals_whole(device):
    """The same row alone (keys split over workgroups and joined) and among many (not split)."""
    say("split over keys")
    q, k, v, m, do = make(1, 1, 1, 600, 6000, 64, "fp32", "int64 holes", device)
    want = reference(q, k, v, m, False, 0.125, do)["out"]
    for rows in (slice(0, 1), slice(5, 30), slice(100, 140), slice(0, 600)):
        with torch.no_grad():
            close(attention(q[:, :, rows], k, v, m), tuple(t[:, :, rows] for t in want), f"out {rows}")


@pytest.mark.parametrize("causal,Hq,Hk", [(False, 2, 2), (True, 4, 2)])
def test_gradients_against_differences(causal, Hq, Hk, device):
    """The directional derivative of sum(w out) from the gradients, against central differences of the
    fp32 forward. Tolerance: the differences' own error in 64 bits (h^2 terms), the forward's tolerance
    divided by h, and the gradients' tolerance along the direction."""
    say(f"differences {causal} {Hq} {Hk}")
    # a small case: the tolerance grows with the number of terms, the derivative with its square root
    q, k, v, m, w = make(1, Hq, Hk, 5, 7, 8, "fp32", "int64", device, scale_do=1.0)
    g = torch.Generator().manual_seed(5)
    dirs = [torch.randn(t.shape, generator=g).to(device) for t in (q, k, v)]
    got = run(q, k, v, m, w, causal)
    h = 2.0 ** -6
    want = reference(q, k, v, m, causal, 8 ** -0.5, w)
    along = sum(float((got[n].double() * d.double()).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    exact = sum(float((want[n][0] * d.double()).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    tol = sum(float((want[n][1] * d.double().abs()).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    value, value64 = [], []
    for sign in (1, -1):
        moved = [t + sign * h * d for t, d in zip((q, k, v), dirs)]
        ref, ref_tol = reference(*moved, m, causal, 8 ** -0.5, w)["out"]
        with torch.no_grad():
            value.append(float((w.double() * attention(*moved, m, causal=causal).double()).sum()))
        value64.append(float((w.double() * ref).sum()))
        tol += float((w.double().abs() * ref_tol).sum()) / (2 * h)
    tol += abs((value64[0] - value64[1]) / (2 * h) - exact)
    assert abs(along - (value[0] - value[1]) / (2 * h)) <= tol
    say(f"   {along:.6f} against {(value[0] - value[1]) / (2 * h):.6f}, tolerance {tol:.2e}")


def test_only_some_inputs_need_gradients(device):
    say("partial gradients")
    q, k, v, m, do = make(1, 2, 2, 40, 40, 64, "bf16", "int64", device)
    want = run(q, k, v, m, do, False)
    v2 = v.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(attention(q, k, v2, m), v2, do)[0], want["dv"])
    q2 = q.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(attention(q2, k, v, m), q2, do)[0], want["dq"])
    # one tensor in all three places
    x = q.detach().requires_grad_()
    (dx,) = torch.autograd.grad(attention(x, x, x, m), x, do)
    parts = run(q, q, q, m, do, False)
    total = sum(parts[n].float() for n in ("dq", "dk", "dv"))
    tol = 2.0 ** -7 * sum(parts[n].float().abs() for n in ("dq", "dk", "dv"))  # two sums rounded to bf16
    assert bool(((dx.float() - total).abs() <= tol).all())


def test_opcheck_and_compile(device):
    say("opcheck, compile")
    q, k, v, m, do = make(2, 4, 2, 20, 30, 64, "bf16", "int64", device)
    ql = q.detach().requires_grad_()
    torch.library.opcheck(torch.ops.sparton.attention_fwd, (ql, k, v, m, True, 0.125),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))

    def f(a, b, c):
        return attention(a, b, c, m, causal=True) * 2

    cf = torch.compile(f, backend="aot_eager", fullgraph=True)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    for a, b in zip(torch.autograd.grad(cf(*leaves), leaves, do), torch.autograd.grad(f(*leaves), leaves, do)):
        assert torch.equal(a, b)


def test_autocast(device):
    say("autocast")
    q, k, v, m, do = make(2, 2, 2, 40, 40, 64, "fp32", "int64", device)
    ql = q.detach().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = attention(ql, k, v, m)
    assert out.dtype == torch.bfloat16 and torch.equal(out, attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), m))
    (dq,) = torch.autograd.grad(out, ql, do.bfloat16())
    assert dq.dtype == torch.float32 and torch.isfinite(dq).all()


@pytest.mark.parametrize("Sq,Sk", [(70, 70), (1, 4000)])
def test_graph_replays(Sq, Sk, device):
    """Forward and backward captured into one graph: every replay on new inputs is the eager result."""
    say(f"graph {Sq} {Sk}")
    sets = [make(2, 4, 2, Sq, Sk, 64, "bf16", "int64 holes", device, seed=s) for s in range(3)]
    held = [t.detach().clone() for t in sets[0]]

    def step():
        q, k, v, m, do = held
        out, lse = torch.ops.sparton.attention_fwd(q, k, v, m, False, 0.125)
        return (out, *torch.ops.sparton.attention_bwd(do, q, k, v, m, out, lse, False, 0.125))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for s in (1, 2, 0, 1):
        for t, new in zip(held, sets[s]):
            t.copy_(new)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for t in outs:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_on_another_stream(device):
    say("another stream")
    q, k, v, m, do = make(2, 4, 4, 200, 200, 64, "bf16", "int64", device)
    want = run(q, k, v, m, do, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, m, do, False)
    torch.cuda.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_rows_outside_a_slice_are_left_alone(device):
    """Gradients and outputs are written row by row: a head dimension below the kernels' block and a row
    count below a tile leave what lies behind them untouched (through the C ABI, into larger buffers)."""
    import ctypes
    from sparton_amd import _lib
    say("rows behind the last one")
    B, H, S, D = 2, 2, 37, 24
    L = _lib.load()
    q, k, v, m, do = make(B, H, H, S, S, D, "bf16", "int64 empty", device)
    big = lambda: torch.full((B, S + 30, H, 64), 5.0, dtype=torch.bfloat16, device=device)
    bufs = dict(o=big(), d_q=big(), d_k=big(), d_v=big())
    lse = torch.empty(B, H, S, device=device)
    d = _lib.AttentionDesc(B=B, Hq=H, Hk=H, Sq=S, Sk=S, D=D, mask_batch=S, scale=D ** -0.5, causal=0, dtype=1, mask_dtype=0)
    for n, t in (("q", q), ("k", k), ("v", v), ("d_o", do)):
        getattr(d, n)[:] = [t.stride(0), t.stride(1), t.stride(2)]
    for n, t in bufs.items():
        getattr(d, n)[:] = [t.stride(0), t.stride(2), t.stride(1)]
    st = torch.cuda.current_stream().cuda_stream
    n1, n2 = L.sparton_attention_workspace_bytes(ctypes.byref(d)), L.sparton_attention_bwd_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(max(n1, n2, 1), dtype=torch.uint8, device=device)
    assert L.sparton_attention_fwd(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), m.data_ptr(),
                                   bufs["o"].data_ptr(), lse.data_ptr(), ws.data_ptr(), n1, st) == 0
    assert L.sparton_attention_bwd(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), m.data_ptr(),
                                   bufs["o"].data_ptr(), lse.data_ptr(), do.data_ptr(), bufs["d_q"].data_ptr(),
                                   bufs["d_k"].data_ptr(), bufs["d_v"].data_ptr(), ws.data_ptr(), n2, st) == 0
    torch.cuda.synchronize()
    want = run(q, k, v, m, do, False)
    for (n, t), r in zip(bufs.items(), ("out", "dq", "dk", "dv")):
        assert bool((t[:, S:] == 5.0).all()) and bool((t[..., D:] == 5.0).all()), n
        assert torch.equal(t[:, :S, :, :D].transpose(1, 2), want[r]), n


@pytest.mark.parametrize("case", [
    # B, Hq, Hk, Sq, Sk, D, dtype, mask, causal: few and many workgroups on either side
    (1, 2, 2, 300, 2100, 64, "bf16", "int64", False),
    (1, 4, 2, 150, 1500, 128, "fp16", "int64 holes", True),
    (1, 3, 3, 1100, 90, 32, "bf16", "bool", False),
    (2, 2, 1, 257, 400, 96, "bf16", "int64 left", True),
    (20, 12, 12, 129, 131, 64, "bf16", "int64 holes empty", True),
    (17, 12, 12, 140, 70, 128, "fp16", "none", False),
], ids=str)
def test_attention_group_sizes(case, device):
    say(f"case {case}")
    B, Hq, Hk, Sq, Sk, D, dt, mask, causal = case
    check(*make(B, Hq, Hk, Sq, Sk, D, dt, mask, device), causal)


@pytest.mark.parametrize("D", [20, 64])
def test_output_changed_in_place(D, device):
    """An output that its user overwrites: the gradients are right, or the backward says what happened."""
    say(f"in place, {D}")
    q, k, v, m, do = make(2, 2, 2, 33, 40, D, "bf16", "int64", device)
    want = run(q, k, v, m, do, False)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, m)
    out.mul_(0.5)
    try:
        grads = torch.autograd.grad(out, leaves, do * 2)  # powers of two: the same bits
    except RuntimeError as e:
        assert "inplace" in str(e)
    else:
        assert all(torch.equal(g, want[n]) for g, n in zip(grads, ("dq", "dk", "dv")))


@pytest.mark.parametrize("B,Sq", [(200, 33), (1, 33), (1, 1)])  # whole rows, and rows split over the keys
def test_fp16_keys_far_below_the_largest(B, Sq, device):
    """40000 keys of 2^-26 of the first one's weight hold 0.06% of each row, and here all of its value.

    Probabilities of the second product are fp16 with a factor 2^7, relative to a maximum that is at most the
    row's: normal ones are off by u = 2^-11 of their value, others by 2^-25 2^-7. The scores are exact."""
    say(f"fp16, small probabilities {B} {Sq}")
    Sk, D = 40001, 64
    q, k = torch.zeros(1, 1, Sq, D), torch.zeros(1, 1, Sk, D)
    q[..., 0], k[..., 0, 0] = 16.0, 9.0  # scores 18 and 0: exp(-18) = 2^-25.97
    v = torch.randint(500, 1500, (1, 1, Sk, D), generator=torch.Generator().manual_seed(0)).float()
    v[:, :, 0] = 0.0
    q, k, v = (t.half().to(device) for t in (q, k, v))
    with torch.no_grad():
        got = attention(*(t.expand(B, -1, -1, -1) for t in (q, k, v)))
    s = 0.125 * (q.double() @ k.double().transpose(-1, -2).contiguous())
    p = torch.softmax(s, -1)
    want = p @ v.double()
    # as in the reference's tolerances: ep of a probability and its row's sum, the sums over the keys, the output
    ep = 2.0 ** -22 * (1 + s.abs() + torch.logsumexp(s, -1, keepdim=True)) + (Sk + 4) * 2.0 ** -24
    ep = ep + (p * ep).sum(-1, keepdim=True)
    u = 2.0 ** -11
    tol = u * want + (p * (u + ep + (Sk + 4) * 2.0 ** -24) + 2.0 ** -32) @ v.double()
    assert bool((tol < 0.03 * want).all())
    close(got, (want.expand(B, -1, -1, -1), tol.expand(B, -1, -1, -1)), "out")


@pytest.mark.parametrize("D", [20, 64])
def test_heads_innermost_in_memory(D, device):
    """[B,S,D,H] in memory, inputs and upstream gradient: the same bits as [B,S,H,D], padded head size or not."""
    say(f"heads innermost, {D}")
    q, k, v, m, do = make(2, 4, 4, 35, 41, D, "bf16", "int64", device)
    last = lambda t: t.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    want, got = run(q, k, v, m, do, False), run(*map(last, (q, k, v)), m, last(do), False)
    assert last(q).stride(1) == 1 and all(torch.equal(got[n], want[n]) for n in want)
    out, lse = torch.ops.sparton.attention_fwd(last(q), last(k), last(v), m, False, D ** -0.5)
    grads = torch.ops.sparton.attention_bwd(last(do), q, k, v, m, last(out), lse, False, D ** -0.5)
    for n, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_causal_keys_that_are_not_finite(dt, device):
    """One value of one key: what it may reach, and what it may not. The mask's keys are another matter."""
    say(f"causal, not finite, {dt}")
    j, d = 100, 7
    q, k, v, m, do = make(2, 4, 2, 150, 150, 64, dt, "none", device)
    want = run(q, k, v, m, do, True)
    for bad in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[0, 0, j, d], v2[0, 0, j, d] = bad, bad
        got = run(q, k, v2, m, do, True)
        # forward: its own column of the rows that share the key head, and there of every row that sees it
        assert not bool(torch.isfinite(got["out"][0, :2, j:, d]).any())
        other = [c for c in range(64) if c != d]
        assert torch.equal(got["out"][0, :2][..., other], want["out"][0, :2][..., other])
        with torch.no_grad():  # a key's scores are dropped, not multiplied
            assert torch.equal(attention(q, k2, v, causal=True)[0, :2, :j], want["out"][0, :2, :j])
        for res in (got, run(q, k2, v, m, do, True)):
            for n, heads in (("out", 2), ("dq", 2), ("dk", 1), ("dv", 1)):  # the other key head, the other batch row
                assert torch.equal(res[n][0, heads:], want[n][0, heads:]) and torch.equal(res[n][1], want[n][1]), n
        m2 = torch.ones(2, 150, dtype=torch.bool, device=device)
        m2[0, j] = False
        masked = run(q, k, v, m2, do, True)
        for n, t in run(q, k2, v2, m2, do, True).items():
            assert torch.equal(t, masked[n]), n


# Every kernel that the launch rules choose from (tests/test_operators_boundary.py counts them): workgroups of 32,
# 64 and 128 rows, whole and split over the keys, and of 64 and 128 keys, for each type and head block.
SHAPES = [  # B, Hq, Hk, Sq, Sk, mask, causal; B of the first two times 12 heads is what 128 rows need
    (None, 12, 12, 101, 97, "int64 holes empty", False),
    (None, 24, 12, 131, 135, "int64 left", True),
    (2, 2, 2, 70, 150, "bool holes", True),
    (1, 2, 1, 41, 1100, "int64", False),
    (1, 2, 2, 140, 2500, "int64 holes", True),
    (2, 4, 2, 9, 201, "int64", True),
    (1, 4, 2, 5, 1501, "int64 holes", False),
]
EVERY = [(B or (22 if dt != "fp32" else 43), Hq, Hk, Sq, Sk, D, dt, mask, causal)
         for dt in DT for D in (24, 64, 104) for B, Hq, Hk, Sq, Sk, mask, causal in SHAPES]


@pytest.mark.parametrize("case", EVERY, ids=["-".join(str(x).replace(" ", "_") for x in c) for c in EVERY])
def test_attention_on_every_kernel(case, device):
    B, Hq, Hk, Sq, Sk, D, dt, mask, causal = case
    say(f"attention {case}")
    check(*make(B, Hq, Hk, Sq, Sk, D, dt, mask, device), causal)


@pytest.mark.parametrize("case", [  # at most 32 keys a row: every row's lie in one tile
    (3, 4, 2, 31, 31, 64, "bf16", "none", True),
    (40, 12, 6, 32, 32, 64, "bf16", "int64", True),     # groups of 128 rows, four query heads' rows in some
    (5, 2, 2, 9, 9, 64, "fp16", "none", False),
    (2, 2, 2, 4, 4, 128, "fp16", "none", True),
    (30, 12, 12, 19, 23, 104, "bf16", "bool left", True),
    (3, 4, 4, 45, 26, 32, "fp16", "int64 empty", False),
    (25, 8, 8, 17, 30, 20, "bf16", "int64 holes", True),
    (2, 3, 3, 70, 300, 64, "bf16", "few", False),        # only 20 keys of 300 take part
    (1, 3, 3, 70, 300, 128, "bf16", "few", True),
], ids=str)
def test_gradients_of_rows_with_few_keys(case, device):
    """There do . v and delta nearly cancel (with one key ds is 0), so delta must not carry the output's rounding:
    as in the reference's tolerances, but for delta, which is then sum_j p_ij (do_i . v_j), each term off by ep and
    by the product's sums, and n sums in fp32."""
    say(f"few keys {case}")
    B, Hq, Hk, Sq, Sk, D, dt, mask, causal = case
    q, k, v, m, do = make(B, Hq, Hk, Sq, Sk, D, dt, "none" if mask == "few" else mask, device, scale_do=1.0)
    if mask == "few":
        m = torch.zeros(B, Sk, dtype=torch.int64, device=device)
        m[:, 35:55] = 1
    got = run(q, k, v, m, do, causal)
    u, tiny = torch.finfo(q.dtype).eps / 2, 2.0 ** -34 if dt == "fp16" else 0.0
    sub = 2.0 ** -25 if dt == "fp16" else 2.0 ** -126
    q, k, v, do = (t.double() for t in (q, k, v, do))
    G, scale = Hq // Hk, D ** -0.5
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    on = allowed_pairs(B, Sq, Sk, m, causal, device)
    kt, vt = k.transpose(-1, -2).contiguous(), v.transpose(-1, -2).contiguous()
    s = scale * (q @ kt)
    L = torch.logsumexp(torch.where(on, s, -math.inf), -1, keepdim=True)
    some = on.any(-1, keepdim=True)
    p = torch.where(on, torch.exp(s - torch.where(some, L, 0.0)), 0.0)
    ep = torch.where(on, (D + 2) * U32 * scale * (q.abs() @ kt.abs())
                     + 2.0 ** -22 * (1 + s.abs() + torch.where(some, L, 0.0).abs()), 0.0)
    ep = ep + (p * ep).sum(-1, keepdim=True) + (Sk + 4) * U32
    dp, e_dp = do @ vt, (D + 2) * U32 * (do.abs() @ vt.abs())
    delta = (p * dp).sum(-1, keepdim=True)
    e_delta = (p * ((ep + (Sk + 4) * U32) * dp.abs() + e_dp)).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_ds = (u + ep + 4 * U32) * ds.abs() + p * (e_dp + e_delta)
    e_ds = e_ds + tiny * torch.maximum(ds.abs().amax(-1, keepdim=True), ds.abs().amax(-2, keepdim=True)) * on
    dq = scale * (ds @ k)
    close(got["dq"], (dq, u * dq.abs() + scale * ((e_ds + (Sk + 4) * U32 * ds.abs()) @ k.abs()) + sub), "dq")
    shared = lambda t: t.reshape(B, Hk, G, Sk, D).sum(2)
    dk = shared(scale * (ds.transpose(-1, -2).contiguous() @ q))
    tol = shared(scale * ((e_ds + (G * Sq + 4) * U32 * ds.abs()).transpose(-1, -2).contiguous() @ q.abs()))
    close(got["dk"], (dk, u * dk.abs() + tol + sub), "dk")
