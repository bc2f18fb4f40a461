"""The RMS norm, the embedding and the gated product together: gradients differentiated again, calls at once on two
streams, captured graphs that share a memory pool, a layer's run of them captured with its backward, and tensors whose
offsets pass 32 bits. Bitwise against the same operators' plain calls, which the tests of each operator check against
64 bits."""
import pytest
import torch

from _parity import say
from sparton_amd.embedding import embedding
from sparton_amd.feed_forward import gated_linear, gated_linear_8bit, quantize_rows
from sparton_amd.norm import rms_norm, rms_norm_8bit

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def randn(*shape, device, seed, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def calls(device, seed=0):
    """name -> (function of its leaves, leaves)"""
    ids = torch.randint(0, 500, (2500,), generator=torch.Generator().manual_seed(seed)).to(device)
    ids[::3] = 7
    rows = [randn(300, 768, device=device, seed=seed + i) for i in range(2)]
    vec = randn(768, device=device, seed=seed + 2)
    table = randn(500, 256, device=device, seed=seed + 3)
    gated = lambda M: [randn(M, 128, device=device, seed=seed + 4)] + [randn(200, 128, device=device, seed=seed + 5 + i, scale=0.1)
                                                                      for i in range(2)]
    return {
        "rms_norm": (lambda x, w: rms_norm(x, w), [rows[0], vec]),
        "rms_norm with the sum": (lambda x, r, w: torch.cat(rms_norm(x, w, residual=r)), [*rows, vec]),
        "embedding": (lambda w: embedding(ids, w, 2.0, 7), [table]),
        "gated": (lambda x, g, u: gated_linear(x, g, u), gated(300)),
        "gated, few rows": (lambda x, g, u: gated_linear(x, g, u, activation="gelu"), gated(5)),
    }


def both(f, leaves):
    """The output and every leaf's gradient."""
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = f(*leaves)
    return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))


NAMES = ["rms_norm", "rms_norm with the sum", "embedding", "gated", "gated, few rows"]


@pytest.mark.parametrize("name", NAMES)
def test_a_second_derivative_is_refused(name, device):
    say(f"second derivative of {name}")
    f, leaves = calls(device)[name]
    want = both(f, leaves)
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = f(*leaves)
    up = torch.ones_like(out, requires_grad=True)
    grads = torch.autograd.grad(out, leaves, up, create_graph=True)
    for g, w in zip(grads, want[1:]):
        assert g.requires_grad and torch.equal(g.detach(), w)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(grads[0].float().sum(), leaves[0])


def test_calls_at_once_on_two_streams(device):
    say("two streams")
    first, second = calls(device, 0), calls(device, 100)
    want = [{n: both(*c[n]) for n in NAMES} for c in (first, second)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for s, c, g in zip(streams, (first, second), got):
            with torch.cuda.stream(s):
                g.append({n: both(*c[n]) for n in NAMES})
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for run in g:
            for n in NAMES:
                assert all(torch.equal(a, b) for a, b in zip(run[n], w[n])), n


def layer(ids, table, r, w, wg, wu, dh):
    """tokens -> rows -> norm with the sum -> gated product, and all gradients, by the registered operators."""
    ops = torch.ops.sparton
    x = ops.embedding_fwd(ids, table, 1.0, 0)
    y, h, q = ops.rms_norm_fwd(x, r, w, 1e-6)
    out, g, u = ops.gated_fwd(y, wg, wu, None, None, "silu")
    dy, dwg, dwu, _, _ = ops.gated_bwd(dh, y, wg, wu, g, u, "silu", False, False)
    dx, dw = ops.rms_norm_bwd(dy, None, h, w, q)
    y8, scale, _ = ops.rms_norm_8bit(x, r, w, 1e-6)
    return out, h, ops.embedding_bwd(dx, ids, table.shape[0], 1.0, 0), dx, dw, dwg, dwu, y8.view(torch.uint8), scale


def layer_inputs(device, seed, M):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 90, (M,), generator=g).to(device), randn(90, 192, device=device, seed=seed + 1),
            randn(M, 192, device=device, seed=seed + 2), randn(192, device=device, seed=seed + 3),
            randn(320, 192, device=device, seed=seed + 4, scale=0.1), randn(320, 192, device=device, seed=seed + 5, scale=0.1),
            randn(M, 320, device=device, seed=seed + 6)]


@pytest.mark.parametrize("M", [3, 700])
def test_a_layers_run_against_autograd(M, device):
    """The same run through the functions, differentiated."""
    say(f"layer of {M}")
    ids, table, r, w, wg, wu, dh = layer_inputs(device, 5, M)
    want = layer(ids, table, r, w, wg, wu, dh)
    leaves = [t.detach().requires_grad_() for t in (table, r, w, wg, wu)]
    y, h = rms_norm(embedding(ids, leaves[0], padding_idx=0), leaves[2], residual=leaves[1])
    out = gated_linear(y, leaves[3], leaves[4])
    got = (out.detach(), h.detach(), *torch.autograd.grad(out, leaves, dh))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and in plain fp32 autograd: 16-bit roundings on the way (of the rows, dg and du, dy, dx), 2^-8 each at most
    f = [t.detach().float().requires_grad_() for t in (table, r, w, wg, wu)]
    s = torch.nn.functional.embedding(ids, f[0], padding_idx=0) + f[1]
    y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * f[2]
    ref = torch.nn.functional.silu(y @ f[3].t()) * (y @ f[4].t())
    for a, b in zip((got[0], *got[2:]), (ref.detach(), *torch.autograd.grad(ref, f, dh.float()))):
        assert float((a.float() - b).norm()) <= 6 * 2.0 ** -8 * float(b.norm())


@pytest.mark.parametrize("M", [3, 700])
def test_two_graphs_of_one_pool(M, device):
    """The run captured for two input sets into graphs that share a memory pool, replayed in turn on changing inputs,
    with eager calls between them."""
    say(f"two graphs of {M}")
    sets = [[layer_inputs(device, 10 * s, M) for s in (a, a + 1, a + 2)] for a in (0, 5)]
    held = [[t.clone() for t in s[0]] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[[t.clone() for t in layer(*i)] for i in s] for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(layer(*h))
        graphs.append(g)
    for which, i in ((0, 1), (1, 2), (1, 0), (0, 2), (1, 1), (0, 0)):
        for t, new in zip(held[which], sets[which][i]):
            t.copy_(new)
        for t in outs[which]:
            t.fill_(7)
        graphs[which].replay()
        layer(*sets[1 - which][i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[which], want[which][i])), (which, i)


def test_8_bits_graph_replays(device):
    say("8 bits, graph")
    x, w = randn(200, 256, device=device, seed=1), randn(256, device=device, seed=2)
    weights = [t for i in (3, 4) for t in quantize_rows(randn(300, 256, device=device, seed=i, scale=0.1))]
    step = lambda t: gated_linear_8bit(*rms_norm_8bit(t, w), *weights)
    other = randn(200, 256, device=device, seed=9)
    with torch.no_grad():
        want = [step(t).clone() for t in (x, other)]
        held = x.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(held)
        for t, v in ((other, want[1]), (x, want[0]), (other, want[1])):
            held.copy_(t)
            graph.replay()
            step(x)
            torch.cuda.synchronize()
            assert torch.equal(out, v)


# ---- offsets past 32 bits --------------------------------------------------------------------

def test_rms_norm_of_more_than_32_bits(device):
    say("rms_norm, 2^31 elements")
    D, M = 4096, 2 ** 31 // 4096 + 101
    x, r = (torch.empty(M, D, dtype=BF16, device=device).normal_() for _ in range(2))
    w = randn(D, device=device, seed=1).requires_grad_()
    tail = slice(M - 120, M)
    leaves, small = [x.requires_grad_(), r.requires_grad_(), w], [t.detach()[tail].clone().requires_grad_() for t in (x, r)] + [w]
    (y, h), (yt, ht) = rms_norm(leaves[0], w, residual=leaves[1]), rms_norm(small[0], w, residual=small[1])
    assert torch.equal(y.detach()[tail], yt.detach()) and torch.equal(h.detach()[tail], ht.detach())
    y8, scale, _ = rms_norm_8bit(x.detach(), w.detach(), residual=r.detach())
    t8, ts, _ = rms_norm_8bit(x.detach()[tail], w.detach(), residual=r.detach()[tail])
    assert torch.equal(y8.view(torch.uint8)[tail], t8.view(torch.uint8)) and torch.equal(scale[tail], ts)
    del y8, h
    dy = torch.zeros_like(y)
    dy[tail] = randn(120, D, device=device, seed=2)
    dx, dw = torch.autograd.grad(y, (leaves[0], w), dy)
    dxt, dwt = torch.autograd.grad(yt, (small[0], w), dy[tail])
    assert torch.equal(dx[tail], dxt) and not bool(dx[:1000].any())
    # the same 120 terms in two orders in fp32, then rounded to bf16: half a step (2^-8) each
    xhat = yt.detach().float() / w.detach().float()
    terms = (dy[tail].float() * xhat).abs().sum(0)
    tol = 2.0 ** -7 * (1 + 2.0 ** -7) * dwt.float().abs() + 2 * 120 * 2.0 ** -24 * terms * (1 + 2.0 ** -6)
    assert bool(((dw.float() - dwt.float()).abs() <= tol).all())


def test_embedding_of_more_than_32_bits(device):
    """Rows, and a table, of more than 2^31 elements."""
    say("embedding, 2^31 elements")
    D, N = 4096, 2 ** 31 // 4096 + 1000
    ids = torch.arange(N, device=device) % 1000
    w = randn(1000, D, device=device, seed=1).requires_grad_()
    out = embedding(ids, w)
    for lo in (0, N // 2, N - 2000):
        assert torch.equal(out.detach()[lo:lo + 2000], w.detach()[ids[lo:lo + 2000]])
    dy = torch.zeros_like(out)
    dy[-1000:] = randn(1000, D, device=device, seed=2)
    (dw,) = torch.autograd.grad(out, w, dy)
    want = torch.zeros_like(dw).index_copy_(0, ids[-1000:], dy[-1000:])  # one place each
    assert torch.equal(dw, want)
    del out, dy
    V = N
    table = torch.zeros(V, D, dtype=BF16, device=device)
    rows = torch.tensor([V - 1, 3, V - 2, V - 1], device=device)
    table[rows] = randn(4, D, device=device, seed=3)
    table.requires_grad_()
    out = embedding(rows, table)
    assert torch.equal(out.detach(), table.detach()[rows])
    up = randn(4, D, device=device, seed=4)
    (dt,) = torch.autograd.grad(out, table, up)
    assert torch.equal(dt[V - 2], up[2]) and torch.equal(dt[3], up[1])
    assert torch.equal(dt[V - 1], (up[0].float() + up[3].float()).to(BF16))
    assert int((dt != 0).any(-1).sum()) == 3


def test_gated_of_more_than_32_bits(device):
    """Small integers, whose every result is exact (test_gpu_gated.py); the gradient comes from the last rows."""
    say("gated, 2^31 elements")
    M, D, F, n = 40000, 8, 60000, 100
    assert M * F > 2 ** 31
    ints = lambda *s: torch.randint(-1, 2, s, generator=torch.Generator().manual_seed(sum(s))).to(BF16).to(device)
    x, wg, wu = (t.requires_grad_() for t in (ints(M, D), ints(F, D), ints(F, D) * 1))
    h = gated_linear(x, wg, wu, activation="relu")
    X, G, U = x.detach()[-n:].double(), wg.detach().double(), wu.detach().double()
    g, u = X @ G.t().contiguous(), X @ U.t().contiguous()
    assert torch.equal(h.detach()[-n:], (g.relu() * u).to(BF16))
    dh = torch.zeros(M, F, dtype=BF16, device=device)
    dh[-n:] = ints(n, F)
    dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), dh)
    du, dg = dh[-n:].double() * g.relu(), dh[-n:].double() * u * (g > 0)
    assert torch.equal(dx[-n:], (dg @ G + du @ U).to(BF16)) and not bool(dx[:-n].any())
    assert torch.equal(dwg, (dg.t().contiguous() @ X).to(BF16)) and torch.equal(dwu, (du.t().contiguous() @ X).to(BF16))
