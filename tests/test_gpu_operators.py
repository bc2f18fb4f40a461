"""Attention, LayerNorm and the preference loss together: gradients differentiated again, calls at once
on two streams, captured graphs that share a memory pool, the same tensor in several places, and
tensors whose offsets pass 32 bits. Bitwise against the same operators' plain calls, which the tests
of each operator check against 64 bits."""
import pytest
import torch

from _parity import say
from sparton_amd.attention import attention
from sparton_amd.loss import preference_loss, preference_margin
from sparton_amd.norm import layer_norm

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def randn(*shape, device, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def calls(device, seed=0):
    """name -> (function of its leaves, leaves)"""
    att = lambda Sq, Sk: [randn(2, S, 4, 64, device=device, seed=seed + i).transpose(1, 2)
                          for i, S in enumerate((Sq, Sk, Sk))]
    mask = (torch.arange(3000, device=device)[None, :] < torch.tensor([[2900], [1700]], device=device)).long()
    rows = [randn(300, 768, device=device, seed=seed + 3 + i) for i in range(2)]
    vecs = [randn(768, device=device, seed=seed + 5 + i) for i in range(2)]
    reps = [randn(6, 30522, device=device, seed=seed + 7 + i).relu() * 0.1 for i in range(3)]
    return {
        "attention": (lambda q, k, v: attention(q, k, v, causal=True), att(200, 200)),
        "attention, few rows": (lambda q, k, v: attention(q, k, v, mask), att(3, 3000)),
        "layer_norm": (lambda x, r, w, b: layer_norm(x, w, b, residual=r), rows + vecs),
        "preference_loss": (lambda q, p, n: preference_loss(q, p, n).loss, reps),
    }


def both(f, leaves):
    """The output and every leaf's gradient."""
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = f(*leaves)
    return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))


NAMES = ["attention", "attention, few rows", "layer_norm", "preference_loss"]


@pytest.mark.parametrize("name", NAMES)
def test_a_second_derivative_is_refused(name, device):
    say(f"second derivative of {name}")
    f, leaves = calls(device)[name]
    want = both(f, leaves)
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = f(*leaves)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=True)
    for g, w in zip(grads, want[1:]):
        assert g.requires_grad and torch.equal(g.detach(), w)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(grads[0].float().sum(), leaves[0])


@pytest.mark.parametrize("name", NAMES)
def test_a_backward_called_by_hand(name, device):
    """Outside the autograd engine, with and without grad mode."""
    say(f"grad_fn of {name}")
    f, leaves = calls(device)[name]
    want = both(f, leaves)[1:]
    out = f(*[t.detach().requires_grad_() for t in leaves])
    grads = [torch.ones_like(out)] + [None] * (name == "preference_loss")  # that node's second output: the margins
    for mode in (False, True):
        with torch.set_grad_enabled(mode):
            got = [g for g in out.grad_fn(*grads) if g is not None]
        assert all(torch.equal(g.detach(), w) for g, w in zip(got, want)) and len(got) >= len(want)


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


def test_two_graphs_of_one_pool(device):
    """Forward calls of two input sets captured into two graphs that share a memory pool, replayed in
    turn with eager calls between them."""
    say("two graphs")
    sets = [calls(device, 0), calls(device, 100)]
    extra = calls(device, 200)

    def step(c):
        with torch.no_grad():
            return {n: f(*leaves) for n, (f, leaves) in c.items()}

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(c) for c in sets]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(step(c))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        for t in outs[i].values():
            t.fill_(7.0)
        graphs[i].replay()
        step(extra)
        torch.cuda.synchronize()
        for n in NAMES:
            assert torch.equal(outs[i][n], want[i][n]), (i, n)


def test_one_tensor_in_several_places(device):
    """A tensor given twice gets the sum of its places' gradients."""
    say("one tensor twice")
    x = randn(2, 70, 4, 64, device=device, seed=1).transpose(1, 2)
    parts = both(lambda a, b, c: attention(a, b, c), [x, x, x])
    leaf = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(attention(leaf, leaf, leaf), leaf, torch.ones_like(x))
    total = sum(p.float() for p in parts[1:])
    # two sums of bf16 tensors, each rounded to bf16 (2^-8 of a partial sum at most)
    assert bool(((dx.float() - total).abs() <= 2.0 ** -7 * sum(p.float().abs() for p in parts[1:])).all())

    h = randn(90, 768, device=device, seed=2, dtype=torch.float32)
    w = randn(768, device=device, seed=3, dtype=torch.float32)
    parts = both(lambda a, r: layer_norm(a, w, residual=r), [h, h])
    leaf = h.detach().requires_grad_()
    (dh,) = torch.autograd.grad(layer_norm(leaf, w, residual=leaf), leaf, torch.ones_like(h))
    assert torch.equal(dh, parts[1] + parts[2])

    q, p = (randn(5, 999, device=device, seed=4 + i, dtype=torch.float32) for i in range(2))
    leaf = p.detach().requires_grad_()
    out = preference_loss(q, leaf, leaf)
    (dp,) = torch.autograd.grad(out.loss, leaf)
    assert not bool(out.margin.any()) and not bool(dp.any())  # c q - c q


# ---- offsets past 32 bits --------------------------------------------------------------------

@pytest.mark.parametrize("Sq,causal", [(300, True), (1, False)])
def test_attention_in_a_large_buffer(Sq, causal, device):
    say(f"large strides, {Sq} rows")
    B, S, D = 2, 280, 64
    step = 2 ** 23 + 8                        # elements between rows: the last row starts past 2^31
    assert (S - 1) * step > 2 ** 31
    buf = torch.empty(B * S * step // 2, dtype=BF16, device=device)
    view = lambda at, n: buf.as_strided((B, 1, n, D), (8 * D, 8, step, 1), at)
    small = [randn(B, 1, n, D, device=device, seed=i) for i, n in enumerate((min(Sq, S), S, S))]
    large = [view(i * D, t.shape[2]) for i, t in enumerate(small)]
    for t, s in zip(large, small):
        t.copy_(s)
    f = lambda q, k, v: attention(q, k, v, causal=causal)
    for a, b in zip(both(f, large), both(f, small)):
        assert torch.equal(a, b)


def test_attention_with_more_output_than_32_bits(device):
    say("2^25 rows")
    S = 2 ** 25 + 77
    q = torch.empty(1, 1, S, 64, dtype=BF16, device=device).normal_()
    k, v = (randn(1, 1, 1, 64, device=device, seed=i) for i in (1, 2))
    with torch.no_grad():
        out = attention(q, k, v)  # one key: every row is its value
    for lo in range(0, S, 2 ** 22):
        part = out[0, 0, lo:lo + 2 ** 22]
        assert bool((part == v[0, 0]).all())


def test_layer_norm_of_more_than_32_bits(device):
    say("2^31 elements")
    D, M = 4096, 2 ** 31 // 4096 + 101
    x = torch.empty(M, D, dtype=BF16, device=device).normal_()
    w = randn(D, device=device, seed=1).requires_grad_()
    tail = slice(M - 120, M)
    xl, xt = x.requires_grad_(), x.detach()[tail].clone().requires_grad_()
    y, yt = layer_norm(xl, w), layer_norm(xt, w)
    assert torch.equal(y.detach()[tail], yt.detach())
    dy = torch.zeros_like(y)
    dy[tail] = randn(120, D, device=device, seed=2)
    dx, dw = torch.autograd.grad(y, (xl, w), dy)
    dxt, dwt = torch.autograd.grad(yt, (xt, w), dy[tail])
    assert torch.equal(dx[tail], dxt) and not bool(dx[:1000].any())
    # the same 120 terms in two orders in fp32, then rounded to bf16: half a step (2^-8) each
    xhat = torch.nn.functional.layer_norm(xt.detach().float(), (D,))
    terms = (dy[tail].float() * xhat).abs().sum(0)
    tol = 2.0 ** -7 * (1 + 2.0 ** -7) * dwt.float().abs() + 2 * 120 * 2.0 ** -24 * terms
    assert bool(((dw.float() - dwt.float()).abs() <= tol).all())


def test_preference_loss_of_more_than_32_bits(device):
    say("2^31 elements of reps")
    B, V, n = 8592, 250002, 3
    assert B * V > 2 ** 31
    q, p, r = (torch.zeros(B, V, dtype=BF16, device=device) for _ in range(3))
    for i, t in enumerate((q, p, r)):
        t[-n:] = randn(n, V, device=device, seed=i).relu() * 0.02
    leaves = [t.requires_grad_() for t in (q, p, r)]
    tails = [t.detach()[-n:].clone() for t in leaves]
    out = preference_loss(*leaves)
    m = preference_margin(*tails)
    # V products and sums in fp32, in two orders
    terms = (tails[0].double() * (tails[1].double() - tails[2].double()).abs()).sum(1)
    assert bool(((out.margin[-n:] - m).abs() <= 2 * V * 2.0 ** -24 * terms).all())
    assert not bool(out.margin[:-n].any())
    grads = torch.autograd.grad(out.loss, leaves)
    c = -torch.sigmoid(-out.margin[-n:].double())[:, None] / B
    want = (c * (tails[1].double() - tails[2].double()), c * tails[0].double(), -c * tails[0].double())
    for g, w in zip(grads, want):
        # one rounding to bf16 (2^-8), and a few in fp32 on the way
        assert bool(((g[-n:].double() - w).abs() <= (2.0 ** -8 + 2.0 ** -18) * w.abs()).all())
        assert not bool(g[:1000].any())
