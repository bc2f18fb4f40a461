"""What a compiled program runs of the gated product: without gradients no g and u are written, and a backward computes
the gradients that are asked for. On the CPU with tensors without data, which take the compiler's path; on the GPU
through torch.compile, against the eager calls."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from _parity import say
from sparton_amd.feed_forward import gated_linear

NAMES = ["x", "w_gate", "w_up", "b_gate", "b_up"]


class Calls(TorchDispatchMode):
    """The framework's operators that are called, with their arguments."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "sparton":
            self.seen.append((func.name().split("::")[1], args))
        return func(*args, **(kwargs or {}))


def inputs(asked, device="cpu", make=torch.empty):
    shapes = dict(x=(20, 64), w_gate=(48, 64), w_up=(48, 64), b_gate=(48,), b_up=(48,))
    return [make(s, device=device).requires_grad_(n in asked) for n, s in shapes.items()]


def test_without_gradients_g_and_u_are_not_written():
    for asked, enabled, op in (([], True, "gated_infer"), (NAMES, False, "gated_infer"), (["b_up"], True, "gated_fwd")):
        with FakeTensorMode(), Calls() as calls, torch.set_grad_enabled(enabled):
            h = gated_linear(*inputs(asked))
            gated_linear(*inputs(asked)[:3])
        assert h.shape == (20, 48) and h.requires_grad == (op == "gated_fwd")
        assert [n for n, _ in calls.seen] == [op, op if "b_up" not in asked else "gated_infer"]


@pytest.mark.gpu
@pytest.mark.parametrize("asked", [[], NAMES])
def test_a_compiled_forward(asked, device):
    say(f"compiled forward, {asked}")
    args = inputs(asked, device, torch.randn)
    f = lambda *t: gated_linear(*t) * 2
    with torch.no_grad():
        want = f(*args)
        assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(*args), want)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*args)
    assert torch.equal(got.detach(), want) and got.requires_grad == bool(asked)


ASKED = [["x"], ["w_up"], ["w_gate", "b_up"], ["b_gate"], ["b_gate", "b_up"], ["x", "b_up"], NAMES]


@pytest.mark.parametrize("asked", ASKED)
def test_a_backward_computes_what_is_asked_for(asked):
    with FakeTensorMode(), Calls() as calls:
        args = inputs(asked)
        leaves = [t for t in args if t.requires_grad]
        grads = torch.autograd.grad(gated_linear(*args).sum(), leaves)
    assert [g.shape for g in grads] == [t.shape for t in leaves]
    (name, args), = calls.seen[1:]
    flags = [*args[7:], True, True][:4]  # the last two have defaults
    assert name == "gated_bwd" and flags == ["b_gate" in asked, "b_up" in asked, "x" in asked,
                                             bool({"w_gate", "w_up"} & set(asked))]


@pytest.mark.gpu
@pytest.mark.parametrize("asked", ASKED)
def test_a_compiled_backward(asked, device):
    say(f"compiled backward of {asked}")
    args = inputs(asked, device, torch.randn)
    leaves = [t for t in args if t.requires_grad]
    dh = torch.randn(20, 48, device=device)
    f = lambda *t: gated_linear(*t) * 2
    want = torch.autograd.grad(f(*args), leaves, dh)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(*args), leaves, dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    every = torch.ops.sparton.gated_bwd(dh, *args[:3], *torch.ops.sparton.gated_fwd(*args, "silu")[1:], "silu", True, True)
    some = torch.ops.sparton.gated_bwd(dh, *args[:3], *torch.ops.sparton.gated_fwd(*args, "silu")[1:], "silu",
                                       "b_gate" in asked, "b_up" in asked, "x" in asked, "w_gate" in asked)
    here = ["x" in asked, "w_gate" in asked, "w_gate" in asked, "b_gate" in asked, "b_up" in asked]
    assert all(torch.equal(a, b) if h else a.numel() == 0 for a, b, h in zip(some, every, here))


@pytest.mark.gpu
def test_a_compiled_backbone(device):
    """A gated encoder, switched whole, as one graph, with and without gradients; tolerances of test_backbone_gated.py."""
    import copy
    from transformers import EuroBertConfig, EuroBertModel
    from sparton_amd.backbone import use_in_backbone
    say("compiled backbone")
    torch.manual_seed(0)
    ref = EuroBertModel(EuroBertConfig(vocab_size=300, hidden_size=128, num_hidden_layers=2, num_attention_heads=4,
                                       num_key_value_heads=2, intermediate_size=256, attn_implementation="eager",
                                       pad_token_id=0)).to(device).eval()
    ours = use_in_backbone(copy.deepcopy(ref), rms_norm=True, feed_forward=True, embedding=True)
    ids = (torch.arange(12).reshape(2, 6) + 5).to(device)
    mask = torch.ones_like(ids)
    mask[1, 4:] = 0
    on = mask.bool()
    compiled = torch.compile(ours, backend="aot_eager", fullgraph=True)
    want = ref(ids, mask).last_hidden_state[on]
    got = compiled(ids, mask).last_hidden_state[on]
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)
    a, b = (dict(zip(dict(m.named_parameters()), torch.autograd.grad(out.square().sum(), list(m.parameters()))))
            for m, out in ((ref, want), (ours, got)))
    floor = 1e-4 * max(g.abs().max().item() for g in a.values())
    assert max((b[n] - g).abs().max().item() / max(g.abs().max().item(), floor) for n, g in a.items()) <= 1e-3
    with torch.no_grad():
        torch.testing.assert_close(compiled(ids, mask).last_hidden_state[on], want, rtol=1e-4, atol=1e-5)
