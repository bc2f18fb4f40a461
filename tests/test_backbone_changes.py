"""What a switched backbone does when its modules are changed afterwards, or hide something that a look at their
submodules does not show: adapters and hooks keep their effect, dropout is not lost. On the CPU, with the operators'
plain forms where a kernel would run.

Both sides compute the same fp32 formula, so rtol 1e-4 and atol 1e-5 as in test_backbone_gated.py."""
import copy
import pickle

import pytest
import torch
from torch import nn
from torch.nn import functional as F

from sparton_amd.backbone import _is_gated_block, _is_pre_norm_layer, use_in_backbone
from sparton_amd.embedding import SpartonEmbedding
from sparton_amd.feed_forward import SpartonGatedMLP, gated_linear_8bit, quantize_rows
from sparton_amd.norm import SpartonRMSNorm
from test_backbone import plain_attention, tiny
from test_backbone_gated import ALL, decoder, plain  # noqa: F401 (a fixture)

IDS = torch.arange(12).reshape(2, 6) + 5


class Adapter(nn.Module):
    """A projection with a low-rank addition, under the name of the one it wraps; `weight` is the base's."""

    def __init__(self, base: nn.Linear):
        super().__init__()
        self.base = base
        self.add = nn.Linear(base.in_features, base.out_features, bias=False)

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + self.add(x)


def same(a, b):
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_an_adapter_put_on_afterwards_counts(name, plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    torch.manual_seed(1)
    adapter = Adapter(getattr(ref.layers[0].mlp, name))
    for m in (ref, ours):
        setattr(m.layers[0].mlp, name, copy.deepcopy(adapter))
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert plain["gated"] == (2 if name == "down_proj" else 1)


@pytest.mark.parametrize("name", ["gate_proj", "up_proj"])
@pytest.mark.parametrize("kind", ["register_forward_hook", "register_forward_pre_hook"])
def test_hooks_of_a_projection_count(name, kind, plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    hook = (lambda m, args, out: out * 1.5) if kind == "register_forward_hook" else (lambda m, args: (args[0] * 1.5,))
    for m in (ref, ours):
        getattr(getattr(m.layers[1].mlp, name), kind)(hook)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)


@pytest.mark.parametrize("before", [False, True])
@pytest.mark.parametrize("kind", ["register_forward_hook", "register_forward_pre_hook", "forward"])
def test_hooks_of_the_activation_count(kind, before, plain):  # noqa: F811
    """Put there before or after the switch; looking at the block does not call them."""
    ref = decoder()
    calls = []

    def scaled(m, args, out=None):
        calls.append(m)
        return (args[0] * 1.5,) if out is None else out * 1.5

    def put(m):
        act = m.layers[0].mlp.act_fn
        if kind == "forward":
            act.forward = lambda x: scaled(act, None, F.silu(x))
        else:
            getattr(act, kind)(scaled)

    ours = copy.deepcopy(ref)
    if before:
        put(ours)
    use_in_backbone(ours, **ALL)
    assert not calls
    if not before:
        put(ours)
    put(ref)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert len(calls) == 2 and plain["gated"] == 1
    with pytest.raises(ValueError, match="activation"):
        SpartonGatedMLP.of(ref.layers[0].mlp)


class ShiftedSiLU(nn.SiLU):
    def forward(self, x):
        return super().forward(x - 1)


class SiLUActivation(nn.Module):  # named as one of transformers'
    def forward(self, x):
        return x.tanh()


OTHERS = dict(subclass=ShiftedSiLU, named=SiLUActivation, tanh=nn.Tanh,
              sequential=lambda: nn.Sequential(nn.SiLU(), nn.Dropout(0.5)).eval(), function=lambda: torch.sin)


@pytest.mark.parametrize("other", OTHERS)
def test_an_activation_put_in_afterwards_runs(other, plain):  # noqa: F811
    """Also where its class derives from one that the kernels compute, or has its name."""
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    for m in (ref, ours):
        if other == "function":  # a registered module's name takes modules alone
            del m.layers[0].mlp.act_fn
        m.layers[0].mlp.act_fn = OTHERS[other]()
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert plain["gated"] == 1
    if other != "function":
        assert not _is_gated_block(ref.layers[0].mlp)
        with pytest.raises(ValueError, match="activation"):
            SpartonGatedMLP.of(ref.layers[0].mlp)


def test_an_activation_of_another_name_put_in_afterwards_runs(plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    for m in (ref, ours):
        m.layers[0].mlp.act_fn = nn.GELU(approximate="tanh")
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert plain["gated"] == 2


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_the_module_of_a_gated_block_too(act, plain):  # noqa: F811
    torch.manual_seed(2)
    gate, up, down = nn.Linear(8, 12), nn.Linear(8, 12), nn.Linear(12, 8)
    fn = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}[act]
    x = torch.randn(3, 8)
    block = SpartonGatedMLP(gate, up, down, act)
    block.gate_proj = Adapter(gate)
    with torch.no_grad():
        same(block(x), down(fn(block.gate_proj(x)) * up(x)))
        block.gate_proj = gate
        gate.register_forward_hook(lambda m, args, out: out + 1)
        same(block(x), down(fn(gate(x)) * up(x)))
    assert plain["gated"] == 0


def test_a_hook_of_the_fused_norm_sees_the_norm(plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    seen = []

    def hook(m, args, out):
        seen.append((len(args), out.shape))
        return out * 1.5

    for m in (ref, ours):
        m.layers[0].post_attention_layernorm.register_forward_hook(hook)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert seen[0] == seen[1] == (1, (2, 6, 128))


def test_a_norm_put_in_afterwards_runs(plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    for m in (ref, ours):
        m.layers[0].post_attention_layernorm = nn.LayerNorm(128)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)


class DropoutBlock(nn.Module):
    def __init__(self, p):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj, self.act_fn = nn.Linear(8, 12), nn.Linear(8, 12), nn.Linear(12, 8), nn.SiLU()
        self.p = p

    def forward(self, x):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(F.dropout(h, self.p, self.training))


class DropoutLayer(nn.Module):
    def __init__(self, p):
        super().__init__()
        self.input_layernorm, self.self_attn = nn.Identity(), nn.Identity()
        self.post_attention_layernorm, self.mlp = nn.Identity(), nn.Identity()
        self.p = p

    def forward(self, hidden_states, **kwargs):
        h = self.self_attn(hidden_states=self.input_layernorm(hidden_states), **kwargs)[0]
        h = hidden_states + F.dropout(h, self.p, self.training)
        return h + self.mlp(self.post_attention_layernorm(h))


@pytest.mark.parametrize("training", [False, True])
def test_dropout_that_is_no_module_is_not_lost(training):
    state = torch.random.get_rng_state()
    for p, ours in ((0.0, True), (0.1, False), (0.01, False)):
        block, layer = DropoutBlock(p).train(training), DropoutLayer(p).train(training)
        assert _is_gated_block(block) == ours and _is_pre_norm_layer(layer) == ours
        assert block.training == training and layer.training == training
    torch.random.set_rng_state(state)
    block = DropoutBlock(0.1)
    state = torch.random.get_rng_state()
    _is_gated_block(block)
    assert torch.equal(state, torch.random.get_rng_state())  # looking leaves the caller's random numbers alone


@pytest.mark.parametrize("which", [1, 3, 5])
def test_a_scale_that_asks_for_a_gradient_is_refused(which):
    x, sx = quantize_rows(torch.randn(3, 16))
    w, sw = quantize_rows(torch.randn(6, 16))
    args = [x, sx, w, sw.clone(), w, sw.clone()]
    args[which] = args[which].clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        gated_linear_8bit(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm/HIP device"):
        gated_linear_8bit(*args)


CALLS = {
    "by position": lambda layer, x, mask, rope: layer(x, mask, None, None, False, rope),
    "mask by position": lambda layer, x, mask, rope: layer(x, mask, position_embeddings=rope),
    "by name": lambda layer, x, mask, rope: layer(hidden_states=x, attention_mask=mask, position_embeddings=rope),
    "no mask": lambda layer, x, mask, rope: layer(x, position_embeddings=rope),
    "as the model": lambda layer, x, mask, rope: layer(x, attention_mask=mask, position_ids=None, past_key_values=None,
                                                       use_cache=False, position_embeddings=rope),
}


@pytest.mark.parametrize("call", CALLS)
def test_a_switched_layer_takes_every_call_of_its_own(call, plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    x = torch.randn(1, 6, 128)
    rope = ref.rotary_emb(x, torch.arange(6)[None])
    with torch.no_grad():
        # causal: what the model gives its layers as a mask, each in its attention's form
        want = CALLS["by name"](ref.layers[0], x, torch.full((6, 6), -1e30).triu(1)[None, None], rope)
        for m in (ours, pickle.loads(pickle.dumps(ours)), copy.deepcopy(ours)):
            before = plain["added"]
            same(CALLS[call](m.layers[0], x, torch.ones(1, 6), rope), want)
            assert plain["added"] == before + 1


def test_a_call_that_the_layer_refuses_is_refused(plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    x = torch.randn(1, 6, 128)
    for m in (ref, ours):
        for args, kw in (((), {}), ((x, None), dict(attention_mask=None)), ((x, None, None, None, False, None, 7), {})):
            with pytest.raises(TypeError):
                m.layers[0](*args, **kw)


def test_a_switched_block_takes_its_input_by_name(plain):  # noqa: F811
    ref = decoder()
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    x = torch.randn(2, 128)
    with torch.no_grad():
        same(ours.layers[0].mlp(x=x), ref.layers[0].mlp(x))
    for args, kw in (((), {}), ((x, x), {}), ((x,), dict(x=x))):
        with pytest.raises(TypeError):
            ours.layers[0].mlp(*args, **kw)


class OtherCall(DropoutLayer):
    """Gives its attention something else than it was given."""

    def __init__(self, kind):
        super().__init__(0.0)
        self.kind = kind

    def forward(self, hidden_states, mask=None, flag=False, **kwargs):
        x = self.input_layernorm(hidden_states)
        calls = dict(same=lambda: self.self_attn(hidden_states=x, mask=mask, flag=flag, **kwargs),
                     position=lambda: self.self_attn(x, mask=mask, flag=flag, **kwargs),
                     dropped=lambda: self.self_attn(hidden_states=x, mask=mask, **kwargs),
                     rest_dropped=lambda: self.self_attn(hidden_states=x, mask=mask, flag=flag),
                     other=lambda: self.self_attn(hidden_states=x, mask=1, flag=flag, **kwargs),
                     more=lambda: self.self_attn(hidden_states=x, mask=mask, flag=flag, more=1, **kwargs))
        h = hidden_states + calls[self.kind]()[0]
        return h + self.mlp(self.post_attention_layernorm(h))


@pytest.mark.parametrize("kind", ["same", "position", "dropped", "rest_dropped", "other", "more"])
def test_a_layer_that_calls_its_attention_in_another_way_keeps_its_forward(kind):
    assert _is_pre_norm_layer(OtherCall(kind)) == (kind == "same")


@pytest.mark.parametrize("before", [False, True])
@pytest.mark.parametrize("name", ["input_layernorm", "post_attention_layernorm"])
def test_a_norms_own_forward_runs(name, before, plain):  # noqa: F811
    """Put on the module, as a wrapper for moved weights does, before or after the switch."""
    ref = decoder()

    def put(m):
        norm = getattr(m.layers[0], name)
        own = norm.forward
        norm.forward = lambda x: own(x) * 1.5

    ours = copy.deepcopy(ref)
    if before:
        put(ours)
    use_in_backbone(ours, **ALL)
    if not before:
        put(ours)
    put(ref)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert plain["added"] == (1 if name == "post_attention_layernorm" else 2)


@pytest.mark.parametrize("change", ["own forward before", "own forward after", "another module after", "hook before",
                                    "hook after"])
def test_an_encoders_layer_norm_changed(change, monkeypatch):
    monkeypatch.setattr("sparton_amd.backbone.attention", plain_attention)
    monkeypatch.setattr("sparton_amd.norm.layer_norm", lambda x, w, b=None, eps=1e-5, residual=None:
                        F.layer_norm(x if residual is None else x + residual, w.shape, w, b, eps))
    ref = tiny("bert").eval()

    def put(m):
        block = m.bert.encoder.layer[0].output
        if change == "another module after":
            block.LayerNorm = nn.LayerNorm(block.LayerNorm.weight.shape[0])
        elif change.startswith("hook"):
            block.LayerNorm.register_forward_pre_hook(lambda m, args: (args[0] + 1.5 * args[0].square(),))
        else:
            own = block.LayerNorm.forward
            block.LayerNorm.forward = lambda x: own(x) * 1.5

    ours = copy.deepcopy(ref)
    if change.endswith("before"):
        put(ours)
    use_in_backbone(ours)
    if change.endswith("after"):
        put(ours)
    put(ref)
    with torch.no_grad():
        same(ours(IDS).logits, ref(IDS).logits)


# ---- a module made of another computes what that one does, or is refused -----------------------

def own_forward(m, f):
    m.forward = f
    return m


class MultipliedBlock(DropoutBlock):
    def forward(self, x):
        return self.down_proj(0.5 * self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class DropoutNorm(nn.RMSNorm):
    def forward(self, x):
        return F.dropout(super().forward(x), 0.1, self.training)


class BiasedNorm(nn.RMSNorm):
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.bias = nn.Parameter(torch.zeros(16))

    def forward(self, x):
        return super().forward(x) + self.bias


class ShiftedEmbedding(nn.Embedding):
    def forward(self, input):
        return super().forward(input + 1)


def other_modules():
    from transformers.models.gemma.modeling_gemma import GemmaRMSNorm
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding
    block, dropped = DropoutBlock(0.0), DropoutBlock(0.0)
    dropped.dropout = nn.Dropout(0.5)
    return {
        "norm of 1 + weight": (SpartonRMSNorm, GemmaRMSNorm(16)),
        "norm with dropout": (SpartonRMSNorm, DropoutNorm(16, eps=1e-5).eval()),
        "norm with a bias": (SpartonRMSNorm, BiasedNorm(16, eps=1e-5)),
        "layer norm": (SpartonRMSNorm, nn.LayerNorm(16)),
        "norm with its own forward": (SpartonRMSNorm, own_forward(nn.RMSNorm(16, eps=1e-5), lambda x: x)),
        "scaled embedding": (SpartonEmbedding, Gemma3TextScaledWordEmbedding(10, 16, 0, embed_scale=4.0)),
        "shifted embedding": (SpartonEmbedding, ShiftedEmbedding(10, 16)),
        "embedding with its own forward": (SpartonEmbedding, own_forward(nn.Embedding(10, 16), lambda x: x)),
        "multiplied block": (SpartonGatedMLP, MultipliedBlock(0.0)),
        "block with dropout": (SpartonGatedMLP, DropoutBlock(0.1)),
        "block with a module more": (SpartonGatedMLP, dropped),
        "block with its own forward": (SpartonGatedMLP, own_forward(block, lambda x: x)),
    }


@pytest.mark.parametrize("name", other_modules())
def test_a_module_that_computes_something_else_is_refused(name):
    cls, module = other_modules()[name]
    with pytest.raises(ValueError, match=cls.__name__):
        cls.of(module)


def test_what_the_kernels_compute_is_taken(plain):  # noqa: F811
    from transformers.models.llama.modeling_llama import LlamaRMSNorm
    x, ids = torch.randn(5, 16), torch.tensor([1, 4, 1])
    for norm in (LlamaRMSNorm(16), nn.RMSNorm(16, eps=1e-5), SpartonRMSNorm(16)):
        with torch.no_grad():
            norm.weight.uniform_(0.5, 1.5)
        ours = SpartonRMSNorm.of(norm)
        same(ours(x), norm(x))
        assert ours.weight is norm.weight
    block = DropoutBlock(0.0)
    same(SpartonGatedMLP.of(block)(x[:, :8]), block(x[:, :8]))
    table = nn.Embedding(10, 16)
    once = SpartonEmbedding.of(table, scale=3.0)
    for ours, factor in ((once, 3), (SpartonEmbedding.of(once), 3), (SpartonEmbedding.of(once, scale=2.0), 6)):
        same(ours(ids), factor * table(ids))


def test_an_embeddings_own_forward_runs(plain):  # noqa: F811
    ref = decoder()
    own = ref.embed_tokens.forward
    ref.embed_tokens.forward = lambda ids: own(ids) * 1.5
    ref.other = nn.Embedding(4, 4)
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    assert type(ours.embed_tokens) is nn.Embedding and isinstance(ours.other, SpartonEmbedding)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)


@pytest.mark.parametrize("training", [False, True])
def test_a_module_made_of_a_gated_block_keeps_its_hooks_and_mode(training, plain):  # noqa: F811
    block, seen = DropoutBlock(0.0).train(training), []
    block.up_proj.train(not training)  # a mode of its own
    block.register_forward_hook(lambda m, args, out: out * 1.5)
    block.register_forward_pre_hook(lambda m, args: seen.append(type(m).__name__))
    ours = SpartonGatedMLP.of(block)
    x = torch.randn(3, 8)
    same(ours(x), block(x))
    assert seen == ["SpartonGatedMLP", "DropoutBlock"] and plain["gated"] == 1
    assert ours.training == training and ours.up_proj.training == block.up_proj.training == (not training)
    assert list(ours.state_dict()) == list(block.state_dict()) and set(dict(ours.named_children())) == {
        "gate_proj", "up_proj", "down_proj"} and block.act_fn is not None
    ours.up_proj = nn.Linear(8, 12)  # the block keeps its own
    assert block.up_proj is not ours.up_proj


@pytest.mark.parametrize("where", ["float64", "bfloat16", "meta"])
def test_modules_are_known_whatever_torchs_defaults_are(where, plain):  # noqa: F811
    ref, norm, block = decoder(), SpartonRMSNorm(16), DropoutBlock(0.0)
    theirs, layer = nn.RMSNorm(16, eps=1e-5), DropoutLayer(0.0)
    ours = copy.deepcopy(ref)
    before = torch.get_default_dtype()
    try:
        if where == "meta":
            torch.set_default_device("meta")
        else:
            torch.set_default_dtype(getattr(torch, where))
        use_in_backbone(ours, **ALL)
        SpartonRMSNorm.of(norm), SpartonRMSNorm.of(theirs), SpartonGatedMLP.of(block)
        assert _is_pre_norm_layer(layer)
    finally:
        torch.set_default_device(None)
        torch.set_default_dtype(before)
    with torch.no_grad():
        same(ours(IDS).last_hidden_state, ref(IDS).last_hidden_state)
    assert plain == dict(rms=5, added=2, gated=2, embedding=1)


def test_a_name_that_the_layer_does_not_take_is_refused(plain):  # noqa: F811
    ref = decoder()

    class Passing(nn.Module):
        """The layer's steps, without other names."""

        def __init__(self, layer):
            super().__init__()
            for n, c in layer.named_children():
                setattr(self, n, c)

        def forward(self, hidden_states, position_embeddings=None, attention_mask=None):
            h = self.self_attn(hidden_states=self.input_layernorm(hidden_states), position_embeddings=position_embeddings,
                               attention_mask=attention_mask)[0]
            h = hidden_states + h
            return h + self.mlp(self.post_attention_layernorm(h))

    ref.layers[0] = Passing(ref.layers[0])
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    x = torch.randn(1, 6, 128)
    rope = ref.rotary_emb(x, torch.arange(6)[None])
    with torch.no_grad():
        want = ref.layers[0](x, rope, torch.full((6, 6), -1e30).triu(1)[None, None])
        same(ours.layers[0](x, rope, torch.ones(1, 6)), want)
    assert plain["added"] == 1
    for m in (ref, ours):
        with pytest.raises(TypeError):
            m.layers[0](x, rope, use_cache=False)
