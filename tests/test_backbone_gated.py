"""The RMS norm, the gated product and the embedding in transformers backbones, tiny and built offline: what
use_in_backbone switches when it is asked to, what it leaves, and a training step on every kernel against the same
model with torch's.

Tolerances, fp32 throughout, as in test_backbone.py: hidden states rtol 1e-4, atol 1e-5; gradients against the
gradient's largest magnitude (with a floor of 1e-4 of the largest of all), at most 1e-3."""
import copy
import pickle

import pytest
import torch
from torch import nn
from torch.nn import functional as F

import sparton_amd
from _parity import say
from sparton_amd.backbone import _is_gated_block, _is_pre_norm_layer, _is_rms_norm, use_in_backbone
from sparton_amd.norm import SpartonRMSNorm
from test_backbone import left_padded, plain_attention, tiny
from test_hf_integration import batch

ALL = dict(rms_norm=True, feed_forward=True, embedding=True)


def decoder(**kw):
    from transformers import LlamaConfig, LlamaModel
    torch.manual_seed(0)
    m = LlamaModel(LlamaConfig(**dict(dict(vocab_size=300, hidden_size=128, num_hidden_layers=2, num_attention_heads=4,
                                           num_key_value_heads=2, intermediate_size=256, attn_implementation="eager",
                                           pad_token_id=0), **kw))).eval()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:  # norms that do something
                p.uniform_(0.5, 1.5)
    return m


@pytest.fixture
def plain(monkeypatch):
    """The operators' plain forms in the kernels' places; counts their calls."""
    calls = dict(rms=0, added=0, gated=0, embedding=0)

    def rms(x, w, eps=1e-6, residual=None):
        calls["rms"] += 1
        calls["added"] += residual is not None
        h = x if residual is None else x + residual
        y = w * h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
        return y if residual is None else (y, h)

    def gated(x, wg, wu, bg=None, bu=None, activation="silu"):
        calls["gated"] += 1
        act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}
        return act[activation](F.linear(x, wg, bg)) * F.linear(x, wu, bu)

    def embed(ids, w, scale=1.0, padding_idx=None):
        calls["embedding"] += 1
        return scale * F.embedding(ids, w, padding_idx)

    monkeypatch.setattr("sparton_amd.backbone.attention", plain_attention)
    monkeypatch.setattr("sparton_amd.norm.rms_norm", rms)
    monkeypatch.setattr("sparton_amd.feed_forward.gated_linear", gated)
    monkeypatch.setattr("sparton_amd.embedding.embedding", embed)
    return calls


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_pytorch_tanh", "relu"])
def test_a_switched_backbone_computes_the_same(act, plain):
    ref = decoder(hidden_act=act, mlp_bias=act == "gelu")
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    assert list(ours.state_dict()) == list(ref.state_dict())
    ids, mask = left_padded(3, 12, seed=1)
    with torch.no_grad():
        a, b = (m(ids, mask).last_hidden_state for m in (ref, ours))
    on = mask.bool()
    torch.testing.assert_close(b[on], a[on], rtol=1e-4, atol=1e-5)
    assert plain == dict(rms=5, added=2, gated=2, embedding=1)
    with torch.no_grad():  # a cache goes through the layers as before
        first = ours(ids[:1, :8], use_cache=True)
        last = ours(ids[:1, 8:], past_key_values=first.past_key_values, use_cache=True).last_hidden_state
        torch.testing.assert_close(last, ref(ids[:1]).last_hidden_state[:, 8:], rtol=1e-4, atol=1e-5)


def test_what_is_not_asked_for_stays(plain):
    ref = decoder()
    for ask in ({}, dict(rms_norm=True), dict(feed_forward=True), dict(embedding=True)):
        m = use_in_backbone(copy.deepcopy(ref), **ask)
        assert any(isinstance(c, SpartonRMSNorm) for c in m.modules()) == ("rms_norm" in ask)
        assert isinstance(m.embed_tokens, sparton_amd.SpartonEmbedding) == ("embedding" in ask)
        assert ("forward" in m.layers[0].mlp.__dict__) == ("feed_forward" in ask)
        assert ("forward" in m.layers[0].__dict__) == ("rms_norm" in ask)


def test_switching_twice_copies_and_pickles(plain):
    ref = decoder()
    m = use_in_backbone(use_in_backbone(copy.deepcopy(ref), **ALL), **ALL)
    ids = torch.arange(12).reshape(2, 6) + 5
    with torch.no_grad():
        want = ref(ids).last_hidden_state
        for twin in (m, copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
            torch.testing.assert_close(twin(ids).last_hidden_state, want, rtol=1e-4, atol=1e-5)
            for layer in twin.layers:
                assert layer.forward.__self__ is layer and layer.mlp.forward.__self__ is layer.mlp
    own = {n: id(p) for n, p in m.named_parameters()}
    assert {n: id(p) for n, p in use_in_backbone(m, **ALL).named_parameters()} == own


def test_a_model_without_them_is_refused_and_stays():
    for ask in (dict(rms_norm=True), dict(feed_forward=True)):
        llm = tiny("bert")
        with pytest.raises(ValueError, match="BertForMaskedLM has no"):
            use_in_backbone(llm, embedding=True, **ask)
        assert llm.config._attn_implementation == "eager"
        assert not any(isinstance(m, (sparton_amd.SpartonLayerNorm, sparton_amd.SpartonEmbedding)) for m in llm.modules())


def test_embeddings_of_an_encoder_and_one_in_two_places(plain):
    """The tied decoder keeps the parameter; a module in two places stays one."""
    ref = tiny("bert")
    ref.again = ref.bert.embeddings.word_embeddings
    ours = use_in_backbone(copy.deepcopy(ref), embedding=True)
    assert ours.again is ours.bert.embeddings.word_embeddings and isinstance(ours.again, sparton_amd.SpartonEmbedding)
    assert ours.again.weight is ours.cls.predictions.decoder.weight and ours.again.padding_idx == ref.again.padding_idx
    kinds = [m for m in ours.modules() if isinstance(m, nn.Embedding)]
    assert len(kinds) == 3 and all(isinstance(m, sparton_amd.SpartonEmbedding) for m in kinds)


class _Norm(nn.Module):
    def __init__(self, f):
        super().__init__()
        self.weight, self.eps, self.f = nn.Parameter(torch.zeros(16)), 1e-5, f

    def forward(self, x):
        return self.f(self.weight, x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps))


class SomeRMSNorm(_Norm):
    pass


def test_modules_are_known_by_what_they_compute():
    """The class's name alone is not trusted: norms of 1 + weight, other activations, blocks with more in them."""
    assert _is_rms_norm(SomeRMSNorm(lambda w, x: w * x)) and _is_rms_norm(nn.RMSNorm(16, eps=1e-5))
    assert not _is_rms_norm(SomeRMSNorm(lambda w, x: (1 + w) * x)) and not _is_rms_norm(_Norm(lambda w, x: w * x))
    assert not _is_rms_norm(nn.RMSNorm(16)) and not _is_rms_norm(nn.RMSNorm((4, 4), eps=1e-5))  # torch's default epsilon
    assert not _is_rms_norm(nn.RMSNorm(16, eps=1e-5, elementwise_affine=False))
    layer = decoder().layers[0]
    assert _is_pre_norm_layer(layer) and _is_gated_block(layer.mlp)

    class Other(type(layer.mlp)):
        def forward(self, x):
            return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))

    class Scaled(type(layer)):
        def forward(self, hidden_states, **kwargs):
            return 0.5 * super().forward(hidden_states, **kwargs)

    layer.mlp.__class__, layer.__class__ = Other, Scaled
    assert not _is_gated_block(layer.mlp) and not _is_pre_norm_layer(layer)
    block = decoder().layers[0].mlp
    block.dropout = nn.Dropout(0.1)
    assert not _is_gated_block(block)
    assert not _is_gated_block(decoder(hidden_act="tanh").layers[0].mlp)


def test_a_block_keeps_its_hooks(plain):
    m = decoder()
    seen = []
    m.layers[0].mlp.register_forward_hook(lambda mod, args, out: seen.append("mlp"))
    m.layers[0].input_layernorm.register_forward_hook(lambda mod, args, out: seen.append("norm"))
    m.embed_tokens.register_forward_hook(lambda mod, args, out: seen.append("embed"))
    use_in_backbone(m, **ALL)(torch.tensor([[3, 4]]))
    assert seen == ["embed", "norm", "mlp"]


# ---- on the kernels -----------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("checkpointing", [False, True])
def test_training_step_on_a_gated_backbone(checkpointing, device):
    """Every gradient of a decoder backbone, on all kernels and on torch's operators."""
    say(f"gated backbone, checkpointing={checkpointing}")
    ref = decoder(use_cache=False, hidden_act="gelu").to(device)
    ours = use_in_backbone(copy.deepcopy(ref), **ALL)
    if checkpointing:
        ours.gradient_checkpointing_enable()
        ours.train()
    ids, mask = (t.to(device) for t in left_padded(4, 40, seed=3))
    ids = ids.masked_fill(mask == 0, 0)
    up = torch.randn(4, 40, 128, generator=torch.Generator().manual_seed(5)).to(device) * mask[..., None]
    grads = []
    for m in (ref, ours):
        out = m(ids, mask).last_hidden_state
        grads.append((out.detach()[mask.bool()], dict(zip(dict(m.named_parameters()), torch.autograd.grad(out, list(m.parameters()), up)))))
    (a, ga), (b, gb) = grads
    torch.testing.assert_close(b, a, rtol=1e-4, atol=1e-5)
    floor = 1e-4 * max(g.abs().max().item() for g in ga.values())
    worst = max((gb[n] - g).abs().max().item() / max(g.abs().max().item(), floor) for n, g in ga.items())
    say(f"   worst gradient error {worst:.2e}")
    assert ga.keys() == gb.keys() and worst <= 1e-3


@pytest.mark.gpu
def test_a_gated_backbone_in_bf16(device):
    """Under autocast over fp32 parameters, and held in bf16: near the fp32 result, gradients finite."""
    say("gated backbone, bf16")
    m = use_in_backbone(decoder(use_cache=False).to(device), **ALL)
    ids, mask = (t.to(device) for t in left_padded(3, 33, seed=4))
    on = mask.bool()
    with torch.no_grad():
        want = m(ids, mask).last_hidden_state[on]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(ids, mask).last_hidden_state[on]
    assert (got.float() - want).abs().max() <= 5e-2 * want.abs().max()
    got.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())
    m.zero_grad()
    m.to(torch.bfloat16)
    got = m(ids, mask).last_hidden_state[on]
    assert got.dtype == torch.bfloat16 and (got.float() - want).abs().max() <= 5e-2 * want.abs().max()
    got.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.dtype == torch.bfloat16 for p in m.parameters())


@pytest.mark.gpu
def test_tokens_one_by_one_on_a_gated_backbone(device):
    say("token by token")
    m = use_in_backbone(decoder().to(device), **ALL)
    ids = torch.randint(0, 300, (2, 20), generator=torch.Generator().manual_seed(0)).to(device)
    with torch.no_grad():
        whole, cache, rows = m(ids).last_hidden_state, None, []
        for n in range(20):
            out = m(ids[:, n:n + 1], past_key_values=cache, use_cache=True)
            cache = out.past_key_values
            rows.append(out.last_hidden_state)
    torch.testing.assert_close(torch.cat(rows, 1), whole, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_norm_and_feed_forward_in_8_bits(device):
    """The norm's e4m3 rows are the product's input. Against the same in 64 bits from the unrounded rows: e4m3's half
    step is 2^-4 of a value (2^-10 of the scale for small ones), random from value to value, in the rows and in both
    weights, so a sum of D such products is off by about sqrt(2) 2^-4 / sqrt(3) of its size, each projection the same;
    their product's norm is held to twice that, 0.2."""
    say("8 bits together")
    from sparton_amd.feed_forward import gated_linear, gated_linear_8bit, quantize_rows
    from sparton_amd.norm import rms_norm, rms_norm_8bit
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(5, 60, 256, generator=g).bfloat16().to(device) for _ in range(2))
    w = (torch.rand(256, generator=g) + 0.5).to(device)
    wg, wu = ((torch.randn(384, 256, generator=g) / 16).bfloat16().to(device) for _ in range(2))
    y8, scale, h = rms_norm_8bit(x, w, 1e-6, r)
    with torch.no_grad():
        y, h2 = rms_norm(x, w, 1e-6, r)
    assert torch.equal(h, h2)
    got = gated_linear_8bit(y8, scale, *quantize_rows(wg), *quantize_rows(wu))
    want = F.silu(y.double() @ wg.double().t().contiguous()) * (y.double() @ wu.double().t().contiguous())
    assert got.shape == (5, 60, 384) and got.dtype == torch.bfloat16
    off = float((got.double() - want).norm() / want.norm())
    say(f"   off by {off:.3f}")
    assert off <= 0.2
