"""The attention and norm kernels in transformers backbones of the reference's families (bert,
distilbert, roberta, xlm-roberta; training/model.py:14-40), tiny and built offline, and a whole
training step on them: backbone -> transform -> head -> SPLADE loss and preference loss -> every
parameter's gradient, against the same model with torch's attention and norms.

Tolerances, fp32 throughout: hidden states rtol 1e-4, atol 1e-5; gradients by the measure of
test_hf_integration.py (error against the gradient's largest magnitude, with a floor of 1e-4 of the
largest of all, at most 1e-3; torch's fp32 CPU result sits within 1e-6 of float64 by it)."""
import copy
import pickle

import pytest
import torch
from torch import nn

import sparton_amd
from _parity import say
from sparton_amd.backbone import attention_forward, key_mask, use_in_backbone
from sparton_amd.loss import preference_loss, preference_margin, splade_loss
from test_hf_integration import backbone_and_head, batch, sparton_projection, tiny_mlm


def tiny(kind, seed=0):
    if kind in ("bert", "xlm-roberta"):
        return tiny_mlm(kind, seed).eval()
    from transformers import DistilBertConfig, DistilBertForMaskedLM, RobertaConfig, RobertaForMaskedLM
    torch.manual_seed(seed)
    if kind == "roberta":
        return RobertaForMaskedLM(RobertaConfig(vocab_size=3001, hidden_size=128, num_hidden_layers=2, num_attention_heads=4,
                                                intermediate_size=256, max_position_embeddings=130,
                                                attn_implementation="eager", hidden_dropout_prob=0.0,
                                                attention_probs_dropout_prob=0.0)).eval()
    return DistilBertForMaskedLM(DistilBertConfig(vocab_size=3001, dim=128, n_layers=2, n_heads=4, hidden_dim=256,
                                                  max_position_embeddings=128, attn_implementation="eager", dropout=0.0,
                                                  attention_dropout=0.0)).eval()


def base(llm):
    return getattr(llm, llm.base_model_prefix)


KINDS = ["bert", "distilbert", "roberta", "xlm-roberta"]


@pytest.mark.parametrize("kind", KINDS)
def test_switching_keeps_parameters_and_names(kind):
    llm = tiny(kind)
    names, own = list(llm.state_dict()), {n: id(p) for n, p in llm.named_parameters()}
    norms = sum(type(m) is nn.LayerNorm for m in llm.modules())
    assert use_in_backbone(llm) is llm and llm.config._attn_implementation == "sparton"
    assert list(llm.state_dict()) == names and {n: id(p) for n, p in llm.named_parameters()} == own
    assert sum(type(m) is sparton_amd.SpartonLayerNorm for m in llm.modules()) == norms > 0
    assert not any(type(m) is nn.LayerNorm for m in llm.modules())
    use_in_backbone(llm)  # a second time changes nothing
    assert list(llm.state_dict()) == names
    twin = copy.deepcopy(llm)  # the copy's blocks run on the copy's own parameters
    for a, b in zip(llm.modules(), twin.modules()):
        if "forward" in a.__dict__:
            assert b.forward.__self__ is b


@pytest.mark.parametrize("kind", KINDS)
def test_a_switched_model_pickles(kind):
    llm = use_in_backbone(tiny(kind))
    twin = pickle.loads(pickle.dumps(llm))
    assert list(twin.state_dict()) == list(llm.state_dict())
    blocks = 0
    for a, b in zip(llm.modules(), twin.modules()):
        assert type(a) is type(b)
        if "forward" in a.__dict__:
            assert b.forward.__self__ is b and b is not a
            blocks += 1
    assert blocks == (0 if kind == "distilbert" else 4)


def test_a_refused_model_stays_as_it_was():
    llm = tiny("bert")
    llm.extra = nn.LayerNorm(16385)  # wider than the kernel's rows
    with pytest.raises(ValueError, match="16384"):
        use_in_backbone(llm)
    assert llm.config._attn_implementation == "eager"
    assert not any(type(m) is sparton_amd.SpartonLayerNorm or "forward" in m.__dict__ for m in llm.modules())


@pytest.mark.parametrize("norm", [lambda: nn.LayerNorm(128, elementwise_affine=False), lambda: nn.Identity()])
def test_a_block_whose_norm_is_another_stays_as_it_is(norm, monkeypatch):
    """Its own forward runs, with the norm that it has."""
    monkeypatch.setattr("sparton_amd.backbone.attention", plain_attention)
    monkeypatch.setattr("sparton_amd.norm.layer_norm", lambda x, w, b=None, eps=1e-5, residual=None:
                        nn.functional.layer_norm(x if residual is None else x + residual, x.shape[-1:], w, b, eps))
    ref = base(tiny("bert"))
    ref.encoder.layer[1].output.LayerNorm = norm()
    ours = use_in_backbone(copy.deepcopy(ref))
    ids = torch.arange(12).reshape(2, 6) + 5
    with torch.no_grad():
        torch.testing.assert_close(ours(ids).last_hidden_state, ref(ids).last_hidden_state, rtol=1e-4, atol=1e-5)


def test_norms_keep_their_hooks(monkeypatch):
    monkeypatch.setattr("sparton_amd.norm.layer_norm", lambda x, w, b=None, eps=1e-5, residual=None:
                        nn.functional.layer_norm(x if residual is None else x + residual, x.shape[-1:], w, b, eps))
    model, seen = nn.Module(), []
    model.norm = ln = nn.LayerNorm(16)
    first = ln.register_forward_hook(lambda m, args, out: seen.append("out"))
    ln.register_forward_pre_hook(lambda m, args: seen.append("in"))
    model.norm = sparton_amd.SpartonLayerNorm.of(ln)
    x = torch.randn(3, 16)
    assert torch.equal(model.norm(x), nn.functional.layer_norm(x, (16,), ln.weight, ln.bias)) and seen == ["in", "out"]
    first.remove()
    model.norm(x)
    assert seen == ["in", "out", "in"]
    ln.weight = nn.Parameter(torch.zeros(16))  # the module that it was made of goes its own way
    assert bool((model.norm.weight == 1).all())


def test_refusals():
    q = torch.zeros(1, 2, 4, 8)
    with pytest.raises(ValueError, match="dropout"):
        attention_forward(nn.Module(), q, q, q, None, dropout=0.1)
    with pytest.raises(ValueError, match="sliding_window"):
        attention_forward(nn.Module(), q, q, q, None, sliding_window=16)
    with pytest.raises(ValueError, match="output_attentions"):
        attention_forward(nn.Module(), q, q, q, None, output_attentions=True)
    with pytest.raises(ValueError, match="per key"):
        attention_forward(nn.Module(), q, q, q, torch.zeros(1, 1, 4, 4))
    from transformers.masking_utils import causal_mask_function, sliding_window_overlay
    with pytest.raises(ValueError, match="pattern"):
        key_mask(1, 4, 4, mask_function=sliding_window_overlay(2))
    with pytest.raises(ValueError, match="room"):
        key_mask(1, 1, 16, q_offset=3, mask_function=causal_mask_function)
    m = torch.ones(1, 4, dtype=torch.long)
    assert key_mask(1, 4, 4, mask_function=causal_mask_function, attention_mask=m) is m
    assert key_mask(1, 4, 4) is None


def test_training_with_attention_dropout_is_refused():
    from transformers import BertConfig, BertModel
    model = use_in_backbone(BertModel(BertConfig(vocab_size=50, hidden_size=32, num_hidden_layers=1, num_attention_heads=2,
                                                 intermediate_size=64)))
    model.embeddings.LayerNorm = nn.LayerNorm(32)  # lets a CPU run reach the attention
    with pytest.raises(ValueError, match="dropout"):
        model.train()(torch.ones(1, 4, dtype=torch.long))


def plain_attention(q, k, v, mask=None, *, causal=False, scale=None):
    """The kernels' formula in torch, for CPU runs."""
    from _attention_ref import allowed_pairs
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    on = allowed_pairs(q.shape[0], q.shape[2], k.shape[2], mask, causal, q.device)
    s = torch.where(on, scale * (q @ k.transpose(-1, -2)), -torch.inf)
    return torch.softmax(s, -1).nan_to_num(0.0) @ v


def tiny_decoder():
    """(with torch's attention, switched), both on the CPU."""
    from transformers import LlamaConfig, LlamaModel
    torch.manual_seed(0)
    ref = LlamaModel(LlamaConfig(vocab_size=300, hidden_size=128, num_hidden_layers=2, num_attention_heads=4,
                                 num_key_value_heads=2, intermediate_size=256, attn_implementation="eager")).eval()
    return ref, use_in_backbone(copy.deepcopy(ref))


def left_padded(B, S, seed):
    g = torch.Generator().manual_seed(seed)
    mask = torch.ones(B, S, dtype=torch.long)
    for b in range(1, B):
        mask[b, :b + 1] = 0
    return torch.randint(0, 300, (B, S), generator=g), mask


def test_the_masks_columns_are_the_keys(monkeypatch):
    """A mask over more columns than there are keys, or fewer: the first ones are the keys', as in torch's attention."""
    m = torch.tensor([[0, 1, 1, 1, 0, 1], [1, 1, 0, 1, 1, 1]])
    assert torch.equal(key_mask(2, 4, 4, attention_mask=m), m[:, :4])
    assert torch.equal(key_mask(2, 2, 3, q_offset=3, kv_offset=2, attention_mask=m), m[:, 2:5])
    assert torch.equal(key_mask(2, 4, 8, attention_mask=m), nn.functional.pad(m, (0, 2)))
    assert torch.equal(key_mask(2, 4, 7, attention_mask=m != 0), nn.functional.pad(m != 0, (0, 1)))
    monkeypatch.setattr("sparton_amd.backbone.attention", plain_attention)
    ref, ours = tiny_decoder()
    ids, mask = left_padded(3, 12, seed=1)
    with torch.no_grad():
        a, b = (m(ids[:, :6], mask).last_hidden_state for m in (ref, ours))
    on = mask[:, :6].bool()
    torch.testing.assert_close(b[on], a[on], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8, torch.int16])
def test_a_mask_of_any_type(dtype):
    """transformers reads a mask's values as true or false; so does a switched model."""
    m = torch.tensor([[0, 1, 1, 1], [1, 1, 0, 1]])
    got = key_mask(2, 4, 4, attention_mask=m.to(dtype))
    assert got.dtype == torch.bool and torch.equal(got, m.bool())
    for own in (torch.bool, torch.uint8, torch.int32, torch.int64):
        assert key_mask(2, 4, 4, attention_mask=m.to(own)).dtype == own


def test_a_mask_of_a_cache_with_room():
    """The cache's length as a tensor: one new token sees what is in use; several rows must be the last ones."""
    from transformers.masking_utils import causal_mask_function
    at = lambda rows, keys, offset, m=None: key_mask(2, rows, keys, q_offset=torch.tensor(offset),
                                                     mask_function=causal_mask_function, attention_mask=m)
    got = at(1, 8, 5)
    assert got.shape == (2, 8) and got.dtype == torch.bool and torch.equal(got[0], torch.arange(8) <= 5)
    m = torch.tensor([[0, 1, 1, 1, 1, 1], [1, 1, 1, 0, 1, 1]])
    want = nn.functional.pad(m, (0, 2)).bool()
    assert torch.equal(at(1, 8, 5, m), want)
    assert torch.equal(key_mask(2, 1, 8, q_offset=torch.tensor(5), mask_function=causal_mask_function, attention_mask=m,
                                device=None), want)
    assert torch.equal(at(1, 8, 3, m), want & (torch.arange(8) <= 3))
    with pytest.raises(ValueError, match="room"):
        at(3, 8, 3)
    with pytest.raises(ValueError, match="room"):
        at(8, 16, 0)
    assert at(3, 8, 5) is None and at(8, 8, 0) is None
    assert torch.equal(at(3, 6, 3, m), m)


@pytest.mark.parametrize("padded", [False, True])
def test_a_token_over_a_static_cache(padded, monkeypatch):
    """Hidden states token by token over a cache allocated ahead, against torch's attention on the same cache."""
    from transformers import StaticCache
    monkeypatch.setattr("sparton_amd.backbone.attention", plain_attention)
    ref, ours = tiny_decoder()
    ids, mask = left_padded(3, 9, seed=2)
    out = {}
    for model in (ref, ours):
        cache, rows = StaticCache(config=ref.config, max_cache_len=16), []
        with torch.no_grad():
            ref(ids[:, :6], mask[:, :6] if padded else None, past_key_values=cache, use_cache=True)
            for n in range(6, 9):
                rows.append(model(ids[:, n:n + 1], mask[:, :n + 1] if padded else None, past_key_values=cache,
                                  use_cache=True).last_hidden_state)
        out[model] = torch.cat(rows, 1)
    torch.testing.assert_close(out[ours], out[ref], rtol=1e-4, atol=1e-5)
    cache = StaticCache(config=ref.config, max_cache_len=16)
    with torch.no_grad():
        ref(ids[:, :6], past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="room"):
            ours(ids[:, 6:8], past_key_values=cache, use_cache=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("padded", [True, False])
def test_backbone_matches_torch(kind, padded, device):
    say(f"backbone {kind} padded={padded}")
    llm = tiny(kind, seed=3).to(device)
    ours = use_in_backbone(copy.deepcopy(llm))
    ids, mask = batch(5, 47, seed=4, device=device)
    mask = mask if padded else torch.ones_like(mask)
    with torch.no_grad():
        ref, got = base(llm)(ids, mask).last_hidden_state, base(ours)(ids, mask).last_hidden_state
        bare = base(ours)(ids).last_hidden_state
    # every position but the padding, whose queries see the same keys and are compared too
    torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-5)
    if not padded:
        torch.testing.assert_close(bare, ref, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_decoder_backbone_is_causal(device):
    """A decoder-only backbone with shared key heads (random, tiny): the registry hands its attention over."""
    from transformers import LlamaConfig, LlamaModel
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=300, hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      intermediate_size=256, attn_implementation="eager", use_cache=False)
    ref = LlamaModel(cfg).to(device).eval()
    ours = use_in_backbone(copy.deepcopy(ref))
    ids, mask = batch(3, 40, seed=1, device=device)
    ids = ids % 300
    with torch.no_grad():
        a, b = ref(ids, mask).last_hidden_state, ours(ids, mask).last_hidden_state
    on = mask.bool()
    torch.testing.assert_close(b[on], a[on], rtol=1e-4, atol=1e-5)
    # token by token over a cache: the rows are the last ones of the keys
    with torch.no_grad():
        whole = ours(ids[:1, :30]).last_hidden_state
        first = ours(ids[:1, :25], use_cache=True)
        last = ours(ids[:1, 25:30], past_key_values=first.past_key_values, use_cache=True).last_hidden_state
    torch.testing.assert_close(last, whole[:, 25:], rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("padded", [False, True])
def test_a_token_over_a_static_cache_on_the_kernels(padded, device):
    """As above, the cache prefilled by torch's attention."""
    from transformers import StaticCache
    say(f"static cache, padded={padded}")
    ref, ours = (m.to(device) for m in tiny_decoder())
    ids, mask = (t.to(device) for t in left_padded(3, 9, seed=2))
    out = {}
    for model in (ref, ours):
        cache, rows = StaticCache(config=ref.config, max_cache_len=200), []
        with torch.no_grad():
            ref(ids[:, :6], mask[:, :6] if padded else None, past_key_values=cache, use_cache=True)
            for n in range(6, 9):
                rows.append(model(ids[:, n:n + 1], mask[:, :n + 1] if padded else None, past_key_values=cache,
                                  use_cache=True).last_hidden_state)
        out[model] = torch.cat(rows, 1)
    torch.testing.assert_close(out[ours], out[ref], rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bert", "xlm-roberta"])
def test_training_step_with_every_operator(kind, device):
    say(f"training step {kind}")
    llm = tiny(kind, seed=6).to(device)
    ours = use_in_backbone(copy.deepcopy(llm))
    q_ids, q_mask = batch(6, 16, seed=7, device=device)
    d_ids, d_mask = batch(12, 60, seed=8, device=device)
    T = 100.0

    def step(model):
        """Gradients of the SPLADE loss over (query, preferred) plus the preference loss over the pairs."""
        backbone, transform, decoder = backbone_and_head(model)
        xf, head = sparton_projection(transform, decoder)
        encode = lambda ids, mask: head(xf(backbone(ids, mask).last_hidden_state), mask)
        q, d = encode(q_ids, q_mask), encode(d_ids, d_mask)
        with torch.no_grad():
            ref = preference_margin(q * 0.9, d[:6], d[6:] * 1.1, T)
        pairs = preference_loss(q, d[:6], d[6:], ref, beta=0.5, temperature=T)
        loss = splade_loss(q, d[:6], T, 1e-3, 1e-3).total + pairs.loss
        model.zero_grad()
        loss.backward()
        return loss.detach(), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}

    (la, ga), (lb, gb) = step(llm), step(ours)
    torch.testing.assert_close(lb, la, rtol=1e-4, atol=1e-6)
    assert ga.keys() == gb.keys()
    floor = 1e-4 * max(g.abs().max().item() for g in ga.values())
    worst = max((gb[n] - g).abs().max().item() / max(g.abs().max().item(), floor) for n, g in ga.items())
    say(f"   loss {lb.item():.6f} (torch's backbone {la.item():.6f}), worst gradient error {worst:.2e}")
    assert worst <= 1e-3


@pytest.mark.gpu
def test_training_step_in_bf16(device):
    """The same under bf16 autocast over fp32 parameters, and held in bf16: it runs, its loss is near the
    fp32 one, and every gradient is finite."""
    say("training step, bf16")
    llm = use_in_backbone(tiny("bert", seed=9).to(device))
    ids, mask = batch(4, 33, seed=10, device=device)
    backbone, transform, decoder = backbone_and_head(llm)
    xf, head = sparton_projection(transform, decoder)

    def reps():
        return head(xf(backbone(ids, mask).last_hidden_state), mask)

    with torch.no_grad():
        want = reps()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = reps()
    assert got.dtype == torch.bfloat16 and (got.float() - want).abs().max() <= 5e-2 * want.abs().max()
    got.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in llm.parameters() if p.grad is not None)
    llm.zero_grad()
    llm.to(torch.bfloat16)
    got = reps()
    assert got.dtype == torch.bfloat16 and (got.float() - want).abs().max() <= 5e-2 * want.abs().max()
    got.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in llm.parameters() if p.grad is not None)
