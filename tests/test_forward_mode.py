"""Forward-mode derivatives of the RMS norm, the embedding and the gated product: none is computed, so one that is asked
for is refused, never dropped, with or without gradients asked for besides."""
import pytest
import torch
from torch.autograd import forward_ad

from sparton_amd.embedding import embedding
from sparton_amd.feed_forward import gated_linear, gated_linear_8bit, quantize_rows
from sparton_amd.norm import rms_norm, rms_norm_8bit


def calls(device):
    """name -> (function, its float tensors)"""
    t = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(sum(s))).to(device)
    ids = torch.tensor([1, 4, 1], device=device)
    q = [x for s in ((3, 16), (6, 16), (6, 16)) for x in quantize_rows(t(*s))]
    return {
        "rms_norm": (rms_norm, [t(3, 16), t(16)]),
        "rms_norm with the sum": (lambda x, r, w: rms_norm(x, w, residual=r), [t(3, 16), t(3, 16), t(16)]),
        "rms_norm_8bit": (lambda x, r, w: rms_norm_8bit(x, w, residual=r), [t(3, 16), t(3, 16), t(16)]),
        "embedding": (lambda w: embedding(ids, w, 2.0), [t(5, 16)]),
        "gated": (gated_linear, [t(3, 16), t(6, 16), t(6, 16), t(6), t(6)]),
        "gated_8bit": (lambda sx, sg, su: gated_linear_8bit(q[0], sx, q[2], sg, q[4], su), [q[1], q[3], q[5]]),
    }


NAMES = list(calls("cpu"))


def refused(name, device, grad):
    f, tensors = calls(device)[name]
    for i, t in enumerate(tensors):
        args = list(tensors)
        with forward_ad.dual_level():
            args[i] = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            with pytest.raises(NotImplementedError):
                f(*args)


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused_by_the_registered_ops(name):
    """Theirs is the path of tensors on the CPU."""
    refused(name, "cpu", False)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name, device):
    refused(name, device, False)
    with torch.no_grad():
        refused(name, device, False)
    if "8bit" not in name:
        refused(name, device, True)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_jvp_is_refused(name, device):
    f, tensors = calls(device)[name]
    for i, t in enumerate(tensors):
        with pytest.raises(RuntimeError, match="forward"):
            torch.func.jvp(lambda x: f(*tensors[:i], x, *tensors[i + 1:]), (t,), (torch.ones_like(t),))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_the_registered_ops_refuse_a_tangent(name, device, monkeypatch):
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    refused(name, device, False)
