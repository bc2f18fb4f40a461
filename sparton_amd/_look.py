"""What a module computes: a small copy of it, on the CPU, against the formula."""
from __future__ import annotations

import copy
from typing import Callable, Dict

import torch
from torch import Tensor, nn

PLAIN = dict(device="cpu", dtype=torch.float32)  # of what is looked with, whatever torch's defaults are


def computes(module: nn.Module, children: Dict[str, nn.Module], x: Tensor, want: Callable[[], Tensor], **kwargs) -> bool:
    """Whether the class's forward, on a copy with these submodules instead, gives `want` for x (and kwargs), in
    evaluation and in training (dropout scales what it keeps)."""
    probe = copy.copy(module)
    probe._modules = dict(children)
    try:
        with torch.no_grad(), torch.random.fork_rng(devices=[]):
            for probe.training in (False, True):
                got = type(module).forward(probe, x, **kwargs)
                if not isinstance(got, Tensor) or not torch.allclose(got, want(), rtol=1e-4, atol=1e-5):
                    return False
            return True
    except Exception:  # whatever it is, it is not what the kernels compute
        return False


def holds_only(module: nn.Module) -> bool:
    """Whether it has no forward, so that there is nothing to agree with."""
    return type(module).forward is nn.Module.forward and "forward" not in module.__dict__
