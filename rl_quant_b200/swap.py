"""Module surgery: nn.Linear <-> QuantLinear (qrt/swap.py:39-74) or W4Linear, nn.RMSNorm <-> RMSNorm.

The swap moves the source layer's Parameter objects into the QuantLinear
(no copies), so optimisers created before or after stay valid, and both
directions carry over the train/eval flag.
"""
from __future__ import annotations

import torch.nn as nn

from .norm import RMSNorm
from .qlinear import QuantLinear
from .w4linear import W4Linear


def get_module(model: nn.Module, path: str) -> nn.Module:
    return model.get_submodule(path)


def set_module(model: nn.Module, path: str, mod: nn.Module) -> None:
    parent_path, _, name = path.rpartition(".")
    parent = model.get_submodule(parent_path) if parent_path else model
    if name.isdigit() and isinstance(parent, (nn.Sequential, nn.ModuleList)):
        parent[int(name)] = mod
    else:
        setattr(parent, name, mod)


def _quantised(path: str, lin: nn.Linear, cfg: dict) -> nn.Module:
    bits = cfg.get("bits", 8)
    if bits == 4:
        extra = set(cfg) - {"bits", "group"}
        if extra:
            raise ValueError(f"{path}: a 4-bit layer takes 'group' only, got {sorted(extra)}")
        return W4Linear(lin, group=cfg.get("group", 64))
    if bits != 8:
        raise ValueError(f"{path}: bits must be 8 or 4, got {bits}")
    return QuantLinear(lin, s_z=cfg.get("s_z"), alpha=cfg.get("alpha"), beta=cfg.get("beta"),
                       act_mode=cfg.get("act_mode", "static"))


def apply(model: nn.Module, plan: dict[str, dict]) -> dict[str, nn.Module]:
    """Swap every ``plan`` path to a QuantLinear, or to a W4Linear where the entry says ``"bits": 4``.
    ``plan = {path: {"s_z": float|None, "alpha": Tensor|None, "beta": Tensor|None, "act_mode": str}}`` or
    ``{path: {"bits": 4, "group": 32|64|128}}``. All or none: the model stays as it was where a layer is refused."""
    swapped: dict[str, nn.Module] = {}
    for path, cfg in plan.items():
        lin = get_module(model, path)
        assert isinstance(lin, nn.Linear), f"{path} is not an nn.Linear: {type(lin)}"
        swapped[path] = _quantised(path, lin, cfg).train(lin.training)
    for path, q in swapped.items():
        set_module(model, path, q)
    return swapped


def apply_norm(model: nn.Module, paths: list[str] | None = None) -> dict[str, nn.RMSNorm]:
    """Swap the named ``nn.RMSNorm`` layers (None: every one) to ``RMSNorm``; returns the originals by path. All or none."""
    if paths is None:
        paths = [n for n, m in model.named_modules() if type(m) is nn.RMSNorm and n]
    originals, swapped = {}, {}
    for path in paths:
        norm = get_module(model, path)
        assert isinstance(norm, nn.RMSNorm), f"{path} is not an nn.RMSNorm: {type(norm)}"
        originals[path], swapped[path] = norm, RMSNorm.from_torch(norm)
    for path, norm in swapped.items():
        set_module(model, path, norm)
    return originals


def restore_norm(model: nn.Module, originals: dict[str, nn.RMSNorm]) -> None:
    """Put the layers that ``apply_norm`` returned back, with the swapped modules' train/eval flag."""
    for path, norm in originals.items():
        norm.train(get_module(model, path).training)
        set_module(model, path, norm)


def restore(model: nn.Module, swapped: dict[str, nn.Module]) -> None:
    """Put plain nn.Linear shells (holding the same Parameters) back."""
    for path, q in swapped.items():
        lin = nn.Linear(q.in_features, q.out_features, bias=q.bias is not None,
                        device=q.weight.device, dtype=q.weight.dtype)
        lin.weight = q.weight
        if q.bias is not None:
            lin.bias = q.bias
        lin.train(q.training)
        set_module(model, path, lin)


def refresh(swapped: dict[str, QuantLinear]) -> None:
    """Requantise every swapped layer after a weight update."""
    for q in swapped.values():
        q.requantize_()
