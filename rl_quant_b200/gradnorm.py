"""Global norm over many tensors, and clipping by it, for the update of a policy (rsl_rl's PPO update clips with
``nn.utils.clip_grad_norm_``; no qrt counterpart).

    n = (sum |g|^2)^(1/2) over all tensors (or sum |g|, or max |g|),  c = min(1, max_norm / (n + 1e-6)),  g' = c g

``clip_grad_norm_`` takes parameters as torch's does, ``clip_grads_`` and ``clip_grads`` the gradients themselves, in
place or into other tensors; ``grad_norm`` is the norm alone. Two kernels for up to 1024 tensors; nothing waits for
the GPU. The coefficient stays on it, so a step with clipping can be captured in a CUDA graph.
"""
from __future__ import annotations

from array import array
from operator import attrgetter

import torch
from torch import Tensor

from . import _native as N

_CODE = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_KIND = {2.0: 2, 1.0: 1, float("inf"): 0}
_dtype, _shape, _layout = attrgetter("dtype"), attrgetter("shape"), attrgetter("layout")
_requires_grad = attrgetter("requires_grad")


def _kind(norm_type) -> int:
    kind = _KIND.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2, 1 or inf, got {norm_type}")
    return kind


def _tensors(grads, what):
    if isinstance(grads, Tensor):
        return [grads]
    grads = list(grads)
    for kind in set(map(type, grads)):
        if not issubclass(kind, Tensor):
            raise TypeError(f"{what} must be tensors, got {kind.__name__}")
    return grads


def _check(grads):
    """One CUDA device and known types; the type codes. (Whole lists at a time: the host's share of a call with hundreds of
    tensors is several times the kernels'.)"""
    dtypes = set(map(_dtype, grads))
    for dt in dtypes:
        if dt not in _CODE:
            raise TypeError(f"a gradient is {dt}; expected float32, float16 or bfloat16")
    for layout in set(map(_layout, grads)):
        if layout is not torch.strided:
            raise TypeError(f"a gradient is {layout}; expected a dense one")
    dev = grads[0].device
    if len(set(map(Tensor.get_device, grads))) != 1 or dev.type != "cuda":
        for t in grads:
            if t.device != dev:
                raise ValueError(f"tensors on {dev} and {t.device}")
        N.require_cuda(grads[0])
    if len(dtypes) == 1:
        return array("i", (_CODE[grads[0].dtype],)) * len(grads)
    return array("i", [_CODE[dt] for dt in map(_dtype, grads)])


def _dense(t) -> bool:
    """The elements fill one block of memory, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for step, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if step != want:
            return False
        want *= size
    return True


def _all_dense(grads):
    """The tensors as dense ones, and whether they all were contiguous."""
    if all(map(Tensor.is_contiguous, grads)):
        return grads, True
    return [t if _dense(t) else t.contiguous() for t in grads], False


def _overlapping(t) -> bool:
    return t.numel() > 1 and any(st == 0 and sz > 1 for st, sz in zip(t.stride(), t.shape))


def _address(table) -> int:
    return table.buffer_info()[0]


def _run(grads, codes, outs, kind, max_norm):
    """The norm; ``outs`` None or where the clipped gradients go (dense, like the gradients)."""
    dev, n = grads[0].device, len(grads)
    src = array("Q", map(Tensor.data_ptr, grads))
    sizes = array("q", map(Tensor.numel, grads))
    lib = N.load()
    ws = torch.empty(lib.glad_grad_norm_workspace_size(n), dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    if outs is None:
        rc = N.on_device(lib.glad_grad_norm, dev.index, _address(src), _address(sizes), _address(codes), n, kind,
                         norm.data_ptr(), ws.data_ptr(), ws.numel())
    else:
        dst = src if outs is grads else array("Q", map(Tensor.data_ptr, outs))
        rc = N.on_device(lib.glad_clip_grads, dev.index, _address(src), _address(dst), _address(sizes), _address(codes), n,
                         kind, max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel())
    if rc:
        N.check(rc, "grad_norm" if outs is None else "clip_grads")
    return norm


def _max_norm(value) -> float:
    value = float(value)
    if not value >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {value}")
    return value


def _refuse_grad(what, tensors):
    N.refuse_tangents(what, *tensors)
    if torch.is_grad_enabled() and any(map(_requires_grad, tensors)):
        raise RuntimeError(f"{what} has no gradient; use torch.no_grad()")


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``grads`` (a tensor or several: float32, float16, bfloat16, mixed or not, any strides, on
    one device) as a float32 tensor of no dimensions. ``norm_type`` 2, 1 or inf. 0 for no tensors. A NaN anywhere makes
    it NaN."""
    kind, grads = _kind(norm_type), _tensors(grads, "grads")
    if not grads:
        return torch.tensor(0.0)
    _refuse_grad("grad_norm", grads)
    codes = _check(grads)
    return _run(_all_dense(grads)[0], codes, None, kind, 0.0)


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None):
    """``(clipped, norm)``: every tensor of ``grads`` times min(1, max_norm / (norm + 1e-6)), in its own type, in new tensors
    or in those of ``out`` (shapes, types and strides of the gradients, which then leave no gaps in memory; their memory is shared with
    no other tensor of the call, but out[i] may be grads[i])."""
    kind, max_norm, grads = _kind(norm_type), _max_norm(max_norm), _tensors(grads, "grads")
    given = None if out is None else _tensors(out, "out")
    if given is not None and len(given) != len(grads):
        raise ValueError(f"{len(given)} tensors in out for {len(grads)} gradients")
    if not grads:
        return [], torch.tensor(0.0)
    _refuse_grad("clip_grads", grads)
    if given is not None:
        _refuse_grad("clip_grads", given)
    codes = _check(grads)
    grads, whole = _all_dense(grads)
    if given is None:
        given = [torch.empty_like(t) for t in grads]
        return given, _run(grads, codes, given, kind, max_norm)
    if list(map(_shape, given)) != list(map(_shape, grads)) or list(map(_dtype, given)) != list(map(_dtype, grads)) or \
            set(map(Tensor.get_device, given)) != {grads[0].get_device()}:
        for t, o in zip(grads, given):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device:
                raise ValueError(f"out {tuple(o.shape)} {o.dtype} on {o.device} does not match the gradient {tuple(t.shape)} "
                                 f"{t.dtype} on {t.device}")
    if not (whole and all(map(Tensor.is_contiguous, given))):
        for t, o in zip(grads, given):
            if o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous()):
                raise ValueError(f"out has strides {o.stride()}, the gradient {t.stride()}")
    norm = _run(grads, codes, given, kind, max_norm)
    torch.autograd.graph.increment_version(given)       # as torch's in-place operators do
    return given, norm


@torch.no_grad()
def clip_grads_(grads, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """``clip_grads`` in place; returns the norm before clipping. Gradients within the limit are not written."""
    kind, max_norm, grads = _kind(norm_type), _max_norm(max_norm), _tensors(grads, "grads")
    if not grads:
        return torch.tensor(0.0)
    N.refuse_tangents("clip_grads_", *grads)
    codes = _check(grads)
    whole, strided = grads, []
    if not all(map(Tensor.is_contiguous, grads)):
        whole = []
        for t in grads:
            if _dense(t):
                whole.append(t)
            elif _overlapping(t):
                raise ValueError(f"a gradient of strides {t.stride()} has elements that share memory")
            else:
                whole.append(t.contiguous())
                strided.append((t, whole[-1]))
    norm = _run(whole, codes, whole, kind, max_norm)
    for t, c in strided:
        t.copy_(c)
    torch.autograd.graph.increment_version(grads)       # as torch's in-place operators do
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` of parameters (one or several) on one device: their ``grad``s are clipped in place,
    the norm before clipping is returned. ``error_if_nonfinite`` waits for the GPU and raises with the gradients unchanged."""
    grads = [p.grad for p in _tensors(parameters, "parameters") if p.grad is not None]
    if error_if_nonfinite and grads:
        with torch.no_grad():
            norm = grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the norm of order {norm_type} of the gradients is {float(norm)}; they were not clipped")
    return clip_grads_(grads, max_norm, norm_type)
