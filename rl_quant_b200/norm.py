"""Root-mean-square norm with the residual's addition, for the blocks around the
quantised linears (no reference counterpart: the reference normalises observations
only, rsl_rl/networks/normalization.py:44-47).

    h = x + residual                     rounded to the residual's type
    y = h / sqrt(mean(h^2) + eps) * weight

``rms_norm`` returns y in x's type and trains (its backward pass is one kernel plus the
reduction of the weight's gradient); ``rms_norm_quant`` returns y in 8 bits with scales,
the input form of ``w4_linear``. ``RMSNorm`` is the module of both.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _native as N

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
MAX_COLS = 32768


def _check(x, weight, residual, eps):
    if x.dtype not in _FLOATS:
        raise TypeError(f"x is {x.dtype}; expected float32, float16 or bfloat16")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"x must have 1..{MAX_COLS} columns, got shape {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    if weight is not None:
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"weight {tuple(weight.shape)} does not match {x.shape[-1]} columns")
        if weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"weight is {weight.dtype}; expected {x.dtype} or float32")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual is {residual.dtype}; expected {x.dtype} or float32")
    for t in (weight, residual):
        if t is not None and t.device != x.device:
            raise ValueError(f"tensors on {x.device} and {t.device}")
    N.require_cuda(x)


def _rows(t):
    """[..., C] as rows of adjacent columns (a view where the strides allow one)."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(1) == 1 or t2.shape[1] == 1 else t2.contiguous()


def _forward(x, weight, residual, eps, rstd):
    """(y, h or None) as rows; ``rstd`` None or f32 [rows] to fill."""
    x2 = _rows(x)
    rows, cols = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r2 = h = None
    if residual is not None:
        r2 = _rows(residual)
        h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    w = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    with N.device_guard(x.device):
        N.check(N.load().glad_rms_norm_forward(
            x2.data_ptr(), N.DTYPES[x.dtype], x2.stride(0), N.ptr(r2), N.DTYPES[h.dtype] if h is not None else 0,
            r2.stride(0) if r2 is not None else 0, N.ptr(w), N.DTYPES[w.dtype] if w is not None else 0, rows, cols,
            eps, y.data_ptr(), N.ptr(h), N.ptr(rstd), N.stream_handle(x.device)), "rms_norm")
    return y, h


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        rstd = torch.empty(x.numel() // x.shape[-1], dtype=torch.float32, device=x.device)
        y, h = _forward(x, weight, residual, eps, rstd)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return (y, h) if h is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:      # only the sum was used
            return (dsum.to(ctx.x_dtype) if need_x and dsum is not None else None, None,
                    dsum if need_r else None, None)
        h2, dy2 = _rows(h), _rows(dy)
        ds2 = _rows(dsum) if dsum is not None else None
        rows, cols = h2.shape
        dev = h.device
        same = h.dtype == ctx.x_dtype       # one gradient serves x and the residual
        dx = torch.empty(h.shape, dtype=ctx.x_dtype, device=dev) if need_x or (need_r and same) else None
        dr = torch.empty(h.shape, dtype=h.dtype, device=dev) if need_r and not same else None
        dw = ws = w = None
        if weight is not None:
            w = weight if weight.is_contiguous() else weight.contiguous()
            if need_w:
                dw = torch.empty(cols, dtype=weight.dtype, device=dev)
                ws = torch.empty(N.load().glad_rms_norm_backward_workspace_size(rows, cols), dtype=torch.uint8,
                                 device=dev)
        with N.device_guard(dev):
            N.check(N.load().glad_rms_norm_backward(
                dy2.data_ptr(), N.DTYPES[ctx.x_dtype], dy2.stride(0), N.ptr(ds2), N.DTYPES[h.dtype],
                ds2.stride(0) if ds2 is not None else 0, h2.data_ptr(), h2.stride(0), N.ptr(w),
                N.DTYPES[w.dtype] if w is not None else 0, rstd.data_ptr(), rows, cols, N.ptr(dx), N.ptr(dr),
                N.ptr(dw), N.ptr(ws), ws.numel() if ws is not None else 0, N.stream_handle(dev)), "rms_norm backward")
        return dx if need_x else None, dw, (dx if same else dr) if need_r else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
             eps: float = 1e-6):
    """y in x's type, or ``(y, h)`` with a residual; h has the residual's type.

    x [..., C] float32, float16 or bfloat16, rows of any stride; weight [C] (None: ones) and residual
    (x's shape) have x's type or float32; C up to 32768. Differentiable in x, weight and residual.
    The sum is rounded to the residual's type first and the norm is of that value."""
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, weight, residual, eps)
    y, h = _forward(x, weight, residual, eps, None)
    return y if h is None else (y, h)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                   eps: float = 1e-6, out_dtype: torch.dtype = torch.int8, group: int = 0,
                   scale: torch.Tensor | None = None):
    """``(q, s)``, or ``(q, s, h)`` with a residual: the norm rounded to int8 or float8_e4m3fn codes, q * s ~ y.

    ``scale`` None: s = max|y| / 127 (448) of each row (``group`` 0, s [..., 1]) or of each ``group`` (32, 64, 128)
    columns of a row (s [..., ceil(C / group)]), 1 where the maximum is 0. ``scale`` a float32 tensor of one value: that
    scale for all (static calibration), returned as s. Inference only: inputs that require a gradient are refused
    while gradients are enabled (``rms_norm`` is the form that trains)."""
    if out_dtype not in (torch.int8, torch.float8_e4m3fn):
        raise TypeError(f"out_dtype is {out_dtype}; expected int8 or float8_e4m3fn")
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group must be 0, 32, 64 or 128, got {group}")
    if scale is not None:
        if group:
            raise ValueError("a given scale is one for the whole tensor (group 0)")
        if scale.numel() != 1 or scale.dtype != torch.float32 or scale.device != x.device:
            raise ValueError("scale must be one float32 value on x's device")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_quant has no gradient; use rms_norm, or torch.no_grad()")
    _check(x, weight, residual, eps)
    x2 = _rows(x)
    rows, cols = x2.shape
    q = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    s = scale
    if s is None:
        s = torch.empty(x.shape[:-1] + (1 if group == 0 else -(-cols // group),), dtype=torch.float32, device=x.device)
    r2 = h = None
    if residual is not None:
        r2 = _rows(residual)
        h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    w = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    with N.device_guard(x.device):
        N.check(N.load().glad_rms_norm_quant(
            x2.data_ptr(), N.DTYPES[x.dtype], x2.stride(0), N.ptr(r2), N.DTYPES[h.dtype] if h is not None else 0,
            r2.stride(0) if r2 is not None else 0, N.ptr(w), N.DTYPES[w.dtype] if w is not None else 0, rows, cols,
            eps, N.DTYPES[out_dtype], group, N.ptr(scale), q.data_ptr(), None if scale is not None else s.data_ptr(),
            N.ptr(h), N.stream_handle(x.device)), "rms_norm_quant")
    return (q, s) if h is None else (q, s, h)


class RMSNorm(nn.Module):
    """``forward(x, residual=None)`` is ``rms_norm``, ``quant(x, residual=None, ...)`` is ``rms_norm_quant``, both with this
    module's weight. Parameter name and shape are those of ``torch.nn.RMSNorm`` over the last dimension."""

    def __init__(self, dim: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = dim, eps
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)

    @classmethod
    def from_torch(cls, norm: nn.RMSNorm) -> "RMSNorm":
        """The same norm over the source module's own Parameter (optimiser references stay valid)."""
        if len(norm.normalized_shape) != 1:
            raise ValueError(f"normalized_shape {tuple(norm.normalized_shape)}: the last dimension only")
        if norm.weight is not None:
            eps = norm.eps if norm.eps is not None else torch.finfo(norm.weight.dtype).eps
        elif norm.eps is None:
            raise ValueError("a norm without weight and eps takes its eps from each input's type; set eps")
        else:
            eps = norm.eps
        m = cls(norm.normalized_shape[0], eps=eps, elementwise_affine=False)
        m.weight = norm.weight
        m.train(norm.training)
        return m

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)

    def quant(self, x, residual=None, out_dtype=torch.int8, group=0, scale=None):
        return rms_norm_quant(x, self.weight, residual, self.eps, out_dtype, group, scale)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}"
