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

_CODE = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
MAX_COLS = 32768


def _check(x, weight, residual, eps):
    dt, shape = x.dtype, x.shape
    if dt not in _CODE:
        raise TypeError(f"x is {dt}; expected float32, float16 or bfloat16")
    if not shape or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"x must have 1..{MAX_COLS} columns, got shape {tuple(shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    dev = x.device
    if weight is not None:
        if weight.shape != shape[-1:]:
            raise ValueError(f"weight {tuple(weight.shape)} does not match {shape[-1]} columns")
        if weight.dtype != dt and weight.dtype != torch.float32:
            raise TypeError(f"weight is {weight.dtype}; expected {dt} or float32")
        if weight.device != dev:
            raise ValueError(f"tensors on {dev} and {weight.device}")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(shape)}")
        if residual.dtype != dt and residual.dtype != torch.float32:
            raise TypeError(f"residual is {residual.dtype}; expected {dt} or float32")
        if residual.device != dev:
            raise ValueError(f"tensors on {dev} and {residual.device}")
    N.require_cuda(x)


def _rows(t):
    """[..., C] as rows of adjacent columns: a view where the strides allow one, a copy of broadcast (overlapping) rows."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    rows, cols = t2.shape
    ld, step = t2.stride()
    return t2 if (step == 1 or cols == 1) and (ld >= cols or rows <= 1) else t2.contiguous()


def _like(t, dtype=None):
    """Contiguous and uninitialised, of t's shape (empty_like is the cheaper call)."""
    if not t.is_contiguous():
        return t.new_empty(t.shape, dtype=dtype)
    return torch.empty_like(t) if dtype is None else torch.empty_like(t, dtype=dtype)


def _forward(x, weight, residual, eps, rstd):
    """(y, h or None); ``rstd`` None or f32 [rows] to fill."""
    x2 = _rows(x)
    rows, cols = x2.shape
    y = _like(x)
    wp, wt, rp, rt, ldr, h, hp = None, 0, None, 0, 0, None, None
    if weight is not None:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        wp, wt = weight.data_ptr(), _CODE[weight.dtype]
    if residual is not None:
        r2 = _rows(residual)
        h = _like(residual)
        rp, rt, ldr, hp = r2.data_ptr(), _CODE[residual.dtype], r2.stride(0), h.data_ptr()
    rc = N.on_device(N.load().glad_rms_norm_forward, x.device.index, x2.data_ptr(), _CODE[x.dtype], x2.stride(0), rp, rt,
                     ldr, wp, wt, rows, cols, eps, y.data_ptr(), hp, None if rstd is None else rstd.data_ptr())
    if rc:
        N.check(rc, "rms_norm")
    return y, h


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
        y, h = _forward(x, weight, residual, eps, rstd)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        x_t, h_t = ctx.x_dtype, h.dtype
        if dy is None:      # only the sum was used
            return (dsum.to(x_t) if need_x and dsum is not None else None, None, dsum if need_r else None, None)
        h2, dy2 = _rows(h), _rows(dy)
        rows, cols = h2.shape
        dx = dr = dw = ws = ds2 = None
        wp, wt, dwp, wsp, wsn, dsp, ldds = None, 0, None, None, 0, None, 0
        if need_x or (need_r and x_t == h_t):       # one gradient serves x and a residual of its type
            dx = _like(dy)
        if need_r:
            dr = dx if x_t == h_t else _like(h)
        if dsum is not None:
            ds2 = _rows(dsum)
            dsp, ldds = ds2.data_ptr(), ds2.stride(0)
        if weight is not None:
            if not weight.is_contiguous():
                weight = weight.contiguous()
            wp, wt = weight.data_ptr(), _CODE[weight.dtype]
            if need_w:
                wsn = N.load().glad_rms_norm_backward_workspace_size(rows, cols)
                dw, ws = torch.empty_like(weight), rstd.new_empty(wsn // 4)
                dwp, wsp = dw.data_ptr(), ws.data_ptr()
        rc = N.on_device(N.load().glad_rms_norm_backward, h.device.index, dy2.data_ptr(), _CODE[x_t], dy2.stride(0), dsp,
                         _CODE[h_t], ldds, h2.data_ptr(), h2.stride(0), wp, wt, rstd.data_ptr(), rows, cols,
                         None if dx is None else dx.data_ptr(), None if dr is None or dr is dx else dr.data_ptr(), dwp,
                         wsp, wsn)
        if rc:
            N.check(rc, "rms_norm backward")
        return dx if need_x else None, dw, dr, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
             eps: float = 1e-6):
    """y in x's type, or ``(y, h)`` with a residual; h has the residual's type.

    x [..., C] float32, float16 or bfloat16, rows of any stride; weight [C] (None: ones) and residual
    (x's shape) have x's type or float32; C up to 32768. Differentiable in x, weight and residual (backward mode).
    The sum is rounded to the residual's type first and the norm is of that value."""
    N.refuse_tangents("rms_norm", x, weight, residual)
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
    columns of a row (s [..., ceil(C / group)]), 1 where that is 0. ``scale`` a float32 tensor of one value: that
    scale for all (static calibration), returned as s. Inference only: inputs that require a gradient are refused
    while gradients are enabled (``rms_norm`` is the form that trains)."""
    if out_dtype != torch.int8 and out_dtype != torch.float8_e4m3fn:
        raise TypeError(f"out_dtype is {out_dtype}; expected int8 or float8_e4m3fn")
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group must be 0, 32, 64 or 128, got {group}")
    if scale is not None:
        if group:
            raise ValueError("a given scale is one for the whole tensor (group 0)")
        if scale.numel() != 1 or scale.dtype != torch.float32 or scale.device != x.device:
            raise ValueError("scale must be one float32 value on x's device")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual, scale)):
        raise RuntimeError("rms_norm_quant has no gradient; use rms_norm, or torch.no_grad()")
    N.refuse_tangents("rms_norm_quant", x, weight, residual, scale)
    _check(x, weight, residual, eps)
    x2 = _rows(x)
    rows, cols = x2.shape
    q = _like(x, out_dtype)
    s, sp, gp = scale, None, None
    if s is None:
        s = x.new_empty(x.shape[:-1] + (-(-cols // group) if group else 1,), dtype=torch.float32)
        sp = s.data_ptr()
    else:
        gp = s.data_ptr()
    wp, wt, rp, rt, ldr, h, hp = None, 0, None, 0, 0, None, None
    if weight is not None:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        wp, wt = weight.data_ptr(), _CODE[weight.dtype]
    if residual is not None:
        r2 = _rows(residual)
        h = _like(residual)
        rp, rt, ldr, hp = r2.data_ptr(), _CODE[residual.dtype], r2.stride(0), h.data_ptr()
    rc = N.on_device(N.load().glad_rms_norm_quant, x.device.index, x2.data_ptr(), _CODE[x.dtype], x2.stride(0), rp, rt, ldr,
                     wp, wt, rows, cols, eps, N.DTYPE_I8 if out_dtype == torch.int8 else N.DTYPE_E4M3, group, gp,
                     q.data_ptr(), sp, hp)
    if rc:
        N.check(rc, "rms_norm_quant")
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
        """The same norm over the source module's own Parameter (optimiser references stay valid). An eps of None is, as
        in torch, that of the type the norm is computed in: float32's for 16-bit layers too."""
        if len(norm.normalized_shape) != 1:
            raise ValueError(f"normalized_shape {tuple(norm.normalized_shape)}: the last dimension only")
        eps = norm.eps
        if eps is None:
            if norm.weight is None:
                raise ValueError("a norm without weight and eps takes its eps from each input's type (float64's, or float32's "
                                 "for the others); set eps")
            eps = torch.finfo(torch.float64 if norm.weight.dtype == torch.float64 else torch.float32).eps
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
