"""Low-rank adapters beside a shared projection, many of them in one batch (no qrt counterpart): what of a 4-bit or int8 layer is
trained, and what differs between the requests or tasks that share the layer.

    y[m] = base[m] + scale[i] * B[i] (A[i] x[m]),   i = index[m]

``lora_linear`` is the operator, with its backward pass; ``LoRALinear`` is an adapter bank over any linear layer of
this package or torch, put in place by ``swap.apply_lora``.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _native as N

_CODE = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
MAX_RANK = 128
MAX_ADAPTERS = 16384
MAX_SIZE = 1 << 24           # rows, inputs, outputs


def _needs_plan(M, L):
    """Whether a forward pass alone needs the order of the rows by adapter laid down first."""
    return M > 4096 or (M > 256 and L > 512)


def _rows(t):
    """[..., C] as rows of adjacent columns: a view where the strides allow one, else a copy."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    rows, cols = t2.shape
    ld, step = t2.stride()
    return t2 if (step == 1 or cols == 1) and (ld >= cols or rows <= 1) else t2.contiguous()


def _forward(x, a, b, index, scale, base, plan, plan_bytes, u):
    """``plan`` and ``u`` are addresses of scratch memory, or None."""
    x2 = _rows(x)
    M, K = x2.shape
    L, r, _ = a.shape
    n = b.shape[1]
    y = x.new_empty(x.shape[:-1] + (n,))
    bp, ldb, ip, ib, sp, sv = None, 0, None, 0, None, 0.0
    if base is not None:
        b2 = _rows(base)
        bp, ldb = b2.data_ptr(), b2.stride(0)
    if index is not None:
        ip, ib = index.data_ptr(), index.element_size()
    if isinstance(scale, torch.Tensor):
        sp = scale.data_ptr()
    else:
        sv = scale
    rc = N.on_device(N.load().glad_lora_forward, x.device.index, x2.data_ptr(), _CODE[x.dtype], x2.stride(0), M, K,
                     a.data_ptr(), b.data_ptr(), n, L, r, ip, ib, plan, plan_bytes, sp, sv, bp, ldb, y.data_ptr(), u)
    if rc:
        N.check(rc, "lora_linear")
    return y


class _LoRA(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, index, scale, base):
        L, r, K = a.shape
        M = x.numel() // K
        # one buffer: the order of the rows, then u
        plan_bytes = N.load().glad_lora_plan_size(M, L) + 15 & -16 if index is not None else 0
        kept = torch.empty(plan_bytes + 4 * M * r, dtype=torch.uint8, device=x.device)
        at = kept.data_ptr()
        plan, u = at if plan_bytes else None, at + plan_bytes if ctx.needs_input_grad[2] else None
        y = _forward(x, a, b, index, scale, base, plan, plan_bytes, u)
        given = isinstance(scale, torch.Tensor)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, a, b, index, scale if given else None, kept)
        ctx.scale, ctx.x_shape, ctx.plan_bytes = 0.0 if given else scale, x.shape, plan_bytes
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_a, need_b, _, _, need_base = ctx.needs_input_grad
        x, a, b, index, scale, kept = ctx.saved_tensors
        dx = da = db = None
        if need_x or need_a or need_b:
            d2 = _rows(dy)
            M, n = d2.shape
            L, r, K = a.shape
            xp = dxp = dap = dbp = up = dup = ip = plan = wsp = None
            ldx = ib = 0
            lib, code = N.load(), _CODE[dy.dtype]
            # one buffer: du, then the adapters transposed (large calls)
            first = 4 * M * r + 15 & -16 if need_a else 0
            ws_bytes = lib.glad_lora_backward_workspace_size(M, K, n, L, r, code, index is not None) if need_x or need_a else 0
            if first or ws_bytes:
                ws = torch.empty(first + ws_bytes, dtype=torch.uint8, device=dy.device)
                dup = ws.data_ptr()
                wsp = dup + first
            if need_x:
                dx = dy.new_empty(ctx.x_shape)
                dxp = dx.data_ptr()
            if need_a:
                x2 = _rows(x)
                xp, ldx = x2.data_ptr(), x2.stride(0)
                da = torch.empty_like(a)
                dap = da.data_ptr()
            if need_b:
                db = torch.empty_like(b)
                dbp, up = db.data_ptr(), kept.data_ptr() + ctx.plan_bytes
            if index is not None:
                ip, ib, plan = index.data_ptr(), index.element_size(), kept.data_ptr()
            rc = N.on_device(lib.glad_lora_backward, dy.device.index, d2.data_ptr(), code, d2.stride(0), xp,
                             ldx, M, K, a.data_ptr(), b.data_ptr(), n, L, r, ip, ib, plan,
                             None if scale is None else scale.data_ptr(), ctx.scale, up, dup, dxp, dap, dbp, wsp, ws_bytes)
            if rc:
                N.check(rc, "lora_linear backward")
        return dx, da, db, None, None, dy if need_base else None


def lora_linear(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor | None = None,
                scale: torch.Tensor | float = 1.0, base: torch.Tensor | None = None) -> torch.Tensor:
    """``base`` [..., N] (None: zeros) plus each row's adapter: scale[i] * b[i] (a[i] x), i = index.

    x [..., K], a [L, r, K], b [L, N, r] and base have one type, float32, float16 or bfloat16; rows of x and base may have any
    stride. index [...] int64 or int32 names the adapter of each row of x; outside 0..L-1 (by custom -1) the row has none. None:
    adapter 0 for all (L = 1). scale a number, or float32 [L]. r up to 128, L up to 16384. Differentiable in x, a, b and
    base (backward mode). Sums are float32 and the result is rounded once; A x (and B^T dy), between the two products, counts with 16
    bits beside bfloat16 rows and with 22 beside others. Large calls of high rank wait for the tensor core with a
    bound; ``w4_status`` tells of a wait that ran out."""
    dt, shape, dev, a_shape, b_shape = x.dtype, x.shape, x.device, a.shape, b.shape
    if dt not in _CODE:
        raise TypeError(f"x is {dt}; expected float32, float16 or bfloat16")
    if len(a_shape) != 3 or len(b_shape) != 3 or b_shape[0] != a_shape[0] or b_shape[2] != a_shape[1]:
        raise ValueError(f"a {tuple(a_shape)} and b {tuple(b_shape)} must be [L, r, K] and [L, N, r]")
    (L, r, K), n = a_shape, b_shape[1]
    if not 1 <= r <= MAX_RANK or not 1 <= L <= MAX_ADAPTERS or not 1 <= K <= MAX_SIZE or not 1 <= n <= MAX_SIZE:
        raise ValueError(f"{L} adapters of rank {r}, {K} inputs and {n} outputs: up to {MAX_ADAPTERS}, {MAX_RANK} and {MAX_SIZE}")
    if not shape or shape[-1] != K:
        raise ValueError(f"x {tuple(shape)} does not match a's {K} inputs")
    M = x.numel() // K
    if M > MAX_SIZE:
        raise ValueError(f"{M} rows: up to {MAX_SIZE}")
    if a.dtype != dt or b.dtype != dt:
        raise TypeError(f"a is {a.dtype} and b {b.dtype}; expected x's {dt}")
    if a.device != dev or b.device != dev:
        raise ValueError(f"tensors on {dev}, {a.device} and {b.device}")
    grad = torch.is_grad_enabled()
    if index is not None:
        if index.dtype != torch.int64 and index.dtype != torch.int32:
            raise TypeError(f"index is {index.dtype}; expected int64 or int32")
        if index.shape != shape[:-1]:
            raise ValueError(f"index {tuple(index.shape)} does not match x {tuple(shape)}")
        if index.device != dev:
            raise ValueError(f"tensors on {dev} and {index.device}")
        if not index.is_contiguous():
            index = index.contiguous()
    elif L != 1:
        raise ValueError(f"{L} adapters need an index")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (L,):
            raise ValueError(f"scale must be a number or float32 [{L}]")
        if scale.device != dev:
            raise ValueError(f"tensors on {dev} and {scale.device}")
        if grad and scale.requires_grad:
            raise RuntimeError("lora_linear has no gradient of scale")
        N.refuse_tangents("lora_linear", scale)
        if not scale.is_contiguous():
            scale = scale.contiguous()
    if base is not None:
        if base.shape != shape[:-1] + (n,):
            raise ValueError(f"base {tuple(base.shape)} does not match {tuple(shape[:-1]) + (n,)}")
        if base.dtype != dt:
            raise TypeError(f"base is {base.dtype}; expected x's {dt}")
        if base.device != dev:
            raise ValueError(f"tensors on {dev} and {base.device}")
    N.refuse_tangents("lora_linear", x, a, b, base)
    N.require_cuda(x)
    if not a.is_contiguous():
        a = a.contiguous()
    if not b.is_contiguous():
        b = b.contiguous()
    if grad and (x.requires_grad or a.requires_grad or b.requires_grad or (base is not None and base.requires_grad)):
        return _LoRA.apply(x, a, b, index, scale, base)
    if index is None or not _needs_plan(M, L):
        return _forward(x, a, b, index, scale, base, None, 0, None)
    size = N.load().glad_lora_plan_size(M, L)
    plan = torch.empty(size, dtype=torch.uint8, device=dev)
    return _forward(x, a, b, index, scale, base, plan.data_ptr(), size, None)


class LoRALinear(nn.Module):
    """A linear layer (``nn.Linear``, ``QuantLinear``, ``W4Linear``) with ``adapters`` low-rank adapters of rank ``rank``:
    ``forward(x)`` is the layer's output plus each row's adapter, times alpha / rank.

    ``select(index)`` names the adapters of the rows from then on (int tensor of x's leading dimensions, or a number for all rows; -1:
    none). The tensor is kept, not copied: new values in it count from the next call on, a captured one's too, while another selection
    needs another capture (an ``InferenceRunner`` makes it by itself). Parameters ``lora_a`` [L, r, K] (random) and ``lora_b`` [L, N, r] (zeros, so a new adapter changes nothing);
    the layer below, ``base``, is kept as it is, and its Parameters are frozen where ``freeze`` is set. Rows are float32, float16 or
    bfloat16; where the layer's output type is not the adapters' own, rows and adapters are cast to it for the call."""

    def __init__(self, base: nn.Module, rank: int = 16, adapters: int = 1, alpha: float | None = None, freeze: bool = True,
                 dtype=None):
        super().__init__()
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"rank must be in 1..{MAX_RANK}, got {rank}")
        if not 1 <= adapters <= MAX_ADAPTERS:
            raise ValueError(f"adapters must be in 1..{MAX_ADAPTERS}, got {adapters}")
        self.base = base
        self.in_features, self.out_features, self.rank, self.adapters = base.in_features, base.out_features, rank, adapters
        self.scale = (rank if alpha is None else alpha) / rank
        w = base.weight
        dtype = dtype or w.dtype
        self.lora_a = nn.Parameter(torch.empty(adapters, rank, self.in_features, dtype=dtype, device=w.device))
        self.lora_b = nn.Parameter(torch.zeros(adapters, self.out_features, rank, dtype=dtype, device=w.device))
        nn.init.normal_(self.lora_a, std=1.0 / math.sqrt(self.in_features))
        self.index: torch.Tensor | int = 0
        if freeze:
            for p in base.parameters():
                p.requires_grad_(False)
        self.train(base.training)

    def select(self, index: torch.Tensor | int | None) -> "LoRALinear":
        if isinstance(index, int) and not -1 <= index < self.adapters:
            raise ValueError(f"adapter {index} of {self.adapters}")
        self.index = -1 if index is None else index
        return self

    def forward(self, x):
        if x.dtype not in _CODE:
            raise TypeError(f"x is {x.dtype}; expected float32, float16 or bfloat16")
        y = self.base(x)
        if isinstance(self.index, int):
            if self.index < 0:
                return y
            a, b, index = self.lora_a[self.index:self.index + 1], self.lora_b[self.index:self.index + 1], None
        else:
            a, b, index = self.lora_a, self.lora_b, self.index
        if a.dtype != y.dtype:
            a, b = a.to(y.dtype), b.to(y.dtype)
        return lora_linear(x.to(y.dtype), a, b, index, self.scale, y)

    def extra_repr(self):
        return f"rank={self.rank}, adapters={self.adapters}, scale={self.scale:g}"
