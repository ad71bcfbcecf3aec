"""4-bit linear of any shape, for few rows to many: int4 weights with one fp16 scale a group of inputs.

The weight format is ``quantize_w4``'s (rl_quant_b200/w4a16.py, the format of the W4A16 actor MLP) with groups of
32, 64 or 128; ``pack_w4`` lays it out once in the order the kernel streams it (include/glad_b200.h, GladW4Weight).
Rows are fp16 or bf16, or 8-bit codes with scales as ``rms_norm_quant`` writes them. Products are exact, sums fp32 and
the group's scale multiplies the group's sum: y = sum_g s[n,g] * (sum_k x[m,k] q[n,k]) + b, rounded once.
"""
from __future__ import annotations

import contextlib
import ctypes
import threading

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _native as N
from .w4a16 import quantize_w4

GROUPS = (32, 64, 128)
_OUT = (torch.float16, torch.bfloat16, torch.float32)


def _shapes(in_features: int, out_features: int, group: int):
    """Shapes of the laid-out weight: tiles (uint8), scales (fp16)."""
    t, u = -(-out_features // 128), -(-in_features // 128)
    return (t, u, 8192), (t, u, 8, 128 // group * 16)


class W4Weight:
    """A laid-out 4-bit weight [out_features, in_features]: ``tiles`` (uint8) and ``scales`` (fp16) on one device."""

    __slots__ = ("_tiles", "_scales", "_shape")

    def __init__(self, tiles, scales, in_features, out_features, group):
        if group not in GROUPS:
            raise ValueError(f"group must be one of {GROUPS}, got {group}")
        if in_features < 2 or in_features % 2:
            raise ValueError(f"in_features must be even, got {in_features}")
        t_shape, s_shape = _shapes(in_features, out_features, group)
        if tiles.dtype != torch.uint8 or tuple(tiles.shape) != t_shape or not tiles.is_contiguous():
            raise ValueError(f"tiles must be contiguous uint8 {t_shape}")
        if scales.dtype != torch.float16 or tuple(scales.shape) != s_shape or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous float16 {s_shape}")
        if tiles.device != scales.device:
            raise ValueError(f"tiles on {tiles.device}, scales on {scales.device}")
        self._tiles, self._scales, self._shape = tiles, scales, (in_features, out_features, group)

    tiles = property(lambda self: self._tiles)
    scales = property(lambda self: self._scales)
    in_features = property(lambda self: self._shape[0])
    out_features = property(lambda self: self._shape[1])
    group = property(lambda self: self._shape[2])


@torch.no_grad()
def pack_w4(packed: torch.Tensor, scales: torch.Tensor, group: int = 64) -> W4Weight:
    """``quantize_w4``'s (packed uint8 [N, K/2], scales fp16 [N, ceil(K/group)]) as a ``W4Weight``."""
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    if packed.dtype != torch.uint8 or packed.dim() != 2 or packed.shape[0] < 1 or packed.shape[1] < 1:
        raise ValueError("packed must be uint8 [N, K/2]")
    n, k = packed.shape[0], 2 * packed.shape[1]
    if scales.dtype != torch.float16 or tuple(scales.shape) != (n, -(-k // group)):
        raise ValueError(f"scales must be float16 [{n}, {-(-k // group)}]")
    (t, u, _), s_shape = _shapes(k, n, group)
    g = 128 // group
    q = torch.zeros(t * 128, u * 128, dtype=torch.uint8, device=packed.device)
    q[:n, 0:k:2] = packed & 15
    q[:n, 1:k:2] = packed >> 4
    # [t, n16, row half, row, unit, kb, j, c, k/2, k%2] -> byte (k/2 + 2 (k%2)) of word j, row half in the nibble
    v = q.view(t, 8, 2, 8, u, 2, 4, 4, 2, 2)
    b = (v[:, :, 0] | (v[:, :, 1] << 4)).permute(0, 3, 1, 4, 2, 6, 5, 8, 7)
    s = torch.zeros(t * 128, u * g, dtype=torch.float16, device=scales.device)
    s[:n, :scales.shape[1]] = scales
    s = s.view(t, 8, 2, 8, u, g).permute(0, 4, 1, 5, 3, 2)
    return W4Weight(b.reshape(t, u, 8192).contiguous(), s.reshape(s_shape).contiguous(), k, n, group)


@torch.no_grad()
def unpack_w4(weight: W4Weight):
    """The inverse of ``pack_w4``: (packed, scales)."""
    (t, u, _), _ = _shapes(weight.in_features, weight.out_features, weight.group)
    n, k, g = weight.out_features, weight.in_features, 128 // weight.group
    b = weight.tiles.view(t, u, 8, 2, 8, 4, 4, 2, 2).permute(0, 2, 4, 1, 3, 6, 5, 8, 7)
    q = torch.stack((b & 15, b >> 4), dim=2).reshape(t * 128, u * 128)[:n, :k]
    packed = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
    s = weight.scales.view(t, u, 8, g, 8, 2).permute(0, 2, 5, 4, 1, 3).reshape(t * 128, u * g)
    return packed, s[:n, :-(-k // weight.group)].contiguous()


def w4_linear(x: torch.Tensor, weight: W4Weight, bias: torch.Tensor | None = None,
              x_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] times the weight's transpose, plus bias: y [..., N].

    x float16 or bfloat16 (``x_scale`` None, ``out_dtype`` x's by default), or int8 / float8_e4m3fn codes with a float32
    ``x_scale`` of one value, [..., 1] (one a row) or [..., ceil(K / group)] (one a row and group of the weight) and
    ``out_dtype`` named. out_dtype float16, bfloat16 or float32; bias [N] has it. Up to 2^20 rows, inputs (an even number)
    and outputs. Inference only."""
    N.refuse_tangents("w4_linear", x, bias, x_scale)
    K, n, group = weight._shape
    shape, dt = x.shape, x.dtype
    if not shape or shape[-1] != K:
        raise ValueError(f"x {tuple(shape)} does not match in_features {K}")
    eight = dt == torch.int8 or dt == torch.float8_e4m3fn
    if not eight and dt != torch.float16 and dt != torch.bfloat16:
        raise TypeError(f"x is {dt}; expected float16, bfloat16, int8 or float8_e4m3fn")
    if out_dtype is None:
        if eight:
            raise ValueError("8-bit rows need out_dtype")
        out_dtype = dt
    if out_dtype not in _OUT:
        raise TypeError(f"out_dtype is {out_dtype}; expected float16, bfloat16 or float32")
    dev = x.device
    per_row = groups = 0
    xp = bp = None
    if eight:
        if x_scale is None:
            raise ValueError("8-bit rows need x_scale")
        if x_scale.dtype != torch.float32:
            raise TypeError(f"x_scale is {x_scale.dtype}; expected float32")
        if x_scale.shape == shape[:-1] + (1,):
            per_row, groups = 1, 1
        elif x_scale.numel() != 1:
            per_row, groups = 1, -(-K // group)
            if x_scale.shape != shape[:-1] + (groups,):
                raise ValueError(f"x_scale {tuple(x_scale.shape)}: one value, {tuple(shape[:-1]) + (1,)} or "
                                 f"{tuple(shape[:-1]) + (groups,)}")
        if x_scale.device != dev:
            raise ValueError(f"tensors on {dev} and {x_scale.device}")
        if not x_scale.is_contiguous():
            x_scale = x_scale.contiguous()
        xp = x_scale.data_ptr()
    elif x_scale is not None:
        raise ValueError("x_scale is for 8-bit rows")
    if weight._tiles.device != dev:
        raise ValueError(f"tensors on {dev} and {weight._tiles.device}")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != out_dtype:
            raise ValueError(f"bias must be {out_dtype} [{n}]")
        if bias.device != dev:
            raise ValueError(f"tensors on {dev} and {bias.device}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bp = bias.data_ptr()
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)
                                    or (x_scale is not None and x_scale.requires_grad)):
        raise RuntimeError("w4_linear has no gradient; use torch.no_grad()")
    N.require_cuda(x)
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    ld, step = x2.stride()
    if step != 1 or (ld < K and x2.shape[0] > 1):       # broadcast (overlapping) rows are copied
        x2 = x2.contiguous()
        ld = K
    y = x.new_empty(shape[:-1] + (n,), dtype=out_dtype)
    w = N.GladW4Weight(weight._tiles.data_ptr(), weight._scales.data_ptr(), K, n, group)
    rc = N.on_device(N.load().glad_w4_linear_forward, dev.index, w, x2.data_ptr(), N.DTYPES[dt], x2.shape[0],
                     ld, xp, per_row, groups, bp, y.data_ptr(), N.DTYPES[out_dtype])
    if rc:
        N.check(rc, "w4_linear")
    return y


# The kernels' status word is one a device and is cleared by reading. So that no reader loses what another one read
# first, each failure found is counted here, and a reader (every InferenceRunner; the direct callers together) keeps the
# counts that it has been told of.
_status_lock = threading.Lock()
_failures: dict[int, tuple[int, int]] = {}      # device index -> (failures found, bits of the last one)
_told: dict[int, int] = {}
_reader = threading.local()


def w4_failures() -> dict[int, int]:
    """Failures found so far by device index: where a new reader starts."""
    with _status_lock:
        return {k: n for k, (n, _) in _failures.items()}


@contextlib.contextmanager
def w4_status_reader(told: dict[int, int]):
    """``w4_status`` calls of this thread inside are those of the reader that keeps ``told``."""
    old, _reader.told = getattr(_reader, "told", None), told
    try:
        yield
    finally:
        _reader.told = old


def w4_status(device=None) -> int:
    """Device status bits of the w4_linear calls on ``device`` since this reader's last call (0: fine); where a bounded
    wait inside a kernel ran out, raises ``DeviceStatusError``. The word is the device's: a failure of anyone's kernels
    is told to every reader once. Covers the work before it in the current stream, which it synchronises."""
    from .fused import DeviceStatusError
    index = device if isinstance(device, int) or device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    word = ctypes.c_uint32(0)
    with _status_lock:                  # reading the word and counting are one step
        with torch.cuda.device(index):
            rc = N.load().glad_w4_linear_status(word, N.stream_handle())
        if rc != N.GLAD_ERR_DEVICE:
            N.check(rc, "w4_status")
        count, bits = _failures.get(index, (0, 0))
        if rc == N.GLAD_ERR_DEVICE:
            count, bits = _failures[index] = (count + 1, word.value)
        told = getattr(_reader, "told", None)
        told = _told if told is None else told
        known, told[index] = told.get(index, 0), count
    if known != count:
        raise DeviceStatusError(f"w4_linear: device status {bits:#x}")
    return 0


def _top(x):
    """float32 x without the lower 16 bits of its significand's 24: a bfloat16 number, x's sign, the rest exact in float32."""
    return (x.view(torch.int32) & -65536).view(torch.float32)


def _linear_f32(x, weight: W4Weight, bias, out_dtype):
    """float32 rows as the sum of three bfloat16 rows of 8 bits each, which is exact (down to bfloat16's smallest numbers),
    so x is not rounded: three times the rows in one ``w4_linear``, its float32 results added from the smallest up."""
    hi = _top(x)
    rest = torch.where(x == hi, 0.0, x - hi)            # 0 and not NaN behind an infinite part
    mid = _top(rest)
    parts = torch.stack((rest - mid, mid, hi)).bfloat16()
    if 3 * (x.numel() // x.shape[-1]) <= 1 << 20:
        lo, mid, hi = w4_linear(parts, weight, out_dtype=torch.float32)
    else:
        lo, mid, hi = (w4_linear(p, weight, out_dtype=torch.float32) for p in parts)
    y = lo + mid + hi
    if bias is not None:
        y = y + bias.float()
    return y.to(out_dtype)


class W4Linear(nn.Module):
    """``nn.Linear`` with 4-bit weights at inference and its own Parameters in training, like ``QuantLinear``:
    with gradients enabled the forward is ``F.linear`` on the source layer's weight and bias; without, ``w4_linear`` on
    the laid-out copy, which ``requantize_`` rewrites in place (captured CUDA graphs stay valid). Rows are float16, bfloat16 or
    float32 (as three bfloat16 rows, not rounded).
    ``forward(q, x_scale)`` takes 8-bit rows, for inference only: refused while a gradient of its weight is asked for."""

    def __init__(self, linear: nn.Linear, group: int = 64):
        super().__init__()
        if group not in GROUPS:
            raise ValueError(f"group must be one of {GROUPS}, got {group}")
        if linear.in_features % 2:
            raise ValueError(f"in_features={linear.in_features} is odd")
        self.in_features, self.out_features, self.group = linear.in_features, linear.out_features, group
        # the source layer's Parameters, transferred (optimiser references stay valid)
        self.weight = linear.weight
        self.bias = linear.bias
        t_shape, s_shape = _shapes(self.in_features, self.out_features, group)
        dev = linear.weight.device
        self.register_buffer("tiles", torch.zeros(t_shape, dtype=torch.uint8, device=dev))
        self.register_buffer("scales", torch.zeros(s_shape, dtype=torch.float16, device=dev))
        self.requantize_()

    @torch.no_grad()
    def requantize_(self):
        """Refresh the 4-bit copy from the current weight, in place."""
        w = pack_w4(*quantize_w4(self.weight, self.group), self.group)
        self.tiles.copy_(w.tiles)
        self.scales.copy_(w.scales)
        return self

    def _apply(self, fn, recurse=True):
        """A cast of the module (``.bfloat16()``) leaves the scales fp16, made anew from the cast weight."""
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float16:
            self.scales = torch.zeros_like(self.scales, dtype=torch.float16)
            self.requantize_()
        return self

    def w4(self) -> W4Weight:
        return W4Weight(self.tiles, self.scales, self.in_features, self.out_features, self.group)

    def forward(self, x, x_scale=None, out_dtype=None):
        if torch.is_grad_enabled():
            if x_scale is None:
                return F.linear(x, self.weight, self.bias)
            if any(t is not None and t.requires_grad for t in (x, x_scale, self.weight, self.bias)):
                raise RuntimeError("W4Linear on 8-bit rows has no gradient; use torch.no_grad()")
        if x.dtype == torch.float32 and x_scale is None:
            N.refuse_tangents("W4Linear", x, self.bias)
            if out_dtype is not None and out_dtype not in _OUT:
                raise TypeError(f"out_dtype is {out_dtype}; expected float16, bfloat16 or float32")
            N.require_cuda(x)
            if not x.dim() or x.shape[-1] != self.in_features:
                raise ValueError(f"x {tuple(x.shape)} does not match in_features {self.in_features}")
            with torch.no_grad():
                return _linear_f32(x, self.w4(), self.bias, out_dtype or x.dtype)
        if out_dtype is None and x_scale is not None:
            out_dtype = self.weight.dtype
        bias = self.bias
        if bias is not None:
            bias = bias.to(out_dtype or x.dtype)
        with torch.no_grad():
            return w4_linear(x, self.w4(), bias, x_scale, out_dtype)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, group={self.group}, bias={self.bias is not None}"
