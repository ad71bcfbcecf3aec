"""Log probabilities of given tokens, entropy and top alternatives of rows of logits, for policies whose actions are tokens
or bins (``fused.ppo_epilogue`` is the counterpart for a Normal head; no qrt counterpart).

    z = (x - max x) / temperature,  log p_j = z_j - ln sum e^z,  H = -sum p ln p

One reading of the logits forward, one backward; the probabilities are never stored.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

_CODE = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
MAX_TOP = 32
MAX_COLS = 1 << 30


class TokenLogProbs(NamedTuple):
    """Results of ``token_log_probs``; what was not asked for is None."""
    log_prob: torch.Tensor
    entropy: torch.Tensor | None
    top_log_prob: torch.Tensor | None
    top_index: torch.Tensor | None


def _rows(t):
    """[..., V] as rows of adjacent columns: a view where the strides allow one, else a copy."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    rows, cols = t2.shape
    ld, step = t2.stride()
    return t2 if (step == 1 or cols == 1) and (ld >= cols or rows <= 1) else t2.contiguous()


def _forward(x, tokens, temperature, entropy, top, ignore_index, stats):
    x2 = _rows(x)
    rows, cols = x2.shape
    shape = x.shape[:-1]
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    lp = x.new_empty(shape, dtype=torch.float32)
    h = x.new_empty(shape, dtype=torch.float32) if entropy else None
    tv = x.new_empty(shape + (top,), dtype=torch.float32) if top else None
    ti = x.new_empty(shape + (top,), dtype=torch.int64) if top else None
    rc = N.on_device(N.load().glad_token_log_probs, x.device.index, x2.data_ptr(), _CODE[x.dtype], x2.stride(0), rows, cols,
                     tokens.data_ptr(), tokens.element_size(), ignore_index, temperature, top, lp.data_ptr(), N.ptr(h),
                     N.ptr(tv), N.ptr(ti), N.ptr(stats))
    if rc:
        N.check(rc, "token_log_probs")
    return lp, h, tv, ti


def _f32(t):
    """A gradient as adjacent float32 values."""
    return None if t is None else t.to(torch.float32).contiguous()


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, temperature, entropy, top, ignore_index):
        stats = x.new_empty(x.shape[:-1] + (2,), dtype=torch.float32)
        lp, h, tv, ti = _forward(x, tokens, temperature, entropy, top, ignore_index, stats)
        ctx.save_for_backward(x, tokens, stats, h, ti)
        ctx.args = temperature, top, ignore_index
        ctx.set_materialize_grads(False)
        if ti is not None:
            ctx.mark_non_differentiable(ti)
        return lp, h, tv, ti

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, gh, gt, _):
        x, tokens, stats, h, ti = ctx.saved_tensors
        temperature, top, ignore_index = ctx.args
        x2 = _rows(x)
        rows, cols = x2.shape
        if not tokens.is_contiguous():
            tokens = tokens.contiguous()
        g, gh, gt = _f32(g), _f32(gh), _f32(gt)
        dx = x.new_empty(x.shape)
        rc = N.on_device(N.load().glad_token_log_probs_backward, x.device.index, x2.data_ptr(), _CODE[x.dtype], x2.stride(0),
                         rows, cols, tokens.data_ptr(), tokens.element_size(), ignore_index, temperature, top,
                         stats.data_ptr(), N.ptr(h), N.ptr(ti), N.ptr(g), N.ptr(gh), N.ptr(gt), dx.data_ptr())
        if rc:
            N.check(rc, "token_log_probs backward")
        return dx, None, None, None, None, None


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0, entropy: bool = False, top: int = 0,
                    ignore_index: int = -100) -> TokenLogProbs:
    """Log probability of ``tokens[...]`` under ``softmax(logits[..., V] / temperature)``, with the distribution's entropy and
    its ``top`` (up to 32) most likely tokens where asked for.

    logits float32, float16 or bfloat16, rows of any stride; tokens int64 or int32. ``log_prob`` [...], ``entropy`` [...] and
    ``top_log_prob`` [..., top] are float32 and differentiable in the logits (backward mode), ``top_index`` [..., top] int64:
    the most likely first, the lower index first among equals. Logits of -inf are masked: probability 0, no gradient (the token itself and
    the alternatives keep their own term, as in torch: d log p_t / d x_t = (1 - p_t) / temperature). A row that is
    masked as a whole has log probability -inf, entropy 0 and no gradient. Rows whose token is ``ignore_index`` count as
    empty whatever they hold: their outputs are 0 (``top_index`` -1), their gradients 0. Any other token outside [0, V) gives NaN, in the row's gradient too."""
    N.refuse_tangents("token_log_probs", logits)
    dt, shape = logits.dtype, logits.shape
    if dt not in _CODE:
        raise TypeError(f"logits are {dt}; expected float32, float16 or bfloat16")
    if not shape or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"logits must have 1..{MAX_COLS} columns, got shape {tuple(shape)}")
    if tokens.dtype != torch.int64 and tokens.dtype != torch.int32:
        raise TypeError(f"tokens are {tokens.dtype}; expected int64 or int32")
    if tokens.shape != shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not match logits {tuple(shape)}")
    if tokens.device != logits.device:
        raise ValueError(f"tensors on {logits.device} and {tokens.device}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6], got {temperature}")
    if not 0 <= top <= MAX_TOP or top > shape[-1]:
        raise ValueError(f"top must be in 0..{MAX_TOP} and at most the {shape[-1]} columns, got {top}")
    N.require_cuda(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, temperature, entropy, top, ignore_index))
    return TokenLogProbs(*_forward(logits, tokens, temperature, entropy, top, ignore_index, None))
