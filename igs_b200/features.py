"""Operators on feature vectors: what stands between an image's tokens and the features
[B,F,D] that ``GaussianSplatting2D`` turns into gaussians.

* ``embed(tokens, table)``: rows of a shared codebook by token;
* ``layer_norm(x, weight, bias)``: every feature vector to mean 0 and variance 1, then an
  affine map;
* ``dropout(x, p, seed)``: a random share of the values to zero, by a counter-based generator.

``fit.ProgressiveSplatter`` calls them (its ``tokens`` / ``norm`` / ``dropout`` options).  The
reference has no counterpart: its features are free parameters (scripts/gs2d_test.py:28-51).

Like the splat they run on CUDA tensors only, on the current stream, asynchronously, and give
the same bits on every call (no floating-point atomics).  Tensors are float32, bfloat16 or
float16; everything is computed in 32 bits and rounded once.  Each is differentiable once.
"""
from __future__ import annotations

import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["embed", "layer_norm", "dropout"]


_F32_MAX = torch.finfo(torch.float32).max


def _require_features(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: igs_b200 runs on CUDA devices only (no CPU path)")
    if t.dtype not in _lib.FEATURE_DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _same_device(name, t, dev):
    if t.device != dev:
        raise RuntimeError(f"all tensors must be on one device; got {dev} and {name} on {t.device}")


def _finite(name, v):
    v = float(v)
    if not abs(v) <= _F32_MAX:
        raise ValueError(f"{name} must be a finite 32-bit number, got {v}")
    return v


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------
class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, empty):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale, ctx.empty = table.shape[0], scale, empty
        return _lib.embed(tokens, table, scale, empty)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return _lib.embed_grad(tokens, grad.contiguous(), ctx.rows, ctx.scale, ctx.empty), None, None, None


def embed(tokens, table, scale=1.0, empty=None):
    """tokens [...] (int32 or int64), table [rows,D] -> [...,D]: ``scale * table[tokens]``, of the
    table's type.

    ``empty``: a token that marks a place without one (any integer, e.g. -1 behind the last token
    of a padded batch): a row of zeros there, and no gradient.  Any other token outside
    ``0 .. rows-1`` gives a row of NaN and no gradient; nothing outside the table is read.

    The gradient of ``table`` is dense, summed in 32 bits in the order of the places (by sorted
    tokens, no atomics).  Rows of the table may be strided (inner stride 1); the result is
    contiguous.
    """
    _require_features("table", table)
    if not isinstance(tokens, torch.Tensor):
        raise TypeError(f"tokens must be a torch.Tensor, got {type(tokens).__name__}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    _same_device("tokens", tokens, table.device)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be [rows,D] with at least one row and column, got {tuple(table.shape)}")
    scale = _finite("scale", scale)
    if empty is not None:
        empty = operator.index(empty)
        if not -(1 << 63) <= empty < 1 << 63:
            raise ValueError(f"empty must fit 64 bits, got {empty}")
    if table.stride(1) != 1 and table.shape[1] > 1:
        table = table.contiguous()
    flat = tokens.reshape(-1).contiguous()
    if _wants_grad(table):
        out = _Embed.apply(table, flat, scale, empty)
    else:
        out = _lib.embed(flat, table, scale, empty)
    return out.view(*tokens.shape, table.shape[1])


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, wdtype, eps):
        y, shift, rstd = _lib.layer_norm(x, weight, bias, wdtype, eps, True)
        ctx.save_for_backward(x, weight, shift, rstd)
        ctx.wdtype = wdtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, shift, rstd = ctx.saved_tensors
        dx, dw, db = _lib.layer_norm_grad(grad.contiguous(), x, weight, ctx.wdtype, shift, rstd, *ctx.needs_input_grad[:3])
        return dx, dw, db, None, None


def _as_rows(x):
    """[...,D] -> [rows,D] with inner stride 1, in place where the strides allow it."""
    D = x.shape[-1]
    if x.stride(-1) == 1 or D == 1:
        try:
            return x.view(-1, D)
        except RuntimeError:
            pass
    return x.contiguous().view(-1, D)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x [...,D] -> ``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (biased
    variance), of x's type.

    ``weight`` and ``bias`` [D], each optional, are of x's type or float32 (both the same).  Rows
    may be strided (inner stride 1); the result is contiguous.  The gradients of ``weight`` and
    ``bias`` are summed over all rows in 32 bits, in a fixed order.
    """
    _require_features("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [...,D] with D >= 1, got {tuple(x.shape)}")
    D = x.shape[-1]
    wdtype = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _require_features(name, t)
        _same_device(name, t, x.device)
        if t.shape != (D,):
            raise ValueError(f"{name} must be [D] = {(D,)}, got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be of x's type ({x.dtype}) or float32, got {t.dtype}")
        if wdtype not in (None, t.dtype):
            raise TypeError(f"weight and bias must be of one type, got {wdtype} and {t.dtype}")
        wdtype = t.dtype
    eps = _finite("eps", eps)
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    wdtype = wdtype or x.dtype
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    rows = _as_rows(x) if x.numel() else x.reshape(0, D)
    if _wants_grad(rows, weight, bias):
        y = _LayerNorm.apply(rows, weight, bias, wdtype, eps)
    else:
        y = _lib.layer_norm(rows, weight, bias, wdtype, eps, False)[0]
    return y.view(x.shape)


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, state):
        ctx.save_for_backward(state)
        ctx.call = (p, seed, offset)
        return _lib.dropout(x, p, seed, offset, state)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (state,) = ctx.saved_tensors
        return _lib.dropout(grad.contiguous(), *ctx.call, state), None, None, None, None


def _word64(name, v):
    v = operator.index(v)
    if not 0 <= v < 1 << 64:
        raise ValueError(f"{name} must be in 0 .. 2^64 - 1, got {v}")
    return v


def dropout(x, p, seed, offset=0):
    """``x / (1 - p)`` where the generator keeps a value, 0 where it does not (whatever was
    there); every value is dropped with probability ``p``, 0 <= p <= 1.

    The mask is a function of (seed, offset, place in the contiguous tensor) and is never stored:
    Philox4x32 with 7 rounds under the key ``seed``, value i taking word i % 4 of the block with
    counter (i // 4, offset).  Calls that should draw different masks take different offsets.

    ``seed``: a number, or an int64 CUDA tensor of two values (seed, offset) that the kernel reads
    when it runs; the argument ``offset`` is then added to the tensor's.  Inside a CUDA graph only
    the tensor form draws a new mask per replay, when something between the replays (or a captured
    operation) changes the tensor.  The backward pass reads it again: pass a tensor that stays as
    it is until then (autograd raises if it was changed in place).
    """
    _require_features("x", x)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in 0 .. 1, got {p}")
    offset = _word64("offset", offset)
    state = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,):
            raise ValueError(f"seed must be a number or an int64 tensor of two values, got {seed.dtype} "
                             f"{tuple(seed.shape)}")
        _same_device("seed", seed, x.device)
        state, seed = seed.contiguous(), 0
    else:
        seed = _word64("seed", seed)
    x = x.contiguous()
    if _wants_grad(x):
        return _Dropout.apply(x, p, seed, offset, state)
    return _lib.dropout(x, p, seed, offset, state)
