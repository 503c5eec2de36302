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
float16; everything is computed in 32 bits and rounded once.  Each is differentiable once, in
reverse mode; forward-mode tangents, ``torch.func`` transforms and ``torch.jit.trace`` raise.
"""
from __future__ import annotations

import operator

import torch

from . import _lib

__all__ = ["embed", "layer_norm", "dropout"]


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
    if empty is not None:
        empty = operator.index(empty)
        if not -(1 << 63) <= empty < 1 << 63:
            raise ValueError(f"empty must fit 64 bits, got {empty}")
    return _lib.features().embed(tokens, table, scale, empty)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x [...,D] -> ``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (biased
    variance), of x's type.

    ``weight`` and ``bias`` [D], each optional, are of x's type or float32 (both the same).  Rows
    may be strided (inner stride 1); the result is contiguous.  The gradients of ``weight`` and
    ``bias`` are summed over all rows in 32 bits, in a fixed order.
    """
    return _lib.features().layer_norm(x, weight, bias, eps)


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
    offset = _word64("offset", offset)
    if isinstance(seed, torch.Tensor):
        return _lib.features().dropout(x, p, 0, offset, seed)
    return _lib.features().dropout(x, p, _word64("seed", seed), offset, None)
