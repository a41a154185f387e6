"""Rotary positions: tables scaled for long contexts, and the rotation of
query and key rows in either pair layout over part or all of a head.

The reference rotates inside its append, in one form (half layout, the whole
128-dim head, FP16 arithmetic: tests/page_gauge_append_extension.cu); that
form stays in ``runtime.AppendExtension`` and ``cache.rope_tables``.  Here
the arithmetic is FP32 from FP32 tables, rounded once.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib


@dataclass(frozen=True)
class RotaryScaling:
    """How the frequencies of a model trained on ``trained_positions`` are
    stretched by ``factor`` for longer contexts:

    * ``linear``: every position is divided by the factor;
    * ``ntk``: the base grows by ``factor ** (d / (d - 2))``, which divides the
      lowest frequency by the factor and leaves the highest;
    * ``parts``: frequencies that turn more than ``fast_turns`` times within the
      trained positions stay, those that turn less than ``slow_turns`` times
      are divided by the factor, those between are blended linearly over the
      pair index, and both tables are multiplied by ``attention_factor``
      (default ``0.1 ln(factor) + 1``).
    """

    kind: str
    factor: float
    trained_positions: int = 8192
    fast_turns: float = 32.0
    slow_turns: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "parts"):
            raise ValueError("rotary scaling must be 'linear', 'ntk' or 'parts'")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError("the rotary scaling factor must be finite and at least 1")
        if self.trained_positions <= 0 or not self.fast_turns > self.slow_turns > 0:
            raise ValueError("trained positions must be positive and fast_turns > slow_turns > 0")


def rotary_frequencies(rotary_dim: int, theta: float = 1.0e6,
                       scaling: RotaryScaling | None = None) -> tuple[torch.Tensor, float]:
    """Angle per position of each of the ``rotary_dim / 2`` pairs (float64)
    and the factor on both tables."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    if not (math.isfinite(theta) and theta > 1.0):
        raise ValueError("theta must be finite and above 1")
    pairs = rotary_dim // 2
    if scaling is not None and scaling.kind == "ntk" and rotary_dim > 2:
        theta = theta * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if scaling is None or scaling.kind == "ntk":
        return inv, 1.0
    if scaling.kind == "linear":
        return inv / scaling.factor, 1.0

    def pair_of(turns: float) -> float:
        return (rotary_dim * math.log(scaling.trained_positions / (turns * 2 * math.pi))
                / (2 * math.log(theta)))

    low = max(math.floor(pair_of(scaling.fast_turns)), 0)
    high = min(math.ceil(pair_of(scaling.slow_turns)), rotary_dim - 1)
    ramp = ((torch.arange(pairs, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    scale = scaling.attention_factor
    if scale is None:
        scale = 0.1 * math.log(scaling.factor) + 1.0
    return inv / scaling.factor * ramp + inv * (1 - ramp), float(scale)


def rotary_tables(positions: int, rotary_dim: int = 128, theta: float = 1.0e6,
                  scaling: RotaryScaling | None = None,
                  device: torch.device | str = "cpu") -> tuple[torch.Tensor, torch.Tensor]:
    """Cosine and sine tables [positions, rotary_dim / 2] in FP32.  The angles
    are 64-bit products: at position 2^17 an FP32 angle would be off by 2^-7."""
    if positions <= 0:
        raise ValueError("positions must be positive")
    inv, scale = rotary_frequencies(rotary_dim, theta, scaling)
    t = torch.arange(positions, dtype=torch.float64, device=device)
    angle = t[:, None] * inv.to(device)
    return (angle.cos() * scale).float(), (angle.sin() * scale).float()


def _refuse_capture(rows: torch.Tensor) -> None:
    """A captured backward pass ends the process where an eager graph of the same
    leaves lives: what accumulates their gradients belongs to the eager stream.
    So neither direction of a rotation with a gradient is captured."""
    with torch.cuda.device(rows.device):
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("a rotation with a gradient cannot be captured; capture the "
                             "rotation and its adjoint under no_grad")


class _Rotate(torch.autograd.Function):
    """The rotation, whose gradient is its transpose.  Rows that the kernel
    leaves (a position outside the tables) are zero, and so are their
    gradients."""

    @staticmethod
    def forward(ctx, query, key, cosine, sine, positions, interleaved, adjoint):
        ctx.save_for_backward(cosine, sine, positions)
        ctx.set_materialize_grads(False)
        ctx.mode = (interleaved, not adjoint)
        out = _lib.torch_ops().rotary(
            query, key, cosine, sine, positions, interleaved, adjoint,
            torch.zeros(query.shape, dtype=query.dtype, device=query.device),
            None if key is None else torch.zeros(key.shape, dtype=key.dtype, device=key.device))
        ctx.mark_non_differentiable(
            *(y for y, need in zip(out, ctx.needs_input_grad) if y is not None and not need))
        return out

    @staticmethod
    def backward(ctx, *grads):
        needed = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[i]]
        # A sum's gradient is one value expanded over the rows.
        if needed:
            _refuse_capture(grads[needed[0]])
        rows = [grads[i] if grads[i].stride(-1) == 1 else grads[i].contiguous() for i in needed]
        result = [None] * 7
        if rows:
            turned = _Rotate.apply(rows[0], rows[1] if len(rows) == 2 else None,
                                   *ctx.saved_tensors, *ctx.mode)
            for i, y in zip(needed, turned):
                result[i] = y
        return tuple(result)


def _rotate_with_gradient(query, key, cosine, sine, positions, interleaved, adjoint, query_out,
                          key_out):
    if query_out is not None or key_out is not None:
        raise ValueError("rows that require gradients are rotated into new tensors")
    if cosine.requires_grad or sine.requires_grad:
        raise ValueError("the rotary tables have no gradient")
    if query.is_cuda:  # others are refused with the arguments
        _refuse_capture(query)
    return _Rotate.apply(query, key, cosine, sine, positions, bool(interleaved), bool(adjoint))


def apply_rotary(query: torch.Tensor, key: torch.Tensor | None, cosine: torch.Tensor,
                 sine: torch.Tensor, positions: torch.Tensor, *, interleaved: bool = False,
                 adjoint: bool = False, query_out: torch.Tensor | None = None,
                 key_out: torch.Tensor | None = None):
    """Rotate ``query`` [T, Hq, D] and ``key`` [T, Hkv, D] (or None) by
    ``positions`` (device int32 [T]); returns (query_out, key_out).

    ``cosine``/``sine`` are FP32 [positions, pairs] (``rotary_tables``); the
    first ``2 * pairs`` dims turn, the others are copied.  Half layout pairs
    dim j with j + pairs, ``interleaved`` 2j with 2j + 1.  ``adjoint`` turns
    back (the gradient of the rotation with respect to its rows, which autograd
    takes for rows that require one; the call then makes its outputs, and neither
    it nor its backward pass is captured into a graph; forward-mode duals are
    refused).  Rows are
    float16, bfloat16 or float32 with a contiguous last dimension and any
    other strides.  The outputs may be the inputs (in place); they must not
    overlap them in any other way.  Rows of a token whose position is outside
    the tables are not written (``runtime.read_device_error`` reports it)."""
    out = (_lib._ops or _lib.torch_ops()).rotary(
        query, key, cosine, sine, positions, interleaved, adjoint, query_out, key_out)
    if out is None:  # rows that require gradients
        out = _rotate_with_gradient(query, key, cosine, sine, positions, interleaved, adjoint,
                                    query_out, key_out)
    return out
