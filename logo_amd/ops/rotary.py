"""Rotary embedding by positions (``csrc/rotary.hip``).

``rotary`` is differentiable and returns new tensors, ``rotary_`` rotates in
place.  Where ``ops.glue.rope`` takes bf16 cos / sin tables of whole heads and
rounds every product as the eager chain of logo/modules/rotary.py:81-106 does,
these take token positions and a ``RotaryPlan``: half or interleaved pairs, the
first part of a head or all of it, frequencies scaled for contexts longer than
the trained ones, bf16, fp16 and fp32, any strides; angles are exact at any
position, products are in fp32 and rounded once.
"""

import math
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _torch_ops

__all__ = ["RotaryPlan", "rotary_plan", "rotary", "rotary_"]

MAX_HEAD_DIM = 256


@dataclass(frozen=True)
class RotaryPlan:
    """How heads are rotated (``rotary_plan`` makes one): the first ``rot_dim``
    of ``head_dim`` elements, in pairs ``(i, i + rot_dim / 2)`` or, with
    ``interleaved``, ``(2 i, 2 i + 1)``; pair i turns by ``turns[i]`` 2^-64 turns
    per position (int64 ``[rot_dim / 2]`` on the device, the bits of an unsigned
    value) and is multiplied by ``amplitude``."""

    head_dim: int
    rot_dim: int
    interleaved: bool
    amplitude: float
    turns: torch.Tensor

    def to(self, device) -> "RotaryPlan":
        return RotaryPlan(self.head_dim, self.rot_dim, self.interleaved, self.amplitude, self.turns.to(device))


def rotary_plan(head_dim: int, theta: float = 10000.0, rot_dim: Optional[int] = None, interleaved: bool = False,
                scaling: Optional[str] = None, factor: float = 1.0, trained_len: Optional[int] = None,
                device=None) -> RotaryPlan:
    """The plan of frequencies ``f_i = theta^(-2 i / rot_dim)`` radians per
    position (logo/modules/rotary.py:58-78), scaled for a context ``factor``
    times the trained one:

    * ``"linear"``: positions interpolated, ``f_i / factor``;
    * ``"ntk"``: the base stretched, ``theta * factor^(rot_dim / (rot_dim - 2))``:
      the fastest pair keeps its frequency, the slowest is divided by ``factor``
      (a single pair keeps its own);
    * ``"yarn"``: pairs that turn more than 32 times over ``trained_len``
      positions keep their frequency, those that turn less than once are divided
      by ``factor``, linearly in the number of turns between; cos and sin are
      multiplied by ``0.1 ln(factor) + 1``."""
    rot = head_dim if rot_dim is None else int(rot_dim)
    if not 1 <= head_dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {MAX_HEAD_DIM}], got {head_dim}")
    if rot < 0 or rot > head_dim or rot % 2:
        raise ValueError(f"rot_dim must be even and at most head_dim ({head_dim}), got {rot}")
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive, got {theta}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"factor must be positive, got {factor}")
    if scaling == "yarn" and (factor < 1 or not trained_len or trained_len < 1):
        raise ValueError("scaling 'yarn' needs trained_len and a factor of at least 1")
    if scaling == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    freqs = [theta ** (-i / rot) for i in range(0, rot, 2)]
    amplitude = 1.0
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    elif scaling == "yarn":
        keep = [min(max((trained_len * f / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0) for f in freqs]
        freqs = [f * k + f / factor * (1.0 - k) for f, k in zip(freqs, keep)]
        amplitude = 0.1 * math.log(factor) + 1.0
    # turns modulo one in 64-bit fixed point, as the bits of an int64
    turns = [int(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64) for f in freqs]
    turns = [t - (1 << 64) if t >> 63 else t for t in turns]
    return RotaryPlan(int(head_dim), rot, bool(interleaved), amplitude,
                      torch.tensor(turns, dtype=torch.int64).to(device=device))


def _args(plan):
    return plan.turns, plan.head_dim, plan.rot_dim, plan.interleaved, plan.amplitude


def rotary(tensors, positions, plan: RotaryPlan):
    """Rotate ``[..., T, H_i, D]`` tensors (one to four of one shape prefix) by
    their tokens' ``positions`` (int32 or int64, broadcast to ``[..., T]``, of
    either sign); returns new contiguous tensors.  Differentiable: the backward
    pass is one launch, the transposed rotation."""
    return _torch_ops.timed("logo_rotary", _torch_ops.ops().rotary, list(tensors), positions, *_args(plan), False)


def rotary_(tensors, positions, plan: RotaryPlan):
    """``rotary`` in place, without gradients; returns the tensors.  At most one
    batch axis, dense rows, and no two rows in the same memory."""
    xs = list(tensors)
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        raise ValueError("rotary_ has no gradient; use rotary")
    _torch_ops.timed("logo_rotary", _torch_ops.ops().rotary_, xs, positions, *_args(plan))
    return xs
