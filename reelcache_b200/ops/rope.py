"""Rotary positions with several axes (csrc/paged/rotate.cu): every token has its own position on each axis (frame,
row, column, ...), every channel pair belongs to one axis.

Pair ``j`` of axis ``a`` (the ``i``-th of its ``sections[a]`` pairs) turns by ``positions[:, a] * theta ** (-i /
sections[a])``. The angle is formed in turns, from a two-float frequency below 2^24 and in FP64 beyond, so its error does
not grow with the position.
"""

from __future__ import annotations

import math
from typing import Sequence

import torch

from ..errors import ConfigurationError, UnsupportedError
from ._ext import ext

LAYOUTS = ("interleaved", "halves")


class AxisRope:
    """A rotation: ``sections`` channel pairs per axis (they add up to ``head_dim // 2``), base ``theta`` and the
    pairs' layout: ``"interleaved"`` neighbours ``(2j, 2j + 1)`` or ``"halves"`` ``(j, j + head_dim / 2)``.

    Keep one per model: :meth:`plan` builds its small device table at its first use on a device (with a copy from the
    host, so outside of graph capture)."""

    def __init__(self, head_dim: int, sections: Sequence[int], *, theta: float = 10000.0, layout: str = "interleaved"):
        self.head_dim, self.sections, self.theta, self.layout = int(head_dim), [int(s) for s in sections], float(theta), layout
        if self.head_dim % 16 or not 16 <= self.head_dim <= 256:
            raise ConfigurationError(f"rotary head_dim {head_dim} must be a multiple of 16, at most 256")
        if not 1 <= len(self.sections) <= 4 or min(self.sections) < 0 or sum(self.sections) != self.head_dim // 2:
            raise ConfigurationError(f"rotary sections {tuple(sections)} must be one to four pair counts adding up to "
                                     f"{self.head_dim // 2}")
        if not (math.isfinite(self.theta) and self.theta > 0):
            raise ConfigurationError(f"rotary theta {theta} must be positive")
        if layout not in LAYOUTS:
            raise ConfigurationError(f"rotary layout {layout!r} must be one of {LAYOUTS}")
        self._plans = {}

    @classmethod
    def wan(cls, head_dim: int, *, theta: float = 10000.0, layout: str = "interleaved") -> "AxisRope":
        """Frame, row and column with the Wan split of the pairs (a third each, the rest to the frame)."""
        third = head_dim // 2 // 3
        return cls(head_dim, (head_dim // 2 - 2 * third, third, third), theta=theta, layout=layout)

    def plan(self, device):
        """The rotation on ``device``, as the kernels take it: turns per position of every pair, in two float32 parts."""
        plan = self._plans.get(device)
        if plan is None:
            exponents = [torch.arange(n, dtype=torch.float64) / max(n, 1) for n in self.sections]
            turns = self.theta ** -torch.cat(exponents) / (2.0 * math.pi)
            high = turns.float()
            table = torch.stack([high, (turns - high.double()).float()]).to(device)
            plan = self._plans[device] = ext().RopePlan(table, turns.to(device), self.sections, self.layout == "halves")
        return plan


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rope: AxisRope):
    """``q[T, heads, head_dim]`` and ``k[T, kv_heads, head_dim]`` (or ``None``) at ``positions[T, axes]`` (int32 or
    float32), rotated in one launch; bf16, fp16 or fp32, FP32 math. Rows may be strided (views of a fused projection).
    Differentiable in ``q`` and ``k`` (in reverse mode). Returns ``(q', k')``, new contiguous tensors of the same type."""
    if not q.is_cuda:
        raise UnsupportedError("rotate needs CUDA tensors")
    if q.shape[-1] != rope.head_dim:
        raise ConfigurationError(f"the rotation is for head_dim {rope.head_dim}, q has {q.shape[-1]}")
    return ext().rotate(q, k, positions, rope.plan(q.device))
