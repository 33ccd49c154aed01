"""Rotary positions with one or several axes (a language model's text; time, height and width of the images and videos among
it) for the queries and keys of an attention, both in one kernel.

Runs on the current stream of the tensors' GPU, keeps nothing between calls and may be captured in a CUDA graph.  Rows are
views with strides of whole 16-byte pieces, such as columns of fused projection rows.  Arguments that cannot be right raise at
the call: ``ValueError`` for a table that cannot be made (head_dim a multiple of 8, rotary_dim of 16, sections that add up) and
for heads of another size, ``T2WError`` for sizes that the kernel does not have (rotary_dim above 4096, tens of thousands of heads)
and for q and k that share memory in place, ``RuntimeError`` for tensors of the wrong type, shape, device or alignment, or that
require a gradient where gradients are recorded.
"""

from __future__ import annotations

import decimal

import torch

from . import ops as O

_TURN = "6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965068423413596429617302656461"


class Rotary:
    """Pair i of a head turns by ``positions[axis_i, row] * f_i``, ``f_i = base ** (-2 i / rotary_dim)`` or ``inv_freq[i]``.

    ``sections``: how many of the ``rotary_dim / 2`` pairs go with each axis of ``positions`` (all with one, unless given),
    the first ``sections[0]`` pairs with axis 0 and so on, or with ``interleaved`` dealt to the axes in turn, as long as an
    axis has any left.
    ``pairs``: "half" pairs values i and i + rotary_dim / 2 of a head, "adjacent" 2 i and 2 i + 1.  Values past
    ``rotary_dim`` (``head_dim`` unless given) stay as they are.

    There is one ladder of frequencies over all pairs, whatever their axes.  Models that start it again for each axis, as image
    towers with height and width do, give it as ``inv_freq``: ``2 * [base ** (-4 * i / rotary_dim) for i in range(rotary_dim // 4)]``
    for two axes with half of the pairs each.

    Angles are whole positions times frequencies in 64-bit fixed point, modulo a turn: as exact at a million as at one."""

    def __init__(self, head_dim: int, sections=None, *, base: float = 10000.0, rotary_dim: int | None = None,
                 pairs: str = "half", interleaved: bool = False, inv_freq=None, device="cuda"):
        rot = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or head_dim % 8 or rot <= 0 or rot % 16 or rot > head_dim:
            raise ValueError("head_dim is a multiple of 8, rotary_dim a multiple of 16 and at most head_dim")
        if pairs not in ("half", "adjacent"):
            raise ValueError('pairs is "half" or "adjacent"')
        n = rot // 2
        sections = [n] if sections is None else [int(s) for s in sections]
        if not sections or min(sections) < 0 or sum(sections) != n:
            raise ValueError(f"the sections add up to the {n} pairs")
        self.head_dim, self.rotary_dim, self.axes, self.adjacent = head_dim, rot, len(sections), pairs == "adjacent"
        if interleaved:
            left, axis = list(sections), []
            while len(axis) < n:
                for a in range(len(left)):
                    if left[a]:
                        axis.append(a)
                        left[a] -= 1
        else:
            axis = [a for a, s in enumerate(sections) for _ in range(s)]
        # Turns per position, to 2^-64, from numbers of 60 digits
        with decimal.localcontext() as c:
            c.prec = 60
            if inv_freq is None:
                if not (base > 0 and base < float("inf")):
                    raise ValueError("base is positive")
                step, f = (decimal.Decimal(base).ln() * -2 / rot).exp(), [decimal.Decimal(1)]
                while len(f) < n:
                    f.append(f[-1] * step)
            else:
                f = [decimal.Decimal(float(x)) for x in inv_freq]
                if len(f) != n or not all(x.is_finite() for x in f):
                    raise ValueError(f"inv_freq holds {n} finite numbers")
            fixed = [int((x / decimal.Decimal(_TURN) * 2 ** 64).to_integral_value()) % 2 ** 64 for x in f]
        self.table = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in fixed] + axis, dtype=torch.int64).to(device)

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inverse: bool = False):
        """The turned ``q [rows, heads, head_dim]`` and ``k [rows, kv_heads, head_dim]`` (bf16 or fp16; k may be None), new
        and contiguous, for ``positions`` (int32 or int64 ``[axes, rows]``, or ``[rows]`` for one axis; rows of text may be
        one line for all axes, ``expand``-ed).  ``inverse`` turns back: by the negative angles, which is also the gradient of
        the forward call."""
        r = O.call("rotary", self._fits(q), k, positions, self.table, self.rotary_dim, self.axes, self.adjacent, inverse)
        return r[0], (r[1] if k is not None else None)

    def apply_(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inverse: bool = False) -> None:
        """The same in place: q and k, which share no memory, are turned where they lie."""
        O.call("rotary_", self._fits(q), k, positions, self.table, self.rotary_dim, self.axes, self.adjacent, inverse)

    def _fits(self, q: torch.Tensor) -> torch.Tensor:
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"heads of {self.head_dim} values, got {tuple(q.shape)}")
        return q
