"""Products with 4-bit weights and group scales, for the projections around a decoder's attention: ``linear``, ``gated``
(the first half of a gated feed-forward in one kernel) and ``feed_forward`` (both halves).

A weight is ``(code - zero) * scale``: codes 0 .. 15, one scale (bf16 or fp16) and one zero (0 .. 15; 8 where there are
none) for each row and each ``group`` (32, 64 or 128) consecutive inputs.  ``quantize`` makes codes, scales and zeros from
a matrix, ``pack`` / ``pack_gated`` lay them out once, when a model is loaded; checkpoints that hold codes of their own
start at ``pack``.

The products run on the current stream of the tensors' GPU, need no workspace, keep nothing between calls and may be captured
in a CUDA graph.  No weight is rounded: sums are fp32 over ``(code - zero) * x``, multiplied by a group's scale after it, and
the output is rounded once; so a group's sum has to fit fp32 before its scale (|x| up to 1e35 always does).  They have no
gradient.

Arguments that cannot be right raise at the call: ``T2WError`` for sizes that the kernels do not have, ``RuntimeError`` for
tensors of the wrong type, shape, device or alignment, ``ValueError`` for weights that cannot be packed.
"""

from __future__ import annotations

import torch

from . import lib as L
from . import ops as O

ACT = {"silu": 0, "gelu_tanh": 1}


class Weight4:
    """A laid-out weight (see ``pack``): ``buffer`` (uint8) on the GPU, ``n`` outputs, ``k`` inputs, ``group``, and whether
    it has ``zeros`` and is a ``gated`` pair.

    Products read the buffer ahead of the stream's earlier kernels, so one that is changed in place needs a
    synchronisation before the next product."""

    __slots__ = ("buffer", "n", "k", "group", "kind")

    def __init__(self, buffer: torch.Tensor, n: int, k: int, group: int, kind: int):
        self.buffer, self.n, self.k, self.group, self.kind = buffer, n, k, group, kind

    @property
    def zeros(self) -> bool:
        return bool(self.kind & 1)

    @property
    def is_gated(self) -> bool:
        return bool(self.kind & 2)

    @property
    def scale_dtype(self) -> torch.dtype:
        return torch.float16 if self.kind & 4 else torch.bfloat16

    def unpack(self):
        """The values, exact, as fp32 ``[n, k]``; of a gated pair the gate's and the up projection's."""
        r = O.call("w4_unpack", self.buffer, self.n, self.k, self.group, self.kind)
        return tuple(r) if self.is_gated else r[0]

    def check(self) -> None:
        """Wait for the GPU and raise ``T2WError`` if a product with this weight has given up on a wait since the last look
        (its outputs are void)."""
        L.check("t2w_w4_linear", O.call("w4_status", self.buffer, self.n, self.k, self.group, self.kind))


def quantize(weight: torch.Tensor, group: int = 128, zeros: bool = False):
    """Codes (uint8 ``[n, k]``), scales (``weight``'s type, ``[n, k / group]``) and zeros (uint8, or None) of a bf16 or fp16
    matrix: each group's largest magnitude / 7 is its scale, or with ``zeros`` its range (0 in it) / 15, rounded to the
    type; codes are the nearest to weight / scale (ties to even).  They are values of their own, without a gradient."""
    if weight.dtype not in (torch.bfloat16, torch.float16) or weight.dim() != 2:
        raise ValueError("a bf16 or fp16 matrix is quantised")
    weight = weight.detach()  # (a parameter's scales would keep the fp32 copies made here for a gradient)
    n, k = weight.shape
    if group not in (32, 64, 128) or k == 0 or k % group:
        raise ValueError(f"groups of 32, 64 or 128 that divide the {k} inputs")
    codes = torch.empty(n, k, device=weight.device, dtype=torch.uint8)
    scales = torch.empty(n, k // group, device=weight.device, dtype=weight.dtype)
    zero = torch.empty(n, k // group, device=weight.device, dtype=torch.uint8) if zeros else None
    step = max(1, (1 << 24) // k)
    for i in range(0, n, step):
        w = weight[i:i + step].float().view(-1, k // group, group)
        if not bool(torch.isfinite(w).all()):
            raise ValueError("the matrix holds values that are not finite")
        if zeros:
            # The range in 64 bits: its ends may be far apart, and the scale is to be the nearest to the true quotient
            low, high = w.amin(2).double().clamp(max=0), w.amax(2).double().clamp(min=0)
            s = ((high - low) / 15).to(weight.dtype)
        else:
            s = (w.abs().amax(2) / 7).to(weight.dtype)
        if not bool(torch.isfinite(s).all()):
            raise ValueError("a group's range has no finite scale in this type")
        inv = s.float().unsqueeze(2)
        q = torch.where(inv > 0, w / inv, 0.0).round()
        if zeros:
            z = torch.where(s > 0, -low / s.double(), 0.0).round().clamp(0, 15).float()
            zero[i:i + step] = z.to(torch.uint8)
            q = q + z.unsqueeze(2)
        else:
            q = q + 8.0
        codes[i:i + step] = q.clamp(0, 15).view(-1, k).to(torch.uint8)
        scales[i:i + step] = s
    return codes, scales, zero


def _pack(first, up) -> Weight4:
    kind, sources = (2 if up is not None else 0), []
    codes, scales = first[0], first[1]
    if codes.dim() != 2 or scales.dim() != 2 or scales.shape[0] != codes.shape[0] or scales.shape[1] == 0:
        raise ValueError("codes are [n, k], scales [n, k / group]")
    (n, k), groups = codes.shape, scales.shape[1]
    if k % groups or k // groups not in (32, 64, 128):
        raise ValueError(f"{groups} scales for {k} inputs: groups are 32, 64 or 128 inputs")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("scales are bf16 or fp16")
    if not codes.is_cuda:
        raise RuntimeError("b200t2w ops take CUDA tensors")
    zeros = first[2] if len(first) > 2 else None
    if up is not None and (up[0].shape != codes.shape or up[1].shape != scales.shape or up[1].dtype != scales.dtype or
                           ((up[2] if len(up) > 2 else None) is None) != (zeros is None)):
        raise ValueError("gate and up projection have the same shape, groups, type of scales, and both zeros or neither")
    for codes_, scales_, *z in (first,) if up is None else (first, up):
        z = z[0] if z else None
        for x in (codes_,) if z is None else (codes_, z):
            if x.dtype != torch.uint8 or (x.numel() and int(x.max()) > 15):
                raise ValueError("codes and zeros are uint8, 0 .. 15")
        if not bool(torch.isfinite(scales_).all()):
            raise ValueError("scales are finite")
        sources += [codes_, scales_, z]
    kind |= (1 if zeros is not None else 0) | (4 if scales.dtype == torch.float16 else 0)
    group = k // groups
    size = L.load().t2w_w4_bytes(n, k, group, kind & 1, up is not None)
    if size < 0:
        raise L.T2WError("t2w_w4_bytes", int(size))
    buffer = torch.empty(size, device=codes.device, dtype=torch.uint8)
    O.call("w4_pack", buffer, n, k, group, kind, *(sources + [None] * 3)[:6])
    torch.cuda.current_stream(codes.device).synchronize()  # products read it ahead of the stream
    return Weight4(buffer, n, k, group, kind)


def pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> Weight4:
    """Lay out codes (uint8 ``[n, k]``, 0 .. 15), scales (bf16 or fp16 ``[n, k / group]``) and zeros (uint8 ``[n, k /
    group]``, 0 .. 15; 8 if None) on their GPU.  Waits for the GPU."""
    return _pack((codes, scales, zeros), None)


def pack_gated(gate, up) -> Weight4:
    """Lay out the two projections of a gated feed-forward, each ``(codes, scales, zeros)`` as ``pack`` takes them, as one
    weight for ``gated``.  Waits for the GPU."""
    return _pack(tuple(gate), tuple(up))


def linear(x: torch.Tensor, w: Weight4, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T (+ bias) (+ residual)`` for ``x [rows, k]`` (bf16 or fp16, rows on 16-byte boundaries), ``bias [n]`` and
    ``residual [rows, n]`` of x's type: ``[rows, n]`` of x's type, rounded once."""
    return O.call("w4_linear", x, w.buffer, w.n, w.k, w.group, w.kind, bias, residual)


def gated(x: torch.Tensor, w: Weight4, act: str = "silu") -> torch.Tensor:
    """``act(x Wgate^T) * (x Wup^T)`` for ``x [rows, k]``, as one kernel; ``act`` is "silu" or "gelu_tanh"."""
    if act not in ACT:
        raise ValueError(f"act is one of {sorted(ACT)}")
    return O.call("w4_gated", x, w.buffer, w.n, w.k, w.group, w.kind, ACT[act])


def feed_forward(x: torch.Tensor, gate_up: Weight4, down: Weight4, residual: torch.Tensor | None = None,
                 act: str = "silu") -> torch.Tensor:
    """A gated feed-forward: ``linear(gated(x, gate_up, act), down, residual=residual)``.  The values between its two kernels
    are of x's type."""
    return linear(gated(x, gate_up, act), down, None, residual)
