"""What stands around the attention call in a video transformer block.

Between the projections and ``Operator.attend`` the models normalise queries and keys and
turn them by rotary positions over (time, height, width); before and after the block stand
a norm with scale and shift, a gate and a residual sum.  The reference leaves these steps to
the model processors (recap/models/{cogvideox,wan,hunyuan}.py) and the models' own blocks;
here each is one pass over its rows, in the kernels of ``librecap_b200.so``:

``rotate_qk``       query/key norm and rotary positions (``AxialRotary``);
``modulated_norm``  the norm before a block: ``norm(x) (1 + scale) + shift``;
``gated_residual``  after a block: ``residual + gate * branch``, with the next block's
                    modulated norm of the sum on the way.

They compute in fp32 and round each output once.  Tensors are bf16, fp16 or fp32 on one
CUDA device, rows contiguous in their last dim, bases and strides multiples of 16 bytes
(``ValueError`` otherwise); a given output holds each element once, each of its strides larger
than what the smaller ones span.  The kernels run on the current stream of that device.  There is
no backward pass, as there is none of ``Operator.attend``, and no forward-mode derivative: inputs that
require a gradient while gradients are being recorded, and dual tensors, raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field
from typing import Sequence

import torch

from . import _lib

MAX_AXES = 4
MAX_PAIRS = 128

_KINDS = {"rms": 1, "layer": 2}  # RECAP_NORM_* of include/recap_b200.h
_RMS_ACROSS = 3


class _RotaryStruct(ctypes.Structure):
    _fields_ = [("axes", ctypes.c_int32), ("pairs", ctypes.c_int32), ("halves", ctypes.c_int32),
                ("reserved", ctypes.c_int32), ("grid", ctypes.c_int32 * MAX_AXES), ("video_offset", ctypes.c_int64),
                ("video_tokens", ctypes.c_int64), ("turns", ctypes.c_uint64 * MAX_PAIRS),
                ("phase", ctypes.c_uint64 * MAX_PAIRS), ("axis", ctypes.c_uint8 * MAX_PAIRS)]


def _per_axis(value, n: int, what: str) -> tuple[float, ...]:
    values = tuple(float(v) for v in value) if isinstance(value, (tuple, list)) else (float(value),) * n
    if len(values) != n:
        raise ValueError(f"{what} needs one value, or one for each of the {n} axes")
    if not all(math.isfinite(v) for v in values):
        raise ValueError(f"{what} must be finite")
    return values


class AxialRotary:
    """Rotary positions of one to four axes.

    ``axis_dims``: how many of the ``head_dim`` values each axis turns (even numbers, in the
    order of the axes); values past their sum are not turned.  Pair ``i`` of axis ``a`` turns
    by ``(position[a] * scale[a] + start[a]) * theta[a] ** (-2 i / axis_dims[a])``; with
    ``ladder="shared"`` the exponent runs over all axes together, ``-2 p / sum(axis_dims)``
    for the p-th pair of the head.  ``pairs``: ``"interleaved"`` pairs values 2p and 2p + 1,
    ``"halves"`` values p and p + sum(axis_dims) / 2.

    With ``grid`` (for video (frames, height, width), the last axis fastest) the positions are
    the grid coordinates of the token index, and the ``text_tokens`` before (``text_first``)
    or after the grid are not turned: the native token order of ``Layout``.  Without it the
    positions come with each call as an integer tensor, of any size: angles are kept as
    64-bit fractions of a turn and wrap without rounding.  The frequencies are doubles, as models
    form them: an angle is within 2^-32 + |position * scale| 2^-53 of a turn of the definition's (theta
    of 1 or more), that is within 2^-31 up to positions of 2^21, 2^-22 up to 2^31.

    The object holds numbers on the host only: it serves every device, stream and graph.
    """

    def __init__(self, head_dim: int, axis_dims: Sequence[int], *, theta=10000.0, grid: Sequence[int] | None = None,
                 text_tokens: int = 0, text_first: bool = False, pairs: str = "interleaved", ladder: str = "axis",
                 scale=1.0, start=0.0):
        dims = tuple(int(d) for d in axis_dims)
        n = len(dims)
        if not 1 <= n <= MAX_AXES:
            raise ValueError(f"rotary positions have 1 to {MAX_AXES} axes")
        if any(d < 2 or d % 2 for d in dims) or sum(dims) > int(head_dim):
            raise ValueError("axis_dims must be even, positive and sum to at most head_dim")
        if head_dim % 8 or not 8 <= head_dim <= 2 * MAX_PAIRS:
            raise ValueError(f"head_dim must be a multiple of 8 up to {2 * MAX_PAIRS}")
        if pairs not in ("interleaved", "halves"):
            raise ValueError(f"unknown pairs {pairs!r}")
        if ladder not in ("axis", "shared"):
            raise ValueError(f"unknown ladder {ladder!r}")
        if pairs == "halves" and sum(dims) % 8:
            raise ValueError("halves need a multiple of 8 turned values")
        thetas = _per_axis(theta, n, "theta")
        if min(thetas) <= 0:
            raise ValueError("theta must be positive")
        if ladder == "shared" and len(set(thetas)) > 1:
            raise ValueError("a shared ladder has one theta")
        scales, starts = _per_axis(scale, n, "scale"), _per_axis(start, n, "start")
        if text_tokens < 0 or (grid is None and (text_tokens or text_first)):
            raise ValueError("text_tokens belong to a grid and are not negative")
        self.head_dim, self.axis_dims, self.pairs, self.ladder = int(head_dim), dims, pairs, ladder
        self.text_tokens, self.text_first = int(text_tokens), bool(text_first)
        self.grid = None
        self.sequence_tokens = None
        c = _RotaryStruct(axes=n, pairs=sum(dims) // 2, halves=pairs == "halves")
        if grid is not None:
            self.grid = tuple(int(g) for g in grid)
            if len(self.grid) != n or min(self.grid) < 1 or math.prod(self.grid) >= 2**31:
                raise ValueError("grid needs one positive size for each axis and under 2^31 tokens")
            c.grid[:n] = self.grid
            c.video_tokens = math.prod(self.grid)
            c.video_offset = self.text_tokens if text_first else 0
            self.sequence_tokens = c.video_tokens + self.text_tokens
        total = sum(dims)
        if ladder == "shared":
            turns = [thetas[0] ** -(2.0 * p / total) / (2.0 * math.pi) for p in range(total // 2)]
        else:
            turns = [theta ** -(2.0 * i / d) / (2.0 * math.pi) for theta, d in zip(thetas, dims) for i in range(d // 2)]
        axis = [a for a, d in enumerate(dims) for _ in range(d // 2)]
        # turns for each unit of position, as 64 bits of a turn; fmod keeps the sign, and with it the bits of small negative ones
        c.turns[:len(turns)] = [round(math.fmod(f * scales[a], 1.0) * 2.0**64) % 2**64 for f, a in zip(turns, axis)]
        if any(starts):
            # added to the top 32 bits of the product, which are cut: up makes up for down
            c.phase[:len(turns)] = [math.ceil(f * starts[a] % 1.0 * 2.0**32) % 2**32 << 32 for f, a in zip(turns, axis)]
        c.axis[:len(turns)] = axis
        self._arguments = (int(head_dim), dims, thetas, self.grid, self.text_tokens, self.text_first, pairs, ladder, scales,
                           starts)
        self._struct = c
        # what a call reads of it: the struct's address, and the bounds it checks
        self._spec = (ctypes.addressof(c), self.head_dim, -1 if grid is None else self.sequence_tokens)

    @classmethod
    def _rebuild(cls, head_dim, dims, theta, grid, text_tokens, text_first, pairs, ladder, scale, start):
        return cls(head_dim, dims, theta=theta, grid=grid, text_tokens=text_tokens, text_first=text_first, pairs=pairs,
                   ladder=ladder, scale=scale, start=start)

    def __reduce__(self):
        # copies and pickles build their own struct: its address is part of the object
        return AxialRotary._rebuild, self._arguments


@dataclass(frozen=True, eq=False)
class Norm:
    """A norm over the last dim: ``"rms"`` (x / sqrt(mean x^2 + eps)) or ``"layer"`` (mean taken off
    first, population variance), times ``weight``, plus ``bias`` (layer norms only).  With
    ``across_heads`` (rms, ``rotate_qk`` only) the mean runs over all heads of a token and the
    weight has a value for each head and dim."""

    kind: str
    weight: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    eps: float = 1e-6
    across_heads: bool = False
    code: int = field(init=False, repr=False, compare=False)  # its RECAP_NORM_* value

    def __post_init__(self) -> None:
        if self.kind not in _KINDS:
            raise ValueError(f"unknown norm {self.kind!r}")
        if self.bias is not None and self.kind != "layer":
            raise ValueError("only a layer norm has a bias")
        if self.across_heads and self.kind != "rms":
            raise ValueError("across_heads is a root mean square norm")
        if not self.eps >= 0.0 or math.isinf(self.eps):
            raise ValueError("eps must be finite and not negative")
        object.__setattr__(self, "code", _RMS_ACROSS if self.across_heads else _KINDS[self.kind])


def rotate_qk(
    query: torch.Tensor,
    key: torch.Tensor | None,
    rotary: AxialRotary | None = None,
    *,
    query_norm: Norm | None = None,
    key_norm: Norm | None = None,
    positions: torch.Tensor | None = None,
    first_token: int = 0,
    out_dtype: torch.dtype | None = None,
    out: tuple[torch.Tensor, torch.Tensor | None] | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Normalise queries and keys and turn them by rotary positions, in one pass.

    ``query`` ``[batch, heads, sequence, dim]`` and ``key`` (the same with its own head count,
    or None) in native token order, dim contiguous, a multiple of 8 up to 256, other strides free.
    ``rotary`` None: norm only.  ``positions`` (a rotary without a grid): int32 or int64
    ``[batch or 1, sequence, axes]`` or ``[sequence, axes]``.  ``first_token``: the place of token 0 in
    the grid's sequence, for a shard or a chunk of it.  The norms are of one kind; a norm across heads
    takes at most 256, 128 and 64 heads of up to 64, 128 and 256 dims.

    Returns new tensors in the inputs' token order, of their dtype or of ``out_dtype`` bfloat16; ``out``
    gives them instead: the inputs themselves (in place) or tensors that do not overlap them, and in either case
    neither the norms' parameters nor the positions."""
    q_out, k_out = (None, None) if out is None else out
    if out is not None and q_out is None:
        raise ValueError("out must match query and key, dim contiguous")
    return _lib.native().rotate_qk(query, key, rotary, query_norm, key_norm, positions, first_token, out_dtype, q_out, k_out)


def modulated_norm(
    x: torch.Tensor,
    norm: Norm,
    *,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The norm before a block: ``norm(x) (1 + scale) + shift``.

    ``x`` ``[batch, tokens, channels]`` or ``[tokens, channels]``, channels contiguous, a multiple of 8 up
    to 16384.  ``scale`` and ``shift``, of one dtype: ``[channels]``, or the dims of ``x`` with size 1
    where they are shared (``[batch, 1, channels]`` of a sample, ``[batch, tokens, channels]`` of every
    token).  The result has the dtype of ``x``, or for float32 rows ``out_dtype``; ``out`` may be ``x``
    itself or a tensor that does not overlap the inputs, the norm's parameters among them."""
    return _lib.native().norm_rows("modulated_norm", x, None, None, None, norm, scale, shift, None, out, out_dtype)[1]


def gated_residual(
    residual: torch.Tensor,
    branch: torch.Tensor,
    gate: torch.Tensor | None = None,
    *,
    branch_norm: Norm | None = None,
    norm: Norm | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """After a block: the sum ``x = residual + gate * branch_norm(branch)`` and, with ``norm``, the
    next block's input ``norm(x) (1 + scale) + shift`` (of the sum before it is rounded).

    ``residual`` and ``branch`` are rows as in ``modulated_norm``; the branch has the residual's dtype, or
    is bf16 or fp16 beside a float32 residual.  ``gate``, ``scale`` and ``shift``, of one dtype, spread
    over the rows as there.  Returns (sum of the residual's dtype, norm of the branch's dtype or None);
    ``out`` gives either or both: the sum may be the residual itself, the norm the branch itself; else they overlap no
    input, the norms' parameters among them."""
    x_out, h_out = (None, None) if out is None else out
    return _lib.native().norm_rows("gated_residual", residual, branch, gate, branch_norm, norm, scale, shift, x_out, h_out,
                                   None)
