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
(``ValueError`` otherwise); the kernels run on the current stream of that device.  There is
no backward pass, as there is none of ``Operator.attend``: inputs that require a gradient
while gradients are being recorded raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass, field
from typing import Sequence

import torch

from . import _lib

MAX_AXES = 4
MAX_PAIRS = 128

# The host structs of include/recap_b200.h as packed bytes: filling one and passing it by address
# costs a fraction of converting thirty ctypes arguments, which a call on few tokens feels.
_ROTATE_ARGS = struct.Struct("<4Q12qQ3qq4Q10i2f")
_NORM_ARGS = struct.Struct("<4Q8q3Q6q4Q10i2f")

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITIONS = {torch.int32: 32, torch.int64: 64}
_KINDS = {"rms": 1, "layer": 2}
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
    64-bit fractions of a turn, so a far position turns as exactly as a near one.

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
        # turns for each unit of position, as 64 bits of a turn
        c.turns[:len(turns)] = [round(f * scales[a] % 1.0 * 2.0**64) % 2**64 for f, a in zip(turns, axis)]
        if any(starts):
            # added to the top 32 bits of the product, which are cut: up makes up for down
            c.phase[:len(turns)] = [math.ceil(f * starts[a] % 1.0 * 2.0**32) % 2**32 << 32 for f, a in zip(turns, axis)]
        c.axis[:len(turns)] = axis
        self._struct = c
        self._address = ctypes.addressof(c)


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


def _refuse_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("this operator has no backward pass: call it under torch.no_grad()")


def _type(dtype: torch.dtype, what: str) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be bfloat16, float16 or float32, not {dtype}")
    return code


def _param(t: torch.Tensor, n: int, device, what: str) -> int:
    """Address of a parameter vector of ``n`` contiguous values."""
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"a {what} must be {n} contiguous values")
    if t.device != device:
        raise ValueError(f"a {what} is on {t.device}, the rows on {device}")
    return t.data_ptr()


def _norm_params(norm: Norm, n: int, device) -> tuple[int, int, int]:
    """(weight address, bias address, their type) of a norm."""
    weight, bias = norm.weight, norm.bias
    if weight is None and bias is None:
        return 0, 0, 0
    _refuse_gradients(weight, bias)
    dtype = (bias if weight is None else weight).dtype
    if weight is not None and bias is not None and bias.dtype != dtype:
        raise ValueError("a norm's weight and bias differ in type")
    return (0 if weight is None else _param(weight, n, device, "norm's weight"),
            0 if bias is None else _param(bias, n, device, "norm's bias"), _type(dtype, "a norm's weight"))


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """First byte and the byte past the last of what a tensor's elements span."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two tensors share no element, as far as that can be told: their spans are apart, or
    they are boxes of one grid (equal strides, each larger than what lies within) that do not meet in
    some dim, as the parts of a packed projection or of a joint sequence."""
    if x.numel() == 0 or y.numel() == 0:
        return True
    (x0, x1), (y0, y1) = _extent(x), _extent(y)
    if x1 <= y0 or y1 <= x0:
        return True
    if x.dim() != y.dim() or x.dtype != y.dtype or (y0 - x0) % x.element_size():
        return False
    dims = [(s, t, n, m) for s, t, n, m in zip(x.stride(), y.stride(), x.shape, y.shape) if n > 1 or m > 1]
    dims.sort(reverse=True)
    away = (y0 - x0) // x.element_size()
    for i, (step, other, n, m) in enumerate(dims):
        if step != other or step == 0:
            return False
        inner_x = 1 + sum((k - 1) * s for s, _, k, _ in dims[i + 1:])
        inner_y = 1 + sum((k - 1) * s for s, _, _, k in dims[i + 1:])
        # y begins `at` steps and `rest` elements from x, with what lies within one step of either in one window
        # of a step: elements are equal only where their steps are
        for at in (away // step, away // step + 1):
            rest = away - at * step
            if max(inner_x, rest + inner_y) - min(0, rest) <= step:
                break
        else:
            return False
        if at >= n or -at >= m:
            return True
        away = rest
    return False


def _same(x: torch.Tensor, y: torch.Tensor) -> bool:
    return x.data_ptr() == y.data_ptr() and x.stride() == y.stride() and x.dtype == y.dtype


def _check_outputs(outs: Sequence[torch.Tensor], inputs: Sequence[torch.Tensor]) -> None:
    """Outputs hold each element once, may be the input of the same place in the list, and
    otherwise overlap neither an input nor one another."""
    for i, o in enumerate(outs):
        if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
            raise ValueError("an output cannot be an expanded tensor")
        for j, x in enumerate(inputs):
            if not (i == j and _same(o, x)) and not _apart(o, x):
                raise ValueError("an output overlaps an input (it may only be that input itself)")
        for p in outs[i + 1:]:
            if not _apart(o, p):
                raise ValueError("the outputs overlap")


def _run(name: str, device: torch.device, *args) -> None:
    """Call an entry point with ``device`` current, on its current stream."""
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(device):
            return _run(name, device, *args)
    rc = getattr(_lib.load(), name)(*args, _lib.raw_stream(index))
    if rc:
        _lib.check(rc, name)


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
    gives them instead: the inputs themselves (in place) or tensors that do not overlap them."""
    # (a call on few tokens takes as long as these checks: each tensor property is read once)
    shape, qs = query.shape, query.stride()
    if len(shape) != 4 or (qs[3] != 1 and shape[3] > 1):
        raise ValueError("query must be [batch, heads, sequence, dim] with dim contiguous")
    b, hq, s, d = shape
    dtype, device = query.dtype, query.device
    grad = torch.is_grad_enabled()
    if d % 8 or not 8 <= d <= 256 or hq < 1:
        raise ValueError("dim must be a multiple of 8 up to 256, and heads positive")
    hk, ks = 0, (0, 0, 0)
    if key is not None:
        shape, ks = key.shape, key.stride()
        if len(shape) != 4 or (ks[3] != 1 and shape[3] > 1):
            raise ValueError("key must be [batch, heads, sequence, dim] with dim contiguous")
        kb_, hk, s_, d_ = shape
        if kb_ != b or s_ != s or d_ != d:
            raise ValueError("query and key differ in batch, sequence or dim")
        if key.dtype != dtype or key.device != device:
            raise ValueError("query and key differ in dtype or device")
        if hk < 1:
            raise ValueError("key has no heads")
        if grad and key.requires_grad:
            _refuse_gradients(key)
    if grad and query.requires_grad:
        _refuse_gradients(query)
    in_type = _type(dtype, "query")
    out_type = in_type
    if out_dtype is not None and out_dtype != dtype:
        if out_dtype != torch.bfloat16:
            raise ValueError("out_dtype is the inputs' dtype or bfloat16")
        out_type = 0

    code = weight_type = qw = qb = kw = kb = 0
    q_eps = k_eps = 0.0
    if query_norm is not None or key_norm is not None:
        if query_norm is None or (key is not None and key_norm is None):
            raise ValueError("query and key are both normalised or neither")
        code, q_eps = query_norm.code, query_norm.eps
        across = code == _RMS_ACROSS
        if across and max(hq, hk) > (256 if d <= 64 else 128 if d <= 128 else 64):
            raise ValueError(f"too many heads of {d} dims for a norm across heads")
        qw, qb, weight_type = _norm_params(query_norm, hq * d if across else d, device)
        if key is not None:
            if key_norm.code != code:
                raise ValueError("the query's and the key's norm differ in kind")
            k_eps = key_norm.eps
            kw, kb, k_type = _norm_params(key_norm, hk * d if across else d, device)
            if kw or kb:
                if (qw or qb) and k_type != weight_type:
                    raise ValueError("the norms' weights differ in type")
                weight_type = k_type

    address = bits = at = 0
    pb = ps = pa = 0
    if rotary is not None:
        address = rotary._address
        if rotary.head_dim != d:
            raise ValueError(f"rotary positions of {rotary.head_dim} dims on heads of {d}")
        if rotary.grid is not None:
            if positions is not None:
                raise ValueError("positions are given by the rotary's grid")
            if first_token < 0 or first_token + s > rotary.sequence_tokens:
                raise ValueError(f"tokens {first_token}..{first_token + s} outside the sequence of "
                                 f"{rotary.sequence_tokens}")
        else:
            if first_token:
                raise ValueError("first_token belongs to a grid")
            if positions is None:
                raise ValueError("a rotary without a grid needs positions")
            bits = _POSITIONS.get(positions.dtype)
            if bits is None:
                raise ValueError("positions must be int32 or int64")
            shape, strides = positions.shape, positions.stride()
            if len(shape) == 2:
                shape, strides = (1, *shape), (0, *strides)
            if len(shape) != 3 or shape[0] not in (1, b) or shape[1] != s or shape[2] != len(rotary.axis_dims):
                raise ValueError("positions must be [batch or 1, sequence, axes]")
            if positions.device != device:
                raise ValueError(f"positions are on {positions.device}, the rows on {device}")
            pb, ps, pa = strides if shape[0] == b else (0, strides[1], strides[2])
            at = positions.data_ptr()
    elif positions is not None or first_token:
        raise ValueError("positions and first_token need a rotary")

    if out is None:
        if out_type == in_type:
            q_out = torch.empty_like(query)
            k_out = None if key is None else torch.empty_like(key)
        else:
            q_out = torch.empty_like(query, dtype=out_dtype)
            k_out = None if key is None else torch.empty_like(key, dtype=out_dtype)
    else:
        q_out, k_out = out
        pairs = [(q_out, query)] if key is None else [(q_out, query), (k_out, key)]
        for o, x in pairs:
            if o is None or o.shape != x.shape or o.device != device or o.stride(3) != 1 and d > 1:
                raise ValueError("out must match query and key, dim contiguous")
            if o.dtype != q_out.dtype or (out_dtype is not None and o.dtype != out_dtype):
                raise ValueError("out differs in dtype")
        if q_out.dtype != dtype and q_out.dtype != torch.bfloat16:
            raise ValueError("out has the inputs' dtype or bfloat16")
        out_type = _TYPES[q_out.dtype]
        _check_outputs([o for o, _ in pairs], [x for _, x in pairs])
    if not query.is_cuda:
        raise ValueError("rotate_qk runs on CUDA tensors only")
    if b == 0 or s == 0:
        return q_out, k_out
    qos = q_out.stride()
    k_ptr = ko_ptr = 0
    kos = (0, 0, 0)
    if key is not None:
        k_ptr, ko_ptr, kos = key.data_ptr(), k_out.data_ptr(), k_out.stride()
    _run("recap_rotate_qk", device, _ROTATE_ARGS.pack(
        query.data_ptr(), k_ptr, q_out.data_ptr(), ko_ptr, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], qos[0], qos[1],
        qos[2], kos[0], kos[1], kos[2], at, pb, ps, pa, first_token, qw, qb, kw, kb, b, hq, hk, s, d, in_type, out_type,
        code, weight_type, bits, q_eps, k_eps), address)
    return q_out, k_out


def _rows(t: torch.Tensor, shape, device, what: str) -> tuple[int, int]:
    """Element strides (batch, token) of rows ``[batch, tokens, channels]`` or ``[tokens, channels]``."""
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the rows on {device}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{what} needs contiguous channels")
    return (0, st[0]) if len(st) == 2 else (st[0], st[1])


def _modulation(t: torch.Tensor, rows, device, what: str) -> tuple[int, int, int]:
    """Address and element strides (batch, token; 0 where shared) of a modulation of rows of a shape: one
    vector ``[channels]``, or the rows' dims with size 1 where it is shared."""
    shape, st = t.shape, t.stride()
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the rows on {device}")
    if not shape or shape[-1] != rows[-1] or (st[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{what} needs {rows[-1]} contiguous channels")
    if len(shape) == 1:
        return t.data_ptr(), 0, 0
    if len(shape) == len(rows):
        token = shape[-2]
        if token == rows[-2] or token == 1:
            step = 0 if token == 1 else st[-2]
            if len(shape) == 2:
                return t.data_ptr(), 0, step
            batch = shape[0]
            if batch == 1 or batch == rows[0]:
                return t.data_ptr(), 0 if batch == 1 else st[0], step
    raise ValueError(f"{what} has shape {tuple(shape)}, which does not spread over {tuple(rows)}")


def _norm_rows(what: str, x, branch, gate, branch_norm, norm, scale, shift, x_out, h, h_dtype):
    shape = x.shape
    if len(shape) not in (2, 3):
        raise ValueError("rows are [batch, tokens, channels] or [tokens, channels]")
    c = shape[-1]
    if c % 8 or not 8 <= c <= 16384:
        raise ValueError("channels must be a multiple of 8 up to 16384")
    device = x.device
    x_type, h_type = _type(x.dtype, "rows"), _type(h_dtype, "the norm's output")
    if h_type != x_type and x_type != 2:
        raise ValueError("only float32 rows have a norm or a branch of another type")
    if torch.is_grad_enabled():
        _refuse_gradients(x, branch, gate, scale, shift)
    xs = _rows(x, shape, device, "rows")
    bs = (0, 0) if branch is None else _rows(branch, shape, device, "branch")
    mod_dtype = None
    mods = []
    for t, name in ((scale, "scale"), (shift, "shift"), (gate, "gate")):
        if t is None:
            mods.append((0, 0, 0))
            continue
        if mod_dtype is None:
            mod_dtype = t.dtype
        elif t.dtype != mod_dtype:
            raise ValueError("scale, shift and gate differ in type")
        mods.append(_modulation(t, shape, device, name))
    sc, sh, ga = mods
    mod_type = 0 if mod_dtype is None else _type(mod_dtype, "modulations")
    norm_code = branch_code = w = wb = w_type = bw = bb = b_type = 0
    eps = branch_eps = 0.0
    if norm is not None:
        norm_code, eps = norm.code, norm.eps
        if norm_code == _RMS_ACROSS:
            raise ValueError("a norm across heads belongs to rotate_qk")
        w, wb, w_type = _norm_params(norm, c, device)
    if branch_norm is not None:
        branch_code, branch_eps = branch_norm.code, branch_norm.eps
        if branch_code == _RMS_ACROSS:
            raise ValueError("a norm across heads belongs to rotate_qk")
        bw, bb, b_type = _norm_params(branch_norm, c, device)
    if x_out is not None or h is not None:
        _check_row_outputs(x, branch, (scale, shift, gate), norm, x_out, h, h_dtype)
    b_ptr = xo_ptr = h_ptr = 0
    xos = hs = (0, 0)
    if branch is not None:
        if x_out is None:
            x_out = torch.empty_like(x)
            st = x_out.stride()
            xos = (0, st[0]) if len(st) == 2 else (st[0], st[1])
        else:
            xos = _rows(x_out, shape, device, "out")
        b_ptr, xo_ptr = branch.data_ptr(), x_out.data_ptr()
    if norm is not None:
        if h is None:
            like = x if branch is None else branch
            h = torch.empty_like(like) if like.dtype == h_dtype else torch.empty_like(like, dtype=h_dtype)
            st = h.stride()
            hs = (0, st[0]) if len(st) == 2 else (st[0], st[1])
        else:
            hs = _rows(h, shape, device, "out")
        h_ptr = h.data_ptr()
    if not x.is_cuda:
        raise ValueError(f"{what} runs on CUDA tensors only")
    b, s = (1, shape[0]) if len(shape) == 2 else (shape[0], shape[1])
    if b == 0 or s == 0:
        return x_out, h
    _run("recap_norm_rows", device, _NORM_ARGS.pack(
        x.data_ptr(), b_ptr, xo_ptr, h_ptr, *xs, *bs, *xos, *hs, sc[0], sh[0], ga[0], sc[1], sc[2], sh[1], sh[2], ga[1],
        ga[2], w, wb, bw, bb, b, s, c, x_type, h_type, norm_code, branch_code, w_type, b_type, mod_type, eps,
        branch_eps))
    return x_out, h


def _check_row_outputs(x, branch, mods, norm, x_out, h, h_dtype) -> None:
    """Given outputs: of the right type, each its own input of the same kind or apart from every input."""
    outs, own = [], []
    if x_out is not None:
        if x_out.dtype != x.dtype:
            raise ValueError("the sum has the residual's dtype")
        outs.append(x_out)
        own.append(x)
    if h is not None:
        if h.dtype != h_dtype:
            raise ValueError("the norm's out differs in dtype")
        outs.append(h)
        own.append(x if branch is None else branch)
    for o in outs:
        if o.shape != x.shape or o.device != x.device:
            raise ValueError("out must have the rows' shape and device")
    _check_outputs(outs, own)
    for o, mine in zip(outs, own):
        for t in (x, branch, *mods):
            if t is not None and t is not mine and not _apart(o, t):
                raise ValueError("an output overlaps an input (it may only be that input itself)")


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
    itself or a tensor that does not overlap the inputs."""
    if out is not None and out_dtype is None:
        out_dtype = out.dtype
    return _norm_rows("modulated_norm", x, None, None, None, norm, scale, shift, None, out,
                      x.dtype if out_dtype is None else out_dtype)[1]


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
    ``out`` gives either or both: the sum may be the residual itself, the norm the branch itself."""
    if norm is None and (scale is not None or shift is not None):
        raise ValueError("scale and shift belong to a norm")
    x_out, h = out if out is not None else (None, None)
    if norm is None and h is not None:
        raise ValueError("out of a norm that is not asked for")
    return _norm_rows("gated_residual", residual, branch, gate, branch_norm, norm, scale, shift, x_out, h, branch.dtype)
