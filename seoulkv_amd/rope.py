"""Rotary positions of query and key heads.

The reference takes keys and queries that are rotated already (post-RoPE,
``api.py:13-40``); a decoder around a record cache needs the rotation itself.
``RotaryTable`` holds the angle per position of every pair of a head,
``rotary`` turns rows of heads to their positions, and
:meth:`seoulkv_amd.records.RecordCache.write` turns keys and queries on their
way into a cache.  ``norm_rotary`` norms the heads first, in the same pass;
``norm_rotary_grad`` is its gradient.

For a pair ``(a, b)`` at angle ``t = position * inverse_frequency``:

    (a, b) -> scale * (a cos t - b sin t, b cos t + a sin t)

Pair ``i`` of ``rotary_dim / 2`` is elements ``(i, i + rotary_dim / 2)`` in the
``"half"`` layout, ``(2 i, 2 i + 1)`` in ``"interleaved"``; elements past
``rotary_dim`` stay as they are.  Angles are exact to 2^-64 of a turn per
position, so far positions cost no accuracy.
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch
from torch.autograd import forward_ad

from seoulkv_amd import _hip

MAX_HEAD_DIM = 1024
LAYOUTS = ("half", "interleaved")
DEFAULT_EPS = 1e-6
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# 1 / (2 pi)
_TURN = Fraction("0.15915494309189533576888376337251436203445964574045644874766734405889679763422653509")


def scaled_frequencies(rotary_dim: int, base: float = 10000.0, scaling=None) -> tuple[list[float], float]:
    """The angle per position of every pair, and the factor on the result.

    ``scaling``: ``None``; ``("linear", f)``: positions divided by ``f``;
    ``("ntk", f)``: the base raised by ``f ** (d / (d - 2))``; ``("yarn", f,
    original)`` or ``("yarn", f, original, fast, slow)``: pairs that turn more
    than ``fast`` (32) times within ``original`` positions stay, those with
    fewer than ``slow`` (1) turns are divided by ``f``, with a ramp between,
    and the result is scaled by ``0.1 ln f + 1``."""
    kind = None if scaling is None else scaling[0]
    if kind not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {kind!r}")
    if kind is not None and len(scaling) not in ((3, 5) if kind == "yarn" else (2,)):
        raise ValueError(f"wrong number of values for scaling {kind!r}")
    factor = 1.0 if kind is None else float(scaling[1])
    if not (math.isfinite(factor) and factor > 0) or not (math.isfinite(base) and base > 1):
        raise ValueError("base must be finite and above 1, the factor finite and positive")
    n = rotary_dim
    if kind == "ntk" and n > 2:
        base *= factor ** (n / (n - 2))
    inv = [base ** (-2 * i / n) for i in range(n // 2)]
    if kind == "linear":
        inv = [x / factor for x in inv]
    if kind != "yarn":
        return inv, 1.0
    original, fast, slow = (float(x) for x in (*scaling[2:], 32.0, 1.0)[:3])
    if not (original > 0 and fast > slow > 0):
        raise ValueError("yarn needs original > 0 and fast > slow > 0")

    def pair_of(turns):  # the (fractional) pair that turns so often in `original` positions
        return n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), n - 1)
    ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n // 2)]
    return [x / factor * r + x * (1 - r) for x, r in zip(inv, ramp)], 0.1 * math.log(factor) + 1


def _turns(inv) -> torch.Tensor:
    """Angles in radians as 2^-64 turns, modulo a turn: the bits of int64."""
    turns = [round(Fraction(x) * _TURN * 2**64) % 2**64 for x in inv]
    return torch.tensor([t - 2**64 if t >> 63 else t for t in turns], dtype=torch.int64)


class RotaryTable:
    """Angles per position of a head's pairs, on one device; built once and used
    for every call (it forms exact fractions on the host and copies them).

    ``rotary_dim``: elements that turn (even).  ``inverse_frequencies``: the
    ``rotary_dim / 2`` angles per position in radians, instead of ``base`` and
    ``scaling`` (see :func:`scaled_frequencies`); ``scale``: a factor on the
    turned elements beside the scaling's own."""

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, scaling=None,
                 inverse_frequencies=None, scale: float = 1.0, layout: str = "half",
                 device="cuda"):
        if type(rotary_dim) is not int or rotary_dim % 2 or not 2 <= rotary_dim <= MAX_HEAD_DIM:
            raise ValueError(f"rotary_dim must be an even int in [2, {MAX_HEAD_DIM}]")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("a rotary table lives on a ROCm GPU device ('cuda' in PyTorch)")
        if inverse_frequencies is None:
            inv, factor = scaled_frequencies(rotary_dim, base, scaling)
        else:
            if scaling is not None:
                raise ValueError("scaling applies to base, not to given inverse frequencies")
            inv, factor = [float(x) for x in inverse_frequencies], 1.0
        if len(inv) != rotary_dim // 2 or not all(math.isfinite(x) for x in inv):
            raise ValueError(f"expected {rotary_dim // 2} finite inverse frequencies")
        self.scale = factor * float(scale)
        if not math.isfinite(self.scale):
            raise ValueError("scale must be finite")
        self.rotary_dim = rotary_dim
        self.layout = layout
        self.turns = _turns(inv).to(dev)
        self.device = self.turns.device
        # what this constructor enqueued is done before any stream uses it
        torch.cuda.current_stream(self.device).synchronize()
        self._desc = _hip.RotaryDesc(turns=self.turns.data_ptr(), pairs=rotary_dim // 2,
                                     interleaved=int(layout == "interleaved"), scale=self.scale)


def _no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:  # (a generator would take a microsecond)
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} records no gradients: call it under torch.no_grad()")
    # (forward mode goes on under no_grad; -1 outside every dual_level)
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{name} records no forward gradients: give it the primal alone")


def _written(*tensors) -> None:
    """Count a change of the caller's tensors that a kernel wrote, for graphs
    that saved them."""
    tensors = [t for t in tensors if t is not None]
    if tensors:
        torch.autograd.graph.increment_version(tensors)


def rotary(x: torch.Tensor, positions: torch.Tensor, table: RotaryTable, *,
           out: torch.Tensor | None = None, transpose: bool = False) -> torch.Tensor:
    """``x`` [n, heads, dim] or [batch, n, heads, dim] (BF16, FP16 or FP32; the
    last dimension contiguous, other strides free, e.g. the query and key heads
    of a fused projection) turned to ``positions`` (int32 or int64, [n] or
    [batch, n], any sign).  ``out``: a tensor like ``x`` to write, which may
    be ``x`` itself or other heads of its rows; else a new contiguous one.  ``transpose`` applies the
    transposed map: given the gradient with respect to the result it returns
    the gradient with respect to ``x`` (and, for scale 1, undoes the turn).
    Enqueued on PyTorch's current stream; FP32 arithmetic, rounded once."""
    shape, dtype = _checked_rows(x, positions, table)
    _no_grad("rotary", x, out)
    given, out = out, _output_like(x, shape, out)
    if x.numel() == 0:
        return out
    positions = positions.contiguous()
    _hip.call_on(x.device.index, "skv_rotary", table._desc, _hip.rows_desc(x), _hip.rows_desc(out),
                 dtype, *_sizes(shape, positions), bool(transpose))
    _written(given)
    return out


def _checked_rows(x, positions, table) -> tuple[torch.Size, int]:
    """The shape and C type of rows that are turned."""
    if not isinstance(table, RotaryTable):
        raise TypeError("table must be a RotaryTable")
    shape, dtype = x.shape, _DTYPES.get(x.dtype)
    if not x.is_cuda or dtype is None or len(shape) not in (3, 4):
        raise ValueError("expected BF16, FP16 or FP32 x [n, heads, dim] or [batch, n, heads, dim] on a GPU")
    if not table.rotary_dim <= shape[-1] <= MAX_HEAD_DIM:
        raise ValueError(f"head dimension {shape[-1]} outside [{table.rotary_dim}, {MAX_HEAD_DIM}]")
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in (shape[:-2], shape[-3:-2]):
        raise ValueError("expected int32 or int64 positions [n] or [batch, n]")
    if not x.device == positions.device == table.device:
        raise ValueError("x, positions and table must be on one device")
    return shape, dtype


def _output_like(x, shape, out):
    if out is None:
        out = x.new_empty(shape)
    elif out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out must have x's shape, type and device")
    if (x.stride(-1) != 1 or out.stride(-1) != 1) and x.numel():
        raise ValueError("the last dimension of x and out must be contiguous")
    return out


def _sizes(shape, positions):
    """Sizes and positions (contiguous) of rows as the C entry points take them."""
    batch, (n, heads, dim) = shape[0] if len(shape) == 4 else 1, shape[-3:]
    return batch, n, heads, dim, positions.data_ptr(), n if positions.dim() == 2 else 0, positions.dtype == torch.int64


def _head_norm(name, weight, eps, dtype, heads, dim, device) -> tuple[_hip.HeadNorm, torch.Tensor]:
    """The norm's description and the tensor that it points to."""
    if not isinstance(weight, torch.Tensor) or weight.dtype not in (dtype, torch.float32) \
            or weight.shape not in ((dim,), (heads, dim)) or weight.device != device:
        raise ValueError(f"expected {name} [{dim}] or [{heads}, {dim}] of {dtype} or float32 on {device}")
    eps = float(eps)
    if not 2.0**-126 <= eps < math.inf:
        raise ValueError("eps must be positive, a normal FP32 number")
    weight = weight.contiguous()
    return _hip.HeadNorm(weight.data_ptr(), _DTYPES[weight.dtype], int(weight.dim() == 2), eps), weight


def norm_rotary(x: torch.Tensor, positions: torch.Tensor, table: RotaryTable, weight: torch.Tensor, *,
                eps: float = DEFAULT_EPS, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rotary` of ``x / sqrt(mean(x ** 2) + eps) * weight``, the mean over
    each head, in one pass: query and key heads that are normed before they are
    turned.  ``weight`` [dim], or [heads, dim] for heads that differ (the query
    and key heads of a fused projection), of ``x``'s type or FP32; the other
    arguments are :func:`rotary`'s.  FP32 arithmetic, rounded once; squares are
    summed in FP32, so a head whose sum of squares passes its range gives 0."""
    shape, dtype = _checked_rows(x, positions, table)
    norm, weight = _head_norm("weight", weight, eps, x.dtype, *shape[-2:], x.device)
    _no_grad("norm_rotary", x, weight, out)
    given, out = out, _output_like(x, shape, out)
    if x.numel() == 0:
        return out
    positions = positions.contiguous()
    _hip.call_on(x.device.index, "skv_norm_rotary", table._desc, norm, _hip.rows_desc(x), _hip.rows_desc(out),
                 dtype, *_sizes(shape, positions))
    _written(given)
    return out


def norm_rotary_grad(grad: torch.Tensor, x: torch.Tensor, positions: torch.Tensor, table: RotaryTable,
                     weight: torch.Tensor, *, eps: float = DEFAULT_EPS,
                     out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients of :func:`norm_rotary` with respect to ``x`` and ``weight``
    (of their shapes and types), given the gradient ``grad`` with respect to its
    result (``x``'s shape and type, its last dimension contiguous).  ``out``: a
    tensor like ``x`` for the first, which may be ``grad`` or ``x`` itself.  The
    weight's is summed in FP32 in a fixed order, the same bits every time."""
    shape, dtype = _checked_rows(x, positions, table)
    if grad.shape != shape or grad.dtype != x.dtype or grad.device != x.device:
        raise ValueError("grad must have x's shape, type and device")
    norm, weight = _head_norm("weight", weight, eps, x.dtype, *shape[-2:], x.device)
    _no_grad("norm_rotary_grad", grad, x, weight, out)
    given, out = out, _output_like(x, shape, out)
    if x.numel() == 0:
        return out, torch.zeros_like(weight)
    if grad.stride(-1) != 1:
        grad = grad.contiguous()
    dweight = torch.empty_like(weight)
    positions = positions.contiguous()
    sizes = _sizes(shape, positions)
    size = _hip.load_library().skv_norm_grad_workspace(sizes[0] * sizes[1], *shape[-2:], weight.dim() == 2)
    work = torch.empty(size, dtype=torch.uint8, device=x.device)
    _hip.call_on(x.device.index, "skv_norm_rotary_grad", table._desc, norm, _hip.rows_desc(grad), _hip.rows_desc(x),
                 _hip.rows_desc(out), dtype, *sizes, dweight.data_ptr(), work.data_ptr(), size)
    _written(given)
    return out, dweight
