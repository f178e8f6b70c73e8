"""Rotary positions of queries and keys (libflexattn ``fa_rotary``), with gradients.

Pair ``i`` of the first ``rotary_dim`` elements of a head row at position ``p`` is turned by
the angle ``p * f[i]`` radians and scaled by a magnitude ``m``::

    (a, b) -> m (a cos - b sin, b cos + a sin)

The pairs are ``(x[i], x[i + rotary_dim / 2])`` (half layout) or ``(x[2 i], x[2 i + 1])``
(interleaved); elements from ``rotary_dim`` on are copied.  The frequencies are ``f[i] =
base ** (-2 i / rotary_dim)``, stretched for long contexts by one of the scalings below.  The
gradient is the transposed rotation, run by the same kernel with the angle negated, and tangents of
forward-mode differentiation turn like their primals.

The kernel holds each ``f[i]`` as a 64-bit fixed-point fraction of a turn and reduces the angle
with integer arithmetic, so it is as exact at position 2^30 as at position 1.  bf16 and fp32
tensors, any even ``rotary_dim`` up to the head dim, any strides with a contiguous last
dimension (rows that 16-byte accesses do not fit take a slower kernel).  There is no CPU path.
"""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass, field
from fractions import Fraction
from typing import Callable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib as L
from .flash_attn import _DTYPES, has_tangent, on_device

_PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")

# A scaling maps (frequencies, base, rotary_dim) to (frequencies, magnitude).
Scaling = Callable[[List[float], float, int], Tuple[List[float], float]]


def linear_scaling(factor: float) -> Scaling:
    """Positions divided by ``factor``: every frequency shrinks by it."""
    factor = _positive("factor", factor)
    return lambda f, base, rd: ([x / factor for x in f], 1.0)


def ntk_scaling(factor: float) -> Scaling:
    """The base grows to ``base * factor ** (rd / (rd - 2))``: the fastest pair keeps its frequency
    and the slowest one shrinks by ``factor``."""
    factor = _positive("factor", factor)

    def scale(f, base, rd):
        if rd <= 2:
            raise ValueError("ntk_scaling needs a rotary_dim above 2")
        b = base * factor ** (rd / (rd - 2))
        return [b ** (-2.0 * i / rd) for i in range(rd // 2)], 1.0

    return scale


def by_parts_scaling(factor: float, original_length: int, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     magnitude: Optional[float] = None) -> Scaling:
    """Pairs that turn more than ``beta_fast`` times within ``original_length`` positions keep their
    frequency, those that turn fewer than ``beta_slow`` times shrink by ``factor``, with a ramp
    between.  The magnitude defaults to ``0.1 ln(factor) + 1`` (1 for factors up to 1)."""
    factor, length = _positive("factor", factor), _positive("original_length", original_length)
    if not beta_fast > beta_slow > 0:
        raise ValueError("by_parts_scaling needs beta_fast > beta_slow > 0")
    m = float(magnitude) if magnitude is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)

    def scale(f, base, rd):
        lo, hi = (rd * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (beta_fast, beta_slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rd - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(rd // 2)]
        return [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)], m

    return scale


def _positive(name: str, x: float) -> float:
    if not (x > 0 and math.isfinite(x)):
        raise ValueError(f"{name} must be positive, got {x}")
    return float(x)


@dataclass(frozen=True, eq=False)
class RotarySpec:
    """A rotary embedding: what ``rotary_spec`` builds and the kernels take."""

    head_dim: int
    rotary_dim: int
    interleaved: bool
    frequencies: Tuple[float, ...]  # radians per position of each pair
    magnitude: float
    _dev: dict = field(default_factory=dict, repr=False, compare=False)

    def turns(self, device: torch.device) -> torch.Tensor:
        """Fractions of a turn per position, in units of 2^-64 turns, on `device` (cached)."""
        return self._on(device)[0]

    def _on(self, device: torch.device) -> tuple:
        """(turns on `device`, their address, streams that read them)."""
        on = self._dev.get(device)
        if on is None:
            t = self._dev["host"].to(device)
            on = self._dev[device] = (t, t.data_ptr(), set())
        return on

    def __post_init__(self):
        bits = [round(Fraction(f) / (2 * _PI) * (1 << 64)) % (1 << 64) for f in self.frequencies]
        self._dev["host"] = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64)

    def packed(self, device: torch.device) -> tuple:
        """The fields of an FaRotarySpec on `device`, for a call on its current stream."""
        if not self.rotary_dim:
            return (0, int(self.interleaved), 0, self.magnitude)
        t, ptr, streams = self._dev.get(device) or self._on(device)
        stream = torch._C._cuda_getCurrentRawStream(device.index)
        if stream not in streams:  # memory that a dropped spec gives back waits for every stream that read it
            t.record_stream(torch.cuda.current_stream(device))
            streams.add(stream)
        return (self.rotary_dim, int(self.interleaved), ptr, self.magnitude)


def rotary_spec(head_dim: int, *, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                scaling: Optional[Scaling] = None, frequencies: Optional[Sequence[float]] = None,
                magnitude: Optional[float] = None) -> RotarySpec:
    """Describe a rotary embedding of heads of ``head_dim`` elements, the first ``rotary_dim`` (default:
    all) of them turned.  ``scaling`` is ``linear_scaling``, ``ntk_scaling`` or ``by_parts_scaling``;
    ``frequencies`` gives the ``rotary_dim / 2`` frequencies themselves instead."""
    rd = head_dim if rotary_dim is None else int(rotary_dim)
    if head_dim <= 0 or rd < 0 or rd > head_dim or rd % 2:
        raise ValueError(f"rotary_dim must be even and within the head dim {head_dim}, got {rd}")
    m = 1.0
    if frequencies is not None:
        if scaling is not None:
            raise ValueError("give either scaling or frequencies")
        f = [float(x) for x in frequencies]
        if len(f) != rd // 2 or not all(map(math.isfinite, f)):
            raise ValueError(f"frequencies must be {rd // 2} finite numbers")
    else:
        if not base > 1:
            raise ValueError(f"base must be above 1, got {base}")
        f = [float(base) ** (-2.0 * i / rd) for i in range(rd // 2)]
        if scaling is not None and rd:
            f, m = scaling(f, float(base), rd)
    return RotarySpec(int(head_dim), rd, bool(interleaved), tuple(f), float(magnitude) if magnitude is not None else m)


Positions = Union[None, int, torch.Tensor]


def _check_qk(q, k, spec):
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q, k must be (B, H, T, D)")
    if not q.is_cuda or (k is not None and k.device != q.device):
        raise ValueError("rotary_embedding runs on CUDA tensors of one device only (there is no CPU path)")
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
        raise ValueError("q, k must share dtype bf16 or fp32")
    B, _, T, D = q.shape
    if k is not None:
        Bk, _, Tk, Dk = k.shape
        if Bk != B or Tk != T or Dk != D:
            raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)}")
    if D != spec.head_dim:
        raise ValueError(f"head dim {D}, but the rotary_spec is for {spec.head_dim}")


_PACK = L.packer(L.FaRotaryParams)
_NONE = (None, 0, (0, 0, 0, 0), (0, 0, 0, 0))


def _in_out(t: Optional[torch.Tensor]):
    """(output tensor, heads, FaTensor of the input, FaTensor of the output), and the input to keep."""
    if t is None:
        return _NONE, None
    if t.numel() == 0:
        return (torch.empty_like(t), *_NONE[1:]), None
    sb, sh, st, sd = t.stride()
    if sd != 1:
        t = t.contiguous()
        sb, sh, st, sd = t.stride()
    o = torch.empty_like(t)
    ob, oh, ot, od = o.stride()
    if od != 1:  # an overlapping or broadcast input
        o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        ob, oh, ot, od = o.stride()
    return (o, t.shape[1], (t.data_ptr(), sb, sh, st), (o.data_ptr(), ob, oh, ot)), t


def _launch(q, k, spec: RotarySpec, positions: Positions, inverse: bool):
    """Rotated copies of the ones of (q, k) that are given."""
    x = q if q is not None else k
    B, _, T, D = x.shape
    dev = x.device
    (oq, hq, fq, foq), q = _in_out(q)
    (ok, hk, fk, fok), k = _in_out(k)
    if hq or hk:
        pos, pos_stride, offset = 0, 0, 0
        if positions is not None:
            if isinstance(positions, torch.Tensor):
                pos = positions.data_ptr()
                pos_stride = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
            else:
                offset = positions
        block = _PACK.pack(_DTYPES[x.dtype], B, hq, hk, T, D, *fq, *fk, *foq, *fok, pos, pos_stride, offset, inverse,
                           *spec.packed(dev))
        with on_device(dev) as stream:
            L.packed_call("fa_rotary", block, stream)
    return oq, ok


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, spec, positions, inverse):
        ctx.set_materialize_grads(False)
        tensor = isinstance(positions, torch.Tensor)
        if tensor:  # saved, so that a change in place before the backward pass is an error
            ctx.save_for_backward(positions)
            ctx.save_for_forward(positions)
        ctx.args = (spec, None if tensor else positions, inverse)
        return _launch(q, k, spec, positions, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        spec, positions, inverse = ctx.args
        if ctx.saved_tensors:
            positions, = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None
        # linear, so its own gradient is the same operator turned back
        gq, gk = _turn(dq, dk, spec, positions, not inverse)
        return gq, gk, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        spec, positions, inverse = ctx.args
        if ctx.saved_tensors:
            positions, = ctx.saved_tensors
        return _turn(tq, tk, spec, positions, inverse)  # linear: a tangent turns like its primal


def _turn(q, k, spec: RotarySpec, positions: Positions, inverse: bool):
    """_launch, differentiable where something asks for it."""
    tangent = has_tangent(q, k)
    if tangent and q is not None and k is not None and not (has_tangent(q) and has_tangent(k)):
        # a call of its own each: either all outputs of a call have tangents or none
        return _Rotary.apply(q, None, spec, positions, inverse)[0], _Rotary.apply(None, k, spec, positions, inverse)[1]
    if tangent or (torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k))):
        return _Rotary.apply(q, k, spec, positions, inverse)
    return _launch(q, k, spec, positions, inverse)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], rotary: RotarySpec,
                     positions: Positions = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotate ``q`` (B, H, T, D) and ``k`` (B, H_kv, T, D; or None) by their positions; differentiable.

    ``positions`` is an integer tensor (T,) or (B, T) of 32-bit positions, an int (token t sits at
    ``positions + t``) or None (token t at t).  Returns rotated copies ``(q, k)`` in one launch.
    """
    _check_qk(q, k, rotary)
    if isinstance(positions, torch.Tensor):
        B, T = q.shape[0], q.shape[2]
        if positions.is_floating_point() or positions.dtype == torch.bool:
            raise ValueError("positions must be integers")
        if tuple(positions.shape) not in ((T,), (B, T), (1, T)):
            raise ValueError(f"positions must be (T,) or (B, T) = ({B}, {T}), got {tuple(positions.shape)}")
        if positions.dim() == 2 and positions.shape[0] == 1:
            positions = positions[0]
        if positions.device != q.device or positions.dtype != torch.int32 or positions.stride(-1) != 1:
            positions = positions.to(device=q.device, dtype=torch.int32).contiguous()
    elif positions is not None:
        try:
            positions = operator.index(positions)
        except TypeError:
            raise ValueError(f"positions must be a tensor, an int or None, got {type(positions).__name__}") from None
        if not -(1 << 31) <= positions <= (1 << 31) - q.shape[2]:
            raise ValueError("positions must fit 32 bits")
    if has_tangent(q, k) or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        return _turn(q, k, rotary, positions, False)
    return _launch(q, k, rotary, positions, False)
