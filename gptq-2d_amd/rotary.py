"""Rotary positions on the GPU (csrc/rotary.hip; no reference counterpart: the reference quantizes weights only).

Pair i of a head's first ``rotated`` elements, (x[i], x[i + rotated/2]) or with ``interleaved`` (x[2 i], x[2 i + 1]), is
turned by position times f_i:

    y1 = a (x1 cos t - x2 sin t),   y2 = a (x2 cos t + x1 sin t),   t = position f_i,   f_i = base^(-2 i / rotated)

and the elements behind them are passed on.  Frequencies may be scaled for contexts longer than a model was trained on
(`Linear`, `Ntk`, `Bands`, `Yarn`; a is 1 but for the last).  Angles are formed in 64 bits: t is off by 2^-51 |t| at most, 10^-6 at
2^31, before its sine and cosine are rounded to 32 bits.  Sums are in 32 bits and rounded once.

    rotary = Rotary(128, base=500000., scaling=Bands(8., context=8192))
    q, k = rotary(q, k, positions=positions)        # one launch; differentiable in q and k

Derivatives go backward and forward, of any order, and through `torch.func`'s transforms; the rotation is linear, so each of them
is a rotation, by the angles or back.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Sequence

import torch
from torch.autograd import forward_ad

import _hip

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NO_PART = (None, 0, 0, 0, None, 0, 0, 0, 0)
# Whether a transform of torch.func is at work; a torch that does not say so is taken to be at it, which costs a node a call.
_transformed = getattr(torch._C, "_are_functorch_transforms_active", lambda: True)


def _followed(xs) -> bool:
    """Whether forward derivatives of xs are wanted."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(x).tangent is not None for x in xs)


class Linear(NamedTuple):
    """Positions divided by ``factor``: f_i / factor."""
    factor: float


class Ntk(NamedTuple):
    """A larger base: base factor^(r / (r - 2)), so that the lowest frequency is divided by ``factor`` and the highest stays."""
    factor: float


class Bands(NamedTuple):
    """By the turns that a pair makes in ``context`` tokens: fewer than ``low`` f_i / factor, more than ``high`` f_i, in between
    in proportion."""
    factor: float
    context: int
    low: float = 1.
    high: float = 4.


class Yarn(NamedTuple):
    """By the pair's number: f_i where the pair makes ``fast`` turns or more in ``context`` tokens, f_i / factor where it makes
    ``slow`` or fewer, a ramp over the numbers in between (from the whole one below to the whole one above).  The rotated part
    is multiplied by ``amplitude`` (None: 0.1 ln factor + 1, or 1 for a factor of at most 1)."""
    factor: float
    context: int
    fast: float = 32.
    slow: float = 1.
    amplitude: float | None = None


def rotary_frequencies(rotated: int, base: float = 10000., scaling: Linear | Ntk | Bands | Yarn | None = None) -> tuple[list, float]:
    """Radians a position of each of the rotated / 2 pairs, and the factor on what is rotated."""
    if isinstance(scaling, Ntk) and rotated > 2:
        base = base * scaling.factor ** (rotated / (rotated - 2))
    f = [base ** (-2 * i / rotated) for i in range(rotated // 2)]
    if scaling is None or isinstance(scaling, Ntk):
        return f, 1.
    if isinstance(scaling, Linear):
        return [x / scaling.factor for x in f], 1.
    if isinstance(scaling, Bands):
        out = []
        for x in f:
            part = (scaling.context * x / (2 * math.pi) - scaling.low) / (scaling.high - scaling.low)
            part = min(max(part, 0.), 1.)
            out.append((1 - part) * x / scaling.factor + part * x)
        return out, 1.
    if isinstance(scaling, Yarn):
        def number(turns):  # of the pair that makes that many in the context
            return rotated * math.log(scaling.context / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(number(scaling.fast)), 0), min(math.ceil(number(scaling.slow)), rotated - 1)
        out = []
        for i, x in enumerate(f):
            part = min(max((i - low) / max(high - low, 0.001), 0.), 1.)
            out.append(part * x / scaling.factor + (1 - part) * x)
        amplitude = scaling.amplitude
        if amplitude is None:
            amplitude = 0.1 * math.log(scaling.factor) + 1. if scaling.factor > 1 else 1.
        return out, amplitude
    raise ValueError(f"scaling must be Linear, Ntk, Bands, Yarn or None, got {scaling!r}")


class Rotary:
    """Rotation of heads of ``dim`` elements (2 to 1024), of which the first ``rotated`` (even; None: all) turn.  ``frequencies``: radians
    a position of each pair, in the place of those that ``base`` and ``scaling`` give."""

    def __init__(self, dim: int, *, base: float = 10000., rotated: int | None = None, interleaved: bool = False,
                 scaling: Linear | Ntk | Bands | Yarn | None = None, frequencies: Sequence[float] | None = None,
                 device: torch.device | str = "cuda"):
        rotated = dim if rotated is None else rotated
        if not 2 <= rotated <= dim <= 1024 or rotated % 2:
            raise ValueError(f"an even number of a head's {dim} elements turns, at least 2 (of at most 1024), not {rotated}")
        if frequencies is None:
            if base <= 1 or (scaling is not None and scaling.factor <= 0):
                raise ValueError("the base must be above 1 and a scaling's factor above 0")
            if isinstance(scaling, Bands) and not scaling.high > scaling.low:
                raise ValueError("high must be above low")
            if isinstance(scaling, (Bands, Yarn)) and scaling.context < 1:
                raise ValueError("the context must be at least one token")
            frequencies, amplitude = rotary_frequencies(rotated, base, scaling)
        elif scaling is not None or len(frequencies) != rotated // 2:
            raise ValueError(f"frequencies must be {rotated // 2} numbers, without a scaling")
        else:
            amplitude = 1.
        self.dim, self.rotated, self.interleaved, self.amplitude = dim, rotated, bool(interleaved), float(amplitude)
        self.turns = torch.tensor([float(f) / (2 * math.pi) for f in frequencies], dtype=torch.float64, device=device)
        _hip.require_device(self.turns)
        self.device = self.turns.device

    def __call__(self, *xs: torch.Tensor, positions: torch.Tensor):
        """One or two tensors (queries, keys) [..., heads, dim] of one type (fp32, bf16 or fp16) rotated, each with its own
        number of heads, any strides.  ``positions`` (int32 or int64) broadcasts to their leading axes, of which there are one
        or two ([tokens], [batch, tokens]); a position may be negative, and is held as it is up to 2^53, where the angle of a fast pair
        is off by more than a radian."""
        if not 1 <= len(xs) <= 2:
            raise ValueError("one or two tensors are rotated in a call")
        lead, kind, device, grad = xs[0].shape[:-2], xs[0].dtype, self.device, False
        if len(lead) not in (1, 2) or kind not in _TYPES:
            raise ValueError(f"tensors must be [tokens, heads, {self.dim}] or [batch, tokens, heads, {self.dim}], float32, bfloat16 or "
                             f"float16; got {tuple(xs[0].shape)} of {kind}")
        for x in xs:
            shape = x.shape
            if shape[-1] != self.dim or shape[:-2] != lead or shape[-2] > 0x7fff:
                raise ValueError(f"tensors must have heads of {self.dim} elements, at most 32767 of them, and the same axes before "
                                 f"these; got {[tuple(x.shape) for x in xs]}")
            if x.dtype is not kind or x.device != device:
                raise ValueError("tensors must be of one type, on the rotation's device")
            grad = grad or x.requires_grad
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != device:
            raise ValueError("positions must be int32 or int64 on the rotation's device")
        if positions.shape != lead and (positions.dim() > len(lead) or
                                        any(a != b and a != 1 for a, b in zip(positions.shape[::-1], lead[::-1]))):
            raise ValueError(f"positions {tuple(positions.shape)} do not broadcast to {tuple(lead)}")
        if (grad and torch.is_grad_enabled()) or _transformed() or _followed(xs):
            out = _turned(self, False, positions, xs)
        else:
            out = self._rotate(xs, positions, False)
        return out[0] if len(xs) == 1 else out

    def _rotate(self, xs, positions, back):
        lead = xs[0].shape[:-2]
        p = positions if positions.shape == lead else positions.expand(lead)
        batched = len(lead) == 2
        outer, inner = lead if batched else (1, lead[0])
        p_outer, p_inner = p.stride() if batched else (0, p.stride(0))
        out, parts, kept = [], [], []  # kept: copies, until the launch
        for x in xs:
            strides = x.stride()
            if strides[-1] != 1:
                x = x.contiguous()
                strides = x.stride()
                kept.append(x)
            heads = x.size(-2)
            y = torch.empty_like(x, memory_format=torch.contiguous_format)
            out.append(y)
            row = heads * self.dim  # of y, which is contiguous
            if batched:
                parts += (x.data_ptr(), *strides[:3], y.data_ptr(), inner * row, row, self.dim, heads)
            else:
                parts += (x.data_ptr(), 0, strides[0], strides[1], y.data_ptr(), 0, row, self.dim, heads)
        if len(xs) == 1:
            parts += _NO_PART
        _hip.launch("rotary", self.device, *parts, _TYPES[xs[0].dtype], outer, inner, self.dim, self.rotated, self.interleaved,
                    self.turns.data_ptr(), self.amplitude, p.data_ptr(), p.dtype is torch.int64, p_outer, p_inner, back)
        return tuple(out)


class _Rotation(torch.autograd.Function):
    """The rotation (or, `back`, its transpose).  It is linear: its derivative along a direction is the direction rotated, its
    gradient the other rotation."""

    @staticmethod
    def forward(ctx, rotary, back, positions, *xs):
        _Rotation._keep(ctx, rotary, back, positions, xs)
        return rotary._rotate(xs, positions, back)

    @staticmethod
    def _keep(ctx, rotary, back, positions, xs):
        ctx.set_materialize_grads(False)
        ctx.rotary, ctx.back, ctx.shapes = rotary, back, [x.shape for x in xs]
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)

    @staticmethod
    def backward(ctx, *grads):
        grads = [g if wanted else None for g, wanted in zip(grads, ctx.needs_input_grad[3:])]
        there, positions = [g for g in grads if g is not None], ctx.saved_tensors[0]
        turned = iter(_turned(ctx.rotary, not ctx.back, positions, there) if there else ())
        return (None, None, None, *(None if g is None else next(turned) for g in grads))

    @staticmethod
    def jvp(ctx, _rotary, _back, _positions, *tangents):
        there, positions = [t for t in tangents if t is not None], ctx.saved_tensors[0]
        turned = iter(_turned(ctx.rotary, ctx.back, positions, there))
        return tuple(there[0].new_zeros(shape) if t is None else next(turned) for t, shape in zip(tangents, ctx.shapes))


class _Mapped(_Rotation):
    """The same in the form that torch.func's transforms take, of which a call costs more."""

    @staticmethod
    def forward(rotary, back, positions, *xs):
        return rotary._rotate(xs, positions, back)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _Rotation._keep(ctx, *inputs[:3], inputs[3:])

    @staticmethod
    def vmap(info, in_dims, rotary, back, positions, *xs):
        """The mapped axis in front of a leading one, or one with the first of two."""
        n = info.batch_size
        xs = [x.expand(n, *x.shape) if at is None else x.movedim(at, 0) for x, at in zip(xs, in_dims[3:])]
        lead = xs[0].shape[1:-2]
        p = positions[None] if in_dims[2] is None else positions.movedim(in_dims[2], 0)
        p = p.reshape(p.size(0), *[1] * (len(lead) - p.dim() + 1), *p.shape[1:]).expand(n, *lead)
        if len(lead) == 2:
            p, xs = p.flatten(0, 1), [x.flatten(0, 1) for x in xs]
        out = _turned(rotary, back, p, xs)
        if len(lead) == 2:
            out = tuple(y.unflatten(0, (n, lead[0])) for y in out)
        return out, (0,) * len(out)


def _turned(rotary, back, positions, xs):
    """The rotation of xs, which whatever follows them sees."""
    if _transformed():
        return _Mapped.apply(rotary, back, positions, *xs)
    if torch.is_grad_enabled() or _followed(xs):
        return _Rotation.apply(rotary, back, positions, *xs)
    return rotary._rotate(xs, positions, back)
