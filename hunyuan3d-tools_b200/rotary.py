"""Rotary positions for attention queries and keys, in one launch for both.

Stands next to the linear layers: the queries and keys that a stacked projection returns side by side are turned where
they lie (``inplace``), or into new tensors.  ``unet.Attention`` calls it when its ``rotary`` is set
(``unet.use_multiview_rotary``).  The reference's UNet leaves positions to its upstream model; nothing there corresponds.
"""
from __future__ import annotations

import decimal
import math
import struct

import torch

from . import quantize_utils as _qu

# Frequencies are made in 60 digits: a 64-bit fraction of a turn has more than a double keeps.
_DIGITS = decimal.Context(prec=60)
_TWO_PI = decimal.Decimal("6.28318530717958647692528676655900576839433879875021164194988918")


class RotaryPositions:
    """Turns pairs of every head's dimensions by angles proportional to the token's position::

        (u, v) -> (u cos a - v sin a, v cos a + u sin a) * amplitude,   a = position[axis] * frequency

    ``head_dim``: dimensions of a head; the first ``rotary_dim`` of them (all by default) are turned.
    ``interleaved``: pairs are (2i, 2i + 1); otherwise (i, i + rotary_dim / 2).
    ``axes``: dimensions given to each axis of the position, e.g. ``(24, 20, 20)`` for (view, row, column); one axis by
    default.  Pair i of an axis with d dimensions has the frequency ``base ** (-2 i / d)``.
    ``scaling`` stretches the positions for contexts longer than a model was trained for:

    * ``{"kind": "linear", "factor": f}``: every frequency divided by f;
    * ``{"kind": "ntk", "factor": f}``: the base times ``f ** (d / (d - 2))``: the slowest frequency is divided by f, the
      fastest stays;
    * ``{"kind": "by_parts", "factor": f, "original_length": n, "slow": s, "fast": t}``: pairs that turn at least t times
      (default 4) in the original length stay, those below s (default 1) turns are divided by f, linear in between.

    ``amplitude`` multiplies the result (an attention temperature that some scalings ask for).

    The plan is a few numbers on the host: it works with tensors on any GPU and in captured graphs.  Angles are taken modulo
    one turn in 64-bit integers (csrc/rotary.cu), so positions of millions lose nothing.  CUDA fp16 / bf16 only; no
    gradient is recorded."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, axes=None, scaling=None, amplitude=1.0):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        axes = (rotary_dim,) if axes is None else tuple(axes)
        if head_dim <= 0 or rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > head_dim or rotary_dim > 512:
            raise RuntimeError(f"rotary_dim must be even, at most head_dim and 512, got {rotary_dim} of {head_dim}")
        if not axes or len(axes) > 255 or any(d <= 0 or d % 2 for d in axes) or sum(axes) != rotary_dim:
            raise RuntimeError(f"axes must be even numbers of dimensions that add up to {rotary_dim}, got {axes}")
        if not (base > 0 and math.isfinite(base) and math.isfinite(amplitude)):
            raise RuntimeError(f"base must be positive and amplitude finite, got {base} and {amplitude}")
        self.head_dim, self.rotary_dim, self.base, self.interleaved = head_dim, rotary_dim, float(base), bool(interleaved)
        self.axes, self.scaling, self.amplitude = axes, dict(scaling) if scaling else None, float(amplitude)
        with decimal.localcontext(_DIGITS):
            exact = [w for d in axes for w in self._axis_frequencies(d)]
            # a fraction of a turn per unit of position, in 2^-64ths (modulo a whole turn), to the nearest
            turns = [w / _TWO_PI for w in exact]
            turns = [int(((t - t.to_integral_value(decimal.ROUND_FLOOR)) * 2 ** 64).to_integral_value()) % 2 ** 64 for t in turns]
        self.frequencies = [float(w) for w in exact]
        if not all(math.isfinite(w) for w in self.frequencies):
            raise RuntimeError(f"rotary frequencies out of range: base {base}, scaling {scaling}")
        self._turns = struct.pack(f"={len(turns)}Q", *turns)
        self._axis = bytes(a for a, d in enumerate(axes) for _ in range(d // 2))
        self._plan = (self.head_dim, self.rotary_dim, len(axes), self.interleaved, self._turns, self._axis, self.amplitude)

    def _axis_frequencies(self, d):
        """Radians per unit of position of each pair of an axis, as decimals."""
        s = self.scaling or {"kind": "none"}
        kind, base = s.get("kind"), decimal.Decimal(self.base)
        allowed = {"none": set(), "linear": {"factor"}, "ntk": {"factor"},
                   "by_parts": {"factor", "original_length", "slow", "fast"}}
        if kind not in allowed:
            raise RuntimeError(f"unknown rotary scaling {kind!r} (expected 'linear', 'ntk' or 'by_parts')")
        if set(s) - {"kind"} - allowed[kind]:
            raise RuntimeError(f"rotary scaling {kind!r} does not take {sorted(set(s) - {'kind'} - allowed[kind])}")
        if kind == "none":
            factor = decimal.Decimal(1)
        else:
            factor = float(s.get("factor", 0.0))
            if not (factor > 0 and math.isfinite(factor)):
                raise RuntimeError(f"rotary scaling needs a positive factor, got {s.get('factor')}")
            factor = decimal.Decimal(factor)
        if kind == "ntk" and d > 2:
            base *= factor ** (decimal.Decimal(d) / (d - 2))
        ratio = base ** (decimal.Decimal(-2) / d)
        w = [decimal.Decimal(1)]
        while len(w) < d // 2:
            w.append(w[-1] * ratio)
        if kind == "linear":
            return [v / factor for v in w]
        if kind == "by_parts":
            length, slow, fast = s.get("original_length", 0), s.get("slow", 1.0), s.get("fast", 4.0)
            if not (length > 0 and fast > slow):
                raise RuntimeError("rotary scaling 'by_parts' needs original_length > 0 and fast > slow")
            length, slow, fast = (decimal.Decimal(float(v)) for v in (length, slow, fast))
            keep = [min(decimal.Decimal(1), max(decimal.Decimal(0), (length * v / _TWO_PI - slow) / (fast - slow))) for v in w]
            return [v * k + v / factor * (1 - k) for v, k in zip(w, keep)]
        return w

    def __call__(self, q, k=None, positions=None, offset=0, inverse=False, inplace=False):
        """q (B, N, H, D) or (N, H, D), k likewise with its own number of heads, or None; any strides with adjacent head
        dimensions (a (B, H, N, D) tensor is passed transposed).  Returns q, or (q, k): new contiguous tensors, or with
        ``inplace`` the same ones turned (side by side in whatever a projection returned: in each token, sequence or head).
        ``positions``: int64 or int32, (N) or (B, N), with several axes
        (N, axes) or (B, N, axes); ``offset`` + 0, 1, 2 ... when there are none (one axis only).  ``inverse`` turns back:
        the inverse of the turn, and its transpose where the amplitude is 1."""
        y = (_qu._NATIVE or _qu._load_native()).rotary(self._plan, q, k, positions, offset, inverse, inplace)
        if y is None:
            self._refuse(q, k, positions, offset, inplace)
        return y

    def _refuse(self, q, k, positions, offset, inplace):
        """Raises with what is wrong with a call that the native path declined."""
        if torch.jit.is_tracing():
            raise RuntimeError("rotary: the call cannot be traced: the trace would hold its output as a constant")
        tensors = [("q", q)] + ([("k", k)] if k is not None else [])
        for name, t in tensors:
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise RuntimeError(f"rotary: {name} must be a CUDA tensor (no CPU fallback)")
            if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != q.dtype:
                raise RuntimeError(f"rotary: {name} has dtype {t.dtype}, expected fp16 or bf16, the same for q and k")
            if t.dim() not in (3, 4) or t.dim() != q.dim() or t.shape[-1] != self.head_dim or t.shape[:-2] != q.shape[:-2]:
                raise RuntimeError(f"rotary: {name} must be (batch, tokens, heads, {self.head_dim}) or (tokens, heads, "
                                   f"{self.head_dim}), alike for q and k, got {tuple(t.shape)}")
            if t.device != q.device:
                raise RuntimeError(f"rotary: q is on {q.device}, {name} on {t.device}")
            if t.stride(-1) != 1 and self.head_dim > 1:
                raise RuntimeError(f"rotary: the dimensions of a head of {name} must be adjacent, their stride is {t.stride(-1)}")
            if t.requires_grad and torch.is_grad_enabled():
                raise RuntimeError(f"rotary: {name} requires a gradient, and none is recorded here: call under "
                                   "torch.no_grad() or detach it")
            if torch._C._is_fwd_grad_enabled() and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"rotary: {name} carries a forward-mode gradient, and none is recorded here: unpack it first")
        if positions is not None:
            shape, lead, n = tuple(getattr(positions, "shape", ())), tuple(q.shape[:-2]), q.shape[-3]
            ends = ((),) if len(self.axes) == 1 else ()
            ends += ((len(self.axes),),)
            if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int64, torch.int32):
                raise RuntimeError("rotary: positions must be an int64 or int32 tensor")
            if positions.device != q.device:
                raise RuntimeError(f"rotary: q is on {q.device}, positions on {positions.device}")
            if not any(shape in ((n,) + e, lead + e) for e in ends):
                raise RuntimeError(f"rotary: positions have shape {shape}, expected (tokens) or (batch, tokens)"
                                   f"{', and the axes behind' if len(self.axes) > 1 else ''} for q of {tuple(q.shape)}")
            if offset:
                raise RuntimeError("rotary: offset goes with positions that are counted, not with given ones")
        elif len(self.axes) > 1:
            raise RuntimeError("rotary: positions are needed where there are several axes")
        if inplace:
            raise RuntimeError("rotary: in place, no two elements of q and k may share memory, and where they interleave, "
                               "their outer dimensions must have the same strides")
        raise RuntimeError("rotary: a tensor subclass, a layout other than strided, or an argument of another type")

    def __repr__(self):
        return (f"RotaryPositions(head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, base={self.base:g}, "
                f"interleaved={self.interleaved}, axes={self.axes}, scaling={self.scaling}, amplitude={self.amplitude:g})")
