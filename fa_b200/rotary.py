"""Rotary positions: ``Rotary`` turns pairs of a head's elements by angles that
grow with the token's position.

Frequencies: pair i of ``rotary_dim`` / 2 turns by base^(-2i/rotary_dim) per
position; ``scaling`` stretches them for contexts longer than trained on:

* ``"linear"``: all divided by ``factor``;
* ``"banded"``: pairs that turn more than ``high`` times within
  ``original_length`` positions are left, those that turn less than ``low``
  times are divided by ``factor``, those between are blended linearly in the
  number of turns.

``magnitude`` multiplies the rotated elements.  The kernel keeps each
frequency as a 64-bit fraction of a turn, computed in decimal arithmetic and
rounded once, and multiplies it by the position exactly (mod 1): before its sine
is taken, the angle of position p is off by p * 2^-65 turns at most.
"""

from __future__ import annotations

import ctypes as C
import math
import threading
from decimal import Decimal, localcontext

import torch
from torch.autograd import forward_ad

from . import calls, lib

LAYOUTS = {"half": 0, "interleaved": 1}

_PI = Decimal("3.14159265358979323846264338327950288419716939937510")

_first_use = threading.RLock()  # of a Rotary on a device


def indexed(device) -> torch.device:
    """The device with its number: what is kept per device is found by it."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


def differentiated(x: torch.Tensor) -> bool:
    """Whether a derivative of either mode is being taken through x."""
    if x.requires_grad and torch.is_grad_enabled():
        return True
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


class _Turn(torch.autograd.Function):
    """The rotation for autograd: its backward pass is the other direction; it
    is linear, so a tangent is turned as the value is."""

    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        saved = [] if positions is None else [positions]
        ctx.save_for_backward(*saved)
        ctx.save_for_forward(*saved)
        ctx.rotary, ctx.inverse = rotary, inverse
        return calls.load().rotary(x, positions, None, rotary.desc(x.device, inverse))

    @staticmethod
    def jvp(ctx, tangent, *_):
        saved = ctx.saved_tensors
        return ctx.rotary(tangent.contiguous(), saved[0] if saved else None, inverse=ctx.inverse)

    @staticmethod
    def backward(ctx, grad):
        # A gradient may come expanded or transposed; the kernel reads rows of whole 16 bytes.
        saved = ctx.saved_tensors
        return ctx.rotary(grad.contiguous(), saved[0] if saved else None, inverse=not ctx.inverse), None, None, None


class Rotary:
    """``rotary(x, positions) -> y`` with y shaped like x.

    dim:        elements of a head (a multiple of 16).
    rotary_dim: the first elements that are turned (a multiple of 16; default
                all); the rest is copied.
    layout:     "half" pairs elements (i, i + rotary_dim/2), "interleaved"
                (2i, 2i + 1).
    """

    def __init__(self, dim: int = 128, *, rotary_dim: int | None = None, base: float = 10000.0,
                 layout: str = "half", scaling: str | None = None, factor: float = 1.0,
                 original_length: int = 0, low: float = 1.0, high: float = 4.0, magnitude: float = 1.0):
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if dim < 16 or dim > 1024 or dim % 16 or rotary_dim < 16 or rotary_dim > dim or rotary_dim % 16:
            raise ValueError("dim and rotary_dim must be multiples of 16, rotary_dim at most dim, dim at most 1024")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
        if scaling not in (None, "linear", "banded"):
            raise ValueError('scaling must be None, "linear" or "banded"')
        if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor) and math.isfinite(magnitude)):
            raise ValueError("base and factor must be positive and finite, magnitude finite")
        if scaling == "banded" and not (original_length > 0 and high > low):
            raise ValueError("banded scaling needs original_length > 0 and high > low")
        self.dim, self.rotary_dim, self.layout = dim, rotary_dim, layout
        self.magnitude = float(magnitude)
        self.frequencies = []  # angle per position of each pair
        self._turns = []       # the same in turns, mod 1, times 2^64
        with localcontext() as ctx:
            ctx.prec = 50
            factor, low, high, original = (Decimal(float(x)) for x in (factor, low, high, original_length))
            log_base = Decimal(float(base)).ln()
            for i in range(rotary_dim // 2):
                f = (log_base * (-2 * i) / rotary_dim).exp()
                if scaling == "linear":
                    f /= factor
                elif scaling == "banded":
                    turns = original * f / (2 * _PI)
                    keep = min(Decimal(1), max(Decimal(0), (turns - low) / (high - low)))
                    f = f * keep + f / factor * (1 - keep)
                self.frequencies.append(float(f))
                self._turns.append(int((f / (2 * _PI) * 2**64).to_integral_value()) % 2**64)
        self._tables = {}  # device -> int64 tensor of 0.64 fixed-point turns
        self._descs = {}   # (device, inverse) -> (RotaryDesc, its address, its table)

    def __getstate__(self):
        # Copies and pickles make tables of their own: a description is an address.
        return {**self.__dict__, "_tables": {}, "_descs": {}}

    def table(self, device) -> torch.Tensor:
        """The frequencies on ``device`` (made at its first use: outside a stream capture)."""
        device = indexed(device)
        if device.type != "cuda":
            raise ValueError("a Rotary works on CUDA devices")
        with _first_use:  # the copy below lets other threads run
            t = self._tables.get(device)
            if t is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first use of a Rotary on a device cannot be captured: call table(device) before")
                t = torch.tensor([x - 2**64 if x >= 2**63 else x for x in self._turns], dtype=torch.int64).to(device)
                self._tables[device] = t
        return t

    def desc(self, device, inverse: bool = False) -> int:
        """Address of the C description (b200fa_rotary_desc) for ``device``."""
        d = self._descs.get((device, inverse))
        if d is None:
            with _first_use:
                d = self._descs.get((device, inverse))
                if d is None:
                    table = self.table(device)
                    c = lib.RotaryDesc(C.sizeof(lib.RotaryDesc), self.dim, self.rotary_dim, LAYOUTS[self.layout],
                                       int(inverse), self.magnitude, table.data_ptr())
                    d = self._descs[(device, inverse)] = (c, C.addressof(c), table)
        return d[1]

    def __call__(self, x: torch.Tensor, positions: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                 inverse: bool = False) -> torch.Tensor:
        """x: [B,H,N,dim] (the attention operator's layout) or [N,H,dim] (a
        token batch), FP16, BF16 or FP32, last dimension contiguous, any
        other strides of whole 16 bytes.  positions: [N] or [B,N], int32 or
        int64 on x's device; None is 0 .. N-1.  out may be x.  ``inverse``
        turns back; with the magnitude it is the transposed map, so it carries
        a gradient of y to x: that is what autograd runs when x requires a
        gradient or carries a tangent (out must then be None)."""
        if differentiated(x):
            if out is not None:
                raise ValueError("out cannot be given when x requires a gradient or carries a tangent")
            return _Turn.apply(x, positions, self, bool(inverse))
        return calls.load().rotary(x, positions, out, self.desc(x.device, bool(inverse)))
