"""Rotary positions: queries and keys turned pair by pair by angles that grow with their rows' positions.

Their products then depend on the difference of two positions alone: what `relative.py` learns as a bias of the scores comes with the scores
here, for any head dim and without an N x N array.  The reference takes its queries and keys as given (evoformer.py:640-651).  One kernel
(csrc/rotary.hip) turns queries and keys, and, the other way around, their gradients.
"""
from __future__ import annotations

import functools
import math
from decimal import Decimal, localcontext
from typing import Optional, Tuple, Union

import torch
from torch import nn

from . import _lib
from ._transforms import refuse_tangents


@functools.lru_cache(maxsize=4)
def _pi(digits: int) -> Decimal:
    """16 atan(1/5) - 4 atan(1/239) by their series, in a context of so many digits."""
    def atan_of_one_over(n):
        total, term, k = Decimal(0), Decimal(1) / n, 1
        while total + term / k != total:
            total += term / k if k % 4 == 1 else -term / k
            term, k = term / (n * n), k + 2
        return total

    return 16 * atan_of_one_over(5) - 4 * atan_of_one_over(239)


def rotary_turns(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0, original_length: Optional[int] = None,
                 fast: float = 32.0, slow: float = 1.0, device=None) -> torch.Tensor:
    """The fraction of a turn per position of each pair, as a 64-bit whole number: int64 [rotary_dim / 2].

    Pair i turns by base^(-2 i / rotary_dim) radians per position.  For contexts `factor` times as long as those the frequencies were trained on, `scaling` is
      "linear"  every frequency divided by the factor
      "base"    the base times factor^(rotary_dim / (rotary_dim - 2)): the slowest pair's frequency divided by the factor, the fastest's kept
      "parts"   by the turns r that a pair makes over `original_length` positions: kept from r = fast on, divided by the factor up to r = slow,
                in between blended by (r - slow) / (fast - slow)
    Formed with as many digits as the whole numbers have (in doubles the fastest pairs would be off by 2^-56 of a turn per position)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not (math.isfinite(base) and base > 0.0):
        raise ValueError(f"base must be a positive number, got {base}")
    if not (math.isfinite(factor) and factor > 0.0):
        raise ValueError(f"factor must be a positive number, got {factor}")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f'scaling must be "linear", "base" or "parts", got {scaling!r}')
    if scaling is None and factor != 1.0:
        raise ValueError("a factor needs a scaling")
    if scaling == "base" and rotary_dim == 2:
        raise ValueError('scaling "base" needs more than one pair')
    if scaling == "parts":
        if original_length is None or original_length < 1:
            raise ValueError('scaling "parts" needs original_length, the positions that the frequencies were trained on')
        if not (fast > slow and math.isfinite(slow)):
            raise ValueError(f"fast must be above slow, a number, got {fast} and {slow}")
    with localcontext() as context:
        # (64 bits behind the point, as many digits before it as bases and factors below one make, and some for what is lost on the way)
        context.prec = 50 + math.ceil(max(0.0, -math.log10(base)) + 3.0 * max(0.0, -math.log10(factor)))
        turn, factor, slow, fast = 2 * _pi(context.prec), Decimal(float(factor)), Decimal(float(slow)), Decimal(float(fast))
        log_base = Decimal(float(base)).ln()
        if scaling == "base":
            log_base += factor.ln() * rotary_dim / (rotary_dim - 2)
        ratio, turns = (log_base * -2 / rotary_dim).exp(), [1 / turn]
        while len(turns) < rotary_dim // 2:
            turns.append(turns[-1] * ratio)
        if scaling == "linear":
            turns = [x / factor for x in turns]
        elif scaling == "parts":
            kept = [min(Decimal(1), max(Decimal(0), (Decimal(float(original_length)) * x - slow) / (fast - slow))) for x in turns]
            turns = [x * (w + (1 - w) / factor) for x, w in zip(turns, kept)]
        whole = [int((x * 2 ** 64).to_integral_value()) % 2 ** 64 for x in turns]
    # (modulo a turn, which positions in whole numbers do not notice; as signed numbers of the same 64 bits)
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in whole], dtype=torch.int64, device=device)


def rotary_positions(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, turns: torch.Tensor, *, interleaved: bool = False,
                     scale: float = 1.0) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q and k with the first R = 2 len(turns) values of each head turned, dense; q alone if k is None.

    q          [N,H,D], [B,N,H,D] or [B,S,N,H,D], bf16, fp16 or fp32, any strides; k likewise, with heads of its own number
    positions  [N], or [B,N] where there is a B; whole numbers of either sign, shared by the S rows
    turns      int64 [R / 2], as rotary_turns() makes it
    interleaved  pairs are neighbours (2 i, 2 i + 1), not the halves' values (i, i + R / 2)
    scale      of the turned values

    Angles are formed in 64 bits: exact to 2^-25 of a turn for positions up to 2^38.  Gradients: q and k.  Runs on the current stream of the
    tensors' device; GPU only."""
    for name, t in (("q", q), ("k", k), ("positions", positions), ("turns", turns)):
        if not isinstance(t, torch.Tensor) and not (t is None and name == "k"):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not torch.compiler.is_compiling():
        host = _lib.host()
        out = host.rotary(q, k, positions, turns, interleaved, scale)
        if out is not None:
            return out if k is not None else out[0]
        with torch.no_grad():
            wrong = host.rotary_wrong(q, k, positions, turns, interleaved, scale)
        if wrong:
            raise ValueError(wrong)
        if not q.is_cuda:
            raise RuntimeError("rotary_positions runs on the GPU only (no CPU implementation); move its tensors to one cuda device")
        refuse_tangents("rotary_positions", q, k)
    out = torch.ops.evoattn.rotary(q, k, positions, turns, interleaved, scale, False)
    return out if k is not None else out[0]


# ---- the same as a registered operator: what the compiler's tracer and the dispatch modes see ----

@torch.library.custom_op("evoattn::rotary", mutates_args=(), device_types="cuda")
def _op_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, turns: torch.Tensor, interleaved: bool, scale: float,
               inverse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, k) turned; k empty if there is none."""
    return _lib.host().rotary_forward(q, k, positions, turns, interleaved, scale, inverse)


@_op_rotary.register_fake
def _(q, k, positions, turns, interleaved, scale, inverse):
    return q.new_empty(q.shape), q.new_empty((0,) if k is None else k.shape)


def _setup_context(ctx, inputs, output):
    q, k, positions, turns, ctx.interleaved, ctx.scale, ctx.inverse = inputs
    ctx.save_for_backward(positions, turns)
    ctx.with_k = k is not None
    ctx.dtype = q.dtype


def _backward(ctx, dq, dk):
    positions, turns = ctx.saved_tensors
    dq, dk = torch.ops.evoattn.rotary(dq.to(ctx.dtype), dk.to(ctx.dtype) if ctx.with_k else None, positions, turns, ctx.interleaved, ctx.scale, not ctx.inverse)
    return dq, dk if ctx.with_k else None, None, None, None, None, None


_op_rotary.register_autograd(_backward, setup_context=_setup_context)


class RotaryPositions(nn.Module):
    """Frequencies of a head dim, and queries and keys turned by their positions.

    rotary_dim   the part of the head that is turned, from its first value on (None: all of it)
    base, scaling, factor, original_length, fast, slow   as rotary_turns() takes them
    magnitude    what the turned values are multiplied by (None: 0.1 ln(factor) + 1 with scaling "parts" and a factor above 1, which
                 sharpens the attention over the longer context; else 1)
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False, *, scaling: Optional[str] = None,
                 factor: float = 1.0, original_length: Optional[int] = None, fast: float = 32.0, slow: float = 1.0, magnitude: Optional[float] = None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be at most the head dim {head_dim}, got {rotary_dim}")
        turns = rotary_turns(rotary_dim, base, scaling=scaling, factor=factor, original_length=original_length, fast=fast, slow=slow)
        # (whole numbers: .to(dtype) of the module leaves them as they are)
        self.register_buffer("turns", turns, persistent=False)
        self.head_dim, self.interleaved = head_dim, bool(interleaved)
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "parts" and factor > 1.0 else 1.0
        self.magnitude = float(magnitude)

    def forward(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor):
        return rotary_positions(q, k, positions, self.turns, interleaved=self.interleaved, scale=self.magnitude)

    def rotate_slots(self, y: torch.Tensor, shape, positions: torch.Tensor) -> torch.Tensor:
        """A projection's result y as its slices [..., N, slots, H, D] (`shape`) with the first two, queries and keys, turned: where they lie if that can be, so y is not to be used again."""
        slots = _lib.host().rotary_slots(y, list(shape), positions, self.turns, self.interleaved, self.magnitude)
        if slots is not None:
            return slots
        q, k, *rest = y.view(shape).unbind(-3)
        return torch.stack((*self(q, k, positions), *rest), -3)

    def plain(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor):
        """The same in plain torch operations, on any device: what the kernel is tested against.  (In 64 bits for inputs in 64 bits, else in 32.)"""
        R = 2 * self.turns.numel()
        # position times frequency modulo a turn, whole numbers that wrap around; then a signed fraction of a turn
        turn = (positions.long()[..., None] * self.turns).double() * 2.0 ** -64
        turn = turn.view(*((-1,) if positions.dim() == 1 else (positions.shape[0],) + (1,) * (q.dim() - 4) + (-1,)), 1, R // 2) * (2.0 * math.pi)

        def turned(x):
            wide = x.double() if x.dtype == torch.float64 else x.float()
            c, s = (turn.cos() * self.magnitude).to(wide.dtype), (turn.sin() * self.magnitude).to(wide.dtype)
            part = wide[..., :R]
            a, b = (part[..., 0::2], part[..., 1::2]) if self.interleaved else (part[..., :R // 2], part[..., R // 2:])
            y, z = a * c - b * s, b * c + a * s
            both = torch.stack((y, z), -1).flatten(-2) if self.interleaved else torch.cat((y, z), -1)
            return torch.cat((both, wide[..., R:]), -1).to(x.dtype)

        return turned(q) if k is None else (turned(q), turned(k))
