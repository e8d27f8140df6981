"""Attention within sequences of different lengths that lie one after the other, without padding.

The reference's rows all have N residues (evoformer.py:640-651); chains of different lengths are padded to the longest there.  Here they are packed: rows
[T, H, D] and the row at which each sequence begins.  Causal or not, query heads in groups that share a key and value head, as many queries as keys
(training, a prompt) or the last few of them (tokens that are added to a sequence).  Kernels: csrc/packed_mfma.hip, packed_dkdv.hip, packed_few.hip, packed_f32.hip.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._transforms import refuse_tangents


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, key_offsets: Optional[torch.Tensor] = None, *,
                     causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each sequence, [Tq, H, D].

    q            [Tq, H, D] bf16, fp16 or fp32, D up to 128, any strides
    k, v         [Tk, Hk, D], Hk dividing H: query heads h and h' share a key head if h // (H / Hk) == h' // (H / Hk)
    offsets      int32 or int64 [sequences + 1] on the same device, ascending from 0 to at most Tq: sequence s has the queries offsets[s] .. offsets[s + 1] - 1
    key_offsets  likewise for the keys; the queries' if not given
    causal       a sequence's queries are its last ones: the last sees every key, the one before all but the last key, and so on
    scale        positive (2^-64 to 2^64); D^-0.5 if not given

    Rows of no sequence (behind the last) and rows without a key get zeros, as do their gradients; what lies in rows that a query does not see, infinities and NaN among
    it, does not reach its result.  Sums are in fp32.  In 16 bits probabilities are rounded to the inputs' type to multiply values, and scores' gradients to multiply queries (to multiply keys:
    as two values; in fp16 both times powers of two, so that gradients of any size keep their bits); for the backward the call keeps, beside its inputs, the output, what rounding left of it, and a number for each row and head.  Gradients: q, k and v, the same bits with every call.

    Room that a cache leaves between its sequences is a sequence without queries: offsets [0, 1, 1, 2, 2], key_offsets [0, n0, room, room + n1, 2 room].  Calls whose sequences have few queries each
    (by the averages of queries times H / Hk and of keys) and others are served by different kernels: prompts and single tokens are best in calls of their own.

    The offsets' values are not looked at on the host (no synchronisation): where they are not ascending, results are not specified.  Runs on the current stream of the tensors' device; GPU only."""
    for name, t in (("q", q), ("k", k), ("v", v), ("offsets", offsets), ("key_offsets", key_offsets)):
        if not isinstance(t, torch.Tensor) and not (t is None and name == "key_offsets"):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not torch.compiler.is_compiling():
        host = _lib.host()
        out = host.packed_attention(q, k, v, offsets, key_offsets, causal, scale)
        if out is not None:
            return out
        with torch.no_grad():
            wrong = host.packed_wrong(q, k, v, offsets, key_offsets, causal, scale)
        if wrong:
            raise ValueError(wrong)
        if not q.is_cuda:
            raise RuntimeError("packed_attention runs on the GPU only (no CPU implementation); move its tensors to one cuda device")
        refuse_tangents("packed_attention", q, k, v)
    return torch.ops.evoattn.packed(q, k, v, offsets, key_offsets, causal, scale)[0]


def packed_positions(offsets: torch.Tensor, rows: int) -> torch.Tensor:
    """Each row's number within its sequence, int64 [rows], from the sequences' offsets (rows behind the last sequence go on counting from its end)."""
    at = torch.arange(rows, device=offsets.device)
    begins = offsets.long()
    return at - begins[(torch.searchsorted(begins, at, right=True) - 1).clamp_(min=0)]


# ---- the same as registered operators: what the compiler's tracer and the dispatch modes see ----

@torch.library.custom_op("evoattn::packed", mutates_args=(), device_types="cuda")
def _op_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, key_offsets: Optional[torch.Tensor], causal: bool,
               scale: Optional[float]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(o, lse, what rounding left of o)"""
    return _lib.host().packed_forward(q, k, v, offsets, key_offsets, causal, scale)


@_op_packed.register_fake
def _(q, k, v, offsets, key_offsets, causal, scale):
    low = (0, q.shape[1], q.shape[2]) if q.dtype == torch.float32 else (q.shape[0], q.shape[1], (q.shape[2] + 7) // 8 * 8)
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32), q.new_empty(low)


@torch.library.custom_op("evoattn::packed_bwd", mutates_args=(), device_types="cuda")
def _op_packed_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, key_offsets: Optional[torch.Tensor],
                   o: torch.Tensor, lse: torch.Tensor, low: torch.Tensor, causal: bool, scale: Optional[float]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.host().packed_backward(dout, q, k, v, offsets, key_offsets, o, lse, low, causal, scale)


@_op_packed_bwd.register_fake
def _(dout, q, k, v, offsets, key_offsets, o, lse, low, causal, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _setup_context(ctx, inputs, output):
    q, k, v, offsets, key_offsets, ctx.causal, ctx.scale = inputs
    o, lse, low = output
    ctx.save_for_backward(q, k, v, offsets, key_offsets, o, lse, low)
    ctx.mark_non_differentiable(lse, low)
    ctx.set_materialize_grads(False)


def _backward(ctx, dout, *_):
    if dout is None:
        return (None,) * 7
    q, k, v, offsets, key_offsets, o, lse, low = ctx.saved_tensors
    grads = torch.ops.evoattn.packed_bwd(dout.to(q.dtype), q, k, v, offsets, key_offsets, o, lse, low, ctx.causal, ctx.scale)
    return *(g if n else None for g, n in zip(grads, ctx.needs_input_grad)), None, None, None, None


_op_packed.register_autograd(_backward, setup_context=_setup_context)
