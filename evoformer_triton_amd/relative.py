"""Learned relative position bias: a number per head and bucket of the distance between two residues, as a pair bias of the attention.

The reference takes its pair bias as given (evoformer.py:640-651); a model forms part of it from the residues' numbers.  Here the
bias [B,1,H,Nq,Nk] comes from one kernel (csrc/relative_bias.hip), added to a pair bias on the way if there is one, and the table's
gradient from one more and a sum, in a fixed order.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib
from ._transforms import refuse_tangents

_MAX_REACH = 4096


def relative_buckets(max_distance: int, num_buckets: Optional[int] = None, device=None) -> torch.Tensor:
    """The bucket of each distance from -max_distance to max_distance (query's position less key's), uint8 [2 * max_distance + 1];
    distances beyond are clipped.

    Without `num_buckets` every distance has a bucket of its own, 0 for -max_distance.  With it the lower half of the buckets is for distances from 0 on
    and the upper half for negative ones (bucket num_buckets // 2 + i where the same distance the other way has bucket i); the first
    half of either, num_buckets // 4, are one distance each, the others cover ever wider ranges: with near = num_buckets // 4 and far
    = num_buckets // 2 - near, bucket near + i begins at the first distance d with (d / near)^far >= (max_distance / near)^i."""
    if max_distance < 0 or max_distance > _MAX_REACH:
        raise ValueError(f"max_distance must be 0 to {_MAX_REACH}, got {max_distance}")
    if num_buckets is None:
        if max_distance > 127:
            raise ValueError("more than 127 distances either way need num_buckets: a bucket's number is a byte")
        return torch.arange(2 * max_distance + 1, dtype=torch.uint8, device=device)
    if num_buckets < 4 or num_buckets > 256 or num_buckets % 2:
        raise ValueError(f"num_buckets must be even and 4 to 256, got {num_buckets}")
    half, near = num_buckets // 2, num_buckets // 4
    far = half - near
    if max_distance <= near:
        raise ValueError(f"max_distance must be beyond the {near} distances that have buckets of their own, got {max_distance}")
    # (in whole numbers: a border that is a power falls where it belongs)
    begins = [max_distance ** i * near ** far for i in range(1, far)]
    of = [d if d < near else near + sum(d ** far * near ** i >= b for i, b in enumerate(begins, 1)) for d in range(max_distance + 1)]
    return torch.tensor([half + i for i in of[:0:-1]] + of, dtype=torch.uint8, device=device)


def _wrong(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype):
    for name, t in (("table", table), ("buckets", buckets), ("positions", positions), ("key_positions", key_positions), ("chains", chains),
                    ("key_chains", key_chains), ("pair_bias", pair_bias)):
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    with torch.no_grad():
        return _lib.host().relative_bias_wrong(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype)


def relative_position_bias(table: torch.Tensor, buckets: torch.Tensor, positions: torch.Tensor, key_positions: Optional[torch.Tensor] = None, *,
                           chains: Optional[torch.Tensor] = None, key_chains: Optional[torch.Tensor] = None,
                           pair_bias: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out[b,0,h,i,j] = table[bucket, h] (+ pair_bias[b,0,h,i,j]), [B,1,H,Nq,Nk], rounded once.

    table          [rows, H] bf16, fp16 or fp32, up to 256 rows: the learned numbers
    buckets        uint8 [2 R + 1], R up to 4096: the bucket of each clipped distance (`relative_buckets`); one of `rows` or more
                   stands for no bias
    positions      [B, Nq] or [Nq], whole numbers (any: residue numbers with gaps, of several chains); key_positions [B, Nk] or
                   [Nk], the queries' if not given.  One row of queries against many keys is a call like any other
    chains         like positions, and key_chains (the queries' if neither keys' positions nor chains are given): pairs of different
                   chains take the table's last row
    pair_bias      [B or 1, 1, H, Nq, Nk], any strides: added
    dtype          of the result: pair_bias's (which must have it), else the table's, if not given

    Gradients: table (a sum in fp32 in a fixed order) and pair_bias.  Runs on the current stream of the tensors' device; GPU only."""
    if key_positions is None:
        key_positions = positions
        if key_chains is None:
            key_chains = chains
    if not torch.compiler.is_compiling():
        host = _lib.host()
        try:
            out = host.relative_bias(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype)
        except TypeError:      # not tensors: worded below
            out = None
        if out is not None:
            return out
        wrong = _wrong(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype)
        if wrong:
            raise ValueError(wrong)
        if not table.is_cuda:
            raise RuntimeError("relative_position_bias runs on the GPU only (no CPU implementation); move its tensors to one cuda device")
        refuse_tangents("relative_position_bias", table, pair_bias)
    return torch.ops.evoattn.relative_bias(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype)


# ---- the same as registered operators: what the compiler's tracer and the dispatch modes see ----

@torch.library.custom_op("evoattn::relative_bias", mutates_args=(), device_types="cuda")
def _op_relative_bias(table: torch.Tensor, buckets: torch.Tensor, positions: torch.Tensor, key_positions: torch.Tensor, chains: Optional[torch.Tensor],
                      key_chains: Optional[torch.Tensor], pair_bias: Optional[torch.Tensor], dtype: Optional[torch.dtype]) -> torch.Tensor:
    return _lib.host().relative_bias_forward(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype)


def _out_dtype(table, pair_bias, dtype):
    return dtype or (table if pair_bias is None else pair_bias).dtype


@_op_relative_bias.register_fake
def _(table, buckets, positions, key_positions, chains, key_chains, pair_bias, dtype):
    sizes = [t.shape[0] for t in (positions, key_positions, chains, key_chains) if t is not None and t.dim() == 2]
    sizes += [] if pair_bias is None else [pair_bias.shape[0]]
    B = next((n for n in sizes if n != 1), 1)
    return table.new_empty((B, 1, table.shape[1], positions.shape[-1], key_positions.shape[-1]), dtype=_out_dtype(table, pair_bias, dtype))


@torch.library.custom_op("evoattn::relative_bias_bwd", mutates_args=(), device_types="cuda")
def _op_relative_bias_bwd(dout: torch.Tensor, table: torch.Tensor, buckets: torch.Tensor, positions: torch.Tensor, key_positions: torch.Tensor,
                          chains: Optional[torch.Tensor], key_chains: Optional[torch.Tensor], pair_bias: Optional[torch.Tensor], need_table: bool,
                          need_pair: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dtable, dpair_bias); one that was not asked for is empty."""
    return _lib.host().relative_bias_backward(dout, table, buckets, positions, key_positions, chains, key_chains, pair_bias, need_table, need_pair)


@_op_relative_bias_bwd.register_fake
def _(dout, table, buckets, positions, key_positions, chains, key_chains, pair_bias, need_table, need_pair):
    return table.new_empty(table.shape) if need_table else dout.new_empty((0,)), pair_bias.new_empty(pair_bias.shape) if need_pair else dout.new_empty((0,))


def _setup_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.dtype = output.dtype


def _backward(ctx, dout):
    table, buckets, positions, key_positions, chains, key_chains, pair_bias = ctx.saved_tensors
    need_table, need_pair = ctx.needs_input_grad[0], pair_bias is not None and ctx.needs_input_grad[6]
    dtable, dpair = torch.ops.evoattn.relative_bias_bwd(dout.to(ctx.dtype), table, buckets, positions, key_positions, chains, key_chains, pair_bias,
                                                        need_table, need_pair)
    return dtable if need_table else None, None, None, None, None, None, dpair if need_pair else None, None


_op_relative_bias.register_autograd(_backward, setup_context=_setup_context)


class RelativePositionBias(nn.Module):
    """A table of one number per head and bucket, and the bias [B,1,H,Nq,Nk] of residues by their positions.

    max_distance, num_buckets   as relative_buckets() takes them
    other_chain                 one row more, for pairs of different chains (`chains` is then given with each call)
    """

    def __init__(self, no_heads: int, max_distance: int = 32, num_buckets: Optional[int] = None, other_chain: bool = False):
        super().__init__()
        buckets = relative_buckets(max_distance, num_buckets)
        rows = int(buckets.max()) + 1 + bool(other_chain)
        if rows > 256:
            raise ValueError("at most 256 buckets, the one for other chains included")
        self.register_buffer("buckets", buckets, persistent=False)
        self.other_chain = bool(other_chain)
        self.weight = nn.Parameter(torch.zeros(rows, no_heads))

    def forward(self, positions: torch.Tensor, key_positions: Optional[torch.Tensor] = None, *, chains: Optional[torch.Tensor] = None,
                key_chains: Optional[torch.Tensor] = None, pair_bias: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None):
        if chains is not None and not self.other_chain:
            raise ValueError("chains need a table with a row for pairs of different chains (other_chain=True)")
        return relative_position_bias(self.weight, self.buckets, positions, key_positions, chains=chains, key_chains=key_chains, pair_bias=pair_bias, dtype=dtype)

    def plain(self, positions: torch.Tensor, *, chains: Optional[torch.Tensor] = None, pair_bias: Optional[torch.Tensor] = None,
              dtype: Optional[torch.dtype] = None):
        """The bias of residues among themselves in plain torch operations, on any device: what the kernel is tested against."""
        at, reach = (positions if positions.dim() == 2 else positions[None]).long(), self.buckets.numel() // 2
        q, k = at[:, :, None], at[:, None, :]
        d = q - k
        # (a difference that int64 does not hold is far; its sign is the query's)
        far = ((q ^ k) & (q ^ d)) < 0
        bucket = self.buckets.long()[torch.where(far, torch.where(q < 0, -reach, reach), d.clamp(-reach, reach)) + reach]
        if chains is not None:
            c = (chains if chains.dim() == 2 else chains[None]).long()
            bucket = torch.where(c[:, :, None] == c[:, None, :], bucket, self.weight.shape[0] - 1)
        out = self.weight.float()[bucket].permute(0, 3, 1, 2).unsqueeze(1)
        if pair_bias is not None:
            out = out + pair_bias.float()
        return out.to(dtype or (self.weight if pair_bias is None else pair_bias).dtype)
