"""The attention block either side of the kernels: projections in, gate and projection out.

The reference stops at the attention itself and returns O ungated (evoformer.py:735); in an
Evoformer block the steps around it are a LayerNorm, the Q/K/V and gate projections, the
pair-bias projection from the pair representation, sigmoid(gate) * O and the output
projection.  This module does those with this package's LayerNorm and Linear kernels (csrc/linear.hip;
fp32, large products and sizes that it does not take through the library's GEMMs, the weight
gradients summed over slices of the rows, which as single GEMMs would leave most of the chip
idle), and lays the results out so that the attention kernels read them as they fall:

  * in 16-bit on the GPU Q, K, V and the gate come out of one GEMM with the four weights stacked,
    as [B,S,N,4*H*D]; viewed as [B,S,N,4,H,D] each is a slot that the kernels take by its strides
    (per-head rows, a token's 4*H*D elements from the next token's): no permute, no copy, and the
    gradients come back in the same arrangement, so the projection's backward is one GEMM for the
    input and one for the weights (`evoformer._SlotAttention`);
  * elsewhere (fp32, under a tracer, head dims that need padding) they come out of the four
    Linear layers as [B,S,N,H*D], which viewed as [B,S,N,H,D] is the per-head ("ds4sci") layout;
  * the gate is applied in the forward kernel's epilogue and its gradient comes from the
    backward (`evoformer_attention(..., gate=g)`), so sigmoid(g) * O never makes a round trip
    of its own;
  * the gated output [B,S,N,H,D] viewed as [B,S,N,H*D] is the input of the output projection;
  * the pair bias Linear(LayerNorm(z)) comes from one kernel as [B,1,H,N,N] in the dtype of Q, so the attention kernels
    take it from 16-bit tiles; for shapes that kernel does not take, from the separate steps and a permute;
  * a learned relative position bias (`relative.py`) is added to the pair bias, or stands for it, if the block has one;
  * queries and keys are turned by their positions (`rotary.py`), in place in the GEMM's result, if the block is made so;
  * sequences of different lengths can come one after the other instead of padded to the longest (`packed.py`,
    `GatedAttentionBlock.packed`);
  * the projections run in 8 bits (`fp8.py`) if the block is made so.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import nn

from . import _lib
from . import evoformer as _evoformer
from .evoformer import _DTYPES, _HEAD_DIMS, _SlotAttention, _alloc_bytes, _on_device, _ptr, _stream, evoformer_attention
from .fp8 import Fp8Weight, fp8_linear
from .packed import packed_attention, packed_positions
from .relative import RelativePositionBias
from .rotary import RotaryPositions


def _row_slices(rows: int, n_out: int, n_in: int) -> int:
    """Slices of the rows a weight gradient is summed over.  The gradient of an [n_out, n_in] weight is
    one small matrix summed over all rows of the activations: as one library GEMM it has a handful of
    output tiles (four of 128 x 128 for 256 x 256) for a chip of 256 CUs.  Summed per slice of the rows
    as a batched GEMM and added up afterwards it fills the chip (32 768 rows, 256 x 256, bf16: 113 us as
    one GEMM, 33 us in 8 to 128 slices; 131 072 rows: 325 against 38 us in 128)."""
    tiles = -(-n_out // 128) * -(-n_in // 128)
    g = 1
    while g * tiles < 512 and rows % (2 * g) == 0 and rows // (2 * g) >= 256:
        g *= 2
    return g


def _weight_grad(dy2: torch.Tensor, x2: torch.Tensor) -> torch.Tensor:
    """dy2^T x2 ([rows, n_out], [rows, n_in] -> [n_out, n_in]) summed over slices of the rows."""
    rows, g = dy2.shape[0], _row_slices(dy2.shape[0], dy2.shape[1], x2.shape[1])
    if g == 1:
        return dy2.t() @ x2
    part = torch.bmm(dy2.view(g, rows // g, -1).transpose(1, 2), x2.view(g, rows // g, -1))
    return part.sum(0)          # (torch adds 16-bit inputs in fp32 and rounds the sum once)


def _bias_grad(dy2: torch.Tensor) -> torch.Tensor:
    """Column sums of dy2 [rows, n_out] (rows may lie further apart than n_out: some columns of a wider array):
    through the library's kernel (one pass at the rate of HBM, fp32 sums in a
    fixed order) where it takes the shape, else torch's."""
    rows, cols = dy2.shape
    if rows and not torch.compiler.is_compiling() and dy2.is_cuda and dy2.dtype in _DTYPES and dy2.stride(1) == 1 \
            and dy2.stride(0) >= cols and dy2.stride(0) % 8 == 0 and dy2.data_ptr() % 16 == 0:
        lib = _lib.load()
        nbytes = lib.evoattn_colsum_workspace_bytes(rows, cols, _DTYPES[dy2.dtype])
        if nbytes:
            with _on_device(dy2.device):
                out = torch.empty((cols,), device=dy2.device, dtype=dy2.dtype)
                ws = _alloc_bytes(nbytes, dy2.device)
                _lib.check(lib.evoattn_colsum(_ptr(dy2), dy2.stride(0), _ptr(out), _ptr(ws), ws.numel(), rows, cols, _DTYPES[dy2.dtype],
                                              _stream(dy2.device)), "evoattn_colsum")
            return out
    return dy2.sum(0)


class _Projections(torch.autograd.Function):
    """Several Linear layers of one input (Q, K, V and the gate of the normalised representation):
    forward(x, w0, b0, w1, b1, ...) -> (x w0^T + b0, x w1^T + b1, ...).  The gradient of the input
    accumulates inside the GEMMs (`addmm_`) instead of as additions of full-size tensors after
    them; the weight gradients are summed over slices of the rows (see _row_slices)."""

    @staticmethod
    def forward(ctx, x, *params):
        ws, bs = params[0::2], params[1::2]
        ctx.save_for_backward(x, *ws)
        ctx.has_bias = tuple(b is not None for b in bs)
        return tuple(torch.nn.functional.linear(x, w, b) for w, b in zip(ws, bs))

    @staticmethod
    def backward(ctx, *dys):
        x, *ws = ctx.saved_tensors
        x2 = x.reshape(-1, x.shape[-1])
        dx, grads = None, []
        for i, (w, dy) in enumerate(zip(ws, dys)):
            dy2 = dy.reshape(-1, dy.shape[-1])
            if ctx.needs_input_grad[0]:
                dx = dy2 @ w if dx is None else dx.addmm_(dy2, w)
            grads.append(_weight_grad(dy2, x2) if ctx.needs_input_grad[1 + 2 * i] else None)
            grads.append(_bias_grad(dy2) if ctx.has_bias[i] and ctx.needs_input_grad[2 + 2 * i] else None)
        return (None if dx is None else dx.view(x.shape), *grads)


class _Linear(torch.autograd.Function):
    """x W^T + b with the weight gradient summed over slices of the rows (see _row_slices); forward and
    input gradient are the library's GEMMs as torch.nn.functional.linear calls them.  What the compiler's tracer sees, and
    what a call reaches that the C++ node does not stand for (under vmap, func.grad and the like, which refuse it)."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        # (as a matrix: for an input of more dimensions whose rows lie apart torch multiplies and then adds the
        # bias in a pass of its own)
        y = torch.nn.functional.linear(x.reshape(-1, x.shape[-1]), weight, bias)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dy2, x2 = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = (dy2 @ weight).view(x.shape)
        if ctx.needs_input_grad[1]:
            dw = _weight_grad(dy2, x2)
        if ctx.has_bias and ctx.needs_input_grad[2]:
            db = _bias_grad(dy2)
        return dx, dw, db


def _recast(layer: nn.Linear, x: torch.Tensor) -> bool:
    """Whether autocast takes the input or the layer's weight to another type: the layer is torch's then, whose backward knows of it."""
    if not torch.is_autocast_enabled("cuda") or not x.is_cuda:
        return False
    to = torch.get_autocast_dtype("cuda")
    return x.dtype != to or layer.weight.dtype != to


def _linear(layer: nn.Linear, x: torch.Tensor, dx_place: Optional[torch.Tensor] = None) -> torch.Tensor:
    if _recast(layer, x):
        return layer(x)
    # (the same in C++)
    y = None if torch.compiler.is_compiling() else _lib.host().linear(x, layer.weight, layer.bias, dx_place)
    return _Linear.apply(x, layer.weight, layer.bias) if y is None else y


class _StackedProjection:
    """The Q, K, V (and gate) projections of one input as a single GEMM with their weights stacked:
    apply(x, gate_bias, w0, w1, ...) -> x [w0; w1; ...]^T (+ gate_bias on the last layer's columns), shaped
    [..., n * out].  The input is read once instead of n times, its gradient is one GEMM over the whole
    gradient of the result (no additions of n partial gradients), and so is the weight gradient (summed over
    slices of the rows, see _row_slices), cut into the layers' pieces afterwards."""

    @staticmethod
    def apply(x, gate_bias, *weights):
        y = _lib.host().stacked_projection(x, gate_bias, weights)
        if y is not None:
            return y
        w = torch.cat(weights, 0)
        if gate_bias is not None:
            gate_bias = torch.cat([gate_bias.new_zeros(w.shape[0] - gate_bias.shape[0]), gate_bias])
        return _Linear.apply(x, w, gate_bias)


class _LayerNorm:
    """LayerNorm over the last dimension through the library's kernels (evoattn_layernorm_fwd / _bwd): x and y
    cross HBM once in the forward, x, dy and dx once in the backward; the gradients of weight and bias are summed
    in a fixed order.  None where those kernels do not take the call."""

    @staticmethod
    def apply(x, weight, bias, eps):
        return _lib.host().layer_norm(x, weight, bias, eps)


def _layer_norm(layer: nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    # under the tracer, no rows, mixed dtypes, or a row length the kernels do not take: the framework's
    y = None if torch.compiler.is_compiling() else _LayerNorm.apply(x, layer.weight, layer.bias, layer.eps)
    return layer(x) if y is None else y


def _pair_bias(norm: nn.LayerNorm, layer: nn.Linear, z: torch.Tensor) -> Optional[torch.Tensor]:
    """Linear(LayerNorm(z)) permuted to [B,1,H,N,N] in one pass over z (csrc/pair_bias.hip), rounded where the separate steps
    round.  None where that kernel does not take the call."""
    if torch.compiler.is_compiling() or layer.bias is not None or z.dim() != 4:
        return None
    return _lib.host().pair_bias(z, norm.weight, norm.bias, norm.eps, layer.weight)


_NO_PARAMETERS = {"weight": None, "bias": None}
_UNBIASED = ("linear_q", "linear_k", "linear_v", "linear_z")


class Fp8BlockWeights(NamedTuple):
    """A block's projections in 8 bits, for inference: `GatedAttentionBlock.fp8_weights`."""
    projections: Fp8Weight               # Q, K, V (and the gate), stacked
    bias: Optional[torch.Tensor]         # theirs, zeros for a layer without one
    output: Fp8Weight


class GatedAttentionBlock(nn.Module):
    """Row-wise gated self-attention with pair bias (the MSA row attention of an Evoformer
    block).

    m    [B,S,N,c_m]   the representation attended over (S rows of N residues)
    z    [B,N,N,c_z]   optional pair representation; its projection to H channels is the bias
    mask [B,S,N]       optional, 1 = keep, 0 = drop the key (bool or float)
    positions [B,N] or [N], chains alike (optional): the residues' numbers and chains, for a block with a relative position bias; the positions for one with rotary positions too
    weights            Fp8BlockWeights of `fp8_weights()`, for inference with a block in 8 bits; else the weights are rounded with each call
    ->   [B,S,N,c_m]

    fp8                       the projections in 8 bits (fp8_linear): operands rounded to e4m3 with a scale for each block of 128, forward and backward
    relative_distance, relative_buckets, other_chain   a learned relative position bias, as RelativePositionBias takes them
    rotary                    a RotaryPositions of head dim c_hidden: what queries and keys are turned by
    """

    fp8 = False

    def __init__(self, c_m: int, c_hidden: int, no_heads: int, c_z: Optional[int] = None, gating: bool = True,
                 inf: float = 1e9, fp8: bool = False, relative_distance: Optional[int] = None, relative_buckets: Optional[int] = None,
                 other_chain: bool = False, rotary: Optional[RotaryPositions] = None):
        super().__init__()
        if fp8:
            self.fp8 = True
        self.c_hidden, self.no_heads, self.inf = c_hidden, no_heads, inf
        hd = c_hidden * no_heads
        self.layer_norm_m = nn.LayerNorm(c_m)
        self.linear_q = nn.Linear(c_m, hd, bias=False)
        self.linear_k = nn.Linear(c_m, hd, bias=False)
        self.linear_v = nn.Linear(c_m, hd, bias=False)
        self.linear_g = nn.Linear(c_m, hd) if gating else None
        self.linear_o = nn.Linear(hd, c_m)
        if c_z is not None:
            self.layer_norm_z = nn.LayerNorm(c_z)
            self.linear_z = nn.Linear(c_z, no_heads, bias=False)
        else:
            self.layer_norm_z = self.linear_z = None
        if relative_distance is not None:
            self.relative = RelativePositionBias(no_heads, relative_distance, relative_buckets, other_chain)
        elif relative_buckets is not None or other_chain:
            raise ValueError("relative_buckets and other_chain need relative_distance")
        else:
            self.relative = None
        if rotary is not None and rotary.head_dim != c_hidden:
            raise ValueError(f"rotary positions of head dim {rotary.head_dim} in a block of head dim {c_hidden}")
        self.rotary = rotary

    def _stacked_weights(self):
        layers = [self.linear_q, self.linear_k, self.linear_v] + ([self.linear_g] if self.linear_g is not None else [])
        weight, bias = torch.cat([l.weight for l in layers], 0), None
        if any(l.bias is not None for l in layers):     # (Q, K and V have none as they are made, but a caller's layers may)
            bias = torch.cat([l.weight.new_zeros(l.weight.shape[0]) if l.bias is None else l.bias for l in layers])
        return weight, bias

    @torch.no_grad()
    def fp8_weights(self) -> Fp8BlockWeights:
        """The projections rounded once, to be given to inference calls (and made anew after the parameters have changed)."""
        weight, bias = self._stacked_weights()
        return Fp8BlockWeights(Fp8Weight.of(weight), bias, Fp8Weight.of(self.linear_o.weight))

    def operands(self, m: torch.Tensor, z: Optional[torch.Tensor], mask: Optional[torch.Tensor], plain: bool = False,
                 positions: Optional[torch.Tensor] = None, chains: Optional[torch.Tensor] = None, weights: Optional[Fp8BlockWeights] = None):
        """Q, K, V, gate [B,S,N,H,D] (views of the projections), additive mask [B,S,1,1,N],
        bias [B,1,H,N,N].  `plain`: the framework's LayerNorm and Linear throughout (what
        `forward_eager` uses), else the library's LayerNorm kernels and the projections with
        their weight gradients summed over slices of the rows."""
        norm = (lambda layer, t: layer(t)) if plain or not m.is_cuda else _layer_norm
        lin = (lambda layer, t: layer(t)) if plain else _linear
        q, k, v, g = self._heads(norm(self.layer_norm_m, m), positions, plain, weights)
        bias, add_mask = self._bias_and_mask(z, mask, q.dtype, m.shape[:3], norm, lin, positions, chains, plain)
        return q, k, v, g, add_mask, bias

    def _heads(self, x, positions, plain, weights):
        """Q, K (turned by their positions), V and the gate of a normalised input [..., c_m], [..., H, D] each."""
        H, D = self.no_heads, self.c_hidden
        layers = [self.linear_q, self.linear_k, self.linear_v] + ([self.linear_g] if self.linear_g is not None else [])
        if plain or (not self.fp8 and any(_recast(layer, x) for layer in layers)):
            outs = [layer(x) for layer in layers]
        elif self.fp8:
            outs = self._project(x, weights).unflatten(-1, (len(layers), H * D)).unbind(-2)
        else:
            outs = _Projections.apply(x, *(t for layer in layers for t in (layer.weight, layer.bias)))
        q, k, v, *g = (t.view(*x.shape[:-1], H, D) for t in outs)
        rotary = self._modules.get("rotary")
        if rotary is not None:
            q, k = (rotary.plain if plain else rotary)(q, k, positions)
        return q, k, v, g[0] if g else None

    def _slots(self, x, positions, weights):
        """The same, [..., slots, H, D], from one GEMM (see `_slots_ok`)."""
        gated = self.linear_g is not None
        if self.fp8:
            y = self._project(x, weights)
        else:
            projections = [self.linear_q.weight, self.linear_k.weight, self.linear_v.weight] + ([self.linear_g.weight] if gated else [])
            y = _StackedProjection.apply(x, self.linear_g.bias if gated else None, *projections)
        shape, rotary = (*x.shape[:-1], 4 if gated else 3, self.no_heads, self.c_hidden), self._modules.get("rotary")
        return y.view(shape) if rotary is None else rotary.rotate_slots(y, shape, positions)

    def _project(self, x: torch.Tensor, weights: Optional[Fp8BlockWeights]) -> torch.Tensor:
        """Q, K, V (and the gate) side by side, in 8 bits."""
        if weights is not None:
            return fp8_linear(x, weights.projections, weights.bias)
        return fp8_linear(x, *self._stacked_weights())

    def _output(self, o: torch.Tensor, weights: Optional[Fp8BlockWeights], place: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.fp8:
            return fp8_linear(o, self.linear_o.weight if weights is None else weights.output, self.linear_o.bias)
        return _linear(self.linear_o, o, place)

    def _bias_and_mask(self, z, mask, dtype, shape, norm, lin, positions=None, chains=None, plain=False):
        B, S, N = shape
        bias = add_mask = None
        if z is not None and self.linear_z is not None and norm is _layer_norm and lin is _linear and z.dtype == dtype:
            bias = _pair_bias(self.layer_norm_z, self.linear_z, z)
        if bias is None and z is not None and self.linear_z is not None:
            bias = lin(self.linear_z, norm(self.layer_norm_z, z)).permute(0, 3, 1, 2).unsqueeze(1).contiguous().to(dtype)
        relative = self._modules.get("relative")
        if relative is not None:
            bias = (relative.plain if plain else relative)(positions, chains=chains, pair_bias=bias, dtype=dtype)
        if mask is not None:
            add_mask = (self.inf * (mask.to(torch.float32) - 1.0)).view(B, S, 1, 1, N)
        return bias, add_mask

    def _check(self, positions, chains, weights):
        relative, rotary = self._modules.get("relative"), self._modules.get("rotary")      # (a block that was saved before it could have one has none)
        if (positions is None) != (relative is None and rotary is None):
            raise ValueError("a block with a relative position bias or rotary positions needs the residues' positions" if positions is None else
                             "positions are for a block with a relative position bias (relative_distance) or rotary positions (rotary)")
        if chains is not None and (relative is None or not relative.other_chain):
            raise ValueError("chains are for a block with a bucket for pairs of different chains (other_chain=True)")
        if weights is not None and not self.fp8:
            raise ValueError("weights in 8 bits are for a block made with fp8=True")

    def _slots_ok(self, m: torch.Tensor) -> bool:
        """Whether Q, K, V and the gate can come from one GEMM and reach the kernels as slots of its result."""
        if not m.is_cuda or m.dtype not in (torch.bfloat16, torch.float16) or m.numel() == 0 or torch.compiler.is_compiling() \
                or torch.jit.is_tracing() or self.c_hidden not in _HEAD_DIMS:
            return False
        if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != m.dtype:
            return False
        mods = self._modules
        layers = [mods["linear_q"], mods["linear_k"], mods["linear_v"], mods["linear_o"]] + ([mods["linear_g"]] if mods.get("linear_g") is not None else [])
        return all(l.weight.dtype == m.dtype for l in layers) and all(l.bias is None for l in layers[:3])

    def _native(self, m, z, mask):
        """The block as one call and one autograd node (csrc/host.cpp); None where it does not take the call.  (Layers are
        looked up as a module stores them: their attribute access alone takes 15 us of a 100 us forward.)"""
        mods, with_z = self._modules, z is not None and self._modules.get("linear_z") is not None
        inputs = [m, z if with_z else None]
        for name, used in (("layer_norm_m", True), ("linear_q", True), ("linear_k", True), ("linear_v", True), ("linear_g", mods.get("linear_g") is not None),
                           ("linear_o", True), ("layer_norm_z", with_z), ("linear_z", with_z)):
            own = mods[name]._parameters if used else _NO_PARAMETERS
            if "weight" not in own or "bias" not in own:
                return None     # (a layer whose weight is formed from something else)
            if name in _UNBIASED:
                if own["bias"] is not None:
                    return None
                inputs.append(own["weight"])
            else:
                inputs += (own["weight"], own["bias"])
        return _lib.host().block(inputs, mask, self.no_heads, mods["layer_norm_m"].eps, mods["layer_norm_z"].eps if with_z else 0.0, self.inf,
                                 _evoformer.FLAGS)

    def forward(self, m: torch.Tensor, z: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, chains: Optional[torch.Tensor] = None, weights: Optional[Fp8BlockWeights] = None):
        B, S, N, _ = m.shape
        mods = self._modules
        simple = not self.fp8 and mods.get("relative") is None and mods.get("rotary") is None and positions is None and chains is None and weights is None
        if not simple:
            self._check(positions, chains, weights)
        if self._slots_ok(m):
            out = self._native(m, z, mask) if simple else None
            if out is not None:
                return out
            H, D = self.no_heads, self.c_hidden
            P = self._slots(_layer_norm(self.layer_norm_m, m), positions, weights)
            bias, add_mask = self._bias_and_mask(z, mask, m.dtype, (B, S, N), _layer_norm, _linear, positions, chains)
            o, grad_slot = _SlotAttention.apply(P, add_mask, bias, self.linear_g is not None)
            return self._output(o.reshape(B, S, N, H * D), weights, grad_slot.view(B, S, N, H * D))
        q, k, v, g, add_mask, bias = self.operands(m, z, mask, positions=positions, chains=chains, weights=weights)
        o = evoformer_attention(q, k, v, add_mask, bias, layout="ds4sci", gate=g)
        return self._output(o.reshape(B, S, N, self.no_heads * self.c_hidden), weights)

    def packed(self, m: torch.Tensor, offsets: torch.Tensor, positions: Optional[torch.Tensor] = None, causal: bool = False,
               weights: Optional[Fp8BlockWeights] = None) -> torch.Tensor:
        """The block without pair bias on sequences of different lengths that lie one after the other: m [T, c_m] -> [T, c_m].

        offsets    int32 or int64 [sequences + 1], as packed_attention takes them; each sequence attends within itself
        positions  [T], for rotary positions: each row's number within its sequence if not given
        causal     a row sees those up to itself only

        Rows behind the last sequence attend to nothing: theirs is the output projection's bias.  GPU only."""
        if m.dim() != 2:
            raise ValueError(f"packed rows must be [T, c_m], got {tuple(m.shape)}")
        if self._modules.get("relative") is not None:
            raise ValueError("a relative position bias is for rows of one length, not for packed ones")
        if self._modules.get("rotary") is not None and positions is None:
            positions = packed_positions(offsets, m.shape[0])
        self._check(positions, None, weights)
        if not m.is_cuda:
            raise RuntimeError("packed rows run on the GPU only (no CPU implementation)")
        x = _layer_norm(self.layer_norm_m, m)
        if self._slots_ok(m):
            q, k, v, *g = self._slots(x, positions, weights).unbind(1)
        else:
            q, k, v, *g = self._heads(x, positions, False, weights)
        o = packed_attention(q, k, v, offsets, causal=causal)
        if self.linear_g is not None:
            o = torch.sigmoid(g[0]) * o
        return self._output(o.reshape(m.shape[0], self.no_heads * self.c_hidden), weights)

    def forward_eager(self, m: torch.Tensor, z: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                      positions: Optional[torch.Tensor] = None, chains: Optional[torch.Tensor] = None):
        """The same block with plain torch operations (the formula of the reference's oracle,
        test.py:47-57, with the per-head view), nothing rounded to 8 bits: what `forward` is tested against."""
        B, S, N, _ = m.shape
        self._check(positions, chains, None)
        q, k, v, g, add_mask, bias = self.operands(m, z, mask, plain=True, positions=positions, chains=chains)
        qh, kh, vh = (t.permute(0, 1, 3, 2, 4) for t in (q, k, v))              # [B,S,H,N,D]
        s = torch.matmul(qh * self.c_hidden ** -0.5, kh.transpose(-1, -2)).float()
        if bias is not None:
            s = s + bias.float()                                                 # [B,1,H,N,N] over S
        if add_mask is not None:
            s = s + add_mask.float()                                             # [B,S,1,1,N] over H and queries
        o = torch.matmul(torch.softmax(s, -1).to(q.dtype), vh).permute(0, 1, 3, 2, 4)   # [B,S,N,H,D]
        if g is not None:
            o = torch.sigmoid(g) * o
        return self.linear_o(o.reshape(B, S, N, self.no_heads * self.c_hidden))
