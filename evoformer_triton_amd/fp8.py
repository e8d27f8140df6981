"""Linear layers in 8 bits: e4m3 operands with a power-of-two scale for each block of 128 along the contraction.

    y = Q(x) Q(w)^T + b        Q rounds along the axis that a product contracts

Q takes each 128 values from index 0 on with the largest finite magnitude a among them, the least whole e with a <= 448 * 2^e (at
least -127; 0 for zeros), and rounds x / 2^e to e4m3, to nearest, ties to even; infinities and NaN become NaN.  Sums are fp32, the result is
rounded once, to the input's dtype.  The gradients are products of the same kind:

    dx = Q(dy) Q(w)            both rounded along the weight's rows
    dw = Q(dy)^T Q(x)          both rounded along the input's rows, all leading dimensions as one
    db = the sum of dy         not rounded

The reference stops at the attention (evoformer.py:640-651); these stand beside the 16-bit Linear layers of the block around it.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Union

import torch

from . import _lib
from ._transforms import refuse_tangents


_AUTOCAST = (torch.float32, torch.bfloat16, torch.float16)


class Fp8Weight(NamedTuple):
    """A weight [n, k] in 8 bits, for inference.

    values   [n, k up to the next multiple of 128], dense, e4m3 (float8_e4m3fn or its bytes), zero beyond k
    scales   [n, number of blocks up to the next multiple of 4], dense, a byte each (uint8 or float8_e8m0fnu): 127 + the block's exponent;
             255 is not a number, and neither are the values of its block
    k        columns of the weight
    """
    values: torch.Tensor
    scales: torch.Tensor
    k: int

    @classmethod
    def of(cls, weight: torch.Tensor) -> "Fp8Weight":
        """`weight` [n, k] (bf16, fp16 or fp32, on the GPU) rounded along its rows."""
        values, scales = _lib.host().fp8_round(weight.detach())
        return cls(values.view(torch.float8_e4m3fn), scales, weight.shape[1])

    def dequantize(self) -> torch.Tensor:
        """The values that it stands for, fp32 [n, k]."""
        if self.values.dtype not in (torch.float8_e4m3fn, torch.uint8) or self.scales.dtype not in (torch.float8_e8m0fnu, torch.uint8):
            raise ValueError("a weight in 8 bits has values in float8_e4m3fn and scales in float8_e8m0fnu, or their bytes (uint8)")
        v = self.values.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 128))
        e = self.scales.view(torch.uint8)[:, :v.shape[1]].int()
        # (a power's bits, not torch.ldexp: its powers of two are off by a last bit on the GPU, here and there)
        power = torch.where(e == 0, 0x400000, torch.where(e == 255, 0x7fc00000, e << 23)).int().view(torch.float32)
        return (v * power.unsqueeze(-1)).flatten(-2)[:, :self.k]


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight], bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x Q(weight)^T + bias with x rounded on the way, [..., n] in x's dtype.

    x        [..., k] bf16, fp16 or fp32, any strides
    weight   [n, k] bf16, fp16 or fp32 (not necessarily x's dtype): rounded with each call, differentiable.  Or an Fp8Weight, rounded once:
             no gradients
    bias     [n], bf16, fp16 or fp32, added in fp32

    Gradients come in the dtype of what they belong to.  A result or weight gradient in fp32 is summed in fp32 throughout; towards
    16 bits the 8-bit matrix instructions form the sums, to about 1.4e-5 of the result.  Under autocast the input, and so the result, are
    of its type, as a Linear's; weight and bias stay as they are.  Rows, n and k up to 2^26.  Runs on the current
    stream of the tensors' device; GPU only."""
    held = isinstance(weight, Fp8Weight)
    for name, t in (("x", x), ("bias", bias)) + ((("weight.values", weight.values), ("weight.scales", weight.scales)) if held else (("weight", weight),)):
        if not isinstance(t, torch.Tensor) and not (t is None and name == "bias"):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if torch.is_autocast_enabled("cuda") and x.is_cuda and x.dtype in _AUTOCAST:
        x = x.to(torch.get_autocast_dtype("cuda"))
    if torch.compiler.is_compiling():
        if held:
            return torch.ops.evoattn.fp8_linear_held(x, weight.values, weight.scales, weight.k, bias)
        return torch.ops.evoattn.fp8_linear(x, weight, bias)
    host = _lib.host()
    y = host.fp8_linear_held(x, weight.values, weight.scales, weight.k, bias) if held else host.fp8_linear(x, weight, bias)
    if y is not None:
        return y
    wrong = host.fp8_linear_held_wrong(x, weight.values, weight.scales, weight.k, bias) if held else host.fp8_linear_wrong(x, weight, bias)
    if wrong:
        raise ValueError(wrong)
    if not x.is_cuda:
        raise RuntimeError("fp8_linear runs on the GPU only (no CPU implementation); move its tensors to one cuda device")
    refuse_tangents("fp8_linear", x, bias, *(() if held else (weight,)))
    if not held:
        return torch.ops.evoattn.fp8_linear(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("an Fp8Weight is for inference: call under torch.no_grad(), or give the weight itself where gradients are needed")
    return torch.ops.evoattn.fp8_linear_held(x, weight.values, weight.scales, weight.k, bias)


# ---- the same as registered operators: what the compiler's tracer and the dispatch modes see ----

@torch.library.custom_op("evoattn::fp8_linear", mutates_args=(), device_types="cuda")
def _op_fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    return _lib.host().fp8_linear_forward(x, weight, bias)


@_op_fp8_linear.register_fake
def _(x, weight, bias):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("evoattn::fp8_linear_bwd", mutates_args=(), device_types="cuda")
def _op_fp8_linear_bwd(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], need_x: bool, need_weight: bool,
                       need_bias: bool) -> List[torch.Tensor]:
    """[dx, dweight, dbias]; one that was not asked for is empty."""
    return _lib.host().fp8_linear_backward(dy, x, weight, bias, need_x, need_weight, need_bias)


@_op_fp8_linear_bwd.register_fake
def _(dy, x, weight, bias, need_x, need_weight, need_bias):
    return [x.new_empty(x.shape if need_x else (0,)), weight.new_empty(weight.shape if need_weight else (0,)),
            bias.new_empty(bias.shape) if need_bias and bias is not None else x.new_empty((0,))]


def _setup_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _backward(ctx, dy):
    x, weight, bias = ctx.saved_tensors
    need = [*ctx.needs_input_grad[:2], bias is not None and ctx.needs_input_grad[2]]
    grads = torch.ops.evoattn.fp8_linear_bwd(dy.to(x.dtype), x, weight, bias, *need)
    return tuple(g if n else None for g, n in zip(grads, need))


_op_fp8_linear.register_autograd(_backward, setup_context=_setup_context)


@torch.library.custom_op("evoattn::fp8_linear_held", mutates_args=(), device_types="cuda")
def _op_fp8_linear_held(x: torch.Tensor, values: torch.Tensor, scales: torch.Tensor, k: int, bias: Optional[torch.Tensor]) -> torch.Tensor:
    return _lib.host().fp8_linear_held_forward(x, values, scales, k, bias)


@_op_fp8_linear_held.register_fake
def _(x, values, scales, k, bias):
    return x.new_empty((*x.shape[:-1], values.shape[0]))
