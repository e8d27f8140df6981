"""The gated block in 8 bits with layers and modes that a caller may bring: biases on Q, K and V, autocast."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def test_every_projections_bias_counts(gpu_device):
    """A block whose Q, K or V has been given a bias: the stacked product's bias is the layers' biases, one after the other."""
    from evoformer_triton_amd import evoformer_attention, fp8_linear
    from evoformer_triton_amd.block import GatedAttentionBlock
    for dt, gating, names in ((BF16, True, ("linear_k", "linear_v")), (F32, False, ("linear_q",)), (F16, False, ("linear_v",)), (F32, True, ("linear_q", "linear_k", "linear_v"))):
        torch.manual_seed(5)
        block = GatedAttentionBlock(64, 32, 2, gating=gating, fp8=True)
        for name in names:
            layer = nn.Linear(64, 64)
            nn.init.normal_(layer.bias, 1.0)
            setattr(block, name, layer)
        block = block.to(gpu_device).to(dt)
        m = torch.randn(1, 4, 40, 64, device=gpu_device).to(dt)
        y = block(m)
        grads = torch.autograd.grad(y, [getattr(block, n).bias for n in names], torch.randn_like(y))
        assert all(g.shape == (64,) and g.any() for n, g in zip(names, grads) if n != "linear_k")      # (K's moves no softmax)
        x = block.layer_norm_m(m)
        with torch.no_grad():
            one = lambda layer: fp8_linear(x, layer.weight, layer.bias).view(1, 4, 40, 2, 32)  # noqa: E731
            o = evoformer_attention(one(block.linear_q), one(block.linear_k), one(block.linear_v), None, None, layout="ds4sci",
                                    gate=one(block.linear_g) if gating else None)
            want = fp8_linear(o.reshape(1, 4, 40, 64), block.linear_o.weight, block.linear_o.bias)
            # (LayerNorm by torch and by the library, which may round a value to another neighbour and so to another number of 8 bits)
            assert (y - want).float().norm() <= 3e-2 * want.float().norm()
            assert torch.equal(block(m, weights=block.fp8_weights()), y)


def test_autocast_takes_8_bit_layers_to_its_type(gpu_device):
    """As torch's Linear: the input in autocast's type, and so the result; parameters and their gradients keep theirs."""
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    x, w, b = (torch.randn(s, device=gpu_device) for s in ((100, 256), (64, 256), (64,)))
    dy = torch.randn(100, 64, device=gpu_device)
    for to in (BF16, F16):
        for t in (F32, BF16, F16):
            leaves = [v.clone().to(t if v is x else F32).requires_grad_() for v in (x, w, b)]
            with torch.autocast("cuda", to):
                y = fp8_linear(*leaves)
                with torch.no_grad():
                    held = fp8_linear(leaves[0], Fp8Weight.of(w), b)
                compiled = torch.compile(fp8_linear, fullgraph=True, backend="aot_eager")(*leaves)
            want_leaves = [leaves[0].detach().to(to).requires_grad_(), *leaves[1:]]
            want = fp8_linear(*want_leaves)
            assert y.dtype == to and all(torch.equal(a, want) for a in (y, held, compiled))
            grads = torch.autograd.grad(y, leaves, dy.to(to))
            want_grads = torch.autograd.grad(want, want_leaves, dy.to(to))
            assert [g.dtype for g in grads] == [t, F32, F32] and all(torch.equal(a, c.to(a.dtype)) for a, c in zip(grads, want_grads))
    with torch.autocast("cuda", BF16, enabled=False):
        assert fp8_linear(x, w, b).dtype == F32
    with torch.autocast("cpu", BF16):
        assert fp8_linear(x, w, b).dtype == F32


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("c_z,relative", [(None, None), (32, None), (32, 8)])
def test_a_block_in_fp32_under_autocast(gpu_device, fp8, c_z, relative):
    """Projections and attention in autocast's type, gradients in the parameters': what the same layers of torch give, to that type's roundings."""
    from evoformer_triton_amd.block import GatedAttentionBlock
    torch.manual_seed(3)
    block = GatedAttentionBlock(64, 32, 2, c_z=c_z, fp8=fp8, relative_distance=relative).to(gpu_device)
    if relative is not None:
        block.relative.weight.data.normal_()
    m = torch.randn(1, 6, 40, 64, device=gpu_device, requires_grad=True)
    z = torch.randn(1, 40, 40, c_z, device=gpu_device, requires_grad=True) if c_z else None
    at = {"positions": torch.arange(40, device=gpu_device)} if relative else {}
    dout = torch.randn(1, 6, 40, 64, device=gpu_device)
    leaves = [m] + ([z] if c_z else []) + [p for n, p in block.named_parameters() if n != "layer_norm_z.bias"]     # (which moves no softmax)
    with torch.autocast("cuda", BF16):
        y = block(m, z, None, **at)
        assert y.dtype == BF16 and all(t.dtype == BF16 for t in block.operands(m, z, None, **at)[:4])
    grads = torch.autograd.grad(y, leaves, dout.to(BF16))
    want = block.forward_eager(m, z, None, **at)
    want_grads = torch.autograd.grad(want, leaves, dout)
    assert [g.dtype for g in grads] == [F32] * len(grads)
    # a few parts in a hundred in 8 bits (operands within 2^-4 of themselves), of bf16's in 16
    assert (y - want).norm() <= (0.15 if fp8 else 2e-2) * want.norm()
    for a, b in zip(grads, want_grads):
        assert torch.isfinite(a).all() and (a - b).norm() <= (0.4 if fp8 else 5e-2) * b.norm() + 1e-3 * b.numel() ** 0.5
