"""Checkpointed calls: the forward runs again while a backward asks for what was saved, and gives the same gradients."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def _same(call, inputs, leaves, early_stop):
    got = torch.autograd.grad(checkpoint(call, *inputs, use_reentrant=False, early_stop=early_stop).float().square().sum(), leaves)
    want = torch.autograd.grad(call(*inputs).float().square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("early_stop", [True, False])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("options", [dict(c_z=32), dict(), dict(c_z=32, gating=False), dict(c_z=32, fp8=True), dict(fp8=True), dict(c_z=32, relative_distance=4),
                                     dict(c_z=32, fp8=True, relative_distance=4)], ids=str)
def test_a_block(gpu_device, options, dt, early_stop):
    from evoformer_triton_amd.block import GatedAttentionBlock
    torch.manual_seed(0)
    block = GatedAttentionBlock(64, 32, 2, **options).to(gpu_device).to(dt)
    at = {"positions": torch.arange(24, device=gpu_device)} if "relative_distance" in options else {}
    m = torch.randn(2, 3, 24, 64, device=gpu_device).to(dt).requires_grad_()
    z = torch.randn(2, 24, 24, 32, device=gpu_device).to(dt).requires_grad_() if "c_z" in options else None
    leaves = [m] + ([] if z is None else [z]) + list(block.parameters())
    _same(lambda a, b: block(a * 1, b, None, **at), (m, z), leaves, early_stop)


@pytest.mark.parametrize("early_stop", [True, False])
def test_the_operators_one_after_the_other(gpu_device, early_stop):
    from evoformer_triton_amd import evoformer_attention, fp8_linear, relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(1)
    x, w, b, table = (torch.randn(s, generator=g).to(gpu_device).requires_grad_() for s in ((1, 5, 40, 64), (192, 64), (192,), (9, 2)))
    lut, at = relative_buckets(4).to(gpu_device), torch.arange(40, device=gpu_device)

    def call(x, table):
        q, k, v = fp8_linear(x.tanh(), w, b).view(1, 5, 40, 3, 2, 32).unbind(3)
        bias = relative_position_bias(table * 2, lut, at) * 0.5
        return evoformer_attention(q, k, v, None, bias, layout="ds4sci").sin()

    _same(call, (x, table), [x, w, b, table], early_stop)
