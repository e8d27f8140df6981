"""Forward-mode differentiation of the relative position bias and the 8-bit layers: refused, also where no gradient is asked for and the dispatcher would drop the tangent."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls(dev):
    from evoformer_triton_amd import Fp8Weight, fp8_linear, relative_buckets, relative_position_bias
    x, w, b = (torch.randn(s, device=dev) for s in ((70, 140), (30, 140), (30,)))
    held, lut, at = Fp8Weight.of(w), relative_buckets(4).to(dev), torch.arange(24, device=dev)
    table, pair = torch.randn(9, 2, device=dev), torch.randn(1, 1, 2, 24, 24, device=dev)
    return {"x": (lambda t: fp8_linear(t, w, b), x), "weight": (lambda t: fp8_linear(x, t, b), w), "bias": (lambda t: fp8_linear(x, w, t), b),
            "held": (lambda t: fp8_linear(t, held), x), "held bias": (lambda t: fp8_linear(x, held, t), b),
            "table": (lambda t: relative_position_bias(t, lut, at), table), "pair": (lambda t: relative_position_bias(table, lut, at, pair_bias=t), pair),
            "op": (lambda t: torch.ops.evoattn.fp8_linear(t, w, b), x), "held op": (lambda t: torch.ops.evoattn.fp8_linear_held(t, held.values, held.scales, 140, None), x),
            "bias op": (lambda t: torch.ops.evoattn.relative_bias(t, lut, at, at, None, None, None, None), table)}


NAMES = ["x", "weight", "bias", "held", "held bias", "table", "pair", "op", "held op", "bias op"]


@pytest.mark.parametrize("name", NAMES)
def test_a_dual_tensor(gpu_device, name):
    call, t = _calls(gpu_device)[name]
    with forward_ad.dual_level():
        for grad in (torch.no_grad, torch.enable_grad):
            with grad(), pytest.raises(NotImplementedError, match="forward mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
        call(t)                                                              # (without a tangent it is a call like any other)


@pytest.mark.parametrize("name", NAMES[:7])
def test_torch_func(gpu_device, name):
    call, t = _calls(gpu_device)[name]
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(torch.func.vmap(call), (t[None],), (torch.ones_like(t)[None],))
