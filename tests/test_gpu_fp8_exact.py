"""Linear layers in 8 bits where every number is one that the formats hold: a result has to be the formula's, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_values_are_exact_on_the_gpu(gpu_device):
    """What a weight stands for, at every scale there is: e4m3 times a power of two."""
    from evoformer_triton_amd import Fp8Weight
    values = torch.arange(256, dtype=torch.uint8).view(2, 128)
    for byte in range(255):
        for dev in ("cpu", gpu_device):
            got = Fp8Weight(values.to(dev), torch.full((2, 4), byte, dtype=torch.uint8, device=dev), 128).dequantize().cpu()
            want = (values.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127)).float()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7), want.nan_to_num(7)), (byte, dev)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,k,n", [(1, 256, 70), (40, 1300, 300), (200, 250, 130), (300, 640, 200)])
def test_a_scale_that_is_no_number(gpu_device, rows, k, n, dt):
    """A byte of 255: the weight's row has no numbers in that block, and results by it are none."""
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    w = Fp8Weight.of(torch.randn((n, k), generator=torch.Generator().manual_seed(1)).to(gpu_device))
    w.scales[3, 1] = 255
    assert w.dequantize().isnan().nonzero().tolist() == [[3, c] for c in range(128, min(256, k))]
    with torch.no_grad():
        bad = fp8_linear(torch.zeros(rows, k, device=gpu_device, dtype=dt), w).isnan()
    assert bad[:, 3].all() and bad.sum() == rows


@pytest.mark.parametrize("rows", [3000, 9000])
def test_the_registered_backward_fills_no_memory_twice(gpu_device, rows):
    """What a compiled or watched step calls takes the gradients' memory once."""
    import evoformer_triton_amd  # noqa: F401
    k, n = 1024, 768
    x, w, b, dy = (torch.randn(s, device=gpu_device).to(torch.bfloat16) for s in ((rows, k), (n, k), (n,), (rows, n)))
    torch.ops.evoattn.fp8_linear_bwd(dy, x, w, b, True, False, False)

    def taken(need_x):
        before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
        grads = torch.ops.evoattn.fp8_linear_bwd(dy, x, w, b, need_x, False, False)
        return torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before, grads[0]

    total, dx = taken(True)
    up = lambda v: -(-v // 128) * 128  # noqa: E731
    rounded = k * up(n) + rows * up(n) + 16 * (k + rows)                     # w^T and dy along their rows, with scales
    assert dx.shape == x.shape and total < rounded + dx.numel() * 2 * 1.5      # (bytes: less than twice dx's; the product is not cut into slices)
