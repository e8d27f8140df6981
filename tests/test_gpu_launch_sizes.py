"""As many problems as a launch does not hold: refused, where such a launch is cut off without an error and leaves the results of the rest as the memory was."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,D,bias", [(1, 8, False), (3, 8, True), (5, 16, False), (2, 32, False)])
def test_more_problems_than_a_launch_holds(gpu_device, N, D, bias):
    from evoformer_triton_amd import evoformer_attention
    q, k, v = (torch.zeros(1, 2 ** 21 + 300, N, 8, D, device=gpu_device, dtype=torch.bfloat16) for _ in range(3))
    pair = torch.zeros(1, 1, 8, N, N, device=gpu_device, dtype=torch.bfloat16) if bias else None
    try:
        o = evoformer_attention(q, k, v + 1, None, pair, layout="ds4sci")
    except RuntimeError as error:
        assert "overflow" in str(error)
    else:       # (a kernel that takes several problems to a workgroup may hold them)
        assert (o == 1).all()


def test_as_many_as_one_holds(gpu_device):
    from evoformer_triton_amd import evoformer_attention
    S, H = 2 ** 21 - 1, 8
    g = torch.Generator(device=gpu_device).manual_seed(1)
    q, k, v = (torch.randn(1, S, 2, H, 8, device=gpu_device, dtype=torch.bfloat16, generator=g).requires_grad_() for _ in range(3))
    o = evoformer_attention(q, k, v, None, None, layout="ds4sci")
    grads = torch.autograd.grad(o, [q, k, v], torch.ones_like(o))
    for rows in (slice(0, 9), slice(S // 2, S // 2 + 9), slice(S - 9, S)):
        part = [t.detach()[:, rows].contiguous().requires_grad_() for t in (q, k, v)]
        want = evoformer_attention(*part, None, None, layout="ds4sci")
        want_grads = torch.autograd.grad(want, part, torch.ones_like(want))
        for a, b in zip((o, *grads), (want, *want_grads)):
            assert (a[:, rows].float() - b.float()).abs().max() <= 2 ** -6 * b.float().abs().max()     # (few rows take kernels of their own: a bf16 step or two)


def test_a_bias_of_more_batches_than_a_launch_holds(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut, table = relative_buckets(1).to(gpu_device), torch.ones(3, 1, device=gpu_device, requires_grad=True)
    at = torch.zeros(2 ** 24, 1, dtype=torch.int32, device=gpu_device)
    with pytest.raises(RuntimeError, match="overflow"):
        relative_position_bias(table, lut, at)
    assert (relative_position_bias(table.detach(), lut, at[:-1]) == 1).all()
    keys = torch.zeros(2 ** 30, dtype=torch.int32, device=gpu_device)
    out = relative_position_bias(table, lut, at[0], keys, dtype=torch.bfloat16)
    assert (out == 1).all()
    with pytest.raises(RuntimeError, match="overflow"):
        out.sum().backward()
