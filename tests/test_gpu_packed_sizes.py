"""Packed attention of very many rows: every result is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_rows_in_fp32_than_a_join_holds(gpu_device):
    """2^26 rows of sequences with one key each, which the last query of each sees, or all of them."""
    from evoformer_triton_amd import packed_attention
    n, each, H, D = 2 ** 17, 64, 8, 8
    q, v = torch.zeros(n * each, H, D, device=gpu_device), torch.randn(n, H, D, device=gpu_device)
    off, koff = torch.arange(0, n * each + 1, each, device=gpu_device), torch.arange(n + 1, device=gpu_device)
    k = torch.randn_like(v)
    out = packed_attention(q, k, v, off, koff).view(n, each, H, D)
    assert (out[:, -1] == v).all() and not out[:, :-1].any()
    assert (packed_attention(q, k, v, off, koff, causal=False).view(n, each, H, D) == v[:, None]).all()


def test_many_short_sequences_in_16_bits(gpu_device):
    """2^22 rows times heads and more, which no launch has a wave to: no parts are joined.  The sequences at both ends and in the middle against the formula."""
    from evoformer_triton_amd import packed_attention
    from oracle.packed import packed
    n, each, H, D = 10000, 20, 32, 64
    g = torch.Generator(device=gpu_device).manual_seed(8)
    q, k, v = (torch.randn(n * each, H, D, device=gpu_device, generator=g).to(torch.bfloat16) for _ in range(3))
    out = packed_attention(q, k, v, torch.arange(0, n * each + 1, each, device=gpu_device))
    for s in (0, n // 2, n - 2):
        rows = slice(s * each, (s + 2) * each)
        (want,), (bound,) = packed(q[rows], k[rows], v[rows], [0, each, 2 * each], [0, each, 2 * each], True, D ** -0.5)
        assert ((out[rows].double() - want).abs() <= bound).all()


def test_as_many_workgroups_as_their_waves_allow(gpu_device):
    """2^22 workgroups of four waves (of sixteen, which fewer sequences have, a launch holds half as many): one key to each query, whose value is the result."""
    from evoformer_triton_amd import packed_attention
    n, H, D = 2 ** 17, 32, 32
    q = torch.zeros(n, H, D, device=gpu_device, dtype=torch.float16)
    v = torch.randn(n, H, D, device=gpu_device).half()
    assert torch.equal(packed_attention(q, q, v, torch.arange(n + 1, device=gpu_device)), v)
