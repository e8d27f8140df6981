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
