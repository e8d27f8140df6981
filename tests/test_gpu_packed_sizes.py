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


@pytest.mark.parametrize("n,each", [(10000, 20), (10000, 16), (140000, 1)])
def test_many_short_sequences_in_16_bits(gpu_device, n, each):
    """2^22 rows times heads and more, which no launch has a wave to: no parts are joined.  The sequences at both ends and in the middle against the formula."""
    from evoformer_triton_amd import packed_attention
    from oracle.packed import packed
    H, D = 32, 64
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


@pytest.mark.parametrize("T,H,Hk,D,far", [(3, 2 ** 16, 2 ** 16, 128, False), (40, 2 ** 16, 2 ** 15, 128, False), (6, 2 ** 17, 2 ** 17, 61, True)])
def test_more_heads_than_rows_lie_apart(gpu_device, T, H, Hk, D, far):
    """Rows of 2^23 values in 16 bits and more, which the kernels take head by head; the first heads, the last and some between against the formula, with their gradients."""
    from evoformer_triton_amd import packed_attention
    from oracle.packed import packed
    g = torch.Generator(device=gpu_device).manual_seed(8)
    q, k, v, dout = (torch.randn(T, h, D, device=gpu_device, generator=g).to(torch.bfloat16) for h in (H, Hk, Hk, H))
    if far:
        q = torch.cat([q, q], 1)[:, :H]                 # (a slice: rows twice as far apart)
    at = [0, T // 2, T]
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, torch.tensor(at, device=gpu_device))
    got = [out, *torch.autograd.grad(out, leaves, dout)]
    G = H // Hk
    for hk in (0, Hk // 2, Hk - 1):
        heads = slice(hk * G, (hk + 1) * G), slice(hk, hk + 1)
        parts = [t.detach()[:, heads[i]] for t, i in ((q, 0), (k, 1), (v, 1))]
        want, bound = packed(*parts, at, at, True, D ** -0.5, dout[:, heads[0]])
        for name, a, w, b, i in zip(("o", "dq", "dk", "dv"), got, want, bound, (0, 0, 1, 1)):
            assert a.shape[1] == (H, Hk)[i] and ((a[:, heads[i]].double() - w).abs() <= b).all(), name
