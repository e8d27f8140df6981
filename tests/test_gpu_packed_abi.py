"""Packed attention by its C entry points."""
import ctypes

import pytest
import torch

from evoformer_triton_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[70], [3], [1100]])
def test_nothing_is_left_of_an_output_in_fp32(gpu_device, lengths):
    """An array for what rounding leaves is not written in fp32, by rows that are formed anew (a value that is no number and that most rows do not see) either."""
    T, H, D = sum(lengths), 2, 32
    q, k, v = (torch.randn(T, H, D, device=gpu_device) for _ in range(3))
    v[-1] = float("nan")
    off = torch.tensor([0, T], device=gpu_device)
    o, left = torch.empty_like(q), torch.full_like(q, 7.0)
    p = _lib.EvoPacked()
    p.n, p.H, p.Hk, p.D, p.dtype, p.causal, p.offset_bytes, p.scale, p.Tq, p.Tk = 1, H, H, D, _lib.EVO_F32, 1, 8, D ** -0.5, T, T
    p.q_stride_t = p.k_stride_t = p.v_stride_t = H * D
    p.q_stride_h = p.k_stride_h = p.v_stride_h = D
    lib = _lib.load()
    ws = torch.empty(max(1, lib.evoattn_packed_fwd_workspace_bytes(ctypes.byref(p))), device=gpu_device, dtype=torch.uint8)
    for name, t in (("q", q), ("k", k), ("v", v), ("offsets", off), ("key_offsets", off), ("o", o), ("o_low", left), ("workspace", ws)):
        setattr(p, name, t.data_ptr())
    p.workspace_bytes = ws.numel()
    assert lib.evoattn_packed_fwd(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (left == 7.0).all() and torch.isfinite(o[:-1]).all() and torch.isnan(o[-1]).all()
