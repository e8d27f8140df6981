"""What packed attention refuses, and its oracle, without a GPU."""
import ctypes

import pytest
import torch

from evoformer_triton_amd import _lib, packed_attention, packed_positions
from oracle.packed import packed


def test_refusals():
    q, k, off = torch.zeros(6, 4, 8), torch.zeros(6, 2, 8), torch.tensor([0, 6])
    for args, kw, what in (
            ((q[0], k, k, off), {}, r"\[Tq, H, D\]"),
            ((q, k, k[:5], off), {}, "values must have"),
            ((q.double(), k, k, off), {}, "bf16, fp16 or fp32"),
            ((q.half(), k, k, off), {}, "queries' dtype"),
            ((q, torch.zeros(6, 2, 9), torch.zeros(6, 2, 9), off), {}, "head dim"),
            ((torch.zeros(6, 4, 129), torch.zeros(6, 2, 129), torch.zeros(6, 2, 129), off), {}, "1 to 128"),
            ((q, torch.zeros(6, 3, 8), torch.zeros(6, 3, 8), off), {}, "multiple"),
            ((q, torch.zeros(6, 0, 8), torch.zeros(6, 0, 8), off), {}, "multiple"),
            ((q, k, k, off.float()), {}, "int32 or int64"),
            ((q, k, k, off[None]), {}, "sequences"),
            ((q, k, k, off[:0]), {}, "sequences"),
            ((q, k, k, off, torch.tensor([0, 3, 6])), {}, "as long as"),
            ((q, torch.zeros(7, 2, 8), torch.zeros(7, 2, 8), off), {}, "need key_offsets"),
            ((q, k, k, off), {"scale": 0.0}, "positive"),
            ((q, k, k, off), {"scale": -1.0}, "positive"),
            ((q, k, k, off), {"scale": float("nan")}, "positive"),
            ((q, k, k, off), {"scale": float("inf")}, "positive")):
        with pytest.raises(ValueError, match=what):
            packed_attention(*args, **kw)
    with pytest.raises(TypeError, match="offsets must be a tensor"):
        packed_attention(q, k, k, [0, 6])
    with pytest.raises(RuntimeError, match="GPU only"):
        packed_attention(q, k, k, off)


def test_positions():
    assert packed_positions(torch.tensor([0, 3, 3, 5]), 7).tolist() == [0, 1, 2, 0, 1, 0, 1]
    assert packed_positions(torch.tensor([0, 2], dtype=torch.int32), 2).tolist() == [0, 1]


def _block():
    p = _lib.EvoPacked()
    p.n, p.H, p.Hk, p.D, p.dtype, p.offset_bytes, p.scale, p.Tq, p.Tk = 1, 4, 2, 64, _lib.EVO_BF16, 4, 0.125, 100, 100
    p.q_stride_t = p.dout_stride_t = 256
    p.k_stride_t = p.v_stride_t = 128
    p.q_stride_h = p.k_stride_h = p.v_stride_h = p.dout_stride_h = 64
    for f in ("q", "k", "v", "offsets", "key_offsets", "o", "lse", "dout", "dq", "dk", "dv", "workspace"):
        setattr(p, f, 0x10000)    # (never dereferenced by the host-side checks)
    p.workspace_bytes = 1 << 40
    return p


def test_the_c_entry_points_refuse():
    lib = _lib.load()
    for change, code in (({"H": 3}, _lib.EVO_EINVAL), ({"D": 0}, _lib.EVO_EINVAL), ({"D": 136}, _lib.EVO_EUNSUPPORTED), ({"scale": 0.0}, _lib.EVO_EINVAL),
                         ({"dtype": 7}, _lib.EVO_EINVAL), ({"offset_bytes": 2}, _lib.EVO_EINVAL), ({"n": -1}, _lib.EVO_EINVAL), ({"Tq": 1 << 31}, _lib.EVO_EOVERFLOW),
                         ({"q": None}, _lib.EVO_EINVAL), ({"offsets": None}, _lib.EVO_EINVAL), ({"workspace_bytes": 0, "dk": 0x10000}, None)):
        p = _block()
        for name, value in change.items():
            setattr(p, name, value)
        if code is None:      # (the backward's scratch)
            assert lib.evoattn_packed_bwd(ctypes.byref(p), None) == _lib.EVO_EWORKSPACE
            continue
        assert lib.evoattn_packed_fwd(ctypes.byref(p), None) == code, change
        assert lib.evoattn_packed_bwd(ctypes.byref(p), None) == code, change
    assert lib.evoattn_packed_fwd(None, None) == _lib.EVO_EINVAL
    assert lib.evoattn_packed_bwd_workspace_bytes(ctypes.byref(_block())) >= 4 * 100 * 4


def test_the_oracle_is_the_formula():
    """Against autograd in 64 bits, with a mask."""
    g = torch.Generator().manual_seed(3)
    q, k, v, dout = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((9, 4, 8), (11, 2, 8), (11, 2, 8), (9, 4, 8)))
    a, b = [0, 4, 8], [0, 5, 10]
    for causal in (True, False):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = torch.zeros_like(q)
        for s in range(2):
            x, y, z = leaves[0][a[s]:a[s + 1]], *(t[b[s]:b[s + 1]].repeat_interleave(2, 1) for t in leaves[1:])
            score = torch.einsum("ihd,jhd->hij", x, y) * 0.3
            if causal:
                score = score.masked_fill(~torch.ones(4, 5, dtype=torch.bool).tril(1), float("-inf"))
            out = out + torch.nn.functional.pad(torch.einsum("hij,jhd->ihd", score.softmax(-1), z), (0, 0, 0, 0, a[s], 9 - a[s + 1]))
        want = [out, *torch.autograd.grad(out, leaves, dout)]
        got, _ = packed(q, k, v, a, b, causal, 0.3, dout)
        for x, y in zip(got, want):
            assert torch.allclose(x, y, rtol=1e-12, atol=1e-12)


def test_the_c_entry_points_refuse_what_is_not_aligned():
    """16 bits: pieces of 16 bytes, rows that lie apart; and a workspace that is not there or begins between two of them."""
    lib = _lib.load()
    for change, code, ways in (({"q": 0x10008}, _lib.EVO_EALIGN, "fb"), ({"v": 0x10002}, _lib.EVO_EALIGN, "fb"), ({"o_low": 0x10008}, _lib.EVO_EALIGN, "fb"),
                               ({"k_stride_t": 132}, _lib.EVO_EALIGN, "fb"), ({"k_stride_t": 56}, _lib.EVO_EALIGN, "fb"), ({"q_stride_t": 0}, _lib.EVO_EALIGN, "fb"),
                               ({"v_stride_t": 1 << 23}, _lib.EVO_EALIGN, "fb"), ({"q_stride_h": 60}, _lib.EVO_EALIGN, "fb"), ({"D": 60}, _lib.EVO_EALIGN, "fb"),
                               ({"dout": 0x10008}, _lib.EVO_EALIGN, "b"), ({"dout_stride_t": 0}, _lib.EVO_EALIGN, "b"), ({"dk": 0x10004}, _lib.EVO_EALIGN, "b"),
                               ({"workspace": 0x10008}, _lib.EVO_EALIGN, "b"), ({"workspace": None}, _lib.EVO_EWORKSPACE, "b"), ({"lse": None}, _lib.EVO_EINVAL, "b"),
                               ({"dk": None}, _lib.EVO_EINVAL, "b"), ({"H": 1 << 21, "Hk": 1}, _lib.EVO_EOVERFLOW, "fb"), ({"n": 1 << 30}, _lib.EVO_EOVERFLOW, "fb")):
        p = _block()
        for name, value in change.items():
            setattr(p, name, value)
        for way in ways:
            call = lib.evoattn_packed_fwd if way == "f" else lib.evoattn_packed_bwd
            assert call(ctypes.byref(p), None) == code, (change, way)
    # parts of a long walk, in both types
    for dtype in (_lib.EVO_BF16, _lib.EVO_F32):
        p = _block()
        p.dtype, p.Tk = dtype, 1 << 20
        need = lib.evoattn_packed_fwd_workspace_bytes(ctypes.byref(p))
        assert need > 0
        for name, value, code in (("workspace_bytes", need - 1, _lib.EVO_EWORKSPACE), ("workspace", None, _lib.EVO_EWORKSPACE), ("workspace", 0x10004, _lib.EVO_EALIGN)):
            p = _block()
            p.dtype, p.Tk = dtype, 1 << 20
            setattr(p, name, value)
            assert lib.evoattn_packed_fwd(ctypes.byref(p), None) == code, (dtype, name)
    # nothing at all
    for dtype in (_lib.EVO_BF16, _lib.EVO_F32):
        for n, Tq, Tk in ((0, 0, 0), (0, 0, 50), (0, 50, 0), (1, 0, 0), (5, 0, 50)):
            p = _block()
            p.dtype, p.n, p.Tq, p.Tk = dtype, n, Tq, Tk
            assert lib.evoattn_packed_fwd_workspace_bytes(ctypes.byref(p)) >= 0 and lib.evoattn_packed_bwd_workspace_bytes(ctypes.byref(p)) >= 0
            if Tq == 0:
                assert lib.evoattn_packed_fwd(ctypes.byref(p), None) == 0
