"""Packed attention of very many rows: what its launches hold, without a GPU."""
import ctypes

import pytest

from evoformer_triton_amd import _lib


def _block(dtype, n, Tq, Tk, H, Hk, D):
    p = _lib.EvoPacked()
    p.n, p.H, p.Hk, p.D, p.dtype, p.offset_bytes, p.scale, p.Tq, p.Tk = n, H, Hk, D, dtype, 4, 0.125, Tq, Tk
    return p


@pytest.mark.parametrize("rows,parts", [(2 ** 26 - 16, True), (2 ** 26 - 4, True), (2 ** 26 - 3, False), (2 ** 26, False), (2 ** 27 - 16, False)])
def test_parts_in_fp32_are_joined_by_a_launch_that_holds_them(rows, parts):
    """A wave to a row, four of them to a workgroup: from 2^26 rows on that would be 2^32 threads.  (The kernels that split the keys of few queries keep their results in parts, and one part at least.)"""
    p = _block(_lib.EVO_F32, rows // 16, rows, rows * 8, 1, 1, 128)
    need = _lib.load().evoattn_packed_fwd_workspace_bytes(ctypes.byref(p))
    assert (need >= rows * 130 * 4) if parts else need == 0
