"""Which products of up to four blocks are rounded on the way, without a GPU: those whose strips are one piece, or a few that are all under way at once."""
import ctypes

import pytest

from evoformer_triton_amd import _lib


@pytest.mark.parametrize("m,n,k,on_the_way", [
    (16384, 768, 384, 1), (16384, 700, 300, 1), (11000, 320, 512, 1), (65536, 512, 512, 1), (100000, 1024, 384, 1),
    # a second round of workgroups: 564, 532, 516, 500 in five pieces on 104 strips and 640
    (12000, 384, 300, 0), (17000, 700, 384, 0), (22000, 1536, 512, 0), (13312, 1280, 384, 0), (40960, 2048, 300, 0),
    (8192, 1024, 512, 0), (300, 8192, 512, 0), (17000, 700, 256, 1), (64, 8192, 4000, 1), (65, 8192, 513, 0)])
def test_the_rule(m, n, k, on_the_way):
    for dtype in (_lib.EVO_BF16, _lib.EVO_F16):
        p = _lib.EvoFp8Matmul()
        p.m, p.n, p.k, p.ldo, p.dtype = m, n, k, n, dtype
        assert _lib.load().evoattn_fp8_matmul_rounds(ctypes.byref(p)) == on_the_way
