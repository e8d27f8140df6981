"""Launches of 2^32 threads or more, which would be cut off without an error, are refused; without a GPU."""
import ctypes

import pytest

from evoformer_triton_amd import _lib

P = 0x10000


def _relative(**change):
    p = _lib.EvoRelativeBias()
    p.B, p.H, p.Nq, p.Nk, p.rows, p.reach, p.dtype, p.table_dtype, p.pos_bytes = 1, 1, 1, 1, 65, 32, _lib.EVO_F32, _lib.EVO_F32, 8
    for f in ("table", "lut", "pos_q", "pos_k", "out", "dout", "workspace"):
        setattr(p, f, P)
    p.workspace_bytes = 1 << 62
    for k, v in change.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def test_the_relative_bias():
    lib = _lib.load()
    for sizes in (dict(B=2 ** 24), dict(B=2 ** 14, H=2 ** 10), dict(B=2 ** 20, H=2 ** 10, Nk=9), dict(H=2 ** 24 + 5)):
        assert lib.evoattn_relative_bias_fwd(_relative(**sizes), None) == _lib.EVO_EOVERFLOW, sizes
    for sizes in (dict(Nk=2 ** 30), dict(B=2 ** 24), dict(B=2 ** 14, Nk=2 ** 16), dict(H=2 ** 28)):
        assert lib.evoattn_relative_bias_bwd(_relative(dtable=P, **sizes), None) == _lib.EVO_EOVERFLOW, sizes
        assert lib.evoattn_relative_bias_bwd_workspace_bytes(_relative(dtable=P, **sizes)) == 0
    for sizes in (dict(H=64, Nq=2 ** 14, Nk=2 ** 14), dict(H=64, Nq=2 ** 15, Nk=2 ** 15, dtype=_lib.EVO_BF16)):
        assert lib.evoattn_relative_bias_bwd(_relative(dpair=P, **sizes), None) == _lib.EVO_EOVERFLOW, sizes


def _product(m, n, k, **change):
    p = _lib.EvoFp8Matmul()
    p.m, p.n, p.k, p.ldo, p.dtype = m, n, k, n, _lib.EVO_BF16
    for f in ("a", "b", "scales_a", "scales_b", "out", "workspace"):
        setattr(p, f, P)
    p.workspace_bytes = 1 << 62
    return ctypes.byref(p)


def test_8_bit_products_and_rounding():
    lib = _lib.load()
    for m, n, k in ((2 ** 24, 2 ** 16, 600), (2 ** 31 - 513, 300, 513)):
        assert lib.evoattn_fp8_matmul(_product(m, n, k), None) == _lib.EVO_EOVERFLOW, (m, n, k)
    assert lib.evoattn_fp8_matmul_rounding(_product(1, 2 ** 30, 2000), P, 2000, None) == _lib.EVO_EOVERFLOW
    for rows, cols in ((2 ** 31, 1), (2 ** 25, 2 ** 13 + 1), (2 ** 38, 1)):
        assert lib.evoattn_fp8_quantize(P, cols, P, P, None, None, None, rows, cols, _lib.EVO_BF16, None) == _lib.EVO_EOVERFLOW, (rows, cols)
    half = _lib.EvoFp8Rounding(P, 1, 2 ** 30, 1, P, P, None, None, None)
    assert lib.evoattn_fp8_quantize_two(ctypes.byref(half), ctypes.byref(half), _lib.EVO_BF16, None) == _lib.EVO_EOVERFLOW
