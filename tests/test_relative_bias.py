"""The relative position bias without a GPU: its buckets, its refusals, the C ABI's checks and the traced operator's shapes."""
import ctypes
import math

import pytest
import torch

from evoformer_triton_amd import RelativePositionBias, _lib, relative_buckets, relative_position_bias


def test_a_bucket_for_each_distance():
    assert relative_buckets(0).tolist() == [0]
    assert relative_buckets(3).tolist() == list(range(7)) and relative_buckets(127)[-1] == 254


@pytest.mark.parametrize("num,reach", [(4, 2), (8, 16), (16, 64), (32, 128), (32, 127), (64, 4096), (254, 4096)])
def test_widening_buckets_begin_where_the_formula_says(num, reach):
    b = relative_buckets(reach, num).tolist()
    half, near = num // 2, num // 4
    far = half - near
    for d in range(reach + 1):
        i = b[reach + d]
        if d < near:
            assert i == d
        else:   # near (reach / near)^((i - near) / far) <= d, and the next border beyond; apart from rounding, where whole numbers decide
            at = near + far * math.log(d / near) / math.log(reach / near)
            assert near <= i < half and i <= at + 1e-9 and (i == half - 1 or at < i + 1 + 1e-9)
        if d:
            assert b[reach - d] == half + i
    assert b == [min(x, 255) for x in b] and b[-1] == half - 1


def test_borders_that_are_powers():
    b = relative_buckets(128, 32)   # near 8, far 8: borders 8 * 2^(i / 2); every second one a whole number
    assert [b[128 + d].item() for d in (8, 15, 16, 31, 32, 63, 64, 127, 128)] == [8, 9, 10, 11, 12, 13, 14, 15, 15]


@pytest.mark.parametrize("args", [(-1,), (4097, 32), (128,), (16, 3), (16, 2), (16, 258), (16, 7), (4, 16)])
def test_buckets_that_are_refused(args):
    with pytest.raises(ValueError):
        relative_buckets(*args)


def _good():
    return dict(table=torch.zeros(5, 2), buckets=relative_buckets(2), positions=torch.arange(6).view(2, 3), key_positions=torch.arange(8).view(2, 4),
                chains=torch.zeros(2, 3, dtype=torch.long), key_chains=torch.zeros(1, 4, dtype=torch.long), pair_bias=torch.zeros(1, 1, 2, 3, 4))


@pytest.mark.parametrize("change,match", [
    (dict(table=torch.zeros(5)), "table"), (dict(table=torch.zeros(0, 2)), "table"), (dict(table=torch.zeros(5, 2, dtype=torch.float64)), "table"),
    (dict(table=torch.zeros(257, 2)), "256"), (dict(buckets=torch.zeros(5)), "uint8"), (dict(buckets=torch.zeros(4, dtype=torch.uint8)), "uint8"),
    (dict(buckets=torch.zeros(8195, dtype=torch.uint8)), "4096"), (dict(positions=torch.zeros(2, 3)), "whole numbers"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.bool)), "whole numbers"), (dict(positions=torch.zeros(1, 2, 3, dtype=torch.long)), r"\[B, N\]"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.long)), "agree"), (dict(key_chains=None), "neither"), (dict(chains=None), "neither"),
    (dict(chains=torch.zeros(2, 4, dtype=torch.long)), "as long as"), (dict(pair_bias=torch.zeros(1, 2, 3, 4)), "pair bias"),
    (dict(pair_bias=torch.zeros(1, 1, 2, 4, 3)), "pair bias"), (dict(pair_bias=torch.zeros(3, 1, 2, 3, 4)), "agree"),
    (dict(pair_bias=torch.zeros(1, 1, 2, 3, 4, dtype=torch.float64)), "pair bias"), (dict(dtype=torch.float16), "dtype"), (dict(dtype=torch.float64), "bf16"),
    (dict(), "GPU only")])
def test_calls_that_are_refused(change, match):
    args = {**_good(), **change}
    table, buckets, positions = (args.pop(x) for x in ("table", "buckets", "positions"))
    with pytest.raises((ValueError, RuntimeError), match=match):
        relative_position_bias(table, buckets, positions, **args)


def test_what_is_no_tensor_is_refused():
    args = _good()
    with pytest.raises(TypeError, match="positions"):
        relative_position_bias(args["table"], args["buckets"], [0, 1, 2])


def test_the_module():
    m = RelativePositionBias(4, 32)
    assert m.weight.shape == (65, 4) and list(m.state_dict()) == ["weight"]
    assert RelativePositionBias(4, 128, 32, other_chain=True).weight.shape == (33, 4)
    with pytest.raises(ValueError, match="other_chain"):
        m(torch.arange(3), chains=torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="256"):
        RelativePositionBias(4, 4096, 256, other_chain=True)


def test_the_traced_operators_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        cuda = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        out = torch.ops.evoattn.relative_bias(cuda(5, 2, dtype=torch.bfloat16), cuda(5, dtype=torch.uint8), cuda(3, 6, dtype=torch.long), cuda(7, dtype=torch.long),
                                              None, None, None, torch.float16)
        assert out.shape == (3, 1, 2, 6, 7) and out.dtype == torch.float16


def _block(lib, **change):
    p = _lib.EvoRelativeBias()
    p.B, p.H, p.Nq, p.Nk, p.rows, p.reach = 2, 4, 30, 40, 65, 32
    p.dtype, p.table_dtype, p.pos_bytes = _lib.EVO_BF16, _lib.EVO_F32, 8
    for f in ("table", "lut", "pos_q", "pos_k", "out", "dout", "dtable", "workspace"):
        setattr(p, f, 0x10000)
    p.workspace_bytes = 1 << 30
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(B=0), _lib.EVO_EINVAL), (dict(Nk=-1), _lib.EVO_EINVAL), (dict(dtype=3), _lib.EVO_EINVAL), (dict(table_dtype=-1), _lib.EVO_EINVAL),
    (dict(lut=None), _lib.EVO_EINVAL), (dict(pos_bytes=2), _lib.EVO_EINVAL), (dict(chain_q=0x10000), _lib.EVO_EINVAL), (dict(rows=0), _lib.EVO_EINVAL),
    (dict(rows=257), _lib.EVO_EUNSUPPORTED), (dict(reach=4097), _lib.EVO_EUNSUPPORTED), (dict(pos_k_stride_b=-1), _lib.EVO_EINVAL),
    (dict(B=1 << 30, H=1 << 30), _lib.EVO_EOVERFLOW)])
def test_the_c_abi_rejects_before_any_launch(change, code):
    lib = _lib.load()
    p = _block(lib, **change)
    assert lib.evoattn_relative_bias_fwd(ctypes.byref(p), None) == code
    assert lib.evoattn_relative_bias_bwd(ctypes.byref(p), None) == code
    assert lib.evoattn_relative_bias_bwd_workspace_bytes(ctypes.byref(p)) == 0


def test_the_c_abi_needs_its_outputs_and_workspace():
    lib = _lib.load()
    need = lib.evoattn_relative_bias_bwd_workspace_bytes(ctypes.byref(_block(lib)))
    assert need >= 65 * 4 * 4 and need % (65 * 4 * 4) == 0
    for change, code in ((dict(dtable=None), _lib.EVO_EINVAL), (dict(dout=None), _lib.EVO_EINVAL), (dict(workspace=None), _lib.EVO_EWORKSPACE),
                         (dict(workspace_bytes=need - 1), _lib.EVO_EWORKSPACE)):
        assert lib.evoattn_relative_bias_bwd(ctypes.byref(_block(lib, **change)), None) == code, change
    assert lib.evoattn_relative_bias_fwd(ctypes.byref(_block(lib, out=None)), None) == _lib.EVO_EINVAL
    assert lib.evoattn_relative_bias_fwd(None, None) == _lib.EVO_EINVAL
