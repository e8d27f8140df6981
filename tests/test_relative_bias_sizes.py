"""The relative position bias at the largest sizes that 32 bits count, without a GPU."""
import ctypes

import pytest
import torch

from evoformer_triton_amd import _lib, relative_buckets, relative_position_bias

MOST = 2 ** 31 - 1 - 1024


def _block(**change):
    p = _lib.EvoRelativeBias()
    p.B, p.H, p.Nq, p.Nk, p.rows, p.reach = 1, 1, 1, 1, 65, 32
    p.dtype, p.table_dtype, p.pos_bytes = _lib.EVO_BF16, _lib.EVO_F32, 8
    for f in ("table", "lut", "pos_q", "pos_k", "out", "dout", "dtable"):
        setattr(p, f, 0x10000)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("which", ["Nq", "Nk"])
def test_what_32_bits_do_not_count_is_refused(which):
    lib = _lib.load()
    for n in (MOST + 1, 2 ** 31 - 512, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1):
        p = ctypes.byref(_block(**{which: n}))
        assert lib.evoattn_relative_bias_bwd_workspace_bytes(p) == 0
        assert lib.evoattn_relative_bias_bwd(p, None) == lib.evoattn_relative_bias_fwd(p, None) == _lib.EVO_EOVERFLOW
    many = ctypes.byref(_block(B=2 ** 15, H=2 ** 15, Nk=2 ** 22))             # (more workgroups than a launch has)
    assert lib.evoattn_relative_bias_bwd_workspace_bytes(many) == 0 and lib.evoattn_relative_bias_bwd(many, None) == _lib.EVO_EOVERFLOW


def test_the_largest_has_a_workspace_of_its_size():
    lib = _lib.load()
    one = 65 * 4                                                             # bytes of a sum
    most = 64 * (2 ** 24 - 1)                                                # keys of as many workgroups as a launch has
    need = lib.evoattn_relative_bias_bwd_workspace_bytes(ctypes.byref(_block(Nk=most)))
    assert need == most // 64 * one                                          # one for each 64 keys of the row
    need = lib.evoattn_relative_bias_bwd_workspace_bytes(ctypes.byref(_block(Nq=MOST)))
    assert need % one == 0 and 256 <= need // one <= 512                     # rows in as many pieces as there are workgroups
    assert lib.evoattn_relative_bias_bwd(ctypes.byref(_block(Nk=most)), None) == _lib.EVO_EWORKSPACE


@pytest.mark.parametrize("positions,keys", [(MOST + 1, 1), (1, MOST + 1), (2 ** 31 + 5, 2)])
def test_the_call_names_what_is_too_large(positions, keys):
    at = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="too many"):
        relative_position_bias(torch.zeros(5, 2), relative_buckets(2), at.expand(positions), at.expand(keys))


@pytest.mark.parametrize("keys", [False, True])
def test_positions_that_int64_does_not_hold_are_refused(keys):
    """As int64, 2^63 would be the number farthest below zero."""
    at, far = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.uint64)
    with pytest.raises(ValueError, match="uint64"):
        relative_position_bias(torch.zeros(5, 2), relative_buckets(2), *((at, far) if keys else (far, at)))
    for dtype in (torch.uint8, torch.int8, torch.uint16, torch.int16, torch.uint32, torch.int32):
        with pytest.raises(RuntimeError, match="GPU only"):
            relative_position_bias(torch.zeros(5, 2), relative_buckets(2), torch.zeros(3, dtype=dtype), at)
    with pytest.raises(RuntimeError, match="GPU only"):
        relative_position_bias(torch.zeros(5, 2), relative_buckets(2), at, at, chains=far, key_chains=far)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64], ids=str)
def test_the_bias_in_plain_operations_takes_any_whole_type(dtype):
    """Differences of a byte, or of 64 bits, that their type does not hold."""
    from evoformer_triton_amd import RelativePositionBias
    bias = RelativePositionBias(1, 3)
    bias.weight.data.copy_(torch.arange(7.0).view(7, 1))
    i = torch.iinfo(dtype)
    values = [0, 2, 100, i.max, i.max - 1, i.min]
    want = [[max(-3, min(3, a - b)) + 3.0 for b in values] for a in values]
    assert bias.plain(torch.tensor(values, dtype=dtype))[0, 0, 0].tolist() == want
