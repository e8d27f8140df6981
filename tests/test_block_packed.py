"""The block's rotary positions and packed rows without a GPU: what it keeps, what it refuses, its plain form."""
import copy

import pytest
import torch

from evoformer_triton_amd import RotaryPositions
from evoformer_triton_amd.block import GatedAttentionBlock


def test_options_and_refusals():
    plain, block = GatedAttentionBlock(64, 32, 4), GatedAttentionBlock(64, 32, 4, rotary=RotaryPositions(32))
    assert set(block.state_dict()) == set(plain.state_dict())
    with pytest.raises(ValueError, match="head dim"):
        GatedAttentionBlock(64, 32, 4, rotary=RotaryPositions(64))
    m, at = torch.randn(1, 2, 5, 64), torch.arange(5)
    with pytest.raises(ValueError, match="needs the residues' positions"):
        block(m)
    with pytest.raises(ValueError, match="rotary"):
        plain(m, positions=at)
    with pytest.raises(ValueError, match="other_chain"):
        block(m, positions=at, chains=at)
    rows, off = torch.randn(5, 64), torch.tensor([0, 5])
    for b, args, error, match in ((block, (m, off), ValueError, "packed rows"), (GatedAttentionBlock(64, 32, 4, relative_distance=4), (rows, off), ValueError, "relative"),
                                  (plain, (rows, off, at), ValueError, "rotary"), (block, (rows, off), RuntimeError, "GPU only"), (plain, (rows, off), RuntimeError, "GPU only"),
                                  (block, (rows, off, None, False, object()), ValueError, "fp8")):
        with pytest.raises(error, match=match.replace("GPU only", "GPU")):
            b.packed(*args)


def test_a_block_saved_without_the_option():
    old = copy.deepcopy(GatedAttentionBlock(16, 8, 2))
    del old.__dict__["rotary"]
    m = torch.randn(1, 1, 4, 16)
    assert old.forward_eager(m).shape == m.shape
    with pytest.raises(ValueError, match="rotary"):
        old.forward_eager(m, positions=torch.arange(4))
    with pytest.raises(RuntimeError, match="GPU"):
        old.packed(m[0, 0], torch.tensor([0, 4]))


def test_only_differences_of_positions_count():
    torch.manual_seed(0)
    block = GatedAttentionBlock(16, 8, 2, rotary=RotaryPositions(8)).double()
    m, at = torch.randn(1, 2, 6, 16, dtype=torch.float64), torch.arange(6)
    y = block.forward_eager(m, positions=at)
    # (the softmax of the plain form is in fp32)
    assert torch.allclose(block.forward_eager(m, positions=at + 1000), y, rtol=0, atol=1e-5) and not torch.allclose(block.forward_eager(m, positions=2 * at), y, rtol=0, atol=1e-3)
