"""Weights held in 8 bits, without a GPU: which types of a byte they may have."""
import pytest
import torch

from evoformer_triton_amd import Fp8Weight, fp8_linear

OTHERS = (torch.int8, torch.bool, torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz)


def _weight(values, scales):
    return Fp8Weight(torch.zeros(4, 384, dtype=torch.uint8).view(values), torch.full((4, 4), 127, dtype=torch.uint8).view(scales), 300)


@pytest.mark.parametrize("which", ["values", "scales"])
@pytest.mark.parametrize("dtype", OTHERS + (torch.float8_e4m3fn, torch.float8_e8m0fnu), ids=str)
def test_other_numbers_of_a_byte_are_refused(which, dtype):
    """They would be read as e4m3, or as a power of two, which they are not."""
    if (which, dtype) in (("values", torch.float8_e4m3fn), ("scales", torch.float8_e8m0fnu)):
        return
    w = _weight(*((dtype, torch.uint8) if which == "values" else (torch.float8_e4m3fn, dtype)))
    for call in (lambda: fp8_linear(torch.zeros(2, 300), w), w.dequantize):
        with pytest.raises(ValueError, match="8 bits"):
            call()


@pytest.mark.parametrize("values", [torch.uint8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("scales", [torch.uint8, torch.float8_e8m0fnu], ids=str)
def test_their_own_types_are_taken(values, scales):
    w = _weight(values, scales)
    assert w.dequantize().shape == (4, 300)
    with pytest.raises(RuntimeError, match="GPU only"):
        fp8_linear(torch.zeros(2, 300), w)
