"""Frequencies, the plain form and the refusals of rotary positions, without a GPU."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

from evoformer_triton_amd import RotaryPositions, _lib, rotary_positions, rotary_turns


def _radians(turns):
    return [float(Fraction(int(t) % 2 ** 64, 2 ** 64)) * 2 * math.pi for t in turns]


def test_frequencies():
    """A frequency is a whole number of 2^-64 turns: half of one off, 2^-65 * 2 pi = 1.7e-19 radians, beside the arithmetic's 2^-53."""
    for R, base in ((2, 10000.0), (64, 10000.0), (128, 500000.0), (24, 100.0)):
        for x, i in zip(_radians(rotary_turns(R, base)), range(R // 2)):
            assert math.isclose(x, base ** (-2 * i / R), rel_tol=1e-14, abs_tol=2e-19)
    plain = _radians(rotary_turns(64))
    for x, y in zip(_radians(rotary_turns(64, scaling="linear", factor=8.0)), plain):
        assert math.isclose(x, y / 8, rel_tol=1e-14, abs_tol=2e-19)
    wide = _radians(rotary_turns(64, scaling="base", factor=8.0))
    assert math.isclose(wide[0], plain[0], rel_tol=1e-14, abs_tol=2e-19) and math.isclose(wide[-1], plain[-1] / 8, rel_tol=1e-12, abs_tol=2e-19)
    parts = _radians(rotary_turns(64, scaling="parts", factor=8.0, original_length=4096))
    for x, y in zip(parts, plain):
        r = 4096 * y / (2 * math.pi)
        keep = 1.0 if r >= 32 else 0.0 if r <= 1 else (r - 1) / 31
        assert math.isclose(x, y * keep + y / 8 * (1 - keep), rel_tol=1e-13, abs_tol=2e-19)
    # a frequency of a turn or more is its fraction: positions are whole
    assert math.isclose(_radians(rotary_turns(4, base=0.01))[1], math.fmod(10.0, 2 * math.pi), rel_tol=1e-13, abs_tol=2e-19)
    with pytest.raises(ValueError):
        rotary_turns(3)
    for kw in ({"scaling": "other"}, {"factor": 2.0}, {"scaling": "parts", "factor": 2.0}, {"scaling": "linear", "factor": 0.0},
               {"scaling": "parts", "factor": 2.0, "original_length": 100, "fast": 1.0}, {"base": -1.0}, {"base": math.inf}):
        with pytest.raises(ValueError):
            rotary_turns(8, **kw)
    with pytest.raises(ValueError):
        rotary_turns(2, scaling="base", factor=2.0)


def test_the_module():
    r = RotaryPositions(8, 4, scaling="parts", factor=4.0, original_length=64)
    assert math.isclose(r.magnitude, 0.1 * math.log(4.0) + 1.0) and RotaryPositions(8, scaling="linear", factor=4.0).magnitude == 1.0
    kept = r.turns.clone()
    assert torch.equal(r.to(torch.bfloat16).turns, kept) and not r.state_dict()
    with pytest.raises(ValueError, match="at most the head dim"):
        RotaryPositions(8, 10)


def test_the_plain_form():
    x = torch.randn(2, 3, 5, 2, 6, dtype=torch.float64)
    at = torch.tensor([[0, 1, 2, 3, 10 ** 9], [5, 4, -3, 2, 1]])
    for interleaved in (False, True):
        r = RotaryPositions(6, 4, interleaved=interleaved)
        y = r.plain(x, None, at)
        for b in range(2):
            for n in range(5):
                for p, w in enumerate((1.0, 0.01)):
                    i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + 2)
                    turn = Fraction(int(at[b, n]) * (int(r.turns[p]) % 2 ** 64) % 2 ** 64, 2 ** 64)
                    a = float(turn) * 2 * math.pi
                    if abs(int(at[b, n])) < 100:
                        assert math.isclose(math.cos(a), math.cos(int(at[b, n]) * w), abs_tol=1e-12)
                    u, v = x[b, :, n, :, i], x[b, :, n, :, j]
                    assert torch.allclose(y[b, :, n, :, i], u * math.cos(a) - v * math.sin(a), atol=1e-12)
                    assert torch.allclose(y[b, :, n, :, j], v * math.cos(a) + u * math.sin(a), atol=1e-12)
        assert torch.equal(y[..., 4:], x[..., 4:])
        both = r.plain(x, x[..., :1, :], at)
        assert torch.equal(both[0], y) and torch.equal(both[1], y[..., :1, :])
        assert torch.equal(r.plain(x[0, 0], None, at[0]), y[0, 0])


def test_refusals():
    q, turns, at = torch.zeros(6, 4, 8), rotary_turns(8), torch.arange(6)
    for args, what in (
            ((q[0], None, at, turns), r"\[N,H,D\]"),
            ((q.double(), None, at, turns), "bf16, fp16 or fp32"),
            ((q, q.half(), at, turns), "queries' dtype"),
            ((q, q[:5], at, turns), "but for the heads"),
            ((q, q[None], at, turns), "but for the heads"),
            ((q, None, at, turns.float()), "turns must be int64"),
            ((q, None, at, torch.zeros(5, dtype=torch.int64)), "turns must be int64"),
            ((q, None, at.float(), turns), "whole numbers"),
            ((q, None, at.to(torch.uint64), turns), "whole numbers"),
            ((q, None, at[:5], turns), r"\[N\] or \[B, N\]"),
            ((q, None, at.expand(2, 6), turns), r"\[N\] or \[B, N\]"),
            ((q[None], None, at.expand(2, 6), turns), r"\[N\] or \[B, N\]")):
        with pytest.raises(ValueError, match=what):
            rotary_positions(*args)
    with pytest.raises(ValueError, match="finite"):
        rotary_positions(q, None, at, turns, scale=float("nan"))
    with pytest.raises(TypeError, match="positions must be a tensor"):
        rotary_positions(q, None, list(range(6)), turns)
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary_positions(q, None, at, turns)


def test_the_c_entry_point_refuses():
    lib = _lib.load()

    def block(**change):
        p = _lib.EvoRotary()
        p.B, p.S, p.N, p.H, p.Hk, p.D, p.R, p.dtype, p.pos_bytes, p.scale = 1, 1, 10, 4, 2, 32, 32, _lib.EVO_BF16, 8, 1.0
        for f in ("pos", "turns", "q", "k", "out_q", "out_k"):
            setattr(p, f, 0x10000)    # (never dereferenced by the host-side checks)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.evoattn_rotary(ctypes.byref(p), None)

    for change, code in (({"R": 3}, _lib.EVO_EINVAL), ({"R": 34}, _lib.EVO_EINVAL), ({"R": 0}, _lib.EVO_EINVAL), ({"dtype": 9}, _lib.EVO_EINVAL),
                         ({"pos_bytes": 2}, _lib.EVO_EINVAL), ({"q": None}, _lib.EVO_EINVAL), ({"out_k": None}, _lib.EVO_EINVAL), ({"pos": None}, _lib.EVO_EINVAL),
                         ({"N": 0}, _lib.EVO_OK), ({"H": 0, "Hk": 0}, _lib.EVO_OK),
                         ({"B": 1 << 20, "S": 1 << 20}, _lib.EVO_EOVERFLOW), ({"N": 2 ** 31 - 1, "H": 2 ** 20}, _lib.EVO_EOVERFLOW)):
        assert block(**change) == code, change
    assert lib.evoattn_rotary(None, None) == _lib.EVO_EINVAL
