"""Rotary frequencies to their last bit: whole numbers of 2^-64 turns that are off by no more than a half (and a hundredth), by exact arithmetic.  At position 2^38 an angle is then off by 2^-27 of a turn."""
from fractions import Fraction

import pytest

from evoformer_triton_amd import rotary_turns


def _two_pi():
    """Between two fractions 10^-90 apart: 8 (4 atan(1/5) - atan(1/239)), whole-numbered series."""
    one = 10 ** 100

    def atan(n):
        total, term, k = 0, one // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    pi8 = 8 * (4 * atan(5) - atan(239))
    return Fraction(pi8 - 10 ** 10, one), Fraction(pi8 + 10 ** 10, one)


LEAST, MOST = _two_pi()
HALF = Fraction(51, 100)


def _bounds(t):
    """What a frequency in radians lies between if `t` is its nearest whole number of 2^-64 turns."""
    t = int(t) % 2 ** 64
    return (t - HALF) * LEAST / 2 ** 64, (t + HALF) * MOST / 2 ** 64


@pytest.mark.parametrize("R,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (24, 100.0), (32, 1234.5678), (48, 1e6)])
def test_every_pair(R, base):
    n = R // 2
    for i, t in enumerate(rotary_turns(R, base)):        # x^n = base^-i
        low, high = _bounds(t)
        assert low ** n < Fraction(base) ** -i < high ** n, i


def test_scaled():
    R, n, factor, base = 64, 32, 8.0, 10000.0
    for i, t in enumerate(rotary_turns(R, base, scaling="linear", factor=factor)):
        low, high = _bounds(t)
        assert (low * 8) ** n < Fraction(base) ** -i < (high * 8) ** n, i
    R, n = 16, 8
    for i, t in enumerate(rotary_turns(R, base, scaling="base", factor=factor)):      # x = base^(-i / n) factor^(-i / (n - 1))
        low, high = _bounds(t)
        m = n * (n - 1)
        assert low ** m < Fraction(base) ** (-i * (n - 1)) * 8 ** (-i * n) < high ** m, i
    R, length = 64, 4096
    plain = rotary_turns(R, base)
    for i, t in enumerate(rotary_turns(R, base, scaling="parts", factor=factor, original_length=length)):
        def scaled(turns):           # of a plain frequency in turns, which is known to 2^-65: rising with it
            keep = min(Fraction(1), max(Fraction(0), (length * turns - 1) / 31))
            return turns * (keep + (1 - keep) / 8)

        x = int(plain[i])
        low, high = scaled(Fraction(x) / 2 ** 64 - HALF / 2 ** 64), scaled(Fraction(x) / 2 ** 64 + HALF / 2 ** 64)
        assert low * 2 ** 64 - HALF <= int(t) <= high * 2 ** 64 + HALF, i


def test_frequencies_of_many_turns():
    """A base below one: of 2^60 radians the fraction of a turn counts."""
    whole = rotary_turns(4, base=2.0 ** -120)
    turns = 2 ** 60 / ((LEAST + MOST) / 2)
    assert abs(Fraction(int(whole[1]) % 2 ** 64, 2 ** 64) - turns % 1) <= HALF / 2 ** 64
