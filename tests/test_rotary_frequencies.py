"""CPU: frequencies mixed for long contexts, against numbers worked out from the stated rule and not from the function."""
import math
from fractions import Fraction

import pytest

from baselinebenchmark_b200 import rotary_frequencies

#: 2 pi
TURN = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)


# Base 100, four dims: the pairs turn by 1 and by 1/10 radian a position, which is original / (2 pi) and original / (20 pi) turns within the original context.
@pytest.mark.parametrize("original,fast,slow,factor,want", [
    # 1000 / (20 pi) = 15.91549430919 turns, of which (15.91549430919 - 1) / 31 = 0.48114497771571 stays: 0.1 (0.48114497771571 + 0.51885502228429 / 4)
    (1000, 32.0, 1.0, 4.0, (1.0, 0.061085873328678)),
    # 400 / (20 pi) = 6.36619772368 turns, (6.36619772368 - 1) / 31 = 0.17310315237664; 63.66 turns of the first pair stay
    (400, 32.0, 1.0, 8.0, (1.0, 0.027646525832956)),
    # 100 / (2 pi) = 15.91549430919 turns of the first pair, 0.48114497771571 stays; the second turns 1.59154943092 times: 0.59154943092 / 31 = 0.019082239707063
    (100, 32.0, 1.0, 4.0, (0.61085873328678, 0.026431167978030)),
    # 300 / (20 pi) = 4.77464829276 turns between 2 and 10: 0.34683103659443
    (300, 10.0, 2.0, 2.0, (1.0, 0.067341551829721))])
def test_the_part_that_stays_is_linear_in_the_turns(original, fast, slow, factor, want):
    got = rotary_frequencies(4, 100.0, scaling="parts", factor=factor, original=original, fast=fast, slow=slow).tolist()
    # (the numbers have 13 digits and more)
    assert all(abs(g / w - 1) <= 1e-12 for g, w in zip(got, want))


@pytest.mark.parametrize("dim,base,original,fast,slow,factor", [(128, 10000.0, 4096, 32.0, 1.0, 16.0), (64, 500000.0, 8192, 4.0, 1.0, 8.0), (96, 10000.0, 2048, 20.0, 0.5, 3.0)])
def test_parts_in_rational_arithmetic(dim, base, original, fast, slow, factor):
    """Every pair, from its unscaled frequency in 64 bits on; three at least lie between the ends, and neither a squared ramp nor one in the pair's index passes."""
    plain = [base ** (-2 * j / dim) for j in range(dim // 2)]
    got = rotary_frequencies(dim, base, scaling="parts", factor=factor, original=original, fast=fast, slow=slow).tolist()
    between, off = 0, 0
    for j, (f, g) in enumerate(zip(plain, got)):
        f = Fraction(f)
        stay = (original * f / TURN - Fraction(slow)) / (Fraction(fast) - Fraction(slow))
        between += 0 < stay < 1
        stay = min(max(stay, Fraction(0)), Fraction(1))
        want = f * stay + f / Fraction(factor) * (1 - stay)
        # the power is off by an ulp or two (2^-52 each), the part that stays by four roundings of numbers of up to `fast` turns over their difference, the
        # rest by four
        assert abs(Fraction(g) / want - 1) <= Fraction(16 + 8 * (fast + slow) / (fast - slow)) / 2 ** 53
        squared = f * stay ** 2 + f / Fraction(factor) * (1 - stay ** 2)
        off += abs(Fraction(g) / squared - 1) > Fraction(1, 1000)
    assert between >= 3 and off >= 3
    # linear in the pair's index between the pairs of `fast` and `slow` turns: another rule
    index = [dim / 2 * math.log(original / (2 * math.pi * turns), base) for turns in (fast, slow)]
    other = [min(max((index[1] - j) / (index[1] - index[0]), 0), 1) for j in range(dim // 2)]
    assert sum(abs(g / (f * s + f / factor * (1 - s)) - 1) > 1e-3 for f, g, s in zip(plain, got, other)) >= 3
