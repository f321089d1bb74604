"""Rotary tables for scaled contexts: pairs by how often they turn over the original context."""
import math

import pytest

from gofann.kv_cache import rope_tables


def frequencies(n, **kw):
    """Angles a position, from a table of positions 0 and 1 (below pi: the fastest pair has 1)."""
    m = 0.1 * math.log(kw["factor"]) + 1.0
    cos, sin = rope_tables(2, n, scaling="parts", device="cpu", **kw)
    return [math.atan2(float(s), float(c)) for c, s in zip(cos[1] / m, sin[1] / m)]


@pytest.mark.parametrize("rotary,original,base", [(128, 131072, 10000.0), (64, 65536, 10000.0), (128, 4096, 10000.0),
                                                  (128, 8192, 500000.0), (64, 1 << 20, 10000.0), (2, 4096, 10000.0)])
def test_parts_divides_what_turns_seldom_only(rotary, original, base):
    factor, fast, slow = 4.0, 32.0, 1.0
    got = frequencies(rotary, base=base, original=original, factor=factor)
    kept = [base ** (-2 * i / rotary) for i in range(rotary // 2)]
    turns = [original * f / (2 * math.pi) for f in kept]
    # the ramp is linear in the pair index, from the last whole index at `fast` turns to the first one at `slow`
    index = lambda t: rotary * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(index(fast)), 0), math.ceil(index(slow))
    for i, (f, t) in enumerate(zip(kept, turns)):
        ramp = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
        # f32 tables: half a unit of 2^-24 on cos and on sin, which their quotient's angle shows as at most 2^-23,
        # once more for the magnitude's division
        assert abs(got[i] - (f * (1 - ramp) + f / factor * ramp)) < 2.0 ** -22, (i, t)
        if t > fast:
            assert abs(got[i] - f) < 2.0 ** -22 + f / max(hi - lo, 1)  # (the whole index before it at the most)
        if t > slow * base ** (2.0 / rotary):  # more than one index before the ramp's end: not fully divided
            assert got[i] > f / factor + 0.5 * f * (1 - 1 / factor) / (hi - lo) - 2.0 ** -22
