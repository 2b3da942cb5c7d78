"""YaRN's frequencies for contexts whose correction range reaches past the last pair:
its upper end is cut at dim - 1 (Peng et al., "YaRN: Efficient Context Window Extension
of Large Language Models", 2023, and its published code), not at the last pair."""
import math

import pytest

from tests.test_latent_args import table


def by_definition(dim, base, factor, orig, fast, slow):
    """Each pair turns r times in the original context; between the dimensions of `fast` and
    `slow` turns its frequency goes from kept to divided by factor."""
    def dimension(turns):
        return dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(dimension(fast)), 0), min(math.ceil(dimension(slow)), dim - 1)
    if high <= low:
        high = low + 1
    out = []
    for i in range(dim // 2):
        f = 1.0 / base ** (2 * i / dim)
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        out.append(f / factor * ramp + f * (1.0 - ramp))
    return out, high


@pytest.mark.parametrize("dim,base,factor,orig,fast,slow,past", [
    (64, 10000.0, 40.0, 4096, 32.0, 1.0, False),   # the range ends at pair 23
    (64, 10000.0, 4.0, 65536, 32.0, 1.0, True),    # at 33 of 32 pairs
    (64, 10000.0, 8.0, 131072, 32.0, 1.0, True),
    (128, 10000.0, 2.0, 1 << 20, 32.0, 1.0, True),
    (64, 500.0, 4.0, 1 << 24, 32.0, 1.0, True),    # cut at dim - 1
    (4, 10000.0, 40.0, 4096, 32.0, 1.0, True),
    (256, 1e6, 4.0, 32768, 32.0, 1.0, False),
])
def test_the_ramp_ends_where_the_method_ends_it(dim, base, factor, orig, fast, slow, past):
    want, high = by_definition(dim, base, factor, orig, fast, slow)
    assert (high > dim // 2 - 1) == past
    rc, t = table(dim, scaling=2, orig=orig, base=base, factor=factor, fast=fast, slow=slow)
    assert rc == 0
    for i, w in enumerate(want):
        got = t.turns[i] / 2.0 ** 64 * 2.0 * math.pi
        # doubles: a few roundings, the power's exponent off by one of its own (ln base of it); the table: cut to 2^-64 of a turn
        assert abs(got - w) < 2.0 ** -46 * w + 2.0 ** -64 * 2.0 * math.pi, i
