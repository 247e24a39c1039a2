"""Attention over texts of up to 2^20 positions that weigh alike: the sum of probabilities and the values' sums pass
32 bits within one stretch of the join, and saturate where the formulas say.

Results are whole numbers fixed by the formulas: every comparison is exact (tolerance 0).
"""
import numpy as np
import pytest
from test_paged import Case, Device, report

pytestmark = pytest.mark.gpu
ONE_WARP = 300  # rows of no request beside 8 heads' one: with that many CTAs each has one warp for all tiles


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def flat(rng, length, heads, pad, values):
    """All scores 0, values by element."""
    c = Case(rng, [(1, length)], heads, 1, 16, 64, pad=pad)
    c.k[:], c.q[:] = 0, 0
    c.v[:] = np.array(values, np.int16)
    return c


def raise_from(c, position, score):
    """Scores from `position` on are `score` / 256 higher for the last head, by less for the ones before: the
    running maximum moves there, and what was summed up is scaled down to different degrees."""
    p = np.arange(position, int(c.lengths[0]))
    c.k[c.table[0][p // 64], :, p % 64, 0] += score
    c.q[0, :, 0] = 1024 * np.arange(1, c.heads + 1) // c.heads  # up to 4.0, by 1 / sqrt(16)


def check(llmx, torch, oracle, c):
    d = Device(llmx, torch, c, block=1)
    d.call()
    got, want = d.result(), c.want(oracle)
    assert np.array_equal(got, want), report(got, want)
    d.p.error()
    d.p.close()
    return got[0]


SMALL = [1, 20, -20, 7, 0, -1, 13, 2] * 2
TINY = [1, -1, 0, 0, 1, 1, -1, -1] * 2  # no sum of these leaves 32 bits


@pytest.mark.parametrize("length", [32704, 32768, 32832, 40000, 65472, 65536, 65600, 100000, 131072, 131136, 262144])
@pytest.mark.parametrize("rise", [None, 2000])
def test_flat_by_one_warp(llmx, torch, oracle, length, rise):
    """From 512 tiles in a stretch on the sum of probabilities passes 2^31, from 1024 on 2^32, from 2048 on 2^33."""
    c = flat(np.random.default_rng(1), length, 8, ONE_WARP, SMALL)
    if rise:
        raise_from(c, length - 1, rise)
    out = check(llmx, torch, oracle, c)
    assert (out != 0).any() == bool(rise)  # a saturated sum's reciprocal is 0; scaled down it is not


@pytest.mark.parametrize("values", [SMALL, TINY])
@pytest.mark.parametrize("heads,pad", [(1, 0), (8, 0), (8, ONE_WARP)])
def test_longest(llmx, torch, oracle, heads, pad, values):
    """2^20 positions, the most that a request may have: 1024 tiles a warp, or 16384."""
    c = flat(np.random.default_rng(2), 2**20, heads, pad, values)
    check(llmx, torch, oracle, c)
    raise_from(c, 2**20 - 100, 1800)
    check(llmx, torch, oracle, c)


@pytest.mark.parametrize("scores", [(500, 500, 500), (100, 100, 1800)])
def test_flat_stretches(llmx, torch, oracle, scores):
    """Long flat stretches between rises, so that sums that passed 32 bits are scaled and added to again."""
    c = flat(np.random.default_rng(3), 200000, 8, ONE_WARP, SMALL)
    for position, score in zip((70000, 150016, 199990), scores):
        raise_from(c, position, score)
    out = check(llmx, torch, oracle, c)
    assert (out != 0).any() == (scores[-1] == 1800)


# a tile's values saturate from 512 on (64 * 512 = 2^15)
LARGE = [700, -700, 511, -511, 512, -512, 600, -600, 32767, -32768, 300, -300, 0, 1, -1, 450]


@pytest.mark.parametrize("length", [16384, 16448, 16512, 24000, 32704, 40000])
@pytest.mark.parametrize("score", [None, 1000, 2000])
def test_large_values_by_one_warp(llmx, torch, oracle, length, score):
    """From 257 tiles in a stretch on the values' sums pass 2^31, from nothing up or down."""
    c = flat(np.random.default_rng(4), length, 8, ONE_WARP, LARGE)
    if score:
        raise_from(c, length - 1, score)
    out = check(llmx, torch, oracle, c)
    assert (out != 0).any() or score != 2000


@pytest.mark.parametrize("then,rise,last", [(500, 1024, 1000), (450, 600, 1440)])
@pytest.mark.parametrize("first", [10, 260, 300])
@pytest.mark.parametrize("values", [LARGE, [700] * 16, [-700] * 16])
def test_values_that_turn(llmx, torch, oracle, values, first, then, rise, last):
    """Sums below 0 that a stretch takes beyond 2^31, and the other way round."""
    c = flat(np.random.default_rng(5), (first + then) * 64, 8, ONE_WARP, values)
    p = np.arange(first * 64)
    c.v[c.table[0][p // 64], :, p % 64] = -np.clip(np.array(values, np.int32), -32767, 32767).astype(np.int16)
    raise_from(c, first * 64, rise)
    raise_from(c, (first + then) * 64 - 1, last)
    out = check(llmx, torch, oracle, c)
    assert (out != 0).any() or last == 1000


@pytest.mark.parametrize("heads,pad", [(1, 0), (8, ONE_WARP)])
def test_longest_with_large_values(llmx, torch, oracle, heads, pad):
    c = flat(np.random.default_rng(6), 2**20, heads, pad, LARGE)
    check(llmx, torch, oracle, c)
    raise_from(c, 2**20 - 1, 2000)
    check(llmx, torch, oracle, c)
