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
