"""Attention over the paged cache by every way there is: three launches, and one by clusters of 1, 2, 4 or 8 CTAs that
hold all or a part of a request's query rows.

Which one a call takes is an estimate of its time (llmx_selftest_paged_way says it, and makes a handle take
another); results are whole numbers fixed by the formulas, so every comparison is exact (tolerance 0).
"""
import ctypes as C

import numpy as np
import pytest
from test_paged import FILL, LENGTHS, Case, Device, report

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def every_way(d):
    """The ways that the handle's calls of d's sizes can take, each in turn; the default at the end."""
    sizes = len(d.c.plan), d.longest or max(int(d.c.lengths.max()), 1)
    took = []
    for way in [0] + [16 * i + b for i in range(4) for b in range(1, 17)]:
        if d.p.selftest_way(way, *sizes) == way:
            took.append(way)
            yield way
    assert 0 in took and d.p.selftest_way(-1, *sizes) in took


def check(llmx, torch, oracle, c, want=None, **kw):
    """The ways taken; all of them give the oracle's rows, the last one where it is called twice too."""
    d = Device(llmx, torch, c, **kw)
    want = c.want(oracle) if want is None else want
    ways = []
    for way in every_way(d):
        for _ in range(2):
            d.out.fill_(FILL)
            d.call()
            got = d.result()
            assert np.array_equal(got, want), (way, report(got, want))
        ways.append(way)
    d.p.error()
    d.p.close()
    return ways


def test_null_handle(llmx):
    assert llmx.lib().llmx_selftest_paged_way(None, -1, 1, 1, C.byref(C.c_int())) == llmx.ERR_ARG


@gpu
def test_refusals(llmx):
    p, n = llmx.Paged(4, 2, 32, 16, 4, 2, 256, 512), C.c_int(77)
    for way, requests, longest in ((-2, 1, 1), (65, 1, 1), (0, 0, 1), (0, 5, 1), (0, 1, 0), (0, 1, 257)):
        assert llmx.lib().llmx_selftest_paged_way(p.h, way, requests, longest, C.byref(n)) == llmx.ERR_ARG
    assert llmx.lib().llmx_selftest_paged_way(p.h, 0, 1, 1, None) == llmx.ERR_ARG and n.value == 77
    assert p.selftest_way(16 * 3 + 1, 1, 65) == 0  # two tiles do not fill a cluster of 8
    p.close()


@gpu
@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 96, 112, 128])
def test_lengths(llmx, torch, oracle, hd):
    ways = check(llmx, torch, oracle, Case(np.random.default_rng(hd), [(1, n) for n in LENGTHS], hd=hd), block=2)
    assert ways == [0, 1, 17, 33, 49]


@gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (9, 1), (14, 2), (16, 1), (12, 4)])
@pytest.mark.parametrize("block", [1, 3, 8])
def test_heads_and_blocks(llmx, torch, oracle, heads, kv, block):
    rng = np.random.default_rng(heads * 100 + block)
    plan = [(block, 130), (max(1, block - 1), 64), (0, 40), (block, block), (1, 1), (block, block // 2), (block, 620)]
    ways = check(llmx, torch, oracle, Case(rng, plan, heads, kv, 48), block=block)
    most = -(-heads // kv * block // 8)
    assert {0, 1, 17, 33, 49, 48 + most} <= set(ways)  # (all columns in one CTA may not fit)


@gpu
@pytest.mark.parametrize("page", [8, 24, 72, 1024])
def test_pages(llmx, torch, oracle, page):
    check(llmx, torch, oracle, Case(np.random.default_rng(page), [(1, 513), (2, 100), (1, page), (3, page + 1)], 16, 2, 128, page), block=3)


@gpu
@pytest.mark.parametrize("hd,block", [(128, 1), (64, 5)])
def test_values_beyond_eight(llmx, torch, oracle, hd, block):
    rng = np.random.default_rng(4)
    c = Case(rng, [(1, 700), (block, 130), (1, 64)], 16, 2, hd, q_sigma=200, k_sigma=300, v_sigma=300)
    for pool in (c.k, c.v):
        at = rng.random(pool.shape) < 0.2
        pool[at] = rng.choice(np.array([2046, 2047, 2048, 2049, 4000, 32767, -2047, -2048, -2049, -5000, -32768], np.int16), at.sum())
    check(llmx, torch, oracle, c, block=block)


@gpu
@pytest.mark.parametrize("q,k,v", [(-32768, -32768, -32768), (32767, 32767, 32767), (-8192, -2048, 100), (-8193, 2048, 5), (0, 0, -32768)])
@pytest.mark.parametrize("hd", [128, 64])
def test_saturation(llmx, torch, oracle, q, k, v, hd):
    rng = np.random.default_rng(9)
    c = Case(rng, [(1, 64), (3, 590), (1, 1)], 8, 1, hd)
    c.q[:, ::3] = q
    c.k[::2], c.v[::2] = k, v
    check(llmx, torch, oracle, c, block=3)
    c.q[:], c.k[:], c.v[:] = q, k, v
    check(llmx, torch, oracle, c, block=3)


@gpu
@pytest.mark.parametrize("q,v", [(0, 700), (0, -700), (0, 3)])
def test_flat_up_to_the_bound(llmx, torch, oracle, q, v):
    """255 tiles, the most that clusters take, that all weigh the same."""
    rng = np.random.default_rng(11)
    c = Case(rng, [(1, 16320), (2, 16000)], 4, 2, 16, 64)
    c.q[:], c.k[:], c.v[:] = q, 0, v
    c.q[0, ::2] = 900
    c.k[c.table[0][254], :, 63, 0] = 2000  # the last position of the first
    ways = check(llmx, torch, oracle, c, block=2)
    assert 49 in ways


@gpu
def test_void_requests_and_pages(llmx, torch, oracle):
    """A length above the bound, a block above the handle's, a page out of range: reported, the others served."""
    rng = np.random.default_rng(15)
    plan = [(1, 600), (3, 550), (1, 577), (1, 530)]
    for spoil, void in (("length", [1]), ("block", [1, 2]), ("page", [2])):
        c = Case(rng, plan, 8, 2, 32)
        want = c.want(oracle)
        d = Device(llmx, torch, c, block=3)
        if spoil == "length":
            d.lengths[1] = 601
        elif spoil == "block":
            d.offsets[2] = 5  # request 1: 4 rows, request 2: none
        else:
            d.table[2, 36] = c.pages
        n = 0
        for way in every_way(d):
            d.out.fill_(FILL)
            d.call()
            got = d.result()
            for b, (rows, _) in enumerate(plan):
                mine = slice(int(c.offsets[b]), int(c.offsets[b]) + rows)
                if b not in void:
                    assert np.array_equal(got[mine], want[mine]), (way, spoil, b)
                elif spoil != "page":
                    assert (got[mine] == FILL).all(), (way, spoil, b)
            with pytest.raises(llmx.LlmxError) as e:
                d.p.error()
            assert e.value.code == llmx.ERR_RANGE
            d.p.error()
            n += 1
        assert n >= 5


@gpu
def test_more_positions_than_reserved(llmx, torch):
    rng = np.random.default_rng(17)
    c = Case(rng, [(1, 1000)] * 4, 8, 2, 32)
    d = Device(llmx, torch, c, positions=1000)
    for way in every_way(d):
        d.call()
        assert (d.result() == FILL).all(), way
        with pytest.raises(llmx.LlmxError) as e:
            d.p.error()
        assert e.value.code == llmx.ERR_RANGE


@gpu
def test_graph(llmx, torch, oracle):
    """Captured by each way, replayed over other lengths, tables and queries."""
    rng = np.random.default_rng(18)
    cases = [Case(rng, p, 16, 2, 64) for p in ([(2, 520), (1, 64), (1, 300)], [(1, 5), (2, 590), (1, 200)], [(0, 9), (4, 600), (0, 0)])]
    d = Device(llmx, torch, Case(rng, [(4, 600)] * 3, 16, 2, 64), longest=600, positions=1800, block=4)
    for way in every_way(d):
        d.call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            d.call()
        for c in cases + cases[:1]:
            n = Device(llmx, torch, c, handle=d.p)
            d.offsets.copy_(n.offsets)
            d.lengths.copy_(n.lengths)
            d.table[:, :n.table.shape[1]] = n.table
            d.k[:c.pages], d.v[:c.pages], d.q[:c.rows] = n.k, n.v, n.q
            d.out.fill_(FILL)
            graph.replay()
            got = d.result()
            assert np.array_equal(got[:c.rows], c.want(oracle)) and (got[c.rows:] == FILL).all(), way
    d.p.error()


@gpu
@pytest.mark.parametrize("bound", [16000, 20000])
def test_large_bounds_take_three_launches(llmx, bound):
    """What test_paged_long.py relies on, for its requests, heads and blocks."""
    for heads, kv, hd, requests, block in ((4, 2, 16, 24, 8), (4, 2, 128, 24, 8), (1, 1, 48, 7, 8), (16, 1, 48, 7, 8), (12, 4, 48, 7, 8), (16, 2, 128, 4, 8),
                                           (8, 1, 128, 3, 8), (8, 2, 32, 4, 3), (16, 2, 64, 3, 8), (4, 2, 16, 3, 8), (8, 2, 64, 5, 8)):
        p = llmx.Paged(heads, kv, hd, 16, requests, block, bound, 3000)
        assert p.selftest_way(-1, requests, bound) == 0, (heads, kv, hd, requests, block)
        p.close()


@gpu
@pytest.mark.parametrize("requests,split", [(4, 1), (20, 7), (70, 33), (300, 150), (1024, 1000)])
def test_offsets_out_of_order(llmx, torch, oracle, requests, split):
    """Two ascending runs of offsets: the request between them, which ends before it starts, is left out and reported, and
    every other one, whose rows nobody else claims, is served."""
    rng = np.random.default_rng(requests)
    plan = [(int(rng.integers(0, 4)), int(rng.integers(1, 90))) for _ in range(requests)]
    plan[0], plan[split], plan[-1] = (3, 200), (0, 50), (2, 150)
    c = Case(rng, plan, 4, 2, 16, 8)
    first, total = int(c.offsets[split]), c.total
    want = np.concatenate([np.roll(c.want(oracle)[:total], total - first, 0), np.full((2, 4, 16), FILL, np.int16)])
    d = Device(llmx, torch, c, block=3)
    d.q[:total] = torch.roll(d.q[:total], total - first, 0)
    # requests up to split take the rows behind the others'
    offsets = np.where(np.arange(requests + 1) <= split, c.offsets.astype(np.int64) + total - first, c.offsets.astype(np.int64) - first)
    assert offsets[split] == total and offsets[split + 1] == 0
    d.offsets.copy_(torch.from_numpy(offsets.astype(np.int32)))
    for way in every_way(d):
        d.out.fill_(FILL)
        d.call()
        got = d.result()
        assert np.array_equal(got, want), (way, report(got, want))
        with pytest.raises(llmx.LlmxError) as e:
            d.p.error()
        assert e.value.code == llmx.ERR_RANGE
