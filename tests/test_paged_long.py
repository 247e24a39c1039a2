"""Attention over the paged cache where the bound on the lengths is large: the scores of all tiles,
their values and the join are then launches of their own, whatever the lengths in the arrays are.

16000 positions are under 256 tiles of 64, 20000 above (the join keeps what each needs otherwise).
Results are whole numbers fixed by the formulas: every comparison is exact (tolerance 0).
"""
import numpy as np
import pytest
from test_paged import FILL, LENGTHS, Case, Device, report

pytestmark = pytest.mark.gpu
BOUNDS = pytest.mark.parametrize("bound", [16000, 20000])


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def widen(c, bound):
    """Tables as wide as the bound asks for; what is not used holds numbers of no page."""
    more = -(-bound // c.page) - c.table.shape[1]
    if more > 0:
        c.table = np.pad(c.table, ((0, 0), (0, more)), constant_values=-1)
    return c


def device(llmx, torch, c, bound, **kw):
    return Device(llmx, torch, widen(c, bound), longest=bound, **kw)


def check(llmx, torch, oracle, c, bound, **kw):
    d = device(llmx, torch, c, bound, **kw)
    d.call()
    got, want = d.result(), c.want(oracle)
    assert np.array_equal(got, want), report(got, want)
    d.p.error()
    d.p.close()


@BOUNDS
@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 96, 112, 128])
def test_lengths(llmx, torch, oracle, hd, bound):
    check(llmx, torch, oracle, Case(np.random.default_rng(hd), [(1, n) for n in LENGTHS], hd=hd), bound)


@BOUNDS
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (3, 3), (8, 1), (9, 1), (14, 2), (16, 2), (16, 1), (12, 4)])
@pytest.mark.parametrize("block", [1, 3, 8])
def test_heads_and_blocks(llmx, torch, oracle, heads, kv, block, bound):
    rng = np.random.default_rng(heads * 100 + block)
    plan = [(block, 130), (max(1, block - 1), 64), (0, 40), (block, block), (1, 1), (block, block // 2), (block, 300)]
    check(llmx, torch, oracle, Case(rng, plan, heads, kv, 48), bound)


@BOUNDS
@pytest.mark.parametrize("page", [8, 24, 64, 72, 200, 1024])
def test_pages(llmx, torch, oracle, page, bound):
    check(llmx, torch, oracle, Case(np.random.default_rng(page), [(1, 513), (2, 100), (1, page), (3, page + 1)], 16, 2, 128, page), bound)


@BOUNDS
@pytest.mark.parametrize("seed", range(6))
def test_drawn(llmx, torch, oracle, seed, bound):
    rng = np.random.default_rng(100 + seed)
    kv, g, hd = int(rng.integers(1, 5)), int(rng.integers(1, 9)), 16 * int(rng.integers(1, 9))
    plan = [(int(rng.integers(0, 9)), int(rng.integers(0, 700))) for _ in range(int(rng.integers(1, 40)))]
    c = Case(rng, plan, kv * g, kv, hd, 8 * int(rng.integers(1, 9)), pad=int(rng.integers(0, 4)))
    check(llmx, torch, oracle, c, bound, extra=8 * int(rng.integers(0, 3)))


@pytest.mark.parametrize("requests", [33, 128, 300, 1024])
def test_many_requests(llmx, torch, oracle, requests):
    rng = np.random.default_rng(requests)
    plan = [(int(rng.integers(0, 3)), int(rng.integers(0, 90))) for _ in range(requests)]
    check(llmx, torch, oracle, Case(rng, plan, 4, 2, 16, 8), 16400, block=2)


@BOUNDS
def test_values_beyond_eight(llmx, torch, oracle, bound):
    rng = np.random.default_rng(4)
    c = Case(rng, [(1, 200), (4, 130), (2, 64)], 16, 2, 128, q_sigma=200, k_sigma=300, v_sigma=300)
    for pool in (c.k, c.v):
        at = rng.random(pool.shape) < 0.2
        pool[at] = rng.choice(np.array([2046, 2047, 2048, 2049, 4000, 32767, -2047, -2048, -2049, -5000, -32768], np.int16), at.sum())
    check(llmx, torch, oracle, c, bound)


@BOUNDS
@pytest.mark.parametrize("q,k,v", [(-32768, -32768, -32768), (32767, 32767, 32767), (-32768, 32767, 32767), (32767, -32768, -32768),
                                   (-8192, -2048, 100), (-8192, -32768, 2048), (8191, -2048, -2048), (-8193, 2048, 5), (8192, 2047, 2047),
                                   (0, 0, 32767), (0, 0, -32768)])
@pytest.mark.parametrize("hd", [128, 64])
def test_saturation(llmx, torch, oracle, q, k, v, hd, bound):
    rng = np.random.default_rng(9)
    c = Case(rng, [(1, 64), (3, 190), (1, 1)], 8, 1, hd)
    c.q[:, ::3] = q
    c.k[::2], c.v[::2] = k, v
    check(llmx, torch, oracle, c, bound)
    c.q[:], c.k[:], c.v[:] = q, k, v
    check(llmx, torch, oracle, c, bound)


@BOUNDS
def test_wide_queries_in_one_place(llmx, torch, oracle, bound):
    rng = np.random.default_rng(10)
    c = Case(rng, [(2, 150), (1, 40)], 16, 2, 128, k_sigma=2500)
    for r, h, e, x in ((0, 0, 0, -8192), (0, 3, 127, 32767), (1, 8, 64, -32768), (2, 15, 5, 8192)):
        c.q[r, h, e] = x
    c.q[1, 4] = rng.integers(-32768, 32767, 128)
    check(llmx, torch, oracle, c, bound)


@BOUNDS
def test_rising_scores(llmx, torch, oracle, bound):
    """The maximum moves in every tile of one head, in none of another; a third stays at one value."""
    rng = np.random.default_rng(11)
    c = Case(rng, [(1, 15900), (2, 5000), (1, 4097)], 4, 2, 16, 64)
    pos = np.arange(15900)
    c.q[0] = 0
    c.k[c.table[0][pos // 64], 1, pos % 64] = 0
    c.k[c.table[0][pos // 64], 1, pos % 64, 0] = (pos // 16 - 500).astype(np.int16)
    c.q[0, 2, 0], c.q[0, 3, 0] = 512, -512
    c.v[c.table[0][pos // 64], 0, pos % 64, :8] = 700
    check(llmx, torch, oracle, c, bound)


@BOUNDS
def test_void_requests_and_pages(llmx, torch, oracle, bound):
    """A length above the bound, a block above the handle's, a page out of range: reported, the others served."""
    rng = np.random.default_rng(15)
    plan = [(1, 100), (3, 50), (1, 77), (1, 30)]
    for spoil, void in (("length", [1]), ("block", [1, 2]), ("page", [2])):
        c = Case(rng, plan, 8, 2, 32)
        want = c.want(oracle)
        d = device(llmx, torch, c, bound, block=3)
        if spoil == "length":
            d.lengths[1] = bound + 1
        elif spoil == "block":
            d.offsets[2] = 5  # request 1: 4 rows, request 2: none
        else:
            d.table[2, 3] = c.pages
        d.call()
        got = d.result()
        for b, (rows, _) in enumerate(plan):
            mine = slice(int(c.offsets[b]), int(c.offsets[b]) + rows)
            if b not in void:
                assert np.array_equal(got[mine], want[mine]), (spoil, b)
            elif spoil != "page":
                assert (got[mine] == FILL).all(), (spoil, b)
        with pytest.raises(llmx.LlmxError) as e:
            d.p.error()
        assert e.value.code == llmx.ERR_RANGE
        d.p.error()
        d.p.close()


@BOUNDS
def test_more_positions_than_reserved(llmx, torch, bound):
    rng = np.random.default_rng(17)
    c = Case(rng, [(1, 9000)] * 4, 8, 2, 32)
    d = device(llmx, torch, c, bound, positions=9000)
    d.call()
    assert (d.result() == FILL).all()
    with pytest.raises(llmx.LlmxError) as e:
        d.p.error()
    assert e.value.code == llmx.ERR_RANGE


def test_one_handle_by_every_way(llmx, torch, oracle):
    """Calls whose bounds lead to one launch and to three, in turn and with one handle."""
    rng = np.random.default_rng(14)
    big = widen(Case(rng, [(8, 700)] * 5, 8, 2, 64), 20000)
    d = Device(llmx, torch, big, longest=20000, positions=4 * 700 * 5)
    for i, plan in enumerate(([(1, 3)], [(2, 70), (1, 999)], [(0, 0), (1, 0)], [(8, 700)] * 5, [(1, 1000)] * 4)):
        for bound in (0, 16000, 20000, 0)[i % 2:]:
            c = Case(rng, plan, 8, 2, 64)
            e = Device(llmx, torch, widen(c, bound or 1), longest=bound, handle=d.p)
            e.call()
            got, want = e.result(), c.want(oracle)
            assert np.array_equal(got, want), (bound, report(got, want))
    d.p.error()
    d.p.close()


@BOUNDS
def test_graph(llmx, torch, oracle, bound):
    """Captured once on a stream of its own, replayed over other lengths, tables and queries, an eager call between."""
    rng = np.random.default_rng(18)
    cases = [Case(rng, p, 16, 2, 64) for p in ([(2, 120), (1, 64), (1, 300)], [(1, 5), (2, 290), (1, 200)], [(0, 9), (4, 300), (0, 0)])]
    d = device(llmx, torch, Case(rng, [(4, 300)] * 3, 16, 2, 64), bound, positions=900)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.call()
    for c in cases + cases[:1]:
        n = Device(llmx, torch, widen(c, bound), longest=bound, handle=d.p)
        n.call()
        assert np.array_equal(n.result(), c.want(oracle))
        d.offsets.copy_(n.offsets)
        d.lengths.copy_(n.lengths)
        d.table[:, :n.table.shape[1]] = n.table
        d.k[:c.pages], d.v[:c.pages], d.q[:c.rows] = n.k, n.v, n.q
        d.out.fill_(FILL)
        graph.replay()
        got = d.result()
        assert np.array_equal(got[:c.rows], c.want(oracle)) and (got[c.rows:] == FILL).all()


@pytest.mark.parametrize("plan", [[(1, 32768)], [(1, 30000), (8, 16385)], [(1, 9000)] * 9])
def test_long_texts(llmx, torch, oracle, plan):
    rng = np.random.default_rng(len(plan))
    c = Case(rng, plan, 8, 1, 32, 64)
    d = Device(llmx, torch, c)
    d.call()
    got, want = d.result(), c.want(oracle)
    assert np.array_equal(got, want), report(got, want)
