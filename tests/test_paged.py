"""The key-value cache in pages (llmx_paged_*): append and attention.

Results are whole numbers fixed by the formulas, so every comparison with the 64-bit
implementation (the oracle's attention, one sequence at a time) is exact (tolerance 0).
"""
import ctypes as C

import numpy as np
import pytest

gpu = pytest.mark.gpu
FILL = 777


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


class Case:
    """Requests of a step: plan is (rows, length) of each."""

    def __init__(self, rng, plan, heads=4, kv=2, hd=32, page=16, q_sigma=330, k_sigma=500, v_sigma=300, pad=2, spare=3):
        self.plan, self.heads, self.kv, self.hd, self.page = plan, heads, kv, hd, page
        self.offsets = np.concatenate([[0], np.cumsum([r for r, _ in plan])]).astype(np.uint32)
        self.lengths = np.array([n for _, n in plan], np.uint32)
        self.total = int(self.offsets[-1])
        self.rows = self.total + pad
        need = [-(-n // page) for _, n in plan]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(plan), max(need) + 1), -1, np.int32)
        self.table[:, -1] = 2**31 - 1  # entries that no position uses may hold anything
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        draw = lambda shape, sigma: np.clip(np.rint(rng.normal(0, sigma, shape)), -32768, 32767).astype(np.int16)  # noqa: E731
        self.k, self.v = draw((self.pages, kv, page, hd), k_sigma), draw((self.pages, kv, page, hd), v_sigma)
        self.q = draw((self.rows, heads, hd), q_sigma)

    def cache(self, b, pool):
        """[length][kv][hd] of request b."""
        p = np.arange(self.lengths[b])
        return pool[self.table[b][p // self.page], :, p % self.page]

    def want(self, O):
        out = np.full((self.rows, self.heads, self.hd), FILL, np.int16)
        g = self.heads // self.kv
        for b, (rows, length) in enumerate(self.plan):
            k, v = self.cache(b, self.k), self.cache(b, self.v)
            for j in range(rows):
                seen = max(length - rows + 1 + j, 0)
                r = int(self.offsets[b]) + j
                for h in range(self.kv):
                    out[r, h * g:(h + 1) * g] = O.attention_group(self.q[r, h * g:(h + 1) * g], k[:seen, h], v[:seen, h])
        return out


class Device:
    def __init__(self, llmx, torch, c, block=8, longest=0, max_length=None, positions=None, extra=0, handle=None):
        self.llmx, self.torch, self.c, self.longest = llmx, torch, c, longest
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.offsets, self.lengths = dev(c.offsets.view(np.int32)), dev(c.lengths.view(np.int32))
        self.table, self.k, self.v = dev(c.table), dev(c.k), dev(c.v)
        width = c.heads * c.hd
        self.ld = width + extra
        wide = np.full((c.rows, self.ld), 12345, np.int16)
        wide[:, :width] = c.q.reshape(c.rows, width)
        self.q = dev(wide)
        self.out = torch.full((c.rows, self.ld), FILL, dtype=torch.int16, device="cuda")
        most = max(int(c.lengths.max()) if len(c.lengths) else 1, 1)
        block = min(block, 128 // (c.heads // c.kv))
        self.p = handle or llmx.Paged(c.heads, c.kv, c.hd, c.page, len(c.plan), block, max_length or max(most, longest),
                                      positions or max(int(c.lengths.sum()), 1))

    def call(self, stream=None):
        c = self.c
        self.p.attention(self.q.data_ptr(), c.rows, self.offsets.data_ptr(), self.lengths.data_ptr(), len(c.plan),
                         self.table.data_ptr(), c.table.shape[1], self.k.data_ptr(), self.v.data_ptr(), c.pages,
                         self.out.data_ptr(), longest=self.longest or max(int(c.lengths.max()), 1), ld_q=self.ld, ld_out=self.ld,
                         stream=stream if stream is not None else self.torch.cuda.current_stream().cuda_stream)

    def result(self):
        self.torch.cuda.synchronize()
        out = self.out.cpu().numpy()
        width = self.c.heads * self.c.hd
        assert (out[:, width:] == FILL).all()
        return out[:, :width].reshape(self.c.rows, self.c.heads, self.c.hd)


def report(got, want):
    bad = np.argwhere(got != want)
    return f"{len(bad)} differ, first {bad[0]}: {got[tuple(bad[0])]} not {want[tuple(bad[0])]}" if len(bad) else "equal"


def check(llmx, torch, oracle, c, **kw):
    d = Device(llmx, torch, c, **kw)
    d.call()
    got, want = d.result(), c.want(oracle)
    assert np.array_equal(got, want), report(got, want)
    d.p.error()
    d.p.close()
    return got


# ---------------------------------------------------------------------------
# refusals, without a GPU
# ---------------------------------------------------------------------------
GOOD = dict(heads=16, kv=2, hd=128, page=16, requests=4, block=8, length=2048, positions=8192)


@pytest.mark.parametrize("change", [dict(heads=0), dict(kv=0), dict(heads=15), dict(heads=2048), dict(hd=0), dict(hd=24), dict(hd=144),
                                    dict(page=0), dict(page=12), dict(page=65544), dict(requests=0), dict(requests=1025), dict(block=0),
                                    dict(block=9), dict(heads=64, kv=2), dict(length=0), dict(length=2**20 + 1), dict(positions=0),
                                    dict(requests=1024, heads=1024, kv=1024, length=2**20, positions=2**30)])
def test_create_refuses(llmx, change):
    a = {**GOOD, **change}
    h = C.c_void_p(1)
    rc = llmx.lib().llmx_paged_create(0, a["heads"], a["kv"], a["hd"], a["page"], a["requests"], a["block"], a["length"],
                                      a["positions"], None, C.byref(h))
    assert rc == llmx.ERR_ARG and not h.value and llmx.last_error().startswith("paged: ")


def test_null_handles(llmx):
    L = llmx.lib()
    assert L.llmx_paged_create(0, 4, 2, 32, 16, 1, 1, 64, 64, None, None) == llmx.ERR_ARG
    assert L.llmx_paged_destroy(None) == llmx.OK
    assert L.llmx_paged_append(None, None, 1, 0, None, None, 1, None, 1, None, 1, None, None, 1, None, 0, None) == llmx.ERR_ARG
    assert L.llmx_paged_attention(None, None, 1, 0, None, None, 1, 0, None, 1, None, None, 1, None, 0, None) == llmx.ERR_ARG
    assert L.llmx_paged_error(None, None) == llmx.ERR_ARG
    assert L.llmx_paged_device_bytes(None) == 0


@gpu
def test_calls_refuse(llmx):
    p = llmx.Paged(4, 2, 32, 16, 4, 2, 256, 512)
    good = dict(q=256, rows=4, ld_q=0, offsets=256, lengths=256, requests=2, longest=64, table=256, ld_table=4, k=256, v=256, pages=8,
                out=256, ld_out=0)
    call = lambda **kw: llmx.lib().llmx_paged_attention(p.h, *{**good, **kw}.values(), None)  # noqa: E731
    for kw in (dict(q=None), dict(offsets=None), dict(lengths=None), dict(table=None), dict(k=None), dict(v=None), dict(out=None),
               dict(q=264), dict(k=8), dict(v=8), dict(out=264), dict(offsets=258), dict(lengths=257), dict(table=2), dict(ld_q=120),
               dict(ld_q=132), dict(ld_out=120), dict(ld_out=130), dict(requests=5), dict(longest=257), dict(ld_table=3), dict(ld_table=0),
               dict(pages=0), dict(pages=2**31), dict(longest=0, ld_table=15), dict(rows=2**20 + 1)):
        assert call(**kw) == llmx.ERR_ARG, kw
    assert call(rows=0) == llmx.OK and call(requests=0) == llmx.OK
    good = dict(qkv=256, rows=4, ld_qkv=0, offsets=256, lengths=256, requests=2, rope=256, positions=64, table=256, ld_table=4, k=256,
                v=256, pages=8, q=256, ld_q=0)
    call = lambda **kw: llmx.lib().llmx_paged_append(p.h, *{**good, **kw}.values(), None)  # noqa: E731, F811
    for kw in (dict(qkv=None), dict(offsets=None), dict(lengths=None), dict(rope=None), dict(table=None), dict(k=None), dict(v=None),
               dict(q=None), dict(qkv=264), dict(rope=8), dict(k=8), dict(v=8), dict(q=8), dict(ld_qkv=248), dict(ld_qkv=260),
               dict(ld_q=120), dict(ld_q=129), dict(requests=5), dict(ld_table=0), dict(pages=0), dict(rows=2**20 + 1)):
        assert call(**kw) == llmx.ERR_ARG, kw
    assert call(rows=0) == llmx.OK and call(requests=0) == llmx.OK
    p.error()
    p.close()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
LENGTHS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 48, 63, 64, 65, 66, 127, 128, 129, 200, 255, 256, 257, 500]


@gpu
@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 96, 112, 128])
def test_lengths(llmx, torch, oracle, hd):
    """One new token for requests of every length around the tiles' ends."""
    check(llmx, torch, oracle, Case(np.random.default_rng(hd), [(1, n) for n in LENGTHS], hd=hd))


@gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (3, 3), (5, 1), (8, 1), (9, 1), (10, 2), (14, 2), (16, 2), (16, 1), (12, 4)])
@pytest.mark.parametrize("block", [1, 2, 3, 5, 8])
def test_heads_and_blocks(llmx, torch, oracle, heads, kv, block):
    """Blocks of rows, each seeing the positions up to its own; a block longer than its sequence."""
    rng = np.random.default_rng(heads * 100 + block)
    plan = [(block, 130), (max(1, block - 1), 64), (0, 40), (block, block), (1, 1), (block, block // 2), (block, 300)]
    check(llmx, torch, oracle, Case(rng, plan, heads, kv, 48))


@gpu
@pytest.mark.parametrize("page", [8, 16, 24, 32, 40, 64, 72, 128, 200, 1024])
def test_pages(llmx, torch, oracle, page):
    check(llmx, torch, oracle, Case(np.random.default_rng(page), [(1, 513), (2, 100), (1, page), (3, page + 1)], 16, 2, 128, page))


@gpu
@pytest.mark.parametrize("seed", range(8))
def test_drawn(llmx, torch, oracle, seed):
    rng = np.random.default_rng(seed)
    kv, g, hd = int(rng.integers(1, 5)), int(rng.integers(1, 9)), 16 * int(rng.integers(1, 9))
    n = int(rng.integers(1, 40))
    plan = [(int(rng.integers(0, 9)), int(rng.integers(0, 400))) for _ in range(n)]
    c = Case(rng, plan, kv * g, kv, hd, 8 * int(rng.integers(1, 9)), pad=int(rng.integers(0, 4)))
    check(llmx, torch, oracle, c, extra=8 * int(rng.integers(0, 3)), longest=int(c.lengths.max()) + int(rng.integers(0, 7)))


@gpu
@pytest.mark.parametrize("requests", [32, 33, 128, 129, 300, 1024])
def test_many_requests(llmx, torch, oracle, requests):
    rng = np.random.default_rng(requests)
    plan = [(int(rng.integers(0, 3)), int(rng.integers(0, 90))) for _ in range(requests)]
    check(llmx, torch, oracle, Case(rng, plan, 4, 2, 16, 8), block=2)


@gpu
@pytest.mark.parametrize("what", ["keys", "values", "both"])
def test_values_beyond_eight(llmx, torch, oracle, what):
    """Values that a Q4.12 operand saturates: products with 32767 instead of 16 y."""
    rng = np.random.default_rng(4)
    c = Case(rng, [(1, 200), (4, 130), (2, 64)], 16, 2, 128, q_sigma=200, k_sigma=300, v_sigma=300)
    for name, pool in (("keys", c.k), ("values", c.v)):
        if what in (name, "both"):
            at = rng.random(pool.shape) < 0.2
            pool[at] = rng.choice(np.array([2046, 2047, 2048, 2049, 4000, 32767, -2047, -2048, -2049, -5000, -32768], np.int16), at.sum())
    check(llmx, torch, oracle, c)


@gpu
@pytest.mark.parametrize("q,k,v", [(-32768, -32768, -32768), (32767, 32767, 32767), (-32768, 32767, 32767), (32767, -32768, -32768),
                                   (-8192, -2048, 100), (-8192, -32768, 2048), (8191, -2048, -2048), (-8193, 2048, 5), (8192, 2047, 2047),
                                   (0, 0, 32767), (0, 0, -32768)])
@pytest.mark.parametrize("hd", [128, 64])
def test_saturation(llmx, torch, oracle, q, k, v, hd):
    """Banks, totals, tile values and accumulators at their limits; one query head of each kind beside
    ordinary ones."""
    rng = np.random.default_rng(9)
    c = Case(rng, [(1, 64), (3, 190), (1, 1)], 8, 1, hd)
    c.q[:, ::3] = q
    c.k[::2], c.v[::2] = k, v
    check(llmx, torch, oracle, c)
    c.q[:], c.k[:], c.v[:] = q, k, v
    check(llmx, torch, oracle, c)


@gpu
def test_wide_queries_in_one_place(llmx, torch, oracle):
    """A single large query element of a head: the head's scores saturate, its neighbours' do not change."""
    rng = np.random.default_rng(10)
    c = Case(rng, [(2, 150), (1, 40)], 16, 2, 128, k_sigma=2500)
    for r, h, e, x in ((0, 0, 0, -8192), (0, 3, 127, 32767), (1, 8, 64, -32768), (2, 15, 5, 8192)):
        c.q[r, h, e] = x
    c.q[1, 4] = rng.integers(-32768, 32767, 128)
    check(llmx, torch, oracle, c)


@gpu
def test_long(llmx, torch, oracle):
    """A long text: over 512 tiles, so that the sum of probabilities and the accumulator saturate where
    every position weighs the same, and the maximum moves often in another head."""
    rng = np.random.default_rng(11)
    c = Case(rng, [(1, 40000), (2, 9000)], 4, 2, 16, 64)
    c.q[0, 0] = 0  # every probability is 1
    pos = np.arange(40000)
    rising = (pos // 20 - 1000).astype(np.int16)  # scores that rise over the text
    c.k[c.table[0][pos // 64], 1, pos % 64] = 0
    c.k[c.table[0][pos // 64], 1, pos % 64, 0] = rising
    c.q[0, 2:] = 0
    c.q[0, 2, 0], c.q[0, 3, 0] = 256, -256
    c.v[c.table[0][pos // 64], 0, pos % 64, :8] = 700
    check(llmx, torch, oracle, c)


@gpu
def test_offsets_beyond_32_bits(llmx, torch, oracle):
    """Pages whose first element lies beyond 2^31 elements."""
    page, kv, hd = 64, 2, 128
    per = kv * page * hd
    pages = 2**31 // per + 40
    rng = np.random.default_rng(12)
    c = Case(rng, [(1, 200), (2, 130)], 16, kv, hd, page)
    big = torch.zeros((pages, kv, page, hd), dtype=torch.int16, device="cuda")
    where = np.arange(c.pages) * 3 + pages - 3 * c.pages
    big[torch.from_numpy(where).cuda()] = torch.from_numpy(c.k).cuda()
    want = None
    d = Device(llmx, torch, c)
    c.v[:] = c.k  # one array for both
    want = c.want(oracle)
    used = c.table >= 0
    used[:, -1] = False
    moved = c.table.copy()
    moved[used] = where[c.table[used]]
    d.k = d.v = big
    d.table = torch.from_numpy(moved).cuda()
    c.pages = pages
    d.call()
    got = d.result()
    assert np.array_equal(got, want), report(got, want)
    d.p.error()


@gpu
def test_shared_pages(llmx, torch, oracle):
    """Requests whose texts begin alike share pages."""
    rng = np.random.default_rng(13)
    c = Case(rng, [(1, 150), (1, 180), (3, 96)], 16, 2, 128)
    c.table[1, :5] = c.table[0, :5]
    c.table[2, :6] = c.table[1, :6]
    check(llmx, torch, oracle, c)


@gpu
def test_same_handle_again_and_smaller(llmx, torch, oracle):
    """Calls of other sizes with one handle leave nothing behind for the next."""
    rng = np.random.default_rng(14)
    first = Case(rng, [(8, 500)] * 5, 8, 2, 64)
    d = Device(llmx, torch, first, max_length=1000, positions=5000)
    d.call()
    assert np.array_equal(d.result(), first.want(oracle))
    for plan in ([(1, 3)], [(2, 70), (1, 999)], [(0, 0), (1, 0)], [(1, 1000)] * 4):
        c = Case(rng, plan, 8, 2, 64)
        e = Device(llmx, torch, c, handle=d.p)
        e.call()
        assert np.array_equal(e.result(), c.want(oracle))
    d.p.error()


@gpu
def test_void_requests(llmx, torch, oracle):
    """Requests that are out of range are left out and reported; the others are served."""
    rng = np.random.default_rng(15)
    plan = [(1, 100), (3, 50), (1, 77), (1, 30)]
    for spoil in ("length", "block", "order", "end"):
        c = Case(rng, plan, 8, 2, 32)
        want = c.want(oracle)
        d = Device(llmx, torch, c, block=3, max_length=100)
        o = c.offsets.copy()
        if spoil == "length":
            d.lengths[1] = 101
            void = [1]
        elif spoil == "block":
            o[2] = 5  # request 1: 4 rows, request 2: none
            void = [1, 2]
        elif spoil == "order":
            o[2] = 0  # request 1 ends before it starts, request 2 has 5 rows
            void = [1, 2]
        else:
            o[4] = 2**32 - 1
            void = [3]
        d.offsets.copy_(torch.from_numpy(o.view(np.int32)))
        d.call()
        got = d.result()
        for b, (rows, _) in enumerate(plan):
            mine = slice(int(c.offsets[b]), int(c.offsets[b]) + rows)
            if b in void:
                assert (got[mine] == FILL).all(), (spoil, b)
            elif (spoil, b) != ("order", 0):  # its row is claimed by request 2 as well
                assert np.array_equal(got[mine], want[mine]), (spoil, b)
        with pytest.raises(llmx.LlmxError) as e:
            d.p.error()
        assert e.value.code == llmx.ERR_RANGE
        d.p.error()  # reported once


@gpu
def test_page_numbers_out_of_range(llmx, torch, oracle):
    rng = np.random.default_rng(16)
    for number in (-1, 2**31 - 1, None):
        c = Case(rng, [(1, 100), (1, 90)], 8, 2, 32)
        want = c.want(oracle)
        d = Device(llmx, torch, c)
        d.table[1, 2] = c.pages if number is None else number
        d.call()
        assert np.array_equal(d.result()[0], want[0])
        with pytest.raises(llmx.LlmxError) as e:
            d.p.error()
        assert e.value.code == llmx.ERR_RANGE and "page" in str(e.value)


@gpu
def test_more_positions_than_reserved(llmx, torch, oracle):
    rng = np.random.default_rng(17)
    c = Case(rng, [(1, 1000)] * 4, 8, 2, 32)
    d = Device(llmx, torch, c, positions=1000)
    d.call()
    assert (d.result() == FILL).all()
    with pytest.raises(llmx.LlmxError) as e:
        d.p.error()
    assert e.value.code == llmx.ERR_RANGE


@gpu
def test_graph_and_streams(llmx, torch, oracle):
    """Captured once, replayed over other lengths, tables and queries; on another stream than the current one."""
    rng = np.random.default_rng(18)
    cases = [Case(rng, p, 16, 2, 64) for p in ([(2, 120), (1, 64), (1, 300)], [(1, 5), (2, 290), (1, 200)], [(0, 9), (4, 300), (0, 0)])]
    d = Device(llmx, torch, Case(rng, [(4, 300)] * 3, 16, 2, 64), longest=300, positions=900)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
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
        assert np.array_equal(got[:c.rows], c.want(oracle)) and (got[c.rows:] == FILL).all()
    # two handles at once on two streams
    a, b = Device(llmx, torch, cases[0]), Device(llmx, torch, cases[1])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        a.call(s1.cuda_stream)
        b.call(s2.cuda_stream)
    assert np.array_equal(a.result(), cases[0].want(oracle)) and np.array_equal(b.result(), cases[1].want(oracle))


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def rotate(x, turn):
    """x [heads][hd], turn [hd]: rotate_fix16_pair_with_quantized_rope in 64 bits."""
    half = x.shape[1] // 2
    a, b = x[:, :half].astype(np.int64), x[:, half:].astype(np.int64)
    c, s = turn[:half].astype(np.int64), turn[half:].astype(np.int64)
    y = np.concatenate([a * c - b * s, b * c + a * s], 1)
    return np.clip((y + 128) >> 8, -32768, 32767).astype(np.int16)


def append_case(llmx, torch, rng, plan, heads, kv, hd, page, rope=None, in_place=False, extra=0, ld_table=None, positions=None):
    c = Case(rng, plan, heads, kv, hd, page)
    most = max(int(c.lengths.max()), 1)
    rope = llmx.rope_table(hd, most) if rope is None else rope
    width = (heads + 2 * kv) * hd
    x = rng.integers(-32768, 32768, (c.rows, width + extra)).astype(np.int16)
    k, v = c.k.copy(), c.v.copy()
    q = np.full((c.rows, heads * hd), FILL, np.int16)
    if in_place:
        q = x.copy()
    for b, (rows, length) in enumerate(plan):
        for j in range(rows):
            r, p = int(c.offsets[b]) + j, length - rows + j
            if p < 0:
                continue
            row = x[r, :width].reshape(heads + 2 * kv, hd)
            turned = rotate(row[:heads + kv], rope[p])
            q[r, :heads * hd] = turned[:heads].reshape(-1)
            at = int(c.table[b, p // page])
            k[at, :, p % page] = turned[heads:]
            v[at, :, p % page] = row[heads + kv:]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    dx, dk, dv, dr, dt = dev(x), dev(c.k), dev(c.v), dev(rope), dev(c.table)
    do, dl = dev(c.offsets.view(np.int32)), dev(c.lengths.view(np.int32))
    dq = dx if in_place else torch.full((c.rows, heads * hd), FILL, dtype=torch.int16, device="cuda")
    p = llmx.Paged(heads, kv, hd, page, len(plan), 1, most, most)
    p.append(dx.data_ptr(), c.rows, do.data_ptr(), dl.data_ptr(), len(plan), dr.data_ptr(), positions or rope.shape[0], dt.data_ptr(),
             c.table.shape[1], dk.data_ptr(), dv.data_ptr(), c.pages, dq.data_ptr(), ld_qkv=width + extra if extra or in_place else 0,
             ld_q=dq.shape[1] if in_place else 0, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return p, c, (dq.cpu().numpy(), dk.cpu().numpy(), dv.cpu().numpy()), (q, k, v)


@gpu
@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads,kv,page", [(16, 2, 16), (3, 3, 8), (5, 1, 24), (8, 4, 64)])
def test_append(llmx, torch, hd, heads, kv, page):
    """Requests of any number of rows, some in front of their sequence, some empty."""
    rng = np.random.default_rng(hd + heads)
    plan = [(1, 1), (1, 40), (0, 17), (33, 50), (7, 3), (100, 100), (1, 300)]
    for in_place in (False, True):
        p, c, got, want = append_case(llmx, torch, rng, plan, heads, kv, hd, page, in_place=in_place, extra=16 if in_place else 0)
        for g, w, name in zip(got, want, "qkv"):
            assert np.array_equal(g, w), name
        p.error()
        p.close()


@gpu
@pytest.mark.parametrize("requests", [1, 2, 31, 32, 33, 64, 100, 1000, 1024])
def test_append_finds_its_request(llmx, torch, requests):
    rng = np.random.default_rng(requests)
    plan = [(int(rng.integers(0, 4)), int(rng.integers(4, 40))) for _ in range(requests)]
    if requests == 1:
        plan = [(3, 5)]
    p, c, got, want = append_case(llmx, torch, rng, plan, 2, 1, 16, 8)
    for g, w, name in zip(got, want, "qkv"):
        assert np.array_equal(g, w), name
    p.error()


@gpu
def test_append_with_any_table(llmx, torch):
    """A rope table of any values (their sums leave 32 bits)."""
    rng = np.random.default_rng(1)
    rope = rng.choice(np.array([-32768, 32767, 0, 256, -256], np.int16), (60, 64))
    p, c, got, want = append_case(llmx, torch, rng, [(20, 60), (5, 31)], 4, 2, 64, 16, rope=rope)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


@gpu
def test_append_out_of_range(llmx, torch):
    """Rows beyond the rope table are left out and reported, the others appended."""
    rng = np.random.default_rng(2)
    p, c, got, want = append_case(llmx, torch, rng, [(3, 20), (4, 41)], 4, 2, 32, 16, positions=40)
    assert np.array_equal(got[0][:6], want[0][:6]) and (got[0][6] == FILL).all()
    for g, w in zip(got[1:], want[1:]):
        at, inside = int(c.table[1, 2]), 40 % 16
        w[at, :, inside] = (c.k if w is want[1] else c.v)[at, :, inside]
        assert np.array_equal(g, w)
    with pytest.raises(llmx.LlmxError) as e:
        p.error()
    assert e.value.code == llmx.ERR_RANGE


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("shape", ["small", "medium", "qwen-layer"])
def test_attention_sublayer_of_many_requests(llmx, torch, shape):
    """RMSNorm, the shared Q/K/V projection, append, attention and the O projection for requests with
    caches in pages: the rows of Task 18 on a context per request, over several steps of
    blocks of rows."""
    s = llmx.shape(shape)
    model = llmx.Model(s).init_gaussian(5)
    heads, kv, hd, hidden = s.heads, s.kv_heads, s.head_dim, s.hidden
    rng = np.random.default_rng(3)
    blob = model.layer(0)
    qkv_rows = hidden + 2 * kv * hd
    wqkv = np.ascontiguousarray(blob[:qkv_rows * hidden].reshape(qkv_rows, hidden))
    wo = np.ascontiguousarray(blob[qkv_rows * hidden:(qkv_rows + hidden) * hidden].reshape(hidden, hidden))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    dqkv, do = dev(wqkv), dev(wo)
    stream = torch.cuda.current_stream().cuda_stream
    requests, page, most = 3, 8, min(s.max_seq, 60)
    a = llmx.Adapters(hidden, qkv_rows, dqkv.data_ptr(), 0, 1, 8 * requests, stream=stream)
    o = llmx.Adapters(hidden, hidden, do.data_ptr(), 0, 1, 8 * requests, stream=stream)
    p = llmx.Paged(heads, kv, hd, page, requests, 8, most, requests * most, stream=stream)
    width = -(-most // page)
    table = rng.permutation(requests * width).astype(np.int32).reshape(requests, width)
    pages = requests * width
    dk = torch.full((pages, kv, page, hd), 99, dtype=torch.int16, device="cuda")
    dv = torch.full_like(dk, -99)
    rope, dt = dev(llmx.rope_table(hd, most)), dev(table)
    contexts = []
    for _ in range(requests):
        acc = llmx.Accelerator(s)
        acc.upload_model(model)
        contexts.append(acc)
    norm = model.norms()[0]
    at = [0] * requests
    for blocks in ((8, 3, 1), (1, 8, 2), (1, 1, 1), (0, 5, 1), (4, 0, 8)):
        if any(x + n > most for x, n in zip(at, blocks)):
            break
        x = np.clip(np.rint(rng.normal(0, 300, (sum(blocks), hidden))), -32768, 32767).astype(np.int16)
        offsets = np.concatenate([[0], np.cumsum(blocks)])
        want = []
        normed = []
        for r, n in enumerate(blocks):
            mine = x[offsets[r]:offsets[r + 1]]
            if n == 0:
                continue
            normed.append(contexts[r].run_feature(llmx.OP_RMSNORM, mine, norm[None])[0])
            contexts[r].write_hidden(1, mine)
            contexts[r].bind(0, 1)
            contexts[r].task(llmx.OP_ATTENTION, 0, at[r], n)
            want.append(contexts[r].read_hidden(0, n))
            at[r] += n
        xn = dev(np.concatenate(normed))
        rows = xn.shape[0]
        doff, dlen = dev(offsets.astype(np.int32)), dev(np.array(at, np.int32))
        qkv = torch.empty((rows, qkv_rows), dtype=torch.int16, device="cuda")
        att = torch.empty((rows, hidden), dtype=torch.int16, device="cuda")
        out = torch.empty((rows, hidden), dtype=torch.int16, device="cuda")
        a.project(xn.data_ptr(), rows, None, qkv.data_ptr(), stream=stream)
        # queries are rotated where the projection left them
        p.append(qkv.data_ptr(), rows, doff.data_ptr(), dlen.data_ptr(), requests, rope.data_ptr(), most, dt.data_ptr(), width,
                 dk.data_ptr(), dv.data_ptr(), pages, qkv.data_ptr(), ld_q=qkv_rows, stream=stream)
        p.attention(qkv.data_ptr(), rows, doff.data_ptr(), dlen.data_ptr(), requests, dt.data_ptr(), width, dk.data_ptr(), dv.data_ptr(),
                    pages, att.data_ptr(), ld_q=qkv_rows, stream=stream)
        o.project(att.data_ptr(), rows, None, out.data_ptr(), stream=stream)
        torch.cuda.synchronize()
        got = np.clip(x.astype(np.int32) + out.cpu().numpy(), -32768, 32767)
        assert np.array_equal(got, np.concatenate(want)), report(got, np.concatenate(want))
        p.error()
    assert max(at) > 8
    for r, n in enumerate(at):  # the pages hold the contexts' caches
        k, v = contexts[r].read_kv(0, 0, n)
        pos = np.arange(n)
        for cache, pool in ((k, dk), (v, dv)):
            assert np.array_equal(pool.cpu().numpy()[table[r][pos // page], :, pos % page].transpose(1, 0, 2), cache)
    for h in (a, o, p, *contexts):
        h.close()


@gpu
def test_rows_in_front_of_the_first_request(llmx, torch, oracle):
    """offsets[0] above 0: rows in front of the first request's are left as they are, as those behind the last."""
    rng = np.random.default_rng(19)
    c = Case(rng, [(2, 100), (0, 5), (3, 77)], 8, 2, 32, pad=9)
    want = c.want(oracle)
    d = Device(llmx, torch, c)
    d.offsets += 4
    d.q = torch.roll(d.q, 4, 0)
    d.call()
    got = d.result()
    assert (got[:4] == FILL).all() and np.array_equal(got[4:], want[:-4])
    rope = llmx.rope_table(32, 100)
    x = rng.integers(-32768, 32767, (c.rows, 12 * 32)).astype(np.int16)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    dx, dr, dk, dv = dev(x), dev(rope), dev(c.k), dev(c.v)
    q = torch.full((c.rows, 256), FILL, dtype=torch.int16, device="cuda")
    d.p.append(dx.data_ptr(), c.rows, d.offsets.data_ptr(), d.lengths.data_ptr(), 3, dr.data_ptr(), 100, d.table.data_ptr(), c.table.shape[1],
               dk.data_ptr(), dv.data_ptr(), c.pages, q.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    d.p.error()
    k, v = c.k.copy(), c.v.copy()
    out = np.full((c.rows, 256), FILL, np.int16)
    for b, (rows, length) in enumerate(c.plan):
        for j in range(rows):
            r, p = 4 + int(c.offsets[b]) + j, length - rows + j
            turned = rotate(x[r].reshape(12, 32)[:10], rope[p])
            out[r] = turned[:8].reshape(-1)
            k[c.table[b, p // 16], :, p % 16] = turned[8:]
            v[c.table[b, p // 16], :, p % 16] = x[r].reshape(12, 32)[10:]
    assert np.array_equal(q.cpu().numpy(), out) and np.array_equal(dk.cpu().numpy(), k) and np.array_equal(dv.cpu().numpy(), v)


@gpu
def test_append_beyond_32_bits(llmx, torch):
    """Pages whose first element lies beyond 2^31 elements."""
    page, kv, hd = 64, 2, 128
    per = kv * page * hd
    pages = 2**31 // per + 20
    rng = np.random.default_rng(20)
    c = Case(rng, [(5, 200), (100, 130)], 4, kv, hd, page)
    rope = llmx.rope_table(hd, 200)
    x = rng.integers(-32768, 32767, (c.rows, 8 * hd)).astype(np.int16)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    where = pages - c.pages + np.arange(c.pages)
    table = c.table.copy()
    table[:, :-1] = np.where(table[:, :-1] >= 0, table[:, :-1] + pages - c.pages, -1)
    big = [torch.zeros((pages, kv, page, hd), dtype=torch.int16, device="cuda") for _ in range(2)]
    dx, dr, dt = dev(x), dev(rope), dev(table)
    do, dl = dev(c.offsets.view(np.int32)), dev(c.lengths.view(np.int32))
    q = torch.empty((c.rows, 4 * hd), dtype=torch.int16, device="cuda")
    p = llmx.Paged(4, kv, hd, page, 2, 1, 200, 400)
    p.append(dx.data_ptr(), c.rows, do.data_ptr(), dl.data_ptr(), 2, dr.data_ptr(), 200, dt.data_ptr(), table.shape[1], big[0].data_ptr(),
             big[1].data_ptr(), pages, q.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    p.error()
    k, v = np.zeros_like(c.k), np.zeros_like(c.v)
    for b, (rows, length) in enumerate(c.plan):
        for j in range(rows):
            r, at = int(c.offsets[b]) + j, length - rows + j
            row = x[r].reshape(8, hd)
            k[c.table[b, at // page], :, at % page] = rotate(row[4:6], rope[at])
            v[c.table[b, at // page], :, at % page] = row[6:]
    for got, want in zip(big, (k, v)):
        assert np.array_equal(got[torch.from_numpy(where).cuda()].cpu().numpy(), want)
        assert not got[:pages - c.pages].any()


@gpu
def test_decoding_in_one_graph(llmx, torch, oracle):
    """Append and attention captured together and replayed token by token, the lengths counted on the device:
    every request's rows are those of the oracle on the cache so far."""
    rng = np.random.default_rng(21)
    heads, kv, hd, page, steps, most = 8, 2, 64, 16, 40, 130
    start = np.array([0, 1, 15, 60, 90], np.int32)
    b = len(start)
    width = -(-most // page)
    table = rng.permutation(b * width).astype(np.int32).reshape(b, width)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    pools = [rng.integers(-600, 600, (b * width, kv, page, hd)).astype(np.int16) for _ in range(2)]
    dk, dv, dt, dl = dev(pools[0]), dev(pools[1]), dev(table), dev(start)
    do = torch.arange(b + 1, dtype=torch.int32, device="cuda")
    rope = llmx.rope_table(hd, most)
    dr = dev(rope)
    qkv = torch.zeros((b, (heads + 2 * kv) * hd), dtype=torch.int16, device="cuda")
    out = torch.zeros((b, heads * hd), dtype=torch.int16, device="cuda")
    p = llmx.Paged(heads, kv, hd, page, b, 1, most, b * most)

    def step():
        s = torch.cuda.current_stream().cuda_stream
        dl.add_(1)
        p.append(qkv.data_ptr(), b, do.data_ptr(), dl.data_ptr(), b, dr.data_ptr(), most, dt.data_ptr(), width, dk.data_ptr(), dv.data_ptr(),
                 b * width, qkv.data_ptr(), ld_q=qkv.shape[1], stream=s)
        p.attention(qkv.data_ptr(), b, do.data_ptr(), dl.data_ptr(), b, dt.data_ptr(), width, dk.data_ptr(), dv.data_ptr(), b * width,
                    out.data_ptr(), ld_q=qkv.shape[1], stream=s)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    dl.copy_(dev(start))
    dk.copy_(dev(pools[0]))
    dv.copy_(dev(pools[1]))
    for n in range(steps):
        x = np.clip(np.rint(rng.normal(0, 500, qkv.shape)), -32768, 32767).astype(np.int16)
        qkv.copy_(dev(x))
        graph.replay()
        got = out.cpu().numpy().reshape(b, heads, hd)
        for r in range(b):
            at = int(start[r]) + n
            row = x[r].reshape(-1, hd)
            turned = rotate(row[:heads + kv], rope[at])
            page_at = table[r, at // page]
            pools[0][page_at, :, at % page], pools[1][page_at, :, at % page] = turned[heads:], row[heads + kv:]
            pos = np.arange(at + 1)
            k, v = (pool[table[r][pos // page], :, pos % page] for pool in pools)
            for h in range(kv):
                g = heads // kv
                want = oracle.attention_group(turned[h * g:(h + 1) * g], k[:, h], v[:, h])
                assert np.array_equal(got[r, h * g:(h + 1) * g], want), (n, r, h)
    p.error()


@gpu
@pytest.mark.parametrize("rows,before,longest", [(200, 37, 0), (77, 0, 0), (77, 0, 17000)])
def test_prompt_as_blocks(llmx, torch, oracle, rows, before, longest):
    """A prompt's rows in one call: blocks of 8 as requests of their own, with one table."""
    rng = np.random.default_rng(rows)
    ends = list(range(8, rows, 8)) + [rows]
    c = Case(rng, [(n - m, before + n) for m, n in zip([0] + ends, ends)], 16, 2, 64)
    c.table[:] = c.table[-1]
    c.table = np.pad(c.table, ((0, 0), (0, longest // 16 + 1)), constant_values=-1)
    check(llmx, torch, oracle, c, longest=longest)


@gpu
@pytest.mark.parametrize("heads,block,hd", [(5, 5, 80), (9, 7, 48), (7, 8, 128), (3, 3, 16)])
@pytest.mark.parametrize("longest", [0, 20000])
def test_partly_filled_column_blocks(llmx, torch, oracle, heads, block, hd, longest):
    """Query rows that do not fill their blocks of 8, so that some lanes store and others do not between one block's
    matrix instructions and the next one's; requests that leave CTAs of a cluster without a tile.  The same every time."""
    rng = np.random.default_rng(heads)
    c = Case(rng, [(block, 700), (1, 65), (block - 1, 130), (2, 64), (block, 1)], heads, 1, hd)
    c.table = np.pad(c.table, ((0, 0), (0, longest // 16 + 1)), constant_values=-1)
    d, want = Device(llmx, torch, c, longest=longest), c.want(oracle)
    for _ in range(10):
        d.out.fill_(FILL)
        d.call()
        got = d.result()
        assert np.array_equal(got, want), report(got, want)
    d.p.error()
