"""Log probabilities of given tokens, entropy and most likely tokens (llmx_token_logprobs).

Tokens and ranks are compared exactly, log probabilities and entropies with the formulas in
64 bits, within bounds that follow from the arithmetic (bounds())."""
import numpy as np
import pytest

gpu = pytest.mark.gpu
NONE = -(2**31)
NO_TOKEN = 0xFFFFFFFF
MARK = -777


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def oracle(z, tokens, temperature, top):
    """The formulas in 64 bits; also the sums that bounds() needs."""
    rows, vocab = z.shape
    out = dict(logprob=np.full(rows, -np.inf), rank=np.full(rows, NO_TOKEN, np.uint32), entropy=np.zeros(rows),
               top_tokens=np.full((rows, top), NO_TOKEN, np.uint32), top_logprobs=np.full((rows, top), -np.inf))
    out["terms"] = [None] * rows
    for r in range(rows):
        row = z[r].astype(np.int64)
        live = np.nonzero(row != NONE)[0]
        if len(live) == 0:
            continue
        order = live[np.argsort(-row[live], kind="stable")]
        t = np.float64(np.float32(temperature[r]))
        greedy = not t > 1e-6
        d = np.where(np.arange(len(order)) == 0, 0.0, np.inf) if greedy else (row[order[0]] - row[order]) / (65536.0 * t)
        w = np.exp(-d[1:])
        rest = w.sum()
        finite = np.where(w > 0, d[1:], 0)
        weighted = (w * finite).sum()
        lp = -d - np.log1p(rest)
        if not greedy:
            out["entropy"][r] = np.log1p(rest) + weighted / (1 + rest)
            out["terms"][r] = (w, finite, rest, weighted)
        n = min(top, len(order))
        out["top_tokens"][r, :n], out["top_logprobs"][r, :n] = order[:n], lp[:n]
        if tokens is not None and tokens[r] < vocab and row[tokens[r]] != NONE:
            at = int(np.nonzero(order == tokens[r])[0][0])
            out["rank"][r], out["logprob"][r] = at, lp[at]
    return out


def bounds(terms, chunks):
    """How far log1p(rest) and the entropy may be off.  A term's weight: 2^-22 of ex2.approx and the
    rounding of its exponent, d (1/2 ulp of the difference, 1/2 of the scale's remainder, 1/2 of the
    product: 2^-23 d with room).  Its way into a row's sum: 16 additions, one per chunk of the warp's
    share and per new maximum (as many at most, with a product), 5 over the lanes, 2^-24 each.
    A term below 2^-126, the least normal number, is taken for 0 (at d = 87.3 and more)."""
    w, d, rest, weighted = terms
    way = (16 + 3 * chunks + 5) * 2.0**-24
    each = 2.0**-22 + 2.0**-23 * d + way
    off = (w * each).sum() + len(w) * 2.0**-126  # of rest
    off_weighted = (w * d * (each + 2.0**-23 + way)).sum() + d.sum() * 2.0**-126
    log = off / (1 + rest)
    return log, log + (off_weighted + weighted * off / (1 + rest)) / (1 + rest)


class Device:
    def __init__(self, llmx, torch, z, tokens, temperature, top, ld=0, skip=0):
        self.llmx, self.torch, self.z, self.tokens, self.temperature, self.top, self.ld = llmx, torch, z, tokens, temperature, top, ld
        rows, vocab = z.shape
        wide = np.full((rows, ld or vocab), 2**31 - 1, np.int32)  # what lies between rows must not matter
        wide[:, :vocab] = z
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.logits = dev(np.concatenate([np.full(skip, 2**31 - 1, np.int32), wide.reshape(-1), np.full(4, 2**31 - 1, np.int32)]))
        self.at = self.logits.data_ptr() + 4 * skip
        self.d_tokens = dev(tokens.view(np.int32)) if tokens is not None else None
        self.d_temperature = dev(temperature) if temperature is not None else None
        full = lambda n, kind: torch.full((n + 3,), MARK, dtype=kind, device="cuda")  # noqa: E731
        self.logprob, self.rank, self.entropy = full(rows, torch.float32), full(rows, torch.int32), full(rows, torch.float32)
        self.top_tokens, self.top_logprobs = full(rows * top, torch.int32), full(rows * top, torch.float32)
        self.size = llmx.logprobs_workspace_bytes(rows, vocab, top)
        self.work = torch.full((self.size + 64,), 85, dtype=torch.uint8, device="cuda")

    def call(self, stream=None):
        p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        self.llmx.token_logprobs(self.at, self.z.shape[0], self.z.shape[1], p(self.d_tokens), p(self.d_temperature), self.top,
                                 p(self.logprob), p(self.rank), p(self.entropy), p(self.top_tokens), p(self.top_logprobs), p(self.work),
                                 self.size, ld=self.ld, stream=stream if stream is not None else self.torch.cuda.current_stream().cuda_stream)

    def result(self):
        self.torch.cuda.synchronize()
        rows = self.z.shape[0]
        out = {}
        for f, n in (("logprob", rows), ("rank", rows), ("entropy", rows), ("top_tokens", rows * self.top), ("top_logprobs", rows * self.top)):
            a = getattr(self, f).cpu().numpy()
            assert (a[n:] == MARK).all(), f
            out[f] = a[:n]
        assert (self.work[self.size:].cpu() == 85).all()
        for f in ("top_tokens", "top_logprobs"):
            out[f] = out[f].reshape(rows, self.top)
        for f in ("rank", "top_tokens"):
            out[f] = out[f].view(np.uint32)
        return out

    def check(self):
        got = self.result()
        t = self.temperature if self.temperature is not None else np.ones(len(self.z), np.float32)
        want = oracle(self.z, self.tokens, t, self.top)
        assert np.array_equal(got["top_tokens"], want["top_tokens"])
        if self.tokens is not None:
            assert np.array_equal(got["rank"], want["rank"])
        else:
            assert (got["rank"].view(np.int32) == MARK).all() and (got["logprob"] == MARK).all()
        chunks = self.z.shape[1] // 512 + 1
        for r in range(len(self.z)):
            log, ent = bounds(want["terms"][r], chunks) if want["terms"][r] is not None else (0, 0)
            assert abs(got["entropy"][r] - want["entropy"][r]) <= ent + want["entropy"][r] * 2.0**-24, r
            pairs = [(got["top_logprobs"][r], want["top_logprobs"][r])]
            if self.tokens is not None:
                pairs.append((got["logprob"][r:r + 1], want["logprob"][r:r + 1]))
            for g, w in pairs:
                gone = np.isinf(w)
                assert np.array_equal(g[gone], w[gone]) and (np.abs(g[~gone] - w[~gone]) <= log + np.abs(w[~gone]) * 2.0**-24).all(), r
        return got, want


def logits(rng, rows, vocab, spread=2.5, excluded=0.0):
    z = rng.normal(0, spread, (rows, vocab))
    for r in range(rows):
        z[r, rng.integers(0, vocab, 6)] += rng.random(6) * 14
    z = np.clip(np.rint(z * 65536), -(2**31) + 1, 2**31 - 1).astype(np.int32)
    if excluded:
        z[rng.random(z.shape) < excluded] = NONE
    return z


def check(llmx, torch, z, tokens=None, temperature=None, top=5, **kw):
    d = Device(llmx, torch, z, tokens, temperature, top, **kw)
    d.call()
    return d.check()


def draw_tokens(rng, z):
    """Likely tokens, unlikely ones, one outside the vocabulary."""
    rows, vocab = z.shape
    t = np.where(rng.random(rows) < 0.6, z.argmax(1), rng.integers(0, vocab, rows)).astype(np.uint32)
    t[rng.random(rows) < 0.1] = vocab
    return t


def test_refusals(llmx):
    L = llmx.lib()
    good = dict(logits=256, ld=0, vocab=100, rows=2, tokens=256, temperature=256, top=3, logprob=256, rank=256, entropy=256,
                top_tokens=256, top_logprobs=256, work=256, size=llmx.logprobs_workspace_bytes(2, 100, 3))
    call = lambda **kw: L.llmx_token_logprobs(*{**good, **kw}.values(), None)  # noqa: E731
    for kw in (dict(logits=None), dict(entropy=None), dict(work=None), dict(logprob=None), dict(rank=None), dict(top_tokens=None),
               dict(top_logprobs=None), dict(vocab=0), dict(vocab=2**22 + 1), dict(ld=99), dict(rows=2**20 + 1), dict(top=33),
               dict(logits=258), dict(tokens=257), dict(temperature=254), dict(logprob=2), dict(rank=1), dict(entropy=3),
               dict(top_tokens=5), dict(top_logprobs=6), dict(work=128), dict(size=good["size"] - 1)):
        assert call(**kw) == llmx.ERR_ARG, kw
        assert llmx.last_error().startswith("token_logprobs: ")
    assert call(rows=0) == llmx.OK


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 31, 32, 33, 127, 511, 512, 513, 1000, 1024, 4099, 32001, 151936])
@pytest.mark.parametrize("rows", [1, 7])
def test_vocabularies(llmx, torch, vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    z = logits(rng, rows, vocab)
    for top in (0, 1, 5, 32):
        check(llmx, torch, z, draw_tokens(rng, z), (rng.random(rows) + 0.4).astype(np.float32), top)


@gpu
@pytest.mark.parametrize("rows", [2, 3, 64, 200, 1500, 5000])
def test_rows(llmx, torch, rows):
    rng = np.random.default_rng(rows)
    vocab = 997 if rows > 1000 else 6001
    z = logits(rng, rows, vocab, excluded=0.2)
    check(llmx, torch, z, draw_tokens(rng, z), None, 9)


@gpu
@pytest.mark.parametrize("skip,ld", [(0, 1003), (1, 1003), (2, 1004), (3, 1008), (1, 0), (3, 1001)])
def test_alignment_and_strides(llmx, torch, skip, ld):
    rng = np.random.default_rng(skip)
    z = logits(rng, 9, 1001)
    check(llmx, torch, z, draw_tokens(rng, z), None, 4, ld=ld, skip=skip)


@gpu
def test_without_tokens(llmx, torch):
    check(llmx, torch, logits(np.random.default_rng(1), 4, 3000), None, None, 3)


@gpu
def test_excluded(llmx, torch):
    """Rows that exclude nearly every token, every token, or the given one; fewer tokens than asked for."""
    rng = np.random.default_rng(2)
    z = logits(rng, 6, 2000, excluded=0.5)
    z[0] = NONE
    z[1] = NONE
    z[1, 1999] = 5
    z[2] = NONE
    z[2, [7, 600, 1200]] = [-(2**31) + 1, 2**31 - 1, 0]
    z[3, 1:] = NONE
    tokens = np.array([3, 1999, 7, 0, int(np.nonzero(z[4] == NONE)[0][0]), 5], np.uint32)
    for t in (None, np.full(6, 1e5, np.float32), np.full(6, np.inf, np.float32)):
        check(llmx, torch, z, tokens, t, 8)


@gpu
def test_temperatures(llmx, torch):
    """Greedy rows (T <= 1e-6, negative, NaN) beside tiny, large and infinite temperatures."""
    rng = np.random.default_rng(3)
    t = np.array([0, 1e-6, -1, np.nan, 1.1e-6, 0.01, 0.3, 1, 7, 1000, 1e30, np.inf], np.float32)
    z = logits(rng, len(t), 5000, excluded=0.1)
    z[:, 17] = z.max(1)  # two maxima in some rows
    check(llmx, torch, z, np.full(len(t), 17, np.uint32), t, 6)
    check(llmx, torch, z, z.argmax(1).astype(np.uint32), t, 6)


@gpu
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "steps", "far"])
def test_ties_and_orders(llmx, torch, kind):
    """Rows of equal logits, in order, of two values, of equal runs: ties go to the lowest index."""
    rng = np.random.default_rng(4)
    vocab, rows = 20000, 3
    i = np.arange(vocab)
    z = {"equal": np.full((rows, vocab), 70000), "rising": np.tile(i * 50, (rows, 1)), "falling": np.tile(-i * 50, (rows, 1)),
         "two": rng.integers(0, 2, (rows, vocab)) * 65536, "steps": np.tile(i // 300 * 4000, (rows, 1)),
         "far": np.where(rng.random((rows, vocab)) < 0.5, -(2**31) + 1, 2**31 - 1)}[kind].astype(np.int32)
    for top in (1, 32):
        check(llmx, torch, z, np.array([0, 19999, 10007], np.uint32), None, top)


@gpu
def test_nearly_certain(llmx, torch):
    """One token with nearly all the probability: its log probability and the entropy keep their digits."""
    rng = np.random.default_rng(5)
    z = np.rint(rng.normal(0, 1, (4, 30000)) * 65536).astype(np.int32)
    z[np.arange(4), [0, 511, 512, 29999]] = (np.array([18, 25, 40, 90]) * 65536).astype(np.int32)
    got, want = check(llmx, torch, z, z.argmax(1).astype(np.uint32), None, 2)
    # 2^-22 of a term, 2^-23 d <= 2^-16.4 of its exponent's rounding (d < 96), the sums' 2^-17; and
    # terms below 2^-126 are taken for 0, 30000 at most
    assert (np.abs(got["logprob"] - want["logprob"]) <= 3e-5 * np.abs(want["logprob"]) + 30000 * 2.0**-126).all()


@gpu
def test_graph_streams_and_repeats(llmx, torch):
    rng = np.random.default_rng(6)
    z, other = logits(rng, 20, 9000), logits(rng, 20, 9000)
    tokens = draw_tokens(rng, z)
    d = Device(llmx, torch, z, tokens, None, 7)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        d.call()
    torch.cuda.synchronize()
    first, _ = d.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.call()
    mine = d.logits.clone()
    for d.z, data in ((other, Device(llmx, torch, other, tokens, None, 7).logits), (z, mine)):
        d.logits.copy_(data)
        graph.replay()
        d.check()
    for _ in range(5):  # the same bits every time
        d.call()
        again, _ = d.check()
        for f in first:
            assert np.array_equal(first[f], again[f])
    a, b = Device(llmx, torch, z, tokens, None, 7), Device(llmx, torch, other, tokens, None, 7)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        a.call(s1.cuda_stream)
        b.call(s2.cuda_stream)
    a.check()
    b.check()


@gpu
def test_offsets_beyond_32_bits(llmx, torch):
    """Rows that lie 2^27 elements apart, the last ones behind 2^31."""
    rng = np.random.default_rng(8)
    ld, rows, vocab = 2**27 + 1, 19, 700
    z = logits(rng, rows, vocab)
    tokens = draw_tokens(rng, z)
    d = Device(llmx, torch, z, tokens, None, 5)
    big = torch.empty((rows - 1) * ld + vocab, dtype=torch.int32, device="cuda")
    for r in range(rows):
        big[r * ld:r * ld + vocab] = torch.from_numpy(z[r]).cuda()
    d.logits, d.at, d.ld = big, big.data_ptr(), ld
    d.call()
    d.check()


@gpu
@pytest.mark.parametrize("vocab,rows", [(2**22, 3), (1, 2000), (5, 20000)])
def test_largest(llmx, torch, vocab, rows):
    rng = np.random.default_rng(9)
    z = rng.integers(-(2**19), 2**19, (rows, vocab)).astype(np.int32)
    check(llmx, torch, z, rng.integers(0, vocab, rows).astype(np.uint32), None, 3)


@gpu
def test_of_verified_tokens(llmx, torch):
    """What the verification of drafts leaves, asked for at once: the rows' tokens go from one call to the
    next on the device, in one graph."""
    import test_verify as V
    rng = np.random.default_rng(10)
    counts, vocab = [3, 0, 4, 1], 20011
    for temperature in (0.0, 1.0):
        c = V.make(rng, counts, vocab, temperature=[temperature] * 4)
        v = V.Device(llmx, torch, c)
        most, rows = c["most"], len(c["target"])
        where = torch.tensor([r * (most + 1) + j for r, k in enumerate(counts) for j in range(k + 1)], device="cuda")
        d = Device(llmx, torch, c["target"], np.zeros(rows, np.uint32), None, 4)

        def step():
            v.call()
            d.d_tokens.copy_(v.out[where])
            d.call()

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for _ in range(2):
            d.d_tokens.fill_(1)
            graph.replay()
            tokens = v.check()[0]  # (requests, most + 1), 0xffffffff behind the drawn one
            d.tokens = tokens.reshape(-1)[where.cpu().numpy()]
            got, _ = d.check()
            drawn = d.tokens != NO_TOKEN
            assert drawn.sum() >= len(counts) and (got["rank"][~drawn] == NO_TOKEN).all()
            if temperature == 0:  # an accepted draft and a drawn token are the rows' maxima
                assert (got["rank"][drawn] == 0).all()


@gpu
@pytest.mark.parametrize("top", [1, 2, 3, 4, 5, 9])
def test_many_equal_many_rows(llmx, torch, top):
    """More equal tokens than are compared all with all, in many rows at once: warps that have none of the best chunks to
    look through (top below 8) are at the lists' end long before the others.  The same bits in every row and every call."""
    rng = np.random.default_rng(top)
    rows, vocab = 600, 2048
    z = np.tile(rng.integers(-9, 1, vocab) // 2 * 65536, (rows, 1)).astype(np.int32)  # some 200 of each value
    z[:, rng.random(vocab) < 0.3] = 65536
    tokens = np.full(rows, 1500, np.uint32)
    d = Device(llmx, torch, z, tokens, None, top)
    want = oracle(z[:1], tokens[:1], np.ones(1, np.float32), top)
    log, ent = bounds(want["terms"][0], vocab // 512 + 1)
    for _ in range(20):
        d.call()
        got = d.result()
        for f in ("logprob", "rank", "entropy", "top_tokens", "top_logprobs"):
            assert (got[f] == got[f][:1]).all(), f
        assert np.array_equal(got["top_tokens"][0], want["top_tokens"][0]) and got["rank"][0] == want["rank"][0]
        assert abs(got["entropy"][0] - want["entropy"][0]) <= ent + want["entropy"][0] * 2.0**-24
        for g, w in ((got["logprob"][0], want["logprob"][0]), (got["top_logprobs"][0], want["top_logprobs"][0])):
            assert (np.abs(g - w) <= log + np.abs(w) * 2.0**-24).all()
