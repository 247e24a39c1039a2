"""Verification of drafted tokens (llmx_verify_drafts).

Results are whole numbers fixed by the formula, so every comparison with the
64-bit implementation is exact (tolerance 0).
"""
import numpy as np
import pytest

import serving_oracle as S

gpu = pytest.mark.gpu
NONE = S.NONE


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def logits(rng, rows, vocab, spread=2.5):
    z = rng.normal(0, spread, (rows, vocab))
    for r in range(rows):
        z[r, rng.integers(0, vocab, 4)] += rng.random(4) * 12
    return np.clip(np.rint(z * 65536), -(2**31) + 1, 2**31 - 1).astype(np.int32)


def make(rng, counts, vocab, model=True, excluded=0.0, spread=2.5, temperature=None):
    b, drafts = len(counts), int(sum(counts))
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    target = logits(rng, drafts + b, vocab, spread)
    rows = [int(offsets[r]) + r + j for r in range(b) for j in range(counts[r])]
    draft = None
    if model and drafts:
        noise = np.rint(rng.normal(0, 0.5, (drafts, vocab)) * 65536).astype(np.int64)
        draft = np.clip(target[rows].astype(np.int64) + noise, -(2**31) + 1, 2**31 - 1).astype(np.int32)
    source = draft if draft is not None else target[rows]
    # drafted tokens: likely ones of the source rows
    tokens = np.array([int(rng.choice(np.argsort(source[j])[-3:])) for j in range(drafts)], np.uint32)
    if excluded:
        target[rng.random(target.shape) < excluded] = NONE
    t = np.asarray(temperature if temperature is not None else rng.random(b) * 1.5 + 0.3, np.float32)
    return dict(target=target, draft=draft, tokens=tokens, offsets=offsets, most=max(list(counts) + [0]), temperature=t,
                accept_u=rng.integers(0, 2**32, drafts, dtype=np.uint64).astype(np.uint32),
                sample_u=rng.integers(0, 2**32, b, dtype=np.uint64).astype(np.uint32))


class Device:
    """A case's arrays on the device; ld: row stride, skip: elements before the first row."""

    def __init__(self, llmx, torch, c, ld=0, skip=0, with_probs=True):
        self.llmx, self.torch, self.c = llmx, torch, c
        b, drafts, vocab = len(c["offsets"]) - 1, len(c["tokens"]), c["target"].shape[1]
        self.b, self.drafts, self.vocab, self.ld = b, drafts, vocab, ld
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()  # noqa: E731

        def rows(a):
            if a is None:
                return None, None
            wide = np.full((a.shape[0], ld or vocab), 2**31 - 1, np.int32)  # what lies between rows must not matter
            wide[:, :vocab] = a
            t = dev(np.concatenate([np.full(skip, 2**31 - 1, np.int32), wide.reshape(-1)]))
            return t, t.data_ptr() + 4 * skip

        self.keep = []
        (t1, self.target), (t2, self.draft) = rows(c["target"]), rows(c["draft"])
        self.args = [dev(c[f]) for f in ("tokens", "offsets", "accept_u", "sample_u")]
        self.temperature = torch.from_numpy(c["temperature"]).cuda()
        self.keep += [t1, t2]
        self.out = torch.full((b * (c["most"] + 1) + 8,), 777, dtype=torch.int32, device="cuda")
        self.accepted = torch.full((b + 8,), 777, dtype=torch.int32, device="cuda")
        self.probs = torch.full((drafts + 4, 2), 777, dtype=torch.int64, device="cuda") if with_probs else None
        size = llmx.verify_workspace_bytes(b, drafts, vocab)
        self.work = torch.full((size + 64,), 85, dtype=torch.uint8, device="cuda")
        self.size = size

    def call(self, stream=None):
        tokens, offsets, accept_u, sample_u = self.args
        p = lambda t: t.data_ptr() if t is not None and t.numel() else None  # noqa: E731
        self.llmx.verify_drafts(self.target, self.draft, self.vocab, p(tokens), p(offsets), self.b, self.drafts, self.c["most"],
                                p(self.temperature), p(accept_u), p(sample_u), p(self.out), p(self.accepted), p(self.probs),
                                p(self.work), self.size, ld_target=self.ld, ld_draft=self.ld,
                                stream=stream if stream is not None else self.torch.cuda.current_stream().cuda_stream)

    def check(self):
        self.torch.cuda.synchronize()
        c = self.c
        want = S.verify(c["target"], c["draft"], c["tokens"], c["offsets"], c["most"], c["temperature"], c["accept_u"], c["sample_u"])
        out, accepted = self.out.cpu().numpy(), self.accepted.cpu().numpy()
        n = self.b * (c["most"] + 1)
        assert (out[n:] == 777).all() and (accepted[self.b:] == 777).all() and (self.work[self.size:].cpu() == 85).all()
        if self.probs is not None:
            probs = self.probs.cpu().numpy()
            assert (probs[self.drafts:] == 777).all()
            for j, pq in want[2].items():
                assert tuple(probs[j]) == pq, (j, probs[j], pq)
        assert np.array_equal(accepted[:self.b].view(np.uint32), want[1]), (accepted[:self.b], want[1])
        assert np.array_equal(out[:n].view(np.uint32).reshape(want[0].shape), want[0])
        return want


def check(llmx, torch, c, **kw):
    d = Device(llmx, torch, c, **kw)
    d.call()
    return d.check()


def test_weights_are_a_softmax():
    """The weights' error against exp in 64 bits: 2e-7 of the polynomial with its
    rounded steps; the rounding of e (below 32) and of the scale move the exponent by at most
    32 * 2^-24 * 2 octaves (ln 2 each); and one unit of truncation."""
    rng = np.random.default_rng(0)
    for t in (0.25, 0.7, 1.0, 3.0):
        z = logits(rng, 1, 20000)[0]
        w = S.weights(z, t)
        d = (int(z.max()) - z.astype(np.int64)) / 65536 / np.float64(np.float32(t))
        true = np.exp(-d) * 2.0**31
        assert (np.abs(w - true) <= true * (2e-7 + 64 * 2.0**-24 * np.log(2)) + 1).all()
        p = S.shares(w)
        assert abs(int(p.sum()) - 2**40) < 2**20 and p.max() <= 2**40


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 31, 32, 33, 127, 1000, 1023, 1024, 1025, 4099, 16384, 32001, 65536, 151936])
@pytest.mark.parametrize("model", [True, False])
def test_vocabularies(llmx, torch, vocab, model):
    rng = np.random.default_rng(vocab)
    check(llmx, torch, make(rng, [3, 0, 1, 4], vocab, model))


@gpu
@pytest.mark.parametrize("counts", [[0], [1], [7], [0, 0, 0], [5, 0, 2], [12] * 3, [1, 40, 0], [3] * 70, [0] * 300])
def test_counts(llmx, torch, counts):
    rng = np.random.default_rng(len(counts))
    check(llmx, torch, make(rng, counts, 501))
    check(llmx, torch, make(rng, counts, 500, excluded=0.3), with_probs=False)


@gpu
@pytest.mark.parametrize("seed", range(6))
def test_many_requests(llmx, torch, seed):
    """Small vocabularies, many draws: every branch of accept and draw."""
    rng = np.random.default_rng(seed)
    counts = rng.integers(0, 5, 400).tolist()
    c = make(rng, counts, [2, 5, 17, 64, 130, 259][seed], model=seed % 2 == 0, spread=1.0, excluded=0.2 * (seed > 2))
    c["tokens"] = rng.integers(0, c["target"].shape[1], len(c["tokens"])).astype(np.uint32)
    want = check(llmx, torch, c)
    assert len(set(want[1].tolist())) > 1  # accepted and rejected drafts both occur


@gpu
@pytest.mark.parametrize("requests,k,vocab", [(60, 2, 30001), (200, 1, 9000), (20, 2, 151936), (90, 0, 100003), (500, 0, 5000),
                                              (3, 0, 400000), (2, 1, 900001)])
def test_many_long_rows(llmx, torch, requests, k, vocab):
    """More rows than run at once, rows held by clusters of every size, and rows that pass
    through shared memory twice; rows of every alignment."""
    rng = np.random.default_rng(requests + vocab)
    c = make(rng, [k - (r % 3 == 2 and k > 0) for r in range(requests)], vocab, temperature=rng.random(requests) + 0.4)
    c["temperature"][::5] = 0.0
    d = Device(llmx, torch, c)
    d.call()
    d.check()
    for _ in range(5):  # the same again, back to back
        d.call()
    d.check()


@gpu
@pytest.mark.parametrize("ld,skip", [(1001, 0), (1004, 0), (1004, 1), (1003, 3), (2048, 2), (0, 1)])
@pytest.mark.parametrize("vocab", [999, 1000])
def test_strides(llmx, torch, vocab, ld, skip):
    rng = np.random.default_rng(ld + skip)
    check(llmx, torch, make(rng, [2, 3, 0], vocab), ld=ld, skip=skip)


@gpu
@pytest.mark.parametrize("vocab", [3, 130, 40000])
def test_masks(llmx, torch, vocab):
    """Rows that exclude every token, all but one, and the drafted token itself."""
    rng = np.random.default_rng(vocab)
    c = make(rng, [2, 2, 1, 0, 2], vocab, temperature=[1.0, 0.0, 0.5, 1.0, 0.0])
    c["target"][0] = NONE            # request 0: first row empty, nothing can be accepted
    c["target"][4, 1:] = NONE        # request 1, second row: one token left
    c["target"][6, c["tokens"][4]] = NONE  # request 2: the drafted token is excluded
    c["target"][8] = NONE            # request 3: nothing to sample from
    c["draft"][5] = NONE             # request 4, first draft row empty
    c["accept_u"][:] = 0
    want = check(llmx, torch, c)
    assert want[0][0, 0] == S.NO_TOKEN and want[0][3, 0] == S.NO_TOKEN and want[1][2] == 0


@gpu
@pytest.mark.parametrize("vocab", [64, 1001, 33333])
def test_flat_and_extreme_rows(llmx, torch, vocab):
    """Equal logits, the type's ends, and differences that pass 31 bits."""
    rng = np.random.default_rng(vocab)
    c = make(rng, [1] * 6, vocab, temperature=[1.0, 1e-3, 1e4, 0.0, 0.7, 1.0])
    c["target"][0] = 5
    c["target"][1] = 2**31 - 1
    c["target"][2, :] = -(2**31) + 1
    c["target"][2, vocab // 2] = 2**31 - 1
    c["target"][4] = NONE + 1
    c["draft"][0] = -7
    c["draft"][1, ::2] = 2**31 - 1
    c["draft"][1, 1::2] = NONE + 1
    c["target"][6] = 9               # greedy request with ties everywhere
    check(llmx, torch, c)


@gpu
def test_random_numbers_at_their_ends(llmx, torch):
    rng = np.random.default_rng(4)
    for accept in (0, 1, 2**31, 2**32 - 1):
        for sample in (0, 1, 2**32 - 1):
            c = make(rng, [2, 0, 3], 300)
            c["accept_u"][:] = accept
            c["sample_u"][:] = sample
            check(llmx, torch, c)
            c["draft"] = None
            check(llmx, torch, c)


@gpu
@pytest.mark.parametrize("t", [0.0, -1.0, 1e-6, 1.1e-6, 1e-4, 0.05, 50.0, 1e30, float("inf"), float("nan")])
def test_temperatures(llmx, torch, t):
    rng = np.random.default_rng(5)
    c = make(rng, [2, 3, 0, 1], 700, temperature=[t] * 4)
    want = check(llmx, torch, c)
    if not np.float32(t) > np.float32(1e-6):  # greedy: an accepted draft is the first maximum of its row
        for r in range(4):
            row = int(c["offsets"][r]) + r
            for j in range(int(want[1][r]) + 1):
                assert want[0][r, j] == np.argmax(c["target"][row + j])


@gpu
def test_same_distribution_accepts_everything(llmx, torch):
    """p = q: every draft is accepted, whatever the number; a token outside the
    vocabulary is rejected and, with nothing left of p - q, p is drawn from."""
    rng = np.random.default_rng(6)
    c = make(rng, [4, 4, 4], 777)
    rows = [int(c["offsets"][r]) + r + j for r in range(3) for j in range(4)]
    c["draft"] = c["target"][rows].copy()
    c["accept_u"][:] = 2**32 - 1
    want = check(llmx, torch, c)
    assert (want[1] == 4).all()
    c["tokens"][2] = 777
    c["tokens"][5] = 2**32 - 1
    want = check(llmx, torch, c)
    assert want[1].tolist() == [2, 1, 4]


@gpu
def test_offsets_out_of_order(llmx, torch):
    """A request with unusable offsets gets no tokens; the others are served."""
    rng = np.random.default_rng(7)
    c = make(rng, [2, 2, 2, 2], 300)
    for bad in ([0, 2, 1, 6, 8], [0, 2, 4, 99, 8], [0, 2**32 - 1, 4, 6, 8], [0, 8, 8, 8, 8]):
        c["offsets"] = np.array(bad, np.uint32)
        d = Device(llmx, torch, c)
        d.call()
        torch.cuda.synchronize()
        got = d.accepted.cpu().numpy()[:4].view(np.uint32)
        for r in range(4):
            ok = 0 <= bad[r + 1] - bad[r] <= 2 and bad[r + 1] <= 8
            assert (got[r] != S.NO_TOKEN) == ok
        out = d.out.cpu().numpy()[:12].view(np.uint32).reshape(4, 3)
        assert (out[got == S.NO_TOKEN] == S.NO_TOKEN).all()


@gpu
def test_drawn_frequencies(llmx, torch):
    """Draft, verify, draw: the first emitted token follows the target's
    distribution.  Over n requests a frequency of probability p has a standard deviation of
    sqrt(p (1 - p) / n); 5 of them (and 1 count) bound eight tokens' frequencies."""
    rng = np.random.default_rng(9)
    n, vocab = 60000, 8
    zt, zd = rng.normal(0, 1, vocab), rng.normal(0, 1, vocab)
    pd = np.exp(zd) / np.exp(zd).sum()
    c = dict(target=np.repeat(np.rint(zt * 65536).astype(np.int32)[None], 2 * n, 0),
             draft=np.repeat(np.rint(zd * 65536).astype(np.int32)[None], n, 0),
             tokens=rng.choice(vocab, n, p=pd).astype(np.uint32), offsets=np.arange(n + 1, dtype=np.uint32), most=1,
             temperature=np.ones(n, np.float32), accept_u=rng.integers(0, 2**32, n, dtype=np.uint64).astype(np.uint32),
             sample_u=rng.integers(0, 2**32, n, dtype=np.uint64).astype(np.uint32))
    d = Device(llmx, torch, c)
    d.call()
    torch.cuda.synchronize()
    first = d.out.cpu().numpy()[:2 * n].reshape(n, 2)[:, 0]
    p = np.exp(zt) / np.exp(zt).sum()
    freq = np.bincount(first, minlength=vocab) / n
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1 / n).all(), (freq, p)


@gpu
def test_stream_graph_and_reuse(llmx, torch):
    """One workspace for calls of other sizes, on a stream of its own, captured, and again."""
    rng = np.random.default_rng(10)
    side = torch.cuda.Stream()
    cases = [make(rng, counts, 5000) for counts in ([3, 4], [0, 2, 1], [7])]
    devs = [Device(llmx, torch, c) for c in cases]
    big = max(d.size for d in devs)
    work = torch.full((big + 64,), 85, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for d in devs:
        d.work, d.size = work, big
        d.call(side.cuda_stream)
    side.synchronize()
    for d in devs:
        d.check()
    d = devs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d.call(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        d.c["sample_u"] = rng.integers(0, 2**32, d.b, dtype=np.uint64).astype(np.uint32)
        d.args[3].copy_(torch.from_numpy(d.c["sample_u"].view(np.int32)))
        g.replay()
        d.check()


@gpu
def test_offsets_beyond_32_bits(llmx, torch):
    """Rows 2^28 elements apart: the last starts past 2^32 bytes."""
    rng = np.random.default_rng(11)
    c = make(rng, [4, 3], 1000, model=False)
    d = Device(llmx, torch, c)
    far = 1 << 28
    t = torch.empty(8 * far + 1000, dtype=torch.int32, device="cuda")
    for r in range(9):
        t[r * far:r * far + 1000] = torch.from_numpy(c["target"][r]).cuda()
    d.target, d.ld = t.data_ptr(), far
    d.call()
    d.check()
    del t
    torch.cuda.empty_cache()


# ---- refusals (no GPU work) -----------------------------------------------------------
@pytest.mark.parametrize("kw,text", [
    ({"target": None}, "null"), ({"offsets": None}, "null"), ({"temperature": None}, "null"), ({"sample_u": None}, "null"),
    ({"tokens": None}, "null"), ({"accepted": None}, "null"), ({"work": None}, "null"), ({"draft_tokens": None}, "drafts > 0"),
    ({"accept_u": None}, "drafts > 0"), ({"vocab": 0}, "vocab"), ({"vocab": (1 << 22) + 1}, "vocab"), ({"requests": 0}, "requests"),
    ({"requests": 65536}, "requests"), ({"drafts": (1 << 24) + 1}, "drafts"), ({"max_drafts": 1024}, "max_drafts"),
    ({"drafts": 9}, "requests * max_drafts"), ({"ld_target": 99}, "stride"), ({"ld_draft": 99}, "stride"), ({"target": 4098}, "aligned"),
    ({"probs": 4100}, "aligned"), ({"work": 4100}, "256"), ({"size": 8}, "workspace too small")])
def test_refusals(llmx, kw, text):
    a = dict(target=4096, ld_target=0, draft=4096, ld_draft=0, vocab=100, draft_tokens=4096, offsets=4096, requests=2, drafts=4,
             max_drafts=4, temperature=4096, accept_u=4096, sample_u=4096, tokens=4096, accepted=4096, probs=4096, work=4096,
             size=1 << 20)
    a.update(kw)
    rc = llmx.lib().llmx_verify_drafts(a["target"], a["ld_target"], a["draft"], a["ld_draft"], a["vocab"], a["draft_tokens"],
                                       a["offsets"], a["requests"], a["drafts"], a["max_drafts"], a["temperature"],
                                       a["accept_u"], a["sample_u"], a["tokens"], a["accepted"], a["probs"], a["work"],
                                       a["size"], None)
    assert rc == llmx.ERR_ARG and text in llmx.last_error()


def test_workspace_grows_with_the_call(llmx):
    f = llmx.verify_workspace_bytes
    assert 0 < f(1, 0, 10) <= f(1, 7, 10) <= f(64, 448, 151936)


@gpu
@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("vocab", [501, 5000])
def test_many_drafts_accepted(llmx, torch, vocab, model):
    """More drafts accepted than the rows whose numbers stay in shared memory (32): all of them, then
    a rejection at 31, 32, 33 and 39, sampled and greedy."""
    rng = np.random.default_rng(12)
    counts = [40] * 6 + [0, 33]
    c = make(rng, counts, vocab, model, temperature=[0.8, 0.8, 0.8, 0.0, 0.0, 1.2, 1.0, 0.9])
    off = [int(o) for o in c["offsets"]]
    rows = [off[r] + r + j for r in range(len(counts)) for j in range(counts[r])]
    c["tokens"] = np.argmax(c["target"][rows], 1).astype(np.uint32)
    if model:
        c["draft"] = c["target"][rows].copy()
        c["accept_u"][:] = 2**32 - 1  # p = q is accepted whatever the number
    else:
        c["accept_u"][:] = 0
    stop = {1: 31, 2: 32, 4: 33, 5: 39}
    for r, j in stop.items():
        c["target"][off[r] + r + j, c["tokens"][off[r] + j]] = NONE  # and so rejected
    want = check(llmx, torch, c)
    assert want[1].tolist() == [40, 31, 32, 40, 33, 39, 0, 33]


@gpu
def test_offsets_out_of_order_leave_the_others(llmx, torch):
    """Beside requests with unusable offsets, those whose rows nobody else claims get their exact
    tokens and probabilities."""
    rng = np.random.default_rng(13)
    c = make(rng, [2, 2, 2, 2], 300)
    # offsets and the requests with usable ones that share no row
    for bad, alone in (([0, 2, 1, 6, 8], [0, 3]), ([0, 2, 4, 99, 8], [0, 1]), ([0, 2**32 - 1, 4, 6, 8], [2, 3]), ([0, 8, 8, 8, 8], [1, 2, 3]),
                       ([0, 2, 99, 6, 8], [0, 3])):
        c["offsets"] = np.array(bad, np.uint32)
        d = Device(llmx, torch, c)
        d.call()
        torch.cuda.synchronize()
        want = S.verify(c["target"], c["draft"], c["tokens"], c["offsets"], c["most"], c["temperature"], c["accept_u"], c["sample_u"])
        out, accepted = d.out.cpu().numpy()[:12].view(np.uint32).reshape(4, 3), d.accepted.cpu().numpy()[:4].view(np.uint32)
        probs = d.probs.cpu().numpy()
        for r in range(4):
            if want[1][r] == S.NO_TOKEN:
                assert accepted[r] == S.NO_TOKEN and (out[r] == S.NO_TOKEN).all()
            elif r in alone:
                assert accepted[r] == want[1][r] and np.array_equal(out[r], want[0][r])
                for j in range(bad[r], bad[r + 1]):
                    assert tuple(probs[j]) == want[2][j]
        assert all(want[1][r] != S.NO_TOKEN for r in alone)
