"""The shared projection with per-row low-rank adapters (llmx_adapters_*).

Results are whole numbers fixed by the formula, so every comparison with the
64-bit implementation is exact (tolerance 0).
"""
import ctypes as C

import numpy as np
import pytest

import serving_oracle as S

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def whole(rng, shape, sigma):
    return np.clip(np.rint(rng.normal(0, sigma, shape)), -32768, 32767).astype(np.int16)


class Case:
    """A handle with adapters on the device, and what it was made from."""

    def __init__(self, llmx, torch, k, n, ranks, max_rows, seed=0, sigma_w=82, extreme=False, max_rank=None):
        self.llmx, self.torch, self.k, self.n = llmx, torch, k, n
        rng = self.rng = np.random.default_rng(seed)
        self.w = np.full((n, k), -32768, np.int16) if extreme else whole(rng, (n, k), sigma_w)
        self.adapters = {}
        top = max_rank or max(list(ranks) + [1])
        dw = self.dev(self.w)
        self.h = llmx.Adapters(k, n, dw.data_ptr(), len(ranks), top, max_rows, stream=self.stream())
        for s, r in enumerate(ranks):
            self.put(s, r, extreme)
        torch.cuda.synchronize()
        dw.zero_()  # the handle keeps its own layout

    def put(self, s, r, extreme=False):
        rng, t = self.rng, self.torch
        if r == 0:
            self.h.set(s, 0, stream=self.stream())
            self.adapters.pop(s, None)
            return
        down = np.full((r, self.k), 32767, np.int16) if extreme else whole(rng, (r, self.k), 82)
        up = np.full((self.n, r), -32768, np.int16) if extreme else whole(rng, (self.n, r), 400)
        scale = -32768 if extreme else int(rng.integers(-32768, 32767))
        dd, du = self.dev(down), self.dev(up)
        self.h.set(s, r, scale, dd.data_ptr(), du.data_ptr(), stream=self.stream())
        t.cuda.synchronize()
        dd.zero_()
        du.zero_()
        self.adapters[s] = (scale, down, up)

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def run(self, x, slot, wide, pad_x=0, pad_out=0):
        t, rows = self.torch, x.shape[0]
        xs = np.full((rows, self.k + pad_x), 12345, np.int16)
        xs[:, :self.k] = x
        dx = self.dev(xs)
        ds = self.dev(np.asarray(slot, np.int32)) if slot is not None else None
        kind = t.int32 if wide else t.int16
        out = t.full((rows + 1, self.n + pad_out), 777, dtype=kind, device="cuda")
        self.h.project(dx.data_ptr(), rows, ds.data_ptr() if ds is not None else None, out.data_ptr(),
                       self.llmx.OUT_Q16_16 if wide else self.llmx.OUT_Q8_8, ld_x=self.k + pad_x if pad_x else 0,
                       ld_out=self.n + pad_out if pad_out else 0, stream=self.stream())
        t.cuda.synchronize()
        self.h.error(self.stream())
        o = out.cpu().numpy()
        assert (o[rows:] == 777).all() and (o[:, self.n:] == 777).all(), "wrote outside the rows"
        return o[:rows, :self.n]

    def check(self, x, slot, wide, **kw):
        got = self.run(x, slot, wide, **kw)
        want = S.project(x, self.w, slot, self.adapters, wide)
        bad = np.argwhere(got != want)
        assert bad.size == 0, (len(bad), bad[:4].tolist(), got[tuple(bad[0])], want[tuple(bad[0])])


ROWS = [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 48, 64, 65, 100, 128, 129, 200, 257]


@gpu
@pytest.mark.parametrize("rows", ROWS)
def test_rows(llmx, torch, rows):
    """Row counts on both sides of every row tile, each row of its own adapter or none."""
    c = Case(llmx, torch, 264, 300, [5, 16, 0, 33, 17, 1], 257, seed=rows)
    x = whole(c.rng, (rows, 264), 900)
    slot = c.rng.integers(-2, 8, rows)  # -2, -1, 6, 7: none; 2: empty
    c.check(x, slot, wide=rows % 2 == 0)
    c.check(x, None, wide=True)


@gpu
@pytest.mark.parametrize("k,n", [(8, 1), (64, 3), (72, 127), (120, 128), (128, 129), (136, 255), (256, 256), (1000, 1025),
                                 (2048, 2560), (11008, 200), (32768, 40)])
@pytest.mark.parametrize("rows", [1, 8, 21, 70])
def test_sizes(llmx, torch, k, n, rows):
    c = Case(llmx, torch, k, n, [16, 7, 40], rows, seed=k + n)
    x = whole(c.rng, (rows, k), 500)
    c.check(x, c.rng.integers(-1, 3, rows), wide=True)
    c.check(x, c.rng.integers(-1, 3, rows), wide=False)


@gpu
@pytest.mark.parametrize("rank", [1, 2, 15, 16, 17, 31, 32, 48, 64, 100, 112, 127, 128])
def test_ranks(llmx, torch, rank):
    """Ranks around the tensor cores' steps, next to adapters of other ranks in
    the same row tile, and more adapters than one row tile's stage holds."""
    ranks = [rank, max(1, rank // 2), rank, 3, rank]
    c = Case(llmx, torch, 512, 200, ranks, 40, seed=rank, max_rank=max(rank, 3) if rank < 128 else 128)
    x = whole(c.rng, (40, 512), 700)
    c.check(x, np.arange(40) % 5, wide=True)
    c.check(x, np.arange(40) // 8, wide=False)
    c.check(x[:1], [2], wide=True)


@gpu
def test_many_adapters(llmx, torch):
    """Every row of 130 has an adapter of its own, then all share one."""
    c = Case(llmx, torch, 128, 140, [1 + s % 40 for s in range(130)], 130, seed=3)
    x = whole(c.rng, (130, 128), 700)
    c.check(x, c.rng.permutation(130), wide=True)
    c.check(x, np.full(130, 77), wide=True)
    c.check(x, np.full(130, -1), wide=False)


@gpu
@pytest.mark.parametrize("rows", [5, 40, 200, 300])
@pytest.mark.parametrize("more", [0, 1, 3, 60, 147])
def test_tiles_beyond_the_processors(llmx, torch, rows, more):
    """More tiles than processors, with a few, many and no tiles left over to share; an
    accumulator that a call leaves behind would show in the next."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = (sms + more) * 128 - 5
    for k in (64, 640):
        c = Case(llmx, torch, k, n, [9, 20, 33], rows, seed=more)
        for _ in range(2):
            x = whole(c.rng, (rows, k), 700)
            c.check(x, c.rng.integers(-1, 3, rows), wide=True)


@gpu
@pytest.mark.parametrize("n", [100, 4999, 9000, 18900])
@pytest.mark.parametrize("k", [64, 1096, 11008])
def test_fewer_tiles_than_processors(llmx, torch, n, k):
    """Rows over one or several row tiles, tiles whole or cut, of one handle in turn; row
    tiles whose rows have no adapter, the last one's rows fewer."""
    c = Case(llmx, torch, k, n, [9, 20, 33, 16], 150, seed=n)
    for rows in (128, 1, 17, 33, 150, 77, 49, 97, 113):
        x = whole(c.rng, (rows, k), 700)
        c.check(x, c.rng.integers(-1, 4, rows), wide=True)
        c.check(x, np.where(np.arange(rows) < rows // 2, -1, 2), wide=False)


@gpu
@pytest.mark.parametrize("k", [128, 32768])
@pytest.mark.parametrize("rows", [3, 40, 130])
def test_extremes(llmx, torch, k, rows):
    """Every operand at an end of its range: the longest sums, and saturation of
    t, of the Q16.16 and of the Q8.8 result."""
    c = Case(llmx, torch, k, 130, [128, 16], rows, extreme=True)
    for value in (-32768, 32767, 0, 127, 128, -128, 255, -256):
        x = np.full((rows, k), value, np.int16)
        slot = np.arange(rows) % 3 - 1
        c.check(x, slot, wide=True)
        c.check(x, slot, wide=False)


@gpu
def test_byte_patterns(llmx, torch):
    """Random bits in every operand: carries between the byte planes."""
    rng = np.random.default_rng(8)
    c = Case(llmx, torch, 400, 260, [64, 9], 70)
    bits = lambda shape: rng.integers(-32768, 32768, shape).astype(np.int16)  # noqa: E731
    w = bits((260, 400))
    down, up = bits((64, 400)), bits((260, 64))
    dw, dd, du = c.dev(w), c.dev(down), c.dev(up)
    h = llmx.Adapters(400, 260, dw.data_ptr(), 1, 64, 70, stream=c.stream())
    h.set(0, 64, 9, dd.data_ptr(), du.data_ptr(), stream=c.stream())
    c.h, c.w, c.adapters = h, w, {0: (9, down, up)}
    for rows in (1, 16, 70):
        c.check(bits((rows, 400)), np.arange(rows) % 2 - 1, wide=True)


@gpu
@pytest.mark.parametrize("rows", [1, 20, 140])
def test_strides(llmx, torch, rows):
    c = Case(llmx, torch, 200, 77, [16, 5], rows)
    x = whole(c.rng, (rows, 200), 600)
    slot = np.arange(rows) % 3 - 1
    for pad_x, pad_out in ((8, 0), (0, 1), (56, 19)):
        c.check(x, slot, wide=True, pad_x=pad_x, pad_out=pad_out)
        c.check(x, slot, wide=False, pad_x=pad_x, pad_out=pad_out)


@gpu
def test_slots_change(llmx, torch):
    """A slot set again, emptied and set with another rank serves the new adapter only."""
    c = Case(llmx, torch, 256, 300, [40, 16], 12)
    x = whole(c.rng, (12, 256), 700)
    slot = np.arange(12) % 2
    c.check(x, slot, wide=True)
    for r in (3, 40, 0, 17):
        c.put(0, r)
        c.check(x, slot, wide=True)


@gpu
def test_rows_are_independent(llmx, torch):
    """A row's result is the same alone, in a block and among 200 others."""
    c = Case(llmx, torch, 512, 640, [16, 32, 8], 200)
    x = whole(c.rng, (200, 512), 700)
    slot = c.rng.integers(-1, 3, 200)
    full = c.run(x, slot, True)
    for i in (0, 63, 64, 127, 128, 199):
        assert np.array_equal(c.run(x[i:i + 1], slot[i:i + 1], True)[0], full[i])
    order = c.rng.permutation(200)
    assert np.array_equal(c.run(x[order], slot[order], True), full[order])
    assert np.array_equal(c.run(x[:8], slot[:8], True), full[:8])


@gpu
def test_no_rows_and_no_slots(llmx, torch):
    c = Case(llmx, torch, 128, 128, [], 4)
    x = whole(c.rng, (4, 128), 700)
    c.check(x, None, wide=True)
    c.check(x, [0, 1, -1, 5], wide=True)  # no slots: no adapters
    c.h.project(None, 0, None, None, stream=c.stream())  # no rows: nothing to do


@gpu
@pytest.mark.parametrize("rows", [4, 150])
def test_stream_and_graph(llmx, torch, rows):
    """On a stream of its own, back to back with changing inputs, and captured."""
    c = Case(llmx, torch, 384, 520, [16, 24], rows)
    xs = [whole(c.rng, (rows, 384), 700) for _ in range(4)]
    slots = [c.rng.integers(-1, 2, rows).astype(np.int32) for _ in range(4)]
    side = torch.cuda.Stream()
    outs = []
    with torch.cuda.stream(side):
        for x, s in zip(xs, slots):
            dx, ds = c.dev(x), c.dev(s)
            o = torch.empty((rows, 520), dtype=torch.int32, device="cuda")
            c.h.project(dx.data_ptr(), rows, ds.data_ptr(), o.data_ptr(), llmx.OUT_Q16_16, stream=side.cuda_stream)
            outs.append((o, dx, ds))
    side.synchronize()
    for (o, _, _), x, s in zip(outs, xs, slots):
        assert np.array_equal(o.cpu().numpy(), S.project(x, c.w, s, c.adapters, True))
    dx, ds = c.dev(xs[0]), c.dev(slots[0])
    o = torch.empty((rows, 520), dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.h.project(dx.data_ptr(), rows, ds.data_ptr(), o.data_ptr(), llmx.OUT_Q16_16,
                    stream=torch.cuda.current_stream().cuda_stream)
    for x, s in zip(xs, slots):
        dx.copy_(torch.from_numpy(x))
        ds.copy_(torch.from_numpy(s))
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(o.cpu().numpy(), S.project(x, c.w, s, c.adapters, True))


@gpu
def test_offsets_beyond_32_bits(llmx, torch):
    """An output whose last row starts past 2^32 bytes (rows 2^28 elements apart), and
    input rows as far apart."""
    rows, k, n = 9, 64, 130
    c = Case(llmx, torch, k, n, [4], rows)
    far = 1 << 28
    x = whole(c.rng, (rows, k), 700)
    dx = torch.zeros((rows - 1) * far + k, dtype=torch.int16, device="cuda")
    out = torch.zeros((rows - 1) * far + n, dtype=torch.int32, device="cuda")
    for i in range(rows):
        dx[i * far:i * far + k] = torch.from_numpy(x[i]).cuda()
    slot = c.dev(np.arange(rows, dtype=np.int32) % 2 - 1)
    c.h.project(dx.data_ptr(), rows, slot.data_ptr(), out.data_ptr(), llmx.OUT_Q16_16, ld_x=far, ld_out=far,
                stream=c.stream())
    torch.cuda.synchronize()
    want = S.project(x, c.w, np.arange(rows) % 2 - 1, c.adapters, True)
    for i in range(rows):
        assert np.array_equal(out[i * far:i * far + n].cpu().numpy(), want[i])
    del dx, out
    torch.cuda.empty_cache()


# ---- refusals (no GPU work) -----------------------------------------------------------
def create(llmx, **kw):
    a = dict(device=0, in_dim=128, out_dim=64, weight=1 << 20, slots=2, max_rank=16, max_rows=8)
    a.update(kw)
    h = C.c_void_p()
    rc = llmx.lib().llmx_adapters_create(a["device"], a["in_dim"], a["out_dim"], a["weight"], a["slots"], a["max_rank"],
                                         a["max_rows"], None, C.byref(h))
    return rc, llmx.last_error()


@pytest.mark.parametrize("kw,text", [
    ({"in_dim": 0}, "in_dim"), ({"in_dim": 12}, "in_dim"), ({"in_dim": 32776}, "in_dim"), ({"out_dim": 0}, "out_dim"),
    ({"out_dim": (1 << 22) + 1}, "out_dim"), ({"slots": 65537}, "slots"), ({"max_rank": 0}, "max_rank"),
    ({"max_rank": 129}, "max_rank"), ({"max_rows": 0}, "max_rows"), ({"max_rows": 65537}, "max_rows"),
    ({"weight": None}, "null"), ({"weight": (1 << 20) + 8}, "aligned")])
def test_create_refusals(llmx, kw, text):
    rc, message = create(llmx, **kw)
    assert rc == llmx.ERR_ARG and text in message


def test_null_handle(llmx):
    L = llmx.lib()
    assert L.llmx_adapters_set(None, 0, 0, 0, None, None, None) == llmx.ERR_ARG
    assert L.llmx_adapters_project(None, None, 1, 0, None, None, 0, 0, None) == llmx.ERR_ARG
    assert L.llmx_adapters_error(None, None) == llmx.ERR_ARG
    assert L.llmx_adapters_destroy(None) == llmx.OK
    assert L.llmx_adapters_device_bytes(None) == 0


@gpu
def test_call_refusals(llmx, torch):
    c = Case(llmx, torch, 128, 64, [4], 8)
    t = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    p = t.data_ptr()
    for bad in (dict(rows=9), dict(out_format=2), dict(x=None), dict(out=None), dict(x=p + 2), dict(out=p + 1),
                dict(out=p + 2, out_format=1), dict(slot=p + 2), dict(ld_x=120), dict(ld_x=129), dict(ld_out=63)):
        a = dict(x=p, rows=8, slot=p, out=p + 65536, out_format=0, ld_x=0, ld_out=0)
        a.update(bad)
        with pytest.raises(llmx.LlmxError) as e:
            c.h.project(a["x"], a["rows"], a["slot"], a["out"], a["out_format"], a["ld_x"], a["ld_out"])
        assert e.value.code == llmx.ERR_ARG
    for args in ((1, 4, 0, p, p), (0, 5, 0, p, p), (0, 4, 0, None, p), (0, 4, 0, p, None), (0, 4, 0, p + 2, p),
                 (0, 4, 0, p, p + 1)):
        with pytest.raises(llmx.LlmxError) as e:
            c.h.set(*args)
        assert e.value.code == llmx.ERR_ARG
    c.check(whole(c.rng, (8, 128), 700), np.zeros(8), wide=True)  # the handle still serves


@gpu
def test_refusals_leave_no_error_behind(llmx, torch):
    """A handle that the device cannot hold (2^22 x 32768 weights, 275 GB) or whose device does
    not exist is refused; the calls after that, of this handle, of a new one and of another operator, succeed."""
    c = Case(llmx, torch, 128, 64, [4], 8)
    x = whole(c.rng, (8, 128), 700)
    few = torch.zeros(64 * 128, dtype=torch.int16, device="cuda")
    tokens = torch.zeros(8, dtype=torch.int32, device="cuda")

    def refuse(what):
        with pytest.raises(llmx.LlmxError) as e:
            if what == "memory":
                llmx.Adapters(32768, 1 << 22, few.data_ptr(), 0, 0, 1, stream=c.stream())
            else:
                llmx.Adapters(128, 64, few.data_ptr(), 0, 0, 1, device=9999, stream=c.stream())
        assert e.value.code == (llmx.ERR_NOMEM if what == "memory" else llmx.ERR_CUDA)

    for what in ("memory", "device"):
        refuse(what)
        c.put(0, 3)
        refuse(what)
        h = llmx.Adapters(128, 64, few.data_ptr(), 0, 0, 8, stream=c.stream())
        h.close()
        refuse(what)
        assert llmx.lm_head_argmax_device(few.data_ptr(), 8, 128, few.data_ptr(), 64, tokens.data_ptr(), c.stream()) == llmx.OK
        c.check(x, np.zeros(8), wide=True)


def test_definition_is_the_adapter_in_real_numbers():
    """Against W x + s B (A x) in 64 bits.  t is rounded to Q8.8, half a step of 2^-9 for each rank,
    which up multiplies, and y to the format's step; that is the whole difference while t stays
    within +-128.  A scaled A x below 2^-9 is a t of zero: the adapter then adds nothing."""
    rng = np.random.default_rng(21)
    k, n, rows, rank = 512, 60, 9, 16
    x, w = whole(rng, (rows, k), 256), whole(rng, (n, k), 82)
    down, up, scale = whole(rng, (rank, k), 82), whole(rng, (n, rank), 400), 5000
    real = lambda a, bits: a.astype(np.float64) / 2.0**bits  # noqa: E731
    t = real(x, 8) @ real(down, 12).T * (scale / 4096)
    assert np.abs(t).max() < 128
    y = real(x, 8) @ real(w, 12).T + t @ real(up, 12).T
    off = 2.0**-9 * np.abs(real(up, 12)).sum(1)
    for wide, bits in ((True, 16), (False, 8)):
        got = S.project(x, w, np.zeros(rows, int), {0: (scale, down, up)}, wide).astype(np.float64) / 2.0**bits
        # Q8.8 is rounded by way of Q16.16: half a step of each
        step = 2.0**-(bits + 1) + (0 if wide else 2.0**-17)
        assert (np.abs(got - y) <= off + step + 1e-9).all()
    small = {0: (1, down, up)}  # s = 2^-12: |t| below 2^-9
    assert np.abs(real(x, 8) @ real(down, 12).T / 4096).max() < 2.0**-9
    assert np.array_equal(S.project(x, w, np.zeros(rows, int), small, True), S.project(x, w, None, {}, True))


@gpu
@pytest.mark.parametrize("rows", [1000, 4097, 65536])
def test_hundreds_of_row_tiles(llmx, torch, rows):
    c = Case(llmx, torch, 64, 130, [16, 5, 20], rows)
    x = whole(c.rng, (rows, 64), 900)
    c.check(x, c.rng.integers(-1, 3, rows), wide=True)
    c.check(x, None, wide=False)
    c.check(x[:17], np.arange(17) % 3, wide=True)
