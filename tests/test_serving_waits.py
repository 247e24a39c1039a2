"""Waits that run out in the kernels that serve several requests.

Their bound is set so low (llmx_selftest_serving_waits) that warps give up while copies and other
warps are still under way.  The kernels have to end, report what they gave up, and serve the next
call exactly.
"""
import numpy as np
import pytest

import serving_oracle as S
from test_adapters import Case, whole
from test_verify import Device, make

pytestmark = pytest.mark.gpu
POLLS = [0, 1, 2, 3, 4, 6, 9]


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture
def short(llmx):
    """Sets the bound; the default is back after the test."""
    yield llmx.selftest_serving_waits
    llmx.selftest_serving_waits()


def project(llmx, torch, short, k, n, ranks, rows):
    c = Case(llmx, torch, k, n, ranks, rows, seed=k)
    x = whole(c.rng, (rows, k), 700)
    slot = c.rng.integers(-1, len(ranks), rows)
    outcomes = []
    for polls in POLLS:
        short(polls)
        for _ in range(3):
            try:
                c.check(x, slot, wide=True)  # exact, or reported
                outcomes.append(llmx.OK)
            except llmx.LlmxError as e:
                outcomes.append(e.code)
        short()
        c.check(x, slot, wide=True)
    assert set(outcomes) <= {llmx.OK, llmx.ERR_TIMEOUT} and outcomes[:3] == [llmx.ERR_TIMEOUT] * 3


@pytest.mark.parametrize("k,n,ranks,rows", [(64, 100, [9], 1), (2048, 2560, [16, 4], 1), (1096, 4999, [13] * 20, 77),
                                            (2048, 22016, [32] * 16, 16), (2048, 3000, [64] * 4, 300)])
def test_projection(llmx, torch, short, k, n, ranks, rows):
    project(llmx, torch, short, k, n, ranks, rows)


@pytest.mark.parametrize("k,n,ranks,rows", [(11008, 2048, [16, 5], 8), (32768, 200, [128], 2), (4096, 4000, [16] * 3, 40)])
def test_projection_of_many_inputs(llmx, torch, short, k, n, ranks, rows):
    """Adapters' products cut over the blocks of a cluster."""
    project(llmx, torch, short, k, n, ranks, rows)


@pytest.mark.parametrize("counts,vocab", [([3, 0, 2], 997), ([1] * 300, 500), ([0] * 500, 2000),
                                          # requests of two CTAs each
                                          ([3, 0, 2], 4000), ([1] * 60, 4000), ([0], 4000),
                                          # rows and requests of several CTAs
                                          ([3, 0, 2], 50001), ([4], 151936), ([0] * 100, 30001), ([2] * 60, 60002)])
def test_verification(llmx, torch, short, counts, vocab):
    d = Device(llmx, torch, make(np.random.default_rng(vocab), counts, vocab))
    for polls in POLLS:
        short(polls)
        for _ in range(3):
            d.call()
        torch.cuda.synchronize()
        short()
        d.call()
        d.check()


def exact_or_given_up(torch, d):
    """Every request has its tokens, or accepted = 0xffffffff; how many have the latter."""
    torch.cuda.synchronize()
    c = d.c
    want = d.want
    n = d.b * (c["most"] + 1)
    accepted = d.accepted.cpu().numpy()[:d.b].view(np.uint32)
    out = d.out.cpu().numpy()[:n].view(np.uint32).reshape(d.b, -1)
    gone = accepted == S.NO_TOKEN
    assert np.array_equal(accepted[~gone], want[1][~gone]) and np.array_equal(out[~gone], want[0][~gone])
    return int(gone.sum())


@pytest.mark.parametrize("counts,vocab", [([3, 0, 2], 997), ([1] * 300, 500), ([0] * 150, 20000), ([1] * 100, 40001), ([0] * 80, 150001)])
def test_sums_given_up_are_marked(llmx, torch, short, counts, vocab):
    """A row of which any warp gave up has no sum, whatever the other warps did after that."""
    d = Device(llmx, torch, make(np.random.default_rng(vocab), counts, vocab))
    d.call()
    d.want = d.check()
    for polls in POLLS:
        short(polls)
        for _ in range(30):
            d.accepted.fill_(777)
            d.call()
            gone = exact_or_given_up(torch, d)
            assert polls > 0 or gone == d.b


@pytest.mark.parametrize("counts,vocab,ctas", [([3, 0, 2], 4000, 2), ([1] * 60, 4000, 2), ([0], 40000, 16), ([4], 151936, 16),
                                               ([3, 0, 2], 50001, 16), ([0] * 30, 20000, 8), ([2] * 60, 60002, 4)])
@pytest.mark.parametrize("model", [True, False])
def test_draws_given_up_are_marked(llmx, torch, short, counts, vocab, ctas, model):
    """A request of which any CTA lacks the others' sums has no tokens: neither a count without
    its token nor one CTA's token beside another's mark."""
    d = Device(llmx, torch, make(np.random.default_rng(vocab), counts, vocab, model=model))
    for lost in (0, 1, 2, 3, 1 << (ctas - 1), (1 << ctas) - 1, (1 << ctas) - 2, 0x5555, 0xaaaa):
        lost &= (1 << ctas) - 1
        short(None, lost)
        for _ in range(5):
            d.accepted.fill_(777)
            d.out.fill_(777)
            d.call()
            torch.cuda.synchronize()
            if lost:
                assert (d.accepted[:d.b] == -1).all() and (d.accepted[d.b:] == 777).all()
                n = d.b * (d.c["most"] + 1)
                assert (d.out[:n] == -1).all() and (d.out[n:] == 777).all()
            else:
                d.check()
    short()
    d.call()
    d.check()
