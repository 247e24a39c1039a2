"""The serving loop of speculative.py: adapters, blocks and verification together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def server(spec, model, drafts, ranks=(8, 3)):
    s = model.shape
    out = spec.Server(model, 3, len(ranks), max(ranks), drafts)
    rng = np.random.default_rng(2)
    for slot, rank in enumerate(ranks):
        out.set_adapter(slot, 4096, rng.integers(-400, 400, (rank, s.hidden)), rng.integers(-400, 400, (s.vocab, rank)))
    return out


PROMPTS = [[3, 9, 4, 3, 9], [5, 5, 5, 5], [1, 2, 3, 1, 2, 3, 1]]


def test_drafts_change_nothing_but_the_steps(llmx):
    """Greedy: the tokens with drafts are those without, and some drafts are accepted;
    a request without an adapter gets the tokens of the host's greedy loop."""
    pytest.importorskip("torch")
    import speculative as spec
    s = llmx.shape("small")
    model = llmx.Model(s).init_reference_random(7)
    results = []
    for drafts in (0, 1, 4, 7):
        sv = server(spec, model, drafts)
        out, (drafted, taken) = sv.generate(PROMPTS, [0, -1, 1], 14)
        sv.close()
        assert [len(o) for o in out] == [14, 14, 14]
        results.append(out)
        assert (drafted == 0) == (drafts == 0)
    assert all(r == results[0] for r in results)
    acc = llmx.Accelerator(s)
    acc.upload_model(model)
    ex = llmx.Executor(acc, model)
    text = list(PROMPTS[1])
    hidden = ex.run_prompt_block(text, 0)[-1]
    for _ in range(14):
        text.append(model.lm_head_argmax(hidden))
        hidden = ex.run_token(text[-1], len(text) - 1)[0]
    assert text[len(PROMPTS[1]):] == results[0][1]


def test_drawn_with_a_temperature(llmx):
    """The same seed gives the same tokens; a request's tokens do not depend on the others' adapters."""
    pytest.importorskip("torch")
    import speculative as spec
    model = llmx.Model(llmx.shape("small")).init_reference_random(7)
    sv = server(spec, model, 3)
    a, _ = sv.generate(PROMPTS, [0, -1, 1], 20, temperature=1.0, seed=5)
    b, _ = sv.generate(PROMPTS, [0, -1, 1], 20, temperature=1.0, seed=5)
    c, _ = sv.generate(PROMPTS, [-1, -1, -1], 20, temperature=0.0)
    d, _ = sv.generate(PROMPTS, [0, -1, 1], 20, temperature=0.0)
    sv.close()
    assert a == b
    assert c[1] == d[1]


def host_greedy(llmx, model, prompt, count):
    """The host's greedy loop: exact scores, the first maximum."""
    acc = llmx.Accelerator(model.shape)
    acc.upload_model(model)
    ex = llmx.Executor(acc, model)
    text = list(prompt)
    for at in range(0, len(text), llmx.MAX_ROWS):
        hidden = ex.run_prompt_block(text[at:at + llmx.MAX_ROWS], at)[-1]
    for _ in range(count):
        text.append(model.lm_head_argmax(hidden))
        hidden = ex.run_token(text[-1], len(text) - 1)[0]
    acc.close()
    return text[len(prompt):]


@pytest.mark.parametrize("untied", [True, False])
def test_scores_come_from_the_lm_head(llmx, untied):
    """Requests without adapters get the host's greedy tokens, with an LM head of its own as
    with a tied one."""
    pytest.importorskip("torch")
    import speculative as spec
    model = llmx.Model(llmx.shape("small")).init_gaussian(11, lm_head=untied)
    sv = spec.Server(model, 3, 1, 8, 2)
    out, _ = sv.generate(PROMPTS, [-1, -1, -1], 8)
    sv.close()
    assert out == [host_greedy(llmx, model, p, 8) for p in PROMPTS]


@pytest.mark.parametrize("untied", [True, False])
def test_temperature_is_that_of_the_logits(llmx, untied):
    """One drawn token at temperature T lies where the cumulative softmax of the model's logits
    over T passes the random number.  The logits are rounded once, to 2^-12 (tied) or
    2^-16: half a step moves a logit over T by at most 2^-13 / T, a cumulative probability by at
    most twice that; the whole-number weights and shares add less than 1e-6 (2e-7 each, and 64
    tokens' roundings of 2^-31 and 2^-40)."""
    pytest.importorskip("torch")
    import speculative as spec
    model = llmx.Model(llmx.shape("small")).init_gaussian(11, lm_head=untied)
    acc = llmx.Accelerator(model.shape)
    acc.upload_model(model)
    ex = llmx.Executor(acc, model)
    unit = 2.0 ** (16 if untied else 12)  # of a logit, in the products' last places over 2^4
    sv = spec.Server(model, 1, 1, 8, 0)
    drawn = set()
    for prompt in ([3], [9, 4], [5, 5, 7], [1, 2, 3, 1]):
        hidden = ex.run_prompt_block(prompt, 0)[-1].astype(np.int64)
        z = (model.lm_head().astype(np.int64) @ hidden) / (16 * unit)
        for t in (0.5, 1.0, 4.0):
            p = np.exp((z - z.max()) / t)
            p /= p.sum()
            mass = np.concatenate([[0], np.cumsum(p)])
            for seed in range(8):
                u = int(np.random.default_rng(seed).integers(0, 2**32, 1, dtype=np.uint64)[0]) / 2**32
                (out,), _ = sv.generate([prompt], [-1], 1, temperature=t, seed=seed)
                off = 2 * 2.0**-13 / t + 1e-6
                assert mass[out[0]] - off <= u <= mass[out[0] + 1] + off, (prompt, t, seed)
                drawn.add(out[0])
    assert len(drawn) > 4
    sv.close()
    acc.close()


def test_each_request_gets_its_own_adapter(llmx):
    """Adapters that favour tokens of their own: each request's text is that of its slot's adapter,
    with drafts (some accepted) as without, whichever request has which slot."""
    pytest.importorskip("torch")
    import speculative as spec
    model = llmx.Model(llmx.shape("small")).init_gaussian(11, lm_head=True)
    s = model.shape

    def adapter(token):
        """Rank 1: t is some tens, of either sign, and lifts `token` or the next one far above the others."""
        up = np.zeros((s.vocab, 1), np.int64)
        up[token], up[token + 1] = 32767, -32767
        return np.random.default_rng(token).integers(-2000, 2000, (1, s.hidden)), up

    def expect(prompt, token, count):
        """Greedy tokens of a request whose adapter is `token`'s (None: no adapter)."""
        acc = llmx.Accelerator(s)
        acc.upload_model(model)
        ex = llmx.Executor(acc, model)
        text = list(prompt)
        hidden = ex.run_prompt_block(text, 0)[-1].astype(np.int64)
        for _ in range(count):
            y = model.lm_head().astype(np.int64) @ hidden
            if token is not None:
                down, up = adapter(token)
                y = y + up @ np.clip((down @ hidden * 32767 + (1 << 23)) >> 24, -32768, 32767)
            text.append(int(np.argmax(np.clip((y + 8) >> 4, -2**31, 2**31 - 1))))
            hidden = ex.run_token(text[-1], len(text) - 1)[0].astype(np.int64)
        acc.close()
        return text[len(prompt):]

    tokens = [7, 23]
    plain = [expect(p, None, 14) for p in PROMPTS]
    for drafts in (0, 4):
        sv = spec.Server(model, 3, 2, 1, drafts)
        for slot, token in enumerate(tokens):
            sv.set_adapter(slot, 32767, *adapter(token))
        for slots in ([0, -1, 1], [1, 0, -1], [-1, 1, 0]):
            want = [expect(p, None if a < 0 else tokens[a], 14) for p, a in zip(PROMPTS, slots)]
            assert all((w != q) == (a >= 0) for w, q, a in zip(want, plain, slots))  # an adapter changes the text
            out, (drafted, taken) = sv.generate(PROMPTS, slots, 14)
            assert out == want
            assert (taken > 0) == (drafts > 0)
        sv.close()
