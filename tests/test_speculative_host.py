"""The serving loop of speculative.py without a GPU: what it makes of failures, on stand-ins for
the two operators and the contexts."""
import types

import numpy as np
import pytest

import speculative as spec


class Loop:
    """A Server on the host: a step's outcome is what `outcome` writes into tokens and accepted."""

    def __init__(self, monkeypatch, outcome, head_error=None, context_error=None, requests=2, drafts=2, steps=6):
        torch = pytest.importorskip("torch")
        self.calls = 0
        sv = self.server = object.__new__(spec.Server)
        sv.torch, sv.dev, sv.drafts, sv.logit_step = torch, torch.device("cpu"), drafts, 1.0
        sv.s = types.SimpleNamespace(vocab=64, hidden=64, layers=1)
        sv.model = types.SimpleNamespace(embed=lambda tokens: np.zeros((len(tokens), 64), np.int16))

        def fails(error):
            def call(*a):
                if error and self.calls >= error:
                    raise spec.llmx.LlmxError(spec.llmx.ERR_TIMEOUT, "stand-in")
            return call

        sv.contexts = [types.SimpleNamespace(stack=lambda *a, **k: None, synchronize=fails(context_error)) for _ in range(requests)]
        sv.head = types.SimpleNamespace(project=lambda *a, **k: None, error=fails(head_error))
        sv.x, sv.logits, sv.work = (torch.zeros(8, dtype=torch.int32) for _ in range(3))
        sv.tokens = torch.zeros((requests, drafts + 1), dtype=torch.int32)
        sv.accepted = torch.zeros(requests, dtype=torch.int32)
        sv.stream, sv._block = lambda: None, lambda *a: None

        def verify(*a, **k):
            self.calls += 1
            assert self.calls <= steps, "the loop makes no progress"
            outcome(self.calls, sv.tokens, sv.accepted)

        monkeypatch.setattr(spec.llmx, "verify_drafts", verify)

    def run(self, prompts=((1, 2), (3,)), max_new=3, slots=(-1, -1)):
        return self.server.generate([list(p) for p in prompts], list(slots), max_new)


def fine(step, tokens, accepted):
    tokens[:, 0] = 10 + step


def test_tokens_are_appended(monkeypatch):
    out, (drafted, taken) = Loop(monkeypatch, fine).run()
    assert out == [[11, 12, 13], [11, 12, 13]] and taken == 0


def test_verification_that_gave_up_ends_the_loop(monkeypatch):
    def outcome(step, tokens, accepted):
        fine(step, tokens, accepted)
        accepted[1] = -1 if step == 2 else 0

    loop = Loop(monkeypatch, outcome)
    with pytest.raises(spec.llmx.LlmxError) as e:
        loop.run()
    assert e.value.code == spec.llmx.ERR_TIMEOUT and loop.calls == 2


def test_row_without_a_token_ends_the_loop(monkeypatch):
    def outcome(step, tokens, accepted):
        tokens[:, 0] = -1

    loop = Loop(monkeypatch, outcome)
    with pytest.raises(spec.llmx.LlmxError) as e:
        loop.run()
    assert e.value.code == spec.llmx.ERR_RANGE and loop.calls == 1


@pytest.mark.parametrize("where", ["head_error", "context_error"])
def test_logits_of_a_failed_step_are_not_used(monkeypatch, where):
    loop = Loop(monkeypatch, fine, **{where: 2})
    with pytest.raises(spec.llmx.LlmxError) as e:
        loop.run()
    assert e.value.code == spec.llmx.ERR_TIMEOUT and loop.calls == 2


def test_failed_step_leaves_the_texts():
    texts = [[1], [2, 3]]
    tokens = np.array([[7, 8], [9, -1]], np.int32)
    with pytest.raises(spec.llmx.LlmxError):
        spec.append_tokens(texts, [9, 9], tokens, np.array([0, -1], np.int32))
    with pytest.raises(spec.llmx.LlmxError):
        spec.append_tokens(texts, [9, 9], tokens, np.array([0, 1], np.int32))
    assert texts == [[1], [2, 3]]
    assert spec.append_tokens(texts, [9, 2], tokens, np.array([1, -1], np.int32)) == 1  # request 1 is done
    assert texts == [[1, 7, 8], [2, 3]]


def test_refusals(monkeypatch):
    for kw in (dict(prompts=((), (3,))), dict(slots=(0,)), dict(prompts=((1,),))):
        with pytest.raises(ValueError):
            Loop(monkeypatch, fine).run(**kw)


def test_adapters_of_other_sizes_are_refused(monkeypatch):
    """The device kernels read [rank][hidden] and [vocab][rank] of what they are given."""
    sv = Loop(monkeypatch, fine).server
    put = []
    sv.head.set = lambda *a, **k: put.append(a)
    good = dict(slot=0, scale=4096, down=np.zeros((4, 64), np.int64), up=np.zeros((64, 4), np.int64))
    for bad in (dict(up=np.zeros((64, 3), np.int64)), dict(up=np.zeros((63, 4), np.int64)), dict(down=np.zeros((4, 56), np.int64)),
                dict(down=np.zeros((64,), np.int64)), dict(down=np.full((4, 64), 32768)), dict(up=np.full((64, 4), -32769)),
                dict(up=np.zeros((64, 4))), dict(scale=32768), dict(scale=0.5)):
        with pytest.raises(ValueError):
            sv.set_adapter(**{**good, **bad})
    assert not put
