"""OaBatchDecoder when a step fails before its end: nothing has moved, on the device or the host, and the same step again is the step."""
import pytest
import torch

from oa_b200.core import fn_matrix as F
from oa_b200.models import OaGptConfig, OaGptModel
from oa_b200.ops import paged, sampling
from oa_b200.serve import OaBatchDecoder, OaSampling
from oa_b200.serve import batch_decoder as BD

CONFIG = OaGptConfig(64, 32, 2, 4, 64, 96, "rms", "swiglu", 10000.0, False, 1e-5, 0.3)
PROMPT = [5, 9, 61, 3, 3, 17, 40, 2, 8, 33, 21, 7, 7, 50, 12, 1, 30]
HOW = [OaSampling(1.3), OaSampling(0.9, TopK=9)]


def _fails(*_, **__):
    raise RuntimeError("no memory")


def _state(dec):
    c = dec.Cache
    return (c.Lens.tolist(), c.PromptLens.tolist(), c.Taken.tolist(), list(c.Held), c.PromptLen, c.Used, dec._random.get_state().tolist(),
            None if dec.Logits is None else dec.Logits.tolist(), None if dec.LogProbs is None else dec.LogProbs.tolist())


PLACES = [(BD, "block_tail"), (paged, "append"), (paged, "attention"), (sampling, "sample")]


@pytest.fixture
def model():
    F.SetRngSeed(5)
    return OaGptModel(CONFIG)


def _decoder(model):
    dec = OaBatchDecoder(model, 2, 40, max_prompt=20, page_size=16, seed=3)
    dec.SetSampling(HOW)
    return dec


@pytest.mark.parametrize("where", range(len(PLACES)))
@pytest.mark.parametrize("prompt", [[], PROMPT])
def test_the_same_step_again_is_the_step(model, monkeypatch, where, prompt):
    steps = [lambda d: d.Feed([[4, 60, 22], [7]]), lambda d: d.Step(torch.tensor([11, 12], dtype=torch.int32)),
             lambda d: d.Step(torch.tensor([3, 0], dtype=torch.int32), [True, False]), lambda d: d.Feed([[], [9] * 17])]
    plain, other = _decoder(model), _decoder(model)
    plain.SetPrompt(prompt)
    other.SetPrompt(prompt)
    for step in steps:
        before = _state(other)
        for _ in range(2):
            with monkeypatch.context() as m:
                m.setattr(*PLACES[where], _fails)
                with pytest.raises(RuntimeError, match="no memory"):
                    step(other)
            assert _state(other) == before
        assert step(other).tolist() == step(plain).tolist()
        assert _state(other) == _state(plain)
    for dec in (plain, other):
        dec.Release([0, 1])
    assert _state(other) == _state(plain) and other.Cache.Used == -(-len(prompt) // 16)


@pytest.mark.parametrize("where", range(3))
def test_a_prompt_that_fails_leaves_none(model, monkeypatch, where):
    """The prompt before is gone (its pages were given back for the new one's), and nothing is held."""
    dec = _decoder(model)
    dec.SetPrompt(PROMPT)
    with monkeypatch.context() as m:
        m.setattr(*PLACES[where], _fails)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.SetPrompt([1, 2, 3])
    c = dec.Cache
    assert (c.PromptLen, c.Used, c.PromptLens.tolist(), c.Taken.tolist()) == (0, 0, [0], [0])
    plain = _decoder(model)
    plain.SetPrompt(PROMPT[:5])
    dec.SetPrompt(PROMPT[:5])
    assert dec.Feed([[4, 60, 22], [7]]).tolist() == plain.Feed([[4, 60, 22], [7]]).tolist()
    assert c.Used == int(c.Taken) == 3


def test_a_release_that_fails_gives_nothing_back(model, monkeypatch):
    dec = _decoder(model)
    dec.SetPrompt(PROMPT)
    dec.Feed([[4, 60, 22], [7]])
    before = _state(dec)
    with monkeypatch.context() as m:
        m.setattr(paged, "release", _fails)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.Release([0, 1])
        assert _state(dec) == before
    dec.Release([0, 1])
    with monkeypatch.context() as m:
        m.setattr(paged, "release", _fails)
        before = _state(dec)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.SetPrompt([1, 2, 3])
        assert _state(dec) == before
    assert dec.Cache.Used == int(dec.Cache.Taken) == 2


def test_a_generation_that_fails_gives_its_pages_back(model, monkeypatch):
    dec, plain = _decoder(model), _decoder(model)
    calls = [0]
    sample = sampling.sample

    def third_fails(*a):
        calls[0] += 1
        return _fails() if calls[0] == 3 else sample(*a)

    with monkeypatch.context() as m:
        m.setattr(sampling, "sample", third_fails)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.Generate([[1, 2], [3] * 20], 8)
    assert dec.Cache.Used == int(dec.Cache.Taken) == 0 and dec.Cache.Held == [0, 0] and dec.Cache.Lens.tolist() == [0, 0]
    dec._random.manual_seed(3)
    assert dec.Generate([[1, 2], [3] * 20], 8) == plain.Generate([[1, 2], [3] * 20], 8)


@pytest.mark.gpu
@pytest.mark.parametrize("fails_at", [1, 2, 3])                   # an eager step, the recording, and the step behind a graph that is there
def test_steps_that_fail_around_the_recording(monkeypatch, fails_at):
    F.SetRngSeed(5)
    prev = F.GetWeightDtype()
    F.SetWeightDtype(torch.bfloat16)
    try:
        model = OaGptModel(OaGptConfig(256, 128, 2, 2, 256, 128, "rms", "swiglu", 10000.0, False, 1e-5, 0.2))
        plain, other = (OaBatchDecoder(model, 2, 64, max_prompt=32, page_size=16, seed=3) for _ in range(2))
        outs = []
        for dec in (plain, other):
            dec.SetSampling(HOW)
            dec.SetPrompt(PROMPT)
            outs.append(dec.Feed([[4, 60, 22], [7]]))
        for i in range(1, 6):
            if i == fails_at and i < 3:
                before = _state(other)
                with monkeypatch.context() as m:
                    m.setattr(sampling, "sample", _fails)
                    with pytest.raises(RuntimeError, match="no memory"):
                        other.Step(outs[1])
                assert _state(other) == before
            elif i == fails_at:
                before = _state(other)
                with pytest.raises(ValueError, match="one token for each"):
                    other.Step(outs[1][:1])
                with pytest.raises(ValueError, match="64 is the most"):
                    other.Feed([[1] * 80, []])
                assert _state(other) == before
            outs = [dec.Step(out.clone()) for dec, out in zip((plain, other), outs)]
            assert torch.equal(*outs) and _state(other) == _state(plain)
        assert plain._graph is not None and other._graph is not None
    finally:
        F.SetWeightDtype(prev)
