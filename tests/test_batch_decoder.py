"""Decoding of a batch of unequal requests behind a shared prompt, against the recomputation of each request's whole window."""
import pytest
import torch

from oa_b200.core import fn_matrix as F
from oa_b200.core.matrix import OaMatrix
from oa_b200.ml import autograd as AG
from oa_b200.models import OaGptConfig, OaGptModel
from oa_b200.ops import kernels as K
from oa_b200.serve import OaBatchDecoder, OaSampling

CONFIGS = {"rope_swiglu": OaGptConfig(64, 32, 2, 4, 64, 96, "rms", "swiglu", 10000.0, False, 1e-5, 0.3),
           "learned_gelu": OaGptConfig(64, 32, 2, 4, 64, 96, "layer", "gelu", 0.0, True, 1e-5, 0.3)}
PROMPT = [5, 9, 61, 3, 3, 17, 40, 2, 8, 33, 21, 7, 7, 50, 12, 1, 30]              # a page of 16 and one more
TEXTS = [[1], [4, 60, 22], list(range(20)), [63] * 16]


def _full_window(model, ids, n):
    """(greedy continuation, logits of the first new token) of one text."""
    out, first = list(ids), None
    with AG.OaGradNo():
        for _ in range(n):
            t = torch.tensor([out], dtype=torch.int32, device=model.Embed.Weight.Tensor().device)
            logits = model.Forward(OaMatrix(t)).Tensor()[-1].float()
            first = logits if first is None else first
            out.append(int(logits.argmax()))
    return out[len(ids):], first


@pytest.mark.parametrize("prompt", [[], PROMPT])
@pytest.mark.parametrize("kind", list(CONFIGS))
def test_generation_matches_each_requests_own_window(kind, prompt):
    F.SetRngSeed(5)
    model = OaGptModel(CONFIGS[kind])
    dec = OaBatchDecoder(model, 5, 40, max_prompt=20, page_size=16)
    dec.SetPrompt(prompt)
    texts = TEXTS if prompt else [[1, 13], *TEXTS[1:]]            # the recomputation wants windows of two tokens or more
    got = dec.Generate(texts, 9)
    for text, new in zip(texts, got):
        assert new == _full_window(model, prompt + text, 9)[0]
    used = -(-len(prompt) // 16)
    assert dec.Cache.Used == used == int(dec.Cache.Taken) and dec.Cache.Held == [0] * 5 and (dec.Cache.Tables == -1).all()
    assert dec.Generate(texts[::-1], 9) == got[::-1]              # in pages that have been used


def test_a_request_ends_at_its_stop_and_others_go_on():
    F.SetRngSeed(5)
    model = OaGptModel(CONFIGS["rope_swiglu"])
    dec = OaBatchDecoder(model, 4, 40, page_size=16)
    free = dec.Generate(TEXTS, 12)
    stop = free[1][3]
    want = [t[:t.index(stop) + 1] if stop in t else t for t in free]
    assert dec.Generate(TEXTS, 12, stop=stop) == want and len(want[1]) <= 4


def test_requests_come_and_go_while_others_stay():
    F.SetRngSeed(5)
    model = OaGptModel(CONFIGS["rope_swiglu"])
    dec = OaBatchDecoder(model, 3, 40, max_prompt=20, pages=7, page_size=16)
    dec.SetPrompt(PROMPT)
    first = dec.Feed([TEXTS[2], [], TEXTS[0]])
    assert int(first[1]) == -1
    long = [int(first[0])]
    dec.Release([2])
    for i in range(3):                                            # request 0 goes on; 1 begins with three tokens at a time, 2 at the second step
        out = dec.Feed([[long[-1]], TEXTS[3][i * 3:i * 3 + 3], TEXTS[1] if i == 1 else []])
        long.append(int(out[0]))
        if i == 1:
            assert int(out[2]) == _full_window(model, PROMPT + TEXTS[1], 1)[0][0]
    assert long == _full_window(model, PROMPT + TEXTS[2], 4)[0]
    assert int(out[1]) == _full_window(model, PROMPT + TEXTS[3][:9], 1)[0][0]
    assert int(out[2]) == -1
    with pytest.raises(ValueError, match="under way"):
        dec.SetPrompt([])
    dec.Release([0, 1, 2])
    dec.SetPrompt(TEXTS[1])
    assert dec.Generate([TEXTS[0]], 4)[0] == _full_window(model, TEXTS[1] + TEXTS[0], 4)[0]


def test_drawn_tokens_follow_the_seed_and_the_settings():
    F.SetRngSeed(5)
    model = OaGptModel(CONFIGS["rope_swiglu"])
    how = [OaSampling(1.0), OaSampling(0.7, TopK=5), OaSampling(), OaSampling(1.5, TopP=0.8, MinP=0.01)]

    def run(seed):
        dec = OaBatchDecoder(model, 4, 40, page_size=16, seed=seed)
        dec.SetSampling(how)
        return dec.Generate(TEXTS, 10)

    a = run(1)
    assert a == run(1) and a != run(2)
    assert a[2] == _full_window(model, TEXTS[2], 10)[0]
    dec = OaBatchDecoder(model, 4, 40, page_size=16, seed=1)
    dec.SetSampling(how)
    out = dec.Feed(TEXTS)
    assert int(out[1]) in dec.Logits[1].topk(5).indices.tolist()
    assert dec.LogProbs.shape == (4,) and float(dec.LogProbs[2]) == 0.0 and (dec.LogProbs <= 0).all()


def test_refusals():
    model = OaGptModel(CONFIGS["learned_gelu"])
    with pytest.raises(ValueError, match="positions"):
        OaBatchDecoder(model, 2, 80, max_prompt=20)
    with pytest.raises(ValueError, match="positive"):
        OaBatchDecoder(model, 0, 8)
    dec = OaBatchDecoder(model, 2, 24, max_prompt=16, pages=3, page_size=16)
    with pytest.raises(ValueError, match="16 is the most"):
        dec.SetPrompt(PROMPT)
    with pytest.raises(ValueError, match="2 settings|2 requests"):
        dec.SetSampling([OaSampling()])
    for new in ([[1]], [[], []], [[1], [2], [3]]):
        with pytest.raises(ValueError, match="new tokens"):
            dec.Feed(new)
    with pytest.raises(ValueError, match="24 is the most"):
        dec.Feed([[1] * 25, []])
    with pytest.raises(ValueError, match="no room"):
        dec.Feed([[1] * 17, [1] * 17])
    dec.Feed([[1] * 17, [2]])                                     # all three pages
    with pytest.raises(ValueError, match="one token for each"):
        dec.Step(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="under way"):
        dec.Generate([[1]], 2)
    dec.Release([0, 1])
    with pytest.raises(ValueError, match="none of them empty"):
        dec.Generate([[1], []], 2)
    with pytest.raises(ValueError, match="no room"):
        dec.Generate([[1] * 10, [1] * 10], 8)
    assert dec.Cache.Used == 0 and dec.Cache.Held == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("heads", [2, 1])
def test_generation_gpu_bf16(heads, use_graph):
    F.SetRngSeed(5)
    prev = F.GetWeightDtype()
    F.SetWeightDtype(torch.bfloat16)
    try:
        model = OaGptModel(OaGptConfig(256, 128, 2, heads, 256, 128, "rms", "swiglu", 10000.0, False, 1e-5, 0.2))
        prompt = [(7 * i) % 256 for i in range(37)]
        texts = [[1], [200, 3, 4], [(11 * i) % 256 for i in range(40)]]
        dec = OaBatchDecoder(model, 4, 64, max_prompt=48, page_size=16, use_graph=use_graph)
        dec.SetPrompt(prompt)
        so_far = [prompt + t for t in texts]
        out = dec.Feed([*texts, []])
        for step in range(5):
            assert int(out[3]) == -1
            for b in range(3):
                first = _full_window(model, so_far[b], 1)[1]
                assert (dec.Logits[b].float() - first).abs().max().item() < 5e-2 * max(1.0, first.abs().max().item())
                assert int(out[b]) == int(dec.Logits[b].float().argmax())
                so_far[b].append(int(out[b]))
            out = dec.Step(out, [True, True, True, False])
        assert (dec._graph is not None) == use_graph
        dec.Release([0, 1, 2])
        assert int(dec.Cache.Taken) == dec.Cache.Used == 3
    finally:
        F.SetWeightDtype(prev)
    K.check_status()


@pytest.mark.gpu
def test_a_graphed_step_draws_what_an_eager_one_does():
    F.SetRngSeed(5)
    prev = F.GetWeightDtype()
    F.SetWeightDtype(torch.bfloat16)
    try:
        model = OaGptModel(OaGptConfig(256, 128, 2, 2, 256, 128, "rms", "swiglu", 10000.0, False, 1e-5, 0.2))
        got = []
        for use_graph in (False, True):
            dec = OaBatchDecoder(model, 3, 64, max_prompt=32, page_size=32, seed=3, use_graph=use_graph)
            dec.SetSampling([OaSampling(1.0, TopK=40), OaSampling(), OaSampling(0.8, TopP=0.9)])
            dec.SetPrompt(list(range(30)))
            got.append(dec.Generate([[1, 2], [3], [4, 5, 6, 7]], 12))
            got.append(dec.Generate([[9], [8, 7]], 12, stop=got[-1][0][-1]))
        assert got[:2] == got[2:]
    finally:
        F.SetWeightDtype(prev)
    K.check_status()


@pytest.mark.gpu
def test_generation_gpu_f32_learned_positions():
    F.SetRngSeed(5)
    model = OaGptModel(OaGptConfig(256, 128, 2, 4, 256, 128, "layer", "gelu", 0.0, True, 1e-5, 0.2))
    dec = OaBatchDecoder(model, 3, 64, max_prompt=48, page_size=16)
    dec.SetPrompt(PROMPT)
    assert dec.Generate(TEXTS[:3], 9) == [_full_window(model, PROMPT + t, 9)[0] for t in TEXTS[:3]]
    K.check_status()
