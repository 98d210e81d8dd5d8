"""A model on packed sequences: rotary positions, attention, log-probabilities and their gradients together, against the same model on one sequence at a
time, and a training step and scoring of prompts as a program makes them."""
import pytest
import torch

from oa_b200.core import fn_matrix as F
from oa_b200.core.matrix import OaMatrix
from oa_b200.ml import autograd as AG
from oa_b200.ml import fn_loss as L
from oa_b200.ml.optim import OaAdamW
from oa_b200.models import OaGptConfig, OaGptModel
from oa_b200.ops import logprob, packed, paged

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LENGTHS = [5, 1, 70, 0, 33, 129]


def _batch(vocab, device, pad=2):
    g = torch.Generator().manual_seed(1)
    tokens = sum(LENGTHS) + pad
    ids = torch.randint(0, vocab, (tokens,), generator=g, dtype=torch.int32)
    starts = torch.tensor([0] + LENGTHS).cumsum(0).to(torch.int32)
    targets = ids.roll(-1).clone()
    targets[starts[1:].long() - 1] = -100                     # nothing follows a sequence's last token
    targets[sum(LENGTHS) - 1:] = -100
    weight = torch.randn(2, tokens, generator=g)
    weight[:, sum(LENGTHS):] = 0
    return ids.to(device), starts.to(device), targets.to(device), weight.to(device)


def _model(rope, device, heads=2, d=64, dtype=torch.float32, **kw):
    prev = F.GetWeightDtype()
    F.SetWeightDtype(dtype)
    try:
        F.SetRngSeed(3)
        return OaGptModel(OaGptConfig(104, d, 2, heads, 2 * d, 256, "rms" if rope else "layer", "swiglu" if rope else "gelu", 10000.0 if rope else 0.0, not rope, 1e-5, 0.15, **kw))
    finally:
        F.SetWeightDtype(prev)


def _grads(model):
    return [p.Data.GradTensor().float().clone() for p in model.AllParameterPtrs() if p.Data.GradTensor() is not None]


def _weighted(out, weight):
    return F.Sum(F.Mul(out, OaMatrix(weight)))


def _run(model, build):
    for p in model.AllParameterPtrs():
        p.Data.ZeroGrad()
    with AG.OaGradientTape() as tape:
        out, loss = build()
        tape.Backward(loss)
    return out, _grads(model)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rope", [False, True])
def test_packed_is_one_sequence_at_a_time(device, rope):
    """fp32: each of about 14 products one after the other adds at most 256 terms, 256 2^-24 of the sum of their magnitudes: 14 * 1.5e-5 = 2^-12 of the largest
    values, and as much on the way back."""
    model = _model(rope, device)
    ids, starts, targets, weight = _batch(104, device)
    seqs = F.PackedSequences(OaMatrix(starts), ids.numel())
    got, grads = _run(model, lambda: (lambda o: (o, _weighted(o, weight)))(model.TokenLogProbs(OaMatrix(ids), OaMatrix(targets), seqs)))
    assert got.Tensor().shape == (2, ids.numel()) and bool((got.Tensor()[0][targets == -100] == 0).all())

    def one_by_one():
        outs, loss = [], None
        for lo, n in zip(starts.tolist(), LENGTHS):
            if n:
                logits = model.Forward(OaMatrix(ids[lo:lo + n].repeat(2, 1)))      # twice, the second time without weight
                o = L.TokenLogProbs(logits, OaMatrix(targets[lo:lo + n].repeat(2)))
                part = _weighted(o, torch.cat([weight[:, lo:lo + n], torch.zeros_like(weight[:, lo:lo + n])], 1))
                outs.append(o.Tensor()[:, :n])
                loss = part if loss is None else F.Add(loss, part)
        return torch.cat(outs, 1), loss

    want, want_grads = _run(model, one_by_one)
    n = sum(LENGTHS)
    assert float((got.Tensor()[:, :n] - want).abs().max()) <= 2 ** -12 * float(want.abs().max())
    assert len(grads) == len(want_grads)
    # A bias of the keys adds one number to all scores of a query: its gradient is 0, and what stands there is what sums of the key weights' terms (rows of unit size
    # apart) leave when they cancel
    scale = {id(b.Attention.KProj.Bias): b.Attention.KProj.Weight.Data.GradTensor().abs().max() for b in model.Blocks if b.Attention.KProj.Bias is not None}
    for p, a, b in zip(model.AllParameterPtrs(), grads, want_grads):
        assert float((a - b).abs().max()) <= 2 ** -11 * float(scale.get(id(p), b.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seq", [40, 200])
def test_packed_bf16_gradients(hd, seq):
    """bf16, four sequences of one length, packed and as the batch that the model takes otherwise: the same products with the same roundings, but for the attention
    kernels, so that against the fp32 model of the same weights the gradients of both are equally far off.  How far roundings of 2^-8 get amplified is the
    model's affair; over thousands of elements the norms of two such errors are alike, and twice the other's is allowed."""
    model = _model(True, "cuda", heads=2, d=2 * hd, dtype=torch.bfloat16)
    ref = _model(True, "cuda", heads=2, d=2 * hd)
    for a, b in zip(model.AllParameterPtrs(), ref.AllParameterPtrs()):
        b.Data.Tensor().copy_(a.Data.Tensor().float())
    g = torch.Generator().manual_seed(2)
    ids, targets = (torch.randint(0, 104, (4 * seq,), generator=g, dtype=torch.int32).cuda() for _ in range(2))
    weight = torch.randn(2, 4 * seq, generator=g).cuda()
    seqs = F.PackedSequences(OaMatrix(torch.arange(0, 5 * seq, seq, dtype=torch.int32, device="cuda")), 4 * seq)
    dense = lambda m: lambda: (lambda o: (o, _weighted(o, weight)))(L.TokenLogProbs(m.Forward(OaMatrix(ids.reshape(4, seq))), OaMatrix(targets)))      # noqa: E731
    want = _run(ref, dense(ref))[1]
    usual = _run(model, dense(model))[1]
    got = _run(model, lambda: (lambda o: (o, _weighted(o, weight)))(model.TokenLogProbs(OaMatrix(ids), OaMatrix(targets), seqs)))[1]
    for a, b, w in zip(got, usual, want):
        assert float((a - w).norm()) <= 2 * float((b - w).norm())


@pytest.mark.parametrize("device", DEVICES)
def test_a_policy_step(device):
    """log-probabilities, entropy, gradients and an optimizer step run, and change the weights; rows behind the last sequence take no part."""
    model = _model(True, device)
    ids, starts, targets, weight = _batch(104, device)
    opt = OaAdamW(model.AllParameterPtrs(), 1e-3)
    seqs = F.PackedSequences(OaMatrix(starts), ids.numel())
    before = [p.Data.Tensor().clone() for p in model.AllParameterPtrs()]
    opt.ZeroGrad()
    with AG.OaGradientTape() as tape:
        tape.Backward(_weighted(model.TokenLogProbs(OaMatrix(ids), OaMatrix(targets), seqs), weight))
    grads = _grads(model)
    opt.Step()
    assert all(bool(g.isfinite().all()) for g in grads) and any(bool((a != p.Data.Tensor()).any()) for a, p in zip(before, model.AllParameterPtrs()))


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_attention_logprobs_together(device):
    """The raw operators as a program for images and text uses them: several axes, grouped heads, alternatives of the last tokens; and the same tokens decoded
    one by one over pages, turned by `rotary`, appended without a turn."""
    hq, hk, hd, vocab = 4, 2, 64, 300
    g = torch.Generator().manual_seed(5)
    n = 40
    qkv = torch.randn(n, (hq + 2 * hk) * hd, generator=g).to(device)
    pos = torch.stack([torch.arange(n), torch.arange(n) // 7, torch.arange(n) % 7]).to(torch.int32).to(device)
    axes = (0,) * 8 + (1,) * 12 + (2,) * 12
    starts = torch.tensor([0, 15, n], dtype=torch.int32, device=device)
    plan = packed.plan(starts, n)
    turned = qkv.clone()
    packed.rotary(turned, pos, axes, hq + hk, hd, 10000.0, out=turned)
    q, k, v = torch.split(turned, [hq * hd, hk * hd, hk * hd], 1)
    o = packed.attention(q, k, v, plan, hd)
    table = torch.arange(8, dtype=torch.int32, device=device).reshape(2, 4)
    k_pages, v_pages = (torch.zeros(8, hk, 16, hd, device=device) for _ in range(2))
    for b, (lo, hi) in enumerate(((0, 15), (15, n))):
        for t in range(lo, hi):
            row = packed.rotary(qkv[t:t + 1], pos[:, t:t + 1].contiguous(), axes, hq + hk, hd, 10000.0)
            slot = table[b, (t - lo) // 16] * 16 + (t - lo) % 16
            qs = paged.append(torch.cat([row, qkv[t:t + 1, (hq + hk) * hd:]], 1), torch.zeros(1, dtype=torch.int32, device=device), slot.reshape(1), k_pages, v_pages, 0.0)
            one = paged.attention(qs, k_pages, v_pages, table[b:b + 1], torch.tensor([t - lo + 1], dtype=torch.int32, device=device),
                                  torch.tensor([0, 1], dtype=torch.int32, device=device), 1)
            assert float((one - o[t:t + 1]).abs().max()) <= 2 ** -17      # sums of 64 and 40 terms of magnitude 1 in 32 bits, twice
    logits = torch.randn(n, vocab, generator=g).to(device)
    ids = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32).to(device)
    r = logprob.token_logprobs(logits, ids, top=3)
    assert torch.equal(r.top_ids[:, 0].long(), logits.argmax(1)) and bool((r.logprobs <= r.top_logprobs[:, 0] + 1e-6).all())


def test_refusals():
    model = _model(False, "cpu")
    ids, starts, targets, _ = _batch(104, "cpu")
    seqs = F.PackedSequences(OaMatrix(starts), ids.numel())
    with pytest.raises(ValueError, match="tokens, but the sequences"):
        model.ForwardPacked(OaMatrix(ids[:-1]), seqs)
    block = model.Blocks[0]
    x = OaMatrix(torch.zeros(ids.numel(), 64))
    block.SetAttentionMode(1)
    with pytest.raises(ValueError, match="packed sequences are causal"):
        block.Forward(x, packed=seqs)
    with pytest.raises(ValueError, match="pair_axes names axes"):
        F.RotaryAxes(x, OaMatrix(seqs.Positions), (1,) * 16, 2, 32)


@pytest.mark.parametrize("device", DEVICES)
def test_default_positions(device):
    seqs = F.PackedSequences(OaMatrix(torch.tensor([2, 5, 5, 9], dtype=torch.int32, device=device)), 12)
    assert seqs.Positions.tolist() == [[0, 0, 0, 1, 2, 0, 1, 2, 3, 0, 0, 0]]
    assert F.PackedSequences(OaMatrix(torch.tensor([0], dtype=torch.int32, device=device)), 0).Positions.shape == (1, 0)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_of_rotary_axes(device):
    x = OaMatrix(torch.randn(6, 128, generator=torch.Generator().manual_seed(0)).to(device)).SetRequiresGrad(True)
    pos = torch.randint(0, 50, (2, 6), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(device)
    w = torch.randn(6, 128, generator=torch.Generator().manual_seed(2)).to(device)
    axes = (0, 1) * 8
    with AG.OaGradientTape() as tape:
        tape.Backward(_weighted(F.RotaryAxes(x, OaMatrix(pos), axes, 2, 64), w))
    assert torch.equal(x.GradTensor(), packed.rotary(w, pos, axes, 2, 64, 10000.0, backward=True))
    # its transpose: <turn(a), w> = <a, turn back(w)>, sums of 768 terms in 32 bits
    a = x.Tensor()
    lhs, rhs = (packed.rotary(a, pos, axes, 2, 64, 10000.0) * w).sum(), (a * x.GradTensor()).sum()
    assert abs(float(lhs - rhs)) <= 768 * 2.0 ** -23 * float((a.abs() * w.abs()).sum())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_of_rotary_axes_over_the_first_columns(device, dtype):
    """Rows wider than the heads that are turned: the other columns are not in the result, and their gradient is 0."""
    g = torch.Generator().manual_seed(0)
    x = OaMatrix(torch.randn(6, 200, generator=g).to(dtype).to(device)).SetRequiresGrad(True)
    pos = torch.randint(0, 50, (1, 6), generator=g, dtype=torch.int32).to(device)
    w = torch.randn(6, 128, generator=g).to(dtype).to(device)
    with AG.OaGradientTape() as tape:
        y = F.RotaryAxes(x, OaMatrix(pos), (0,) * 32, 2, 64)
        assert y.Tensor().shape == (6, 128)
        tape.Backward(_weighted(y, w))
    got = x.GradTensor()
    assert got.shape == (6, 200) and bool((got[:, 128:] == 0).all())
    assert torch.equal(got[:, :128], packed.rotary(w, pos, (0,) * 32, 2, 64, 10000.0, backward=True))


def _aux(model):
    loss = None
    for b in model.Blocks:
        if b.Moe is not None:
            loss = b.Moe.AuxLoss() if loss is None else F.Add(loss, b.Moe.AuxLoss())
    return loss


def _step(model, ids, starts, targets, weight, tokens):
    """(log-probabilities and entropy, balancing loss, gradients, shares of the experts) of the first `tokens` rows' batch."""
    seqs = F.PackedSequences(OaMatrix(starts), tokens)

    def build():
        out = model.TokenLogProbs(OaMatrix(ids[:tokens].clone()), OaMatrix(targets[:tokens].clone()), seqs)
        loss, aux = _weighted(out, weight[:, :tokens].contiguous()), _aux(model)
        return (out, aux), loss if aux is None else F.Add(loss, aux)

    (out, aux), grads = _run(model, build)
    return out.Tensor().clone(), None if aux is None else aux.Tensor().clone(), grads, [b.Moe.LastLoadFraction() for b in model.Blocks if b.Moe is not None]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("experts", [0, 4])
def test_rows_of_no_sequence_take_no_part(device, experts):
    """fp32: whatever tokens stand behind the last sequence, and whether any do, the real rows' results, the gradients, the experts' shares and their balancing losses are
    those of the sequences.  Sums may be added up in another order: the bounds of test_packed_is_one_sequence_at_a_time."""
    model = _model(True, device, **({"NumExperts": experts, "TopK": 2, "ExpertFf": 48, "AuxAlpha": 0.3} if experts else {}))
    for b in model.Blocks:
        if b.Moe is not None:
            b.Moe.SetZLossBeta(0.2)
    ids, starts, targets, weight = _batch(104, device, pad=90)
    n = sum(LENGTHS)
    want, want_aux, want_grads, want_shares = _step(model, ids, starts, targets, weight, n)
    for fill in (0, 1, 103):
        ids[n:] = fill
        got, aux, grads, shares = _step(model, ids, starts, targets, weight, n + 90)
        assert float((got[:, :n] - want).abs().max()) <= 2 ** -12 * float(want.abs().max())
        assert len(grads) == len(want_grads) and all(float((a - b).abs().max()) <= 2 ** -11 * float(b.abs().max()) for a, b in zip(grads, want_grads))
        assert shares == want_shares
        if experts:
            assert abs(float(aux) - float(want_aux)) <= 2 ** -12 * float(want_aux)


@pytest.mark.gpu
def test_rows_of_no_sequence_take_no_part_bf16():
    """Same number of rows, other tokens behind the last sequence: a row's products do not depend on other rows, so the sequences' results are the same bits, and
    the experts' shares the same counts."""
    model = _model(True, "cuda", d=128, dtype=torch.bfloat16, NumExperts=8, TopK=2, ExpertFf=64, AuxAlpha=0.3)
    ids, starts, targets, weight = _batch(104, "cuda", pad=90)
    n = sum(LENGTHS)
    want = None
    for fill in (0, 1, 103):
        ids[n:] = fill
        got, aux, _, shares = _step(model, ids, starts, targets, weight, n + 90)
        want = want or (got, aux, shares)
        assert torch.equal(got[:, :n], want[0][:, :n]) and shares == want[2]
        # 8 products of shares and mean probabilities, which are sums of 238 and 90 zeros
        assert abs(float(aux) - float(want[1])) <= 2.0 ** -16 * float(want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_moves_what_has_a_gradient(device):
    model = _model(True, device)
    ids, starts, targets, weight = _batch(104, device)
    params = model.AllParameterPtrs()
    opt = OaAdamW(params, 1e-3)
    opt.ZeroGrad()
    _, _, grads, _ = _step(model, ids, starts, targets, weight, ids.numel())
    before = [p.Data.Tensor().clone() for p in params]
    opt.Step()
    assert len(grads) == len(params)
    for p, a, g in zip(params, before, grads):
        assert bool(g.abs().max() > 0) and bool((p.Data.Tensor() != a)[g.abs() > 1e-3 * g.abs().max()].all())


def test_load_over_ranks_is_refused():
    """Where the load is counted over expert-parallel ranks, rows of no sequence cannot be left out of what is balanced by it."""
    model = _model(True, "cpu", NumExperts=4, TopK=2, ExpertFf=48, AuxAlpha=0.3)
    ids, starts, _, _ = _batch(104, "cpu")
    model.Blocks[0].Moe.Dispatcher = object()
    with pytest.raises(ValueError, match="over expert-parallel ranks"):
        model.ForwardPacked(OaMatrix(ids), F.PackedSequences(OaMatrix(starts), ids.numel()))


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_sequences(device):
    seqs = F.PackedSequences(OaMatrix(torch.tensor([2, 5, 5, 9], dtype=torch.int32, device=device)), 12)
    assert seqs.Rows().tolist() == [2 <= i < 9 for i in range(12)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,experts", [(64, 0), (128, 0), (64, 8)])
def test_bf16_training_on_any_number_of_rows(hd, experts):
    """238 rows as they come and with two or ten of no sequence behind them: the same products and zeros, so that gradients differ by the order of sums in 32 bits, then a
    rounding to bf16 on either side."""
    model = _model(True, "cuda", heads=2, d=2 * hd, dtype=torch.bfloat16, **({"NumExperts": experts, "TopK": 2, "ExpertFf": 64} if experts else {}))
    ids, starts, targets, weight = _batch(104, "cuda", pad=10)
    n = sum(LENGTHS)
    assert n % 8
    want = None
    for tokens in (n + 2, n, n + 10, n + 1):
        out, _, grads, _ = _step(model, ids, starts, targets, weight, tokens)
        want = want or (out, grads)
        assert torch.equal(out[:, :n], want[0][:, :n]) and len(grads) == len(want[1])
        for a, b in zip(grads, want[1]):
            assert float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_leaves_its_input_alone_while_autograd_records(device):
    """Whether or not the projection asks for a gradient; given to be consumed, or without recording, it is turned in place."""
    qkv = torch.randn(12, 3 * 64, generator=torch.Generator().manual_seed(3)).to(device)
    seqs = F.PackedSequences(OaMatrix(torch.tensor([0, 5, 12], dtype=torch.int32, device=device)), 12)
    for wants in (False, True):
        x = OaMatrix(qkv.clone()).SetRequiresGrad(wants)
        with AG.OaGradientTape():
            first = F.PackedAttention(x, seqs, 1, 1, 64, rope_theta=100.0).Tensor()
            assert torch.equal(x.Tensor(), qkv)
            assert torch.equal(F.PackedAttention(x, seqs, 1, 1, 64, rope_theta=100.0).Tensor(), first)
            given = OaMatrix(qkv.clone()).SetRequiresGrad(wants)
            assert torch.equal(F.PackedAttention(given, seqs, 1, 1, 64, rope_theta=100.0, consume_input=True).Tensor(), first)
            assert not torch.equal(given.Tensor(), qkv)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 64), (8, 2, 64), (8, 2, 128)])
def test_single_tokens_bf16(hq, hk, hd):
    """Tokens decoded one by one over pages, turned by `rotary`, appended without a turn, against the whole sequences: each side rounds its weights before they meet the values
    and its result once, 2^-8 of the magnitudes for either, and sums of at most 200 terms in 32 bits."""
    lengths = [70, 200]
    n, ps = sum(lengths), 16
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(n, (hq + 2 * hk) * hd, generator=g).bfloat16().cuda()
    pos = torch.stack([torch.arange(n), torch.arange(n) // 7]).to(torch.int32).cuda()
    axes = (0, 1) * (hd // 4)
    starts = torch.tensor([0, 70, n], dtype=torch.int32, device="cuda")
    turned = packed.rotary(qkv, pos, axes, hq + hk, hd, 10000.0)
    q, k = torch.split(turned, [hq * hd, hk * hd], 1)
    v = qkv[:, (hq + hk) * hd:]
    o = packed.attention(q, k, v, packed.plan(starts, n), hd)
    table = torch.arange(26, dtype=torch.int32, device="cuda").reshape(2, 13)
    k_pages, v_pages = (torch.zeros(26, hk, ps, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    got = torch.empty_like(o)
    for b, (lo, hi) in enumerate(((0, 70), (70, n))):
        for t in range(lo, hi):
            row = packed.rotary(qkv[t:t + 1], pos[:, t:t + 1].contiguous(), axes, hq + hk, hd, 10000.0)
            assert torch.equal(row, turned[t:t + 1])
            slot = table[b, (t - lo) // ps] * ps + (t - lo) % ps
            qs = paged.append(torch.cat([row, v[t:t + 1]], 1), torch.zeros(1, dtype=torch.int32, device="cuda"), slot.reshape(1), k_pages, v_pages, 0.0)
            got[t] = paged.attention(qs, k_pages, v_pages, table[b:b + 1], torch.tensor([t - lo + 1], dtype=torch.int32, device="cuda"), one, 1)[0]
    for lo, hi in ((0, 70), (70, n)):
        m = hi - lo
        qd = q[lo:hi].double().reshape(m, hq, hd)
        kd, vd = (x[lo:hi].double().reshape(m, hk, hd).repeat_interleave(hq // hk, 1) for x in (k, v))
        p = torch.softmax((torch.einsum("ihd,jhd->hij", qd, kd) * hd ** -0.5).masked_fill(torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1), float("-inf")), -1)
        y, mag = (torch.einsum("hij,jhd->ihd", p, x).reshape(m, hq * hd) for x in (vd, vd.abs()))
        bound = 2.0 ** -8 * y.abs() + (2.0 ** -8 + 2.0 ** -13) * mag
        for side in (o, got):
            assert bool(((side[lo:hi].double() - y).abs() <= bound).all())


@pytest.mark.gpu
def test_bf16_training_on_any_number_of_rows_with_biases():
    """As above, for the model with layer norms, GELU, biases and learned positions.  A gradient that sums of many terms leave when they cancel (the key bias's is 0) is as near as
    the sums: 2^-8 of the largest term's products, taken from the weight that the bias belongs to."""
    model = _model(False, "cuda", heads=2, d=128, dtype=torch.bfloat16)
    ids, starts, targets, weight = _batch(104, "cuda", pad=10)
    n = sum(LENGTHS)
    scale = {}
    want = None
    for tokens in (n + 2, n, n + 9):
        out, _, grads, _ = _step(model, ids, starts, targets, weight, tokens)
        if want is None:
            want = (out, grads)
            scale = {id(b.Attention.KProj.Bias): b.Attention.KProj.Weight.Data.GradTensor().float().abs().max() for b in model.Blocks if b.Attention.KProj.Bias is not None}
        assert torch.equal(out[:, :n], want[0][:, :n]) and len(grads) == len(want[1])
        for p, a, b in zip(model.AllParameterPtrs(), grads, want[1]):
            assert float((a - b).abs().max()) <= 2.0 ** -7 * float(scale.get(id(p), b.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [0, 8])
def test_scoring_in_a_graph(experts):
    """The plan, positions, rows and all layers recorded once and replayed on other sequences: the bits of calls made one by one, the experts' balancing loss too."""
    model = _model(True, "cuda", d=128, dtype=torch.bfloat16, **({"NumExperts": experts, "TopK": 2, "ExpertFf": 64, "AuxAlpha": 0.3} if experts else {}))
    ids, starts, targets, _ = _batch(104, "cuda", pad=90)
    n = ids.numel()

    def score():
        out = model.TokenLogProbs(OaMatrix(ids), OaMatrix(targets), F.PackedSequences(OaMatrix(starts), n)).Tensor()
        return out, _aux(model).Tensor() if experts else None

    sets = [starts.clone(), torch.tensor([3, 3, 100, 101, 250, 299, 299], dtype=torch.int32, device="cuda"), torch.zeros_like(starts)]
    want = []
    for s in sets:
        starts.copy_(s)
        want.append([None if t is None else t.clone() for t in score()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = score()
    for i in (0, 1, 2, 1):
        starts.copy_(sets[i])
        graph.replay()
        torch.cuda.synchronize()
        rows = slice(int(sets[i][0]), int(sets[i][-1]))
        assert torch.equal(got[0][:, rows], want[i][0][:, rows])
        if experts:
            assert torch.equal(got[1], want[i][1])


def test_axes_are_whole_numbers():
    x, pos = OaMatrix(torch.ones(3, 64)), OaMatrix(torch.ones(2, 3, dtype=torch.int32))
    want = F.RotaryAxes(x, pos, (0, 1) * 16, 1, 64).Tensor()
    assert torch.equal(F.RotaryAxes(x, pos, torch.tensor([0, 1] * 16), 1, 64).Tensor(), want)
    for bad in ((0.5,) * 32, ("0",) * 32):
        with pytest.raises(TypeError):
            F.RotaryAxes(x, pos, bad, 1, 64)
        with pytest.raises(TypeError):
            F.PackedSequences(OaMatrix(torch.tensor([0, 3], dtype=torch.int32)), 3, pos, bad)
