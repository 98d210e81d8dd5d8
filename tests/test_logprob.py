"""Log-probabilities of given tokens, entropy, alternatives and the logits' gradient, on both paths against statements in 64 bits with bounds worked out from
the roundings."""
import math

import pytest
import torch

from oa_b200.ops import logprob as L

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
INF = math.inf


def _logits(rows, vocab, dtype, std=3.0, seed=0):
    g = torch.Generator().manual_seed(seed * 101 + rows * 7 + vocab)
    x = torch.randn(rows, vocab, generator=g) * std
    return x.to(dtype), torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32), torch.randn(rows, generator=g), torch.randn(rows, generator=g)


def _oracle(x, targets, top, scale, ignore):
    y = x.double() * scale
    logp = y - torch.logsumexp(y, 1, keepdim=True)
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, 0.0).sum(1)
    chosen = torch.where(targets == ignore, 0.0, logp.gather(1, targets.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0])
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    return chosen, h, logp, p, order


def _relative(y):
    """Of a weight exp(y - m): its argument's rounding (the product with scale and the difference, 2^-23 of both magnitudes; the multiplication by log2 e inside
    the exponential 2^-23 more) and the exponential's own 2^-21, for the exponents that count (e^-30 of the row and less do not show)."""
    mag = y.abs().masked_fill(y == -INF, 0).amax(1)
    return (2 * mag + 30) * 2.0 ** -23 + 2.0 ** -21


def _check(x, targets, dlogp, dent, device, top=0, scale=1.0, ignore=-100, place=None):
    """`place`: x as it lies on the device, where it matters how."""
    rows, vocab = x.shape
    chosen, h, logp, p, order = _oracle(x, targets, top, scale, ignore)
    xd, td = x.to(device) if place is None else place, targets.to(device)
    r = L.token_logprobs(xd, td, top, scale, ignore)
    e = _relative(x.double() * scale) + (math.log2(vocab) + 60) * 2.0 ** -24      # sums by threads, then as a tree: few hundred terms one after the other
    assert r.top_ids.dtype is torch.int32 and torch.equal(r.top_ids.cpu().long(), order)
    near = lambda name, got, want, bound: _near(name, got, want, bound)      # noqa: E731
    b = e + 2.0 ** -22 * (chosen.abs() + 1)
    near("logprobs", r.logprobs, chosen, torch.where(targets == ignore, 0.0, b))
    want = logp.gather(1, order)
    near("top_logprobs", r.top_logprobs, want, e[:, None] + 2.0 ** -22 * (want.abs() + 1))
    spread = torch.where(p > 0, p * logp.abs(), 0.0).sum(1)
    near("entropy", r.entropy, h, 3 * e * (1 + spread) + 2.0 ** -22)
    near("stats", r.stats.sum(1), torch.logsumexp(x.double() * scale, 1), e + 2.0 ** -22 * (1 + (x.double() * scale).amax(1).abs()))
    for g, k in ((dlogp, None), (dlogp, dent), (None, dent)):
        gg = torch.zeros(rows).double() if g is None else torch.where(targets == ignore, 0.0, g).double()
        kk = torch.zeros(rows).double() if k is None else k.double()
        inner = torch.where(p > 0, logp, 0.0) + h[:, None]
        d = -p * (gg[:, None] + kk[:, None] * inner)
        d[torch.arange(rows), targets.clamp(min=0).long()] += gg
        d = d * scale
        # a weight's error, twice over (it and the row's sum), its logarithm's and the entropy's, then the roundings of sum and product
        t = torch.zeros_like(p)
        t[torch.arange(rows), targets.clamp(min=0).long()] = gg.abs()
        bound = U[x.dtype] * d.abs() + scale * (p * ((2 * e[:, None] + 2.0 ** -21) * (gg.abs()[:, None] + kk.abs()[:, None] * inner.abs())
                                                      + kk.abs()[:, None] * (e + 3 * e * (1 + spread) + 2.0 ** -21 * (1 + h.abs()))[:, None]
                                                      + kk.abs()[:, None] * 2.0 ** -21 * torch.where(p > 0, logp.abs(), 0.0)) + 2.0 ** -22 * t) + 2.0 ** -126
        # a weight below the smallest normal number, 2^-126, may count as 0: its product with the bracket, by at most 2^-126 of that, is then missing
        bound = bound + scale * 2.0 ** -126 * (gg.abs()[:, None] + kk.abs()[:, None] * inner.abs())
        got = L.token_logprobs_backward(xd, td, r, None if g is None else g.to(device), None if k is None else k.to(device), scale, ignore)
        assert got.dtype is x.dtype
        near("dlogits", got, d, bound)
    return r


def _near(name, got, want, bound):
    got = got.cpu().double()
    err = torch.where(got == want, 0.0, (got - want).abs())
    assert not err.isnan().any(), f"{name}: NaN at {err.isnan().nonzero()[:4].tolist()}"
    over = (err > bound).nonzero()
    assert over.numel() == 0, f"{name}: {over.shape[0]} off, first {over[0].tolist()}: {got[tuple(over[0])]} for {want[tuple(over[0])]}, bound {bound[tuple(over[0])]}"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (16, 256), (5, 999), (2, 4096), (3, 32000), (1, 50257), (33, 2049), (2, 201088)])
def test_shapes(device, dtype, rows, vocab):
    _check(*_logits(rows, vocab, dtype), device, top=min(20, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(400, 8191, 1), (700, 1000, 32), (150, 33000, 0), (300, 60001, 5), (1200, 64, 7), (40, 120000, 32)])
def test_many_rows(dtype, rows, vocab, top):
    _check(*_logits(rows, vocab, dtype), "cuda", top=top)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.5, 1.0 / 0.7, 20.0])
def test_scale(device, dtype, scale):
    _check(*_logits(4, 3000, dtype, std=1.0), device, top=3, scale=scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [300, 40000])
def test_far_from_zero(device, dtype, vocab):
    """Rows whose logits are all of the order of 1e4: differences count."""
    x, t, g, h = _logits(3, vocab, dtype)
    _check((x.float() + torch.tensor([[1e4], [-3e4], [500.0]])).to(dtype), t, g, h, device, top=4)


def _order_cases(vocab):
    g = torch.Generator().manual_seed(vocab)
    up = torch.linspace(-8, 8, vocab)
    spikes = torch.randn(vocab, generator=g)
    spikes[::max(vocab // 40, 1)] = 12.0
    tail = torch.full((vocab,), -9.0)
    tail[-5:] = 1.0
    few = torch.full((vocab,), -INF)
    few[vocab // 2], few[vocab - 1] = 0.5, -0.5
    return {"rising": up, "falling": up.flip(0), "equal": torch.full((vocab,), 1.25), "zeros": torch.cat([torch.zeros(vocab // 2), -torch.zeros(vocab - vocab // 2)]),
            "spikes": spikes, "tail": tail, "few": few, "steps": (up * 2).floor(), "blocks": spikes.sort().values.roll(vocab // 3)}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 2500, 33333, 201088])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_orders_and_ties(device, dtype, vocab, top):
    """Equal logits rank by index, whatever order a row's logits come in and however many there are of one."""
    x = torch.stack(list(_order_cases(vocab).values())).to(dtype)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    r = L.token_logprobs(x.to(device), torch.zeros(x.shape[0], dtype=torch.int32, device=device), top)
    for i, name in enumerate(_order_cases(vocab)):
        assert torch.equal(r.top_ids[i].cpu().long(), order[i]), name
    logp = x.double() - torch.logsumexp(x.double(), 1, keepdim=True)
    want = logp.gather(1, order)
    _near("top", r.top_logprobs, want, 2.0 ** -17 + 2.0 ** -22 * want.abs().nan_to_num(posinf=0.0))      # |y| to 24: (48 + 30) 2^-23 and the sums


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [33, 5000, 150001])
def test_masked_and_broken_rows(device, dtype, vocab):
    x, t, g, h = _logits(8, vocab, dtype)
    t[:] = torch.tensor([vocab - 1, 0, 3, 3, 3, -100, vocab, -1])
    x[0, :vocab - 1] = -INF                        # one token left: probability 1
    x[1, 1:] = torch.finfo(dtype).min              # the type's lowest value as the mask
    x[2] = -INF                                    # nothing left
    x[3, vocab // 2] = math.nan
    x[4, vocab // 3] = INF
    x[5, ::2] = -INF
    top = 5
    r = L.token_logprobs(x.to(device), t.to(device), top)
    lp, ent = r.logprobs.cpu(), r.entropy.cpu()
    assert lp[0] == 0 and ent[0] == 0 and lp[1] == 0 and abs(float(ent[1])) < 1e-6
    assert lp[2] == -INF and ent[2] == 0 and bool((r.top_logprobs[2] == -INF).all()) and r.top_ids[2].tolist() == list(range(top))
    assert bool(lp[3:5].isnan().all()) and bool(ent[3:5].isnan().all()) and bool(r.top_logprobs[3:5].isnan().all())
    assert int(r.top_ids[4, 0]) == vocab // 3 and vocab // 2 not in r.top_ids[3].tolist()
    assert lp[5] == 0 and bool(lp[6:].isnan().all()) and not bool(ent[5:].isnan().any())
    assert r.top_ids[0].tolist()[0] == vocab - 1 and r.top_ids[0].tolist()[1:] == list(range(top - 1))
    d = L.token_logprobs_backward(x.to(device), t.to(device), r, g.to(device), h.to(device)).cpu()
    assert bool((d[0] == 0).all()) and bool((d[1] == 0).all()) and bool((d[2] == 0).all())
    assert bool(d[3:5].isnan().all()) and bool(d[6:].isnan().all())
    assert bool((d[5, ::2] == 0).all()) and not bool(d[5].isnan().any())
    # the row of which half is masked: as if the masked tokens were not there
    xs, ts = x[5:6, 1::2].contiguous(), torch.tensor([-100], dtype=torch.int32)
    s = L.token_logprobs(xs, ts, 0)
    want = L.token_logprobs_backward(xs.double().float(), ts, s, None, h[5:6])
    assert torch.allclose(d[5, 1::2].float(), want.float(), rtol=2 * U[dtype] + 1e-4, atol=1e-7) and abs(float(s.entropy[0] - ent[5])) < 1e-4


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [37, 6000, 90001])
def test_layouts(device, dtype, vocab):
    """Rows apart, rows that begin anywhere, columns apart, and the gradient in other rows or in the logits' place.  Sums depend on where a row begins: they are
    added up by 16-byte pieces."""
    x, t, g, h = _logits(5, vocab, dtype)
    td, gd, hd = (v.to(device) for v in (t, g, h))
    for extra, at in ((8, 0), (8, 8), (3, 1), (5, 4)):
        wide = torch.full((5, vocab + extra), math.nan, dtype=dtype, device=device)
        y = wide[:, at:at + vocab]
        y.copy_(x)
        r = _check(x, t, g, h, device, top=6, place=y)
        want = L.token_logprobs_backward(y, td, r, gd, hd)
        out = torch.full((5, vocab + extra + 1), 7.0, dtype=dtype, device=device)
        got = L.token_logprobs_backward(y, td, r, gd, hd, out=out[:, at:at + vocab])
        assert torch.equal(got, want) and bool((out[:, :at] == 7).all()) and bool((out[:, at + vocab:] == 7).all())
        assert torch.equal(L.token_logprobs_backward(y, td, r, gd, hd, out=y), want)
        assert torch.equal(y, want) and bool(wide[:, :at].isnan().all()) and bool(wide[:, at + vocab:].isnan().all())
    _check(x, t, g, h, device, top=6, place=x.to(device).t().contiguous().t())
    row = x[:1].to(device).expand(5, vocab)
    _check(x[:1].expand(5, vocab), t, g, h, device, place=row)


@pytest.mark.parametrize("device", DEVICES)
def test_ignore_index_within_the_vocabulary(device):
    x, t, g, h = _logits(6, 50, torch.float32)
    t[2] = t[4] = 0
    _check(x, t, g, h, device, ignore=0)


def test_gradients_against_differences():
    """The CPU path in 64-bit steps of one logit at a time."""
    x, t, g, h = _logits(2, 9, torch.float32)
    r = L.token_logprobs(x, t, 0, 0.8)
    d = L.token_logprobs_backward(x, t, r, g, h, 0.8)

    def loss(y):
        lp = torch.log_softmax(y * 0.8, 1)
        return (lp.gather(1, t.long()[:, None])[:, 0] * g.double() - (lp.exp() * lp).sum(1) * h.double()).sum()

    for i in range(2):
        for j in range(9):
            step = torch.zeros(2, 9, dtype=torch.float64)
            step[i, j] = 1e-5
            diff = (loss(x.double() + step) - loss(x.double() - step)) / 2e-5
            assert abs(float(diff) - float(d[i, j])) < 2e-6      # third derivatives of order 1 times 1e-10, and 32 bits


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows(device, dtype):
    x, t = torch.zeros(0, 50, dtype=dtype, device=device), torch.zeros(0, dtype=torch.int32, device=device)
    r = L.token_logprobs(x, t, 3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    assert L.token_logprobs_backward(x, t, r, None).shape == (0, 50)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(4, 201088), (64, 32000), (2000, 3000)])
def test_same_bits_graphs_and_streams(rows, vocab):
    x, t, g, h = (v.cuda() for v in _logits(rows, vocab, torch.bfloat16))
    y = _logits(rows, vocab, torch.bfloat16, seed=5)[0].cuda()
    both = lambda z: (lambda r: (*r, L.token_logprobs_backward(z, t, r, g, h)))(L.token_logprobs(z, t, 10))      # noqa: E731
    want = [both(x), both(y)]
    assert all(torch.equal(a, b) for a, b in zip(both(x), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(y)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want[1]))
    a, b = x.clone(), y.clone()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph, z in zip(graphs, (a, b)):
        with torch.cuda.graph(graph):
            outs.append(both(z))
    for first, second in ((0, 1), (1, 0)):
        a.copy_((x, y)[first])
        b.copy_((x, y)[second])
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs[0], want[first])) and all(torch.equal(p, q) for p, q in zip(outs[1], want[second]))


def test_refusals():
    x, t = torch.zeros(3, 20), torch.zeros(3, dtype=torch.int32)
    r = L.token_logprobs(x, t)
    for bad in (x.half(), x.double(), x[0], torch.zeros(3, 0)):
        with pytest.raises(ValueError, match="logits must be"):
            L.token_logprobs(bad, t)
    for bad in (t.long(), t[:2], torch.zeros(3, 1, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="targets must be"):
            L.token_logprobs(x, bad)
        with pytest.raises(ValueError, match="targets must be"):
            L.token_logprobs_backward(x, bad, r, None)
    for top in (-1, 21):
        with pytest.raises(ValueError, match="0 to 20 alternatives"):
            L.token_logprobs(x, t, top)
    with pytest.raises(ValueError, match="0 to 32 alternatives"):
        L.token_logprobs(torch.zeros(3, 100), t, 33)
    for scale in (0.0, -1.0, math.nan, INF):
        with pytest.raises(ValueError, match="scale must be positive"):
            L.token_logprobs(x, t, scale=scale)
        with pytest.raises(ValueError, match="scale must be positive"):
            L.token_logprobs_backward(x, t, r, None, scale=scale)
    for match, args, kw in (("dlogprobs must be", (torch.zeros(2),), {}), ("dlogprobs must be", (torch.zeros(3).bfloat16(),), {}), ("dentropy must be", (None, torch.zeros(6)[::2]), {}),
                            ("out must be", (None,), dict(out=torch.zeros(3, 19))), ("out must be", (None,), dict(out=torch.zeros(20, 3).t())),
                            ("out must be", (None,), dict(out=torch.zeros(1, 20).expand(3, 20))), ("out must be", (None,), dict(out=x.bfloat16()))):
        with pytest.raises(ValueError, match=match):
            L.token_logprobs_backward(x, t, r, *args, **kw)
    for ignore in (1 << 31, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="ignore_index is"):
            L.token_logprobs(x, t, ignore_index=ignore)
    both = torch.zeros(3, 21)
    with pytest.raises(ValueError, match="lie apart"):
        L.token_logprobs_backward(both[:, 1:], t, r, None, out=both[:, :20])
    with pytest.raises(ValueError, match="result.stats must be"):
        L.token_logprobs_backward(x, t, r._replace(stats=torch.zeros(3)), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 37, 64, 250, 1000, 1024, 2047])
def test_many_short_rows(vocab, dtype):
    """Rows enough for eight lanes to each, their number not a multiple of a block's, with rows of every special kind among them."""
    rows = 64 * torch.cuda.get_device_properties(0).multi_processor_count + 13
    x, targets, g, h = _logits(rows, vocab, dtype)
    x[::5, ::2] = -INF
    x[::5, -1] = 0.0
    targets[::7] = -100
    targets[::5] = vocab - 1                 # a target among the masked has log-probability -inf, which no bound is for
    _check(x, targets, g, h, "cuda")
    x[3], x[5, 0], x[6, -1] = -INF, math.nan, INF
    targets[3] = 0
    r = L.token_logprobs(x.cuda(), targets.cuda())
    lp, ent = r.logprobs.cpu(), r.entropy.cpu()
    assert lp[3] == -INF and ent[3] == 0 and ent[5].isnan() and ent[6].isnan() and lp[6].isnan()
    others = torch.ones(rows, dtype=torch.bool)
    others[[3, 5, 6]] = False
    assert lp[others].isfinite().all() and ent[others].isfinite().all()
    wide = torch.full((rows, vocab + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:vocab + 1] = x.cuda()
    odd = L.token_logprobs(wide[:, 1:vocab + 1], targets.cuda())
    e = _relative(torch.where(others[:, None], x, 0).double()) + (math.log2(vocab) + 60) * 2.0 ** -24
    _near("logprobs", odd.logprobs[others.cuda()], lp[others].double(), 2 * (e + 2.0 ** -22 * (lp.abs() + 1))[others])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [250, 32000])
def test_rows_beyond_32_bits(vocab):
    """The last rows of more than 2^31 logits: the bits of a small tensor's, forward and in place backward."""
    n = 64 * torch.cuda.get_device_properties(0).multi_processor_count if vocab == 250 else 704      # enough for the same form, a multiple of 8
    rows = 2 ** 31 // vocab // 8 * 8 + 96 + n                        # so that those rows lie on 16 bytes as in a tensor of their own: how a row is cut depends on it
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    for part in x.split(1 << 18):
        part.normal_(std=3.0)
    first = rows - n
    targets = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    tail = x[first:].clone()
    r = L.token_logprobs(x, targets)
    s = L.token_logprobs(tail, targets[first:].clone())
    for name in ("logprobs", "entropy", "stats"):
        assert torch.equal(getattr(r, name)[first:], getattr(s, name)), name
    want = L.token_logprobs_backward(tail, targets[first:].clone(), s, g[first:].clone(), h[first:].clone())
    L.token_logprobs_backward(x, targets, r, g, h, out=x)
    assert torch.equal(x[first:], want)


@pytest.mark.parametrize("device", DEVICES)
def test_a_scale_given_as_a_tensor(device):
    """It is read at every call, not remembered by which tensor it was."""
    x, t, g, h = (v.to(device) for v in _logits(3, 50, torch.float32))
    scale = torch.tensor(1.0)
    for s in (1.0, 0.25):
        scale.fill_(s)
        got, want = L.token_logprobs(x, t, 2, scale), L.token_logprobs(x, t, 2, s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(L.token_logprobs_backward(x, t, got, g, h, scale), L.token_logprobs_backward(x, t, want, g, h, s))
    for bad in (0.0, -1.0, INF):
        scale.fill_(bad)
        with pytest.raises(ValueError, match="scale must be positive"):
            L.token_logprobs(x, t, 2, scale)
        with pytest.raises(ValueError, match="scale must be positive"):
            L.token_logprobs_backward(x, t, want, g, h, scale)


@pytest.mark.parametrize("device", DEVICES)
def test_results_carry_no_graph(device):
    x, t, g, h = (v.to(device) for v in _logits(3, 50, torch.float32))
    for v in (x, g, h):
        v.requires_grad_(True)
    r = L.token_logprobs(x, t, 2)
    d = L.token_logprobs_backward(x, t, r, g, h)
    for v in (*r, d):
        assert not v.requires_grad and v.grad_fn is None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top", [0, 2])
def test_inference_mode(device, top):
    """Calls within inference mode give what they give elsewhere, and leave nothing of it to calls outside; what one call gives back is that call's alone."""
    x, t, g, h = (v.to(device) for v in _logits(7, 53, torch.float32))
    with torch.inference_mode():
        within = L.token_logprobs(x, t, top)
        grad = L.token_logprobs_backward(x, t, within, g, h)
    outside, again = L.token_logprobs(x, t, top), L.token_logprobs(x, t, top)
    assert all(torch.equal(a, b) for a, b in zip(within, outside)) and torch.equal(grad, L.token_logprobs_backward(x, t, outside, g, h))
    for a, b in zip(outside, again):
        assert not a.is_inference() and a is not b
        if a.dtype.is_floating_point:
            a.requires_grad_(True)
            assert not b.requires_grad and not L.token_logprobs(x, t, top).top_logprobs.requires_grad


def _many():
    """Rows enough for blocks of 128 threads where the vocabulary allows, not a multiple of anything."""
    return 4 * torch.cuda.get_device_properties(0).multi_processor_count + 3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 2049), (torch.bfloat16, 8191), (torch.bfloat16, 32000), (torch.bfloat16, 33600), (torch.bfloat16, 33607),
                                         (torch.float32, 2049), (torch.float32, 8191), (torch.float32, 16800), (torch.float32, 16803)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_many_long_rows(dtype, vocab, top):
    _check(*_logits(_many(), vocab, dtype), "cuda", top=top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [2500, 8192, 16001])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_orders_and_ties_of_many_rows(dtype, vocab, top):
    x = torch.stack(list(_order_cases(vocab).values())).to(dtype)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    logp = (x.double() - torch.logsumexp(x.double(), 1, keepdim=True)).gather(1, order)
    n, many = x.shape[0], _many()
    at = torch.arange(many) % n
    r = L.token_logprobs(x.cuda()[at.cuda()], torch.zeros(many, dtype=torch.int32, device="cuda"), top)
    assert torch.equal(r.top_ids.cpu().long(), order[at])
    _near("top", r.top_logprobs, logp[at], 2.0 ** -17 + 2.0 ** -22 * logp[at].abs().nan_to_num(posinf=0.0))      # as in test_orders_and_ties


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [2050, 9001])
@pytest.mark.parametrize("top", [0, 5])
def test_masked_and_broken_rows_among_many(dtype, vocab, top):
    """Few such rows and many: the same where they are 0, infinite or NaN, the same alternatives, and values as near as either is to the definition."""
    x, t, g, h = _logits(8, vocab, dtype)
    t[:] = torch.tensor([vocab - 1, 0, 3, 3, 3, -100, vocab, -1])
    x[0, :vocab - 1] = -INF
    x[1, 1:] = torch.finfo(dtype).min
    x[2] = -INF
    x[3, vocab // 2] = math.nan
    x[4, vocab // 3] = INF
    x[5, ::2] = -INF
    few = [v.cuda() for v in (x, t, g, h)]
    at = torch.arange(_many(), device="cuda") % 8
    many = [v[at] for v in few]
    got = []
    for a in (few, many):
        r = L.token_logprobs(a[0], a[1], top)
        got.append([*r, L.token_logprobs_backward(a[0], a[1], r, a[2], a[3])])
    # |y| to 15: (30 + 30) 2^-23 and the sums, either way; a gradient up to 6 such errors with g, h and log p to 16, then rounded
    e = 2 * 2.0 ** -16
    for name, a, b in zip(("logprobs", "entropy", "stats", "top_logprobs", "top_ids", "dlogits"), *got):
        a = a[at]
        same = (a == b) | (a.isnan() & b.isnan()) if a.is_floating_point() else a == b
        if name == "top_ids":
            assert bool(same.all())
        else:
            d = (a.double() - b.double()).abs().masked_fill(same, 0)
            bound = e + 2.0 ** -22 * a.double().abs() if name != "dlogits" else 16 * 6 * e * a.double().abs() + 2 * U[dtype] * a.double().abs() + 2.0 ** -100
            assert bool((same | (d <= bound)).all()), name             # the bound of a NaN is NaN: those are the same, or differ by NaN


@pytest.mark.gpu
@pytest.mark.parametrize("top", [5, 9])
def test_several_waves_of_longer_rows(top):
    """Twelve rows to an SM and more of over 4200 pieces: blocks of 128 threads up to eight alternatives, of 256 beyond."""
    _check(*_logits(12 * torch.cuda.get_device_properties(0).multi_processor_count + 3, 17201, torch.float32), "cuda", top=top)
