"""Sampling against a plain statement of its rule in exact arithmetic, and against the distribution it stands for."""
import math
from fractions import Fraction

import pytest
import torch

from oa_b200 import _native as N
from oa_b200.ops import sampling as S

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _exp32(y, device):
    """exp in fp32 as the device has it: the rule's weights are fp32 numbers, and everything behind them is exact."""
    return torch.exp(torch.tensor(y, dtype=torch.float32, device=device)).cpu()


def _oracle(x, u, t, k, p, least, device):
    """(token, log-probability) of one row by sorting; whole-number masses, threshold and running sums in Python's integers and fractions."""
    x = [-math.inf if math.isnan(v) else v for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if not x or x[order[0]] == -math.inf:
        return -1, -math.inf
    if not t > 0:
        return order[0], 0.0
    top = x[order[0]]
    inv = (torch.ones(()) / torch.tensor(t, dtype=torch.float32)).item()
    f32 = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    y = torch.where(f32(x) == top, f32(0.0), (f32(x) - f32(top)) * f32(inv))
    w = torch.where(f32(x) == -math.inf, f32(0.0), _exp32(y.tolist(), device))
    mass = [int(Fraction(v) * (1 << 40)) for v in w.tolist()]
    kept = order[:k] if k > 0 else order
    if p < 1:
        part, run, n = float(f32(p)) * float(sum(mass[i] for i in kept)), 0, 0
        for i in kept:
            if n and not float(run) < part:
                break
            run += mass[i]
            n += 1
        kept = kept[:n]
    kept = sorted(i for i in kept if w[i] >= min(f32(least), f32(1.0)))
    total = sum(mass[i] for i in kept)
    at = min(int(float(f32(u)) * float(total)), total - 1)
    run = 0
    for i in kept:
        run += mass[i]
        if run > at:
            return i, float(y[i]) - math.log(total / 2 ** 40)
    raise AssertionError


def _check(device, x, u, t, k, p, least):
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=device)  # noqa: E731
    tokens, logprobs = S.sample(x.to(device), f(u), f(t), torch.tensor(k, dtype=torch.int32, device=device), f(p), f(least))
    for r in range(x.shape[0]):
        want, lp = _oracle(x[r].float().tolist(), u[r], t[r], k[r], p[r], least[r], device)
        assert int(tokens[r]) == want, f"row {r}"
        # y is the rule's own; the logarithm of the mass is rounded to fp32 twice and the difference once
        assert float(logprobs[r]) == lp or abs(float(logprobs[r]) - lp) <= 2 ** -22 * (1 + abs(lp) + 20), f"row {r}"


RULES = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1), (0.8, 40, 0.8, 0.05), (0.0, 3, 0.5, 0.0), (2.0, 1, 1.0, 0.0),
         (1.0, 0, 0.0, 0.0), (1.0, 10 ** 6, 0.999, 0.0), (1.0, 3, 0.3, 2.0), (-1.0, 0, 1.0, 0.0), (0.05, 0, 0.95, 0.0), (30.0, 0, 0.5, 0.0),
         (1.0, -4, 1.5, 0.0), (1.0, 700, 0.99, 0.001)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 256, 511, 1000, 4099])
def test_every_rule(device, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    n = len(RULES) * 3
    x = (torch.randn(n, vocab, generator=g) * 2.5).to(dtype)
    u = torch.rand(n, generator=g).tolist()
    t, k, p, least = ([r[i] for r in RULES] * 3 for i in range(4))
    _check(device, x, u, t, k, p, least)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [33, 700, 5000])
def test_equal_logits_rank_by_index(device, vocab):
    """All logits equal, two values only, and a few values: the cut falls among equals."""
    g = torch.Generator().manual_seed(vocab)
    n = len(RULES)
    t, k, p, least = ([r[i] for r in RULES] for i in range(4))
    u = torch.rand(n, generator=g).tolist()
    _check(device, torch.full((n, vocab), -3.25), u, t, k, p, least)
    _check(device, torch.randint(0, 2, (n, vocab), generator=g).float(), u, t, k, p, least)
    x = torch.randint(-3, 4, (n, vocab), generator=g).float() * 0.5
    x[x == 0] = -0.0                                              # a zero is a zero
    x[:, ::2] += 0.0
    _check(device, x, u, t, k, p, least)


@pytest.mark.parametrize("device", DEVICES)
def test_masked_and_broken_logits(device):
    """-inf, the type's lowest value, NaN, +inf and rows of nothing."""
    g = torch.Generator().manual_seed(2)
    low = torch.finfo(torch.float32).min
    x = torch.randn(12, 777, generator=g)
    x[0, 5:] = -math.inf
    x[1] = -math.inf
    x[2] = math.nan
    x[3, ::3] = math.nan
    x[4, 1:] = low
    x[5] = low
    x[6, 100] = math.inf
    x[7, 100:104] = math.inf
    x[7, 50] = math.nan
    x[8, :776] = -math.inf
    x[9] *= 1e30
    x[10, 400:] = low
    for rule in RULES:
        n = x.shape[0]
        _check(device, x, torch.rand(n, generator=g).tolist(), *([v] * n for v in rule))


@pytest.mark.parametrize("device", DEVICES)
def test_ends_of_the_random_numbers(device):
    x = torch.tensor([[0.0, 0.0, -math.inf, 0.0]] * 6)
    u = [0.0, 0.3333, 0.33334, 0.6667, 1.0 - 2.0 ** -24, 0.5]
    tokens, logprobs = S.sample(x.to(device), torch.tensor(u, device=device))
    assert tokens.tolist() == [0, 0, 1, 3, 3, 1]
    assert torch.allclose(logprobs.cpu(), torch.full((6,), -math.log(3.0)), rtol=2 ** -22, atol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_strided_rows_and_scalars_left_out(device):
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(5, 1000, generator=g).to(device)
    x, u = wide[:, 3:903], torch.rand(5, generator=g).to(device)
    for a, b in zip(S.sample(x, u), S.sample(x.contiguous(), u)):
        assert torch.equal(a, b)
    flip = wide[:, :900].t().contiguous().t()                     # columns side by side
    for a, b in zip(S.sample(flip, u), S.sample(wide[:, :900].contiguous(), u)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [32000, 50257, 201088, 300001])
def test_large_vocabularies(dtype, vocab):
    """The kernel's cuts against a sort on the device: token, and the log-probability, of every rule."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    n = len(RULES)
    x = (torch.randn(n, vocab, generator=g, device="cuda") * 2.5).to(dtype)
    x[:, 17] += 6
    x[1::4] *= 4                                                  # rows in which a few tokens hold everything
    x[2::4] *= 0.01                                               # rows that are nearly flat
    x[3::4, 1000:] = -math.inf
    u = torch.rand(n, generator=g, device="cuda")
    _check_on_device(x, u, RULES)


def _check_on_device(x, u, rules):
    f = lambda i, dtype=torch.float32: torch.tensor([r[i] for r in rules], dtype=dtype, device="cuda")  # noqa: E731
    t, k, p, least = f(0), f(1, torch.int32), f(2), f(3)
    tokens, logprobs = S.sample(x, u, t, k, p, least)
    for r, (tr, kr, pr, lr) in enumerate(rules):                  # the rule again, with int64 sums along a sorted row
        xs, order = torch.sort(x[r].float(), descending=True, stable=True)
        if tr <= 0:
            assert int(tokens[r]) == int(order[0]) and float(logprobs[r]) == 0
            continue
        y = torch.where(xs == xs[0], 0.0, (xs - xs[0]) * (1.0 / t[r]))
        w = torch.where(xs == -math.inf, 0.0, torch.exp(y))
        mass = (w * 2.0 ** 40).long()
        if kr > 0:
            mass[kr:] = 0
        if pr < 1:
            n = int(((torch.cumsum(mass, 0) - mass).double() < p[r].double() * mass.sum().double()).sum())
            mass[max(n, 1):] = 0
        mass[w < min(lr, 1.0)] = 0
        by_index = torch.zeros_like(mass).scatter_(0, order, mass)
        total = int(mass.sum())
        at = min(int(float(u[r]) * float(total)), total - 1)
        want = int(torch.searchsorted(torch.cumsum(by_index, 0), torch.tensor([at], device="cuda"), right=True))
        assert int(tokens[r]) == want, f"row {r}"
        lp = float(y[int((order == want).nonzero()[0, 0])]) - math.log(total / 2 ** 40)
        assert abs(float(logprobs[r]) - lp) <= 2 ** -22 * (1 + abs(lp) + 20), f"row {r}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [600, 9000, 77777, 201088])
@pytest.mark.parametrize("spread", [1e-6, 0.05, 1.0, 40.0])
def test_cuts_deep_in_a_row(dtype, vocab, spread):
    """Cuts that leave thousands of tokens, from rows in which many are nearly or quite equal to rows that spread far."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rules = [(1.0, 300, 1.0, 0.0), (3.0, 0, 0.9, 0.0), (1.0, 5000, 1.0, 0.0), (1.0, 5000, 0.7, 0.001), (100.0, 0, 0.5, 0.0), (1e4, 0, 0.97, 0.0), (0.5, 0, 0.999999, 0.0),
             (1.0, 70000, 0.9, 0.0), (1.0, 0, 0.999, 0.9999), (2.0, 257, 0.01, 0.0), (1.0, 0, 1.0, 1e-6), (1.0, vocab - 1, 1.0, 0.0)]
    x = (torch.randn(len(rules), vocab, generator=g, device="cuda") * spread).to(dtype)
    u = torch.rand(len(rules), generator=g, device="cuda")
    _check_on_device(x, u, rules)
    _check_on_device((x * 4).round() / 4 + 100, u, rules)         # equal ones, away from zero
    x[:, vocab // 3:] = torch.finfo(dtype).min
    _check_on_device(x, u, rules)


@pytest.mark.gpu
def test_more_tokens_than_a_cluster_holds():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(len(RULES), 500009, generator=g, device="cuda") * 2.5
    _check_on_device(x, torch.rand(len(RULES), generator=g, device="cuda"), RULES)


@pytest.mark.parametrize("device", DEVICES)
def test_tokens_follow_the_distribution(device):
    """16384 numbers spread evenly over [0, 1): each token as often as its probability says, to one count at either end of its stretch."""
    g = torch.Generator().manual_seed(4)
    n, row = 16384, torch.randn(60, generator=g) * 2
    u = (torch.arange(n) + 0.5) / n
    t = torch.full((n,), 0.9)
    tokens, logprobs = S.sample(row.expand(n, 60).contiguous().to(device), u.to(device), t.to(device), None, None, None)
    prob = torch.softmax(row.double() / 0.9, 0)
    count = torch.bincount(tokens.cpu().long(), minlength=60).double()
    assert ((count - prob * n).abs() <= 1.01).all()
    # the scaled logits are fp32, with the product's and the difference's rounding: 2^-22 of at most 10
    assert (logprobs.cpu().double() - prob.log()[tokens.cpu().long()]).abs().max() <= 10 * 2.0 ** -21


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, u = torch.zeros(3, 8, device=device), torch.zeros(3, device=device)
    for bad in [(x[0], u), (x, u[:2]), (x, u.double()), (x, u, u[:2]), (x, u, None, u), (x, u, None, None, u.bfloat16()), (x, u, u.double())]:
        with pytest.raises(ValueError):
            S.sample(*bad)
    empty = S.sample(torch.zeros(0, 8, device=device), torch.zeros(0, device=device))
    assert empty[0].numel() == 0 and empty[1].numel() == 0


@pytest.mark.gpu
def test_refusals_of_the_kernel():
    u = torch.zeros(3, device="cuda")
    with pytest.raises(N.OaKernelError):
        S.sample(torch.zeros(3, 8, device="cuda", dtype=torch.float16), u)
    with pytest.raises(ValueError):
        S.sample(torch.zeros(3, 8, device="cuda"), u.cpu())
