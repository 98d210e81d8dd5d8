"""Packed sequences: the plan's lists, rotary positions with several axes, causal attention with grouped heads and its gradients, on both paths against
statements in 64 bits with bounds worked out from the roundings.

A rounding to a type is off by at most half its step relative to the value: U bf16 2^-8, fp32 2^-24.  In bf16 the weights p and the score gradients dS are
rounded once more before they meet V, dO, K and Q, and delta is worked out from the rounded output.
"""
import math

import pytest
import torch

from oa_b200.ops import kernels as K
from oa_b200.ops import packed as P

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F64 = torch.float64
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
THETA = 10000.0


def _starts(lengths, device, first=0):
    return torch.tensor([first] + lengths).cumsum(0).to(torch.int32).to(device)


def _inputs(lengths, hq, hk, hd, dtype, device, first=0, pad=0, seed=0, fill=math.nan):
    """q, k, v as slices of one projection's rows, and dO; rows of no sequence hold `fill`."""
    g = torch.Generator().manual_seed(seed * 1009 + len(lengths) * 31 + hd)
    tokens = first + sum(lengths) + pad
    qkv = torch.randn(tokens, (hq + 2 * hk) * hd, generator=g).to(dtype)
    dout = torch.randn(tokens, hq * hd, generator=g).to(dtype)
    for t in (qkv, dout):
        t[:first] = fill
        t[tokens - pad:] = fill
    qkv, dout = qkv.to(device), dout.to(device)
    return (*torch.split(qkv, [hq * hd, hk * hd, hk * hd], 1), dout)


def _oracle(q, k, v, dout, starts, hd, scale, dtype, exact_ds=False):
    """{name: (value, bound)} in 64 bits; rows of no sequence are 0 (lse -inf) with bound 0.  exact_ds: delta is the sum of p dP in 32 bits, and dS goes to its
    products as two bf16 numbers, together off by 2^-8 of 2^-8."""
    q, k, v, dout = (t.cpu().double() for t in (q, k, v, dout))
    tokens, hq, hk = q.shape[0], q.shape[1] // hd, k.shape[1] // hd
    u, half = U[dtype], dtype is torch.bfloat16
    up = u if half else 0.0                                       # the extra rounding of p and dS
    out = {n: [torch.zeros(tokens, h * hd, dtype=F64), torch.zeros(tokens, h * hd, dtype=F64)] for n, h in (("o", hq), ("dq", hq), ("dk", hk), ("dv", hk))}
    out["lse"] = [torch.full((hq, tokens), -math.inf, dtype=F64), torch.zeros(hq, tokens, dtype=F64)]
    st = starts.tolist()
    for lo, hi in zip(st, st[1:]):
        n = hi - lo
        if n <= 0:
            continue
        qs, dy = (t[lo:hi].reshape(n, hq, hd).transpose(0, 1) for t in (q, dout))
        ks, vs = (t[lo:hi].reshape(n, hk, hd).transpose(0, 1).repeat_interleave(hq // hk, 0) for t in (k, v))
        late = torch.ones(n, n, dtype=torch.bool).triu(1)
        x = (qs @ ks.transpose(1, 2) * scale).masked_fill(late, -math.inf)
        lse = torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(x - lse)
        y = p @ vs
        # scores: hd products added in 32 bits (each step at most 2^-23 of the sum of magnitudes), then the exponential: 2^-21 and
        # the rounding of its argument; sums of n terms: n 2^-24
        mag = (qs.abs() @ ks.abs().transpose(1, 2)).masked_fill(late, 0) * scale
        far = (x - lse).masked_fill(late, 0).abs().amax()
        dx = mag.amax() * hd * 2 ** -23 + far * 2 ** -22 + 2 ** -20
        sums = (n + hd) * 2.0 ** -23
        e = float(2 * dx + sums)                                  # relative error of a weight: its own score and the row's sum
        bo = u * y.abs() + (up + e) * (p @ vs.abs())
        delta = (dy * y).sum(-1, keepdim=True)
        dp = dy @ vs.transpose(1, 2)
        ds = scale * p * (dp - delta)
        bdelta = (dy.abs() * bo).sum(-1, keepdim=True) + hd * 2 ** -23 * (dy * y).abs().sum(-1, keepdim=True)
        bdp = hd * 2 ** -23 * (dy.abs() @ vs.abs().transpose(1, 2))
        if exact_ds:
            bdelta = (e + n * 2 ** -23) * (p * dp.abs()).sum(-1, keepdim=True) + (p * bdp).sum(-1, keepdim=True)
        bds = scale * p * (bdelta + bdp + 2 ** -22 * (dp.abs() + delta.abs())) + ((up ** 2 if exact_ds else up) + e) * ds.abs()
        sum_ds = sums * ds.abs()
        one = lambda t: t.transpose(0, 1).reshape(n, -1)          # noqa: E731
        group = lambda t: one(t.reshape(hk, hq // hk, n, hd).sum(1))   # noqa: E731
        dq, dk, dv = ds @ ks, ds.transpose(1, 2) @ qs, p.transpose(1, 2) @ dy
        many = (n * (hq // hk)) * 2.0 ** -23
        for name, val, bound in (("o", one(y), one(bo)), ("dq", one(dq), u * one(dq).abs() + one((bds + sum_ds) @ ks.abs())),
                                 ("dk", group(dk), u * group(dk).abs() + group((bds + many * ds.abs()).transpose(1, 2) @ qs.abs())),
                                 ("dv", group(dv), u * group(dv).abs() + (up + e + many) * group(p.transpose(1, 2) @ dy.abs()))):
            out[name][0][lo:hi], out[name][1][lo:hi] = val, bound
        out["lse"][0][:, lo:hi] = lse[..., 0]
        out["lse"][1][:, lo:hi] = dx + sums + 2 ** -21 * (1 + lse[..., 0].abs())
    return out


def _close(name, got, want, bound):
    got = got.cpu().double()
    same = got == want                                            # -inf of rows without a sequence
    err = torch.where(same, 0.0, (got - want).abs())
    assert not err.isnan().any(), f"{name}: NaN at {err.isnan().nonzero()[:5].tolist()}"
    over = (err > bound * 1.0001 + 1e-30).nonzero()
    assert over.numel() == 0, f"{name}: {over.shape[0]} of {err.numel()} off, first {over[0].tolist()}: {got[tuple(over[0])]} for {want[tuple(over[0])]}, " \
                              f"bound {bound[tuple(over[0])]}"


def _both(q, k, v, dout, starts, hd, scale=None):
    plan = P.plan(starts, q.shape[0])
    o, lse = P.attention(q, k, v, plan, hd, scale, return_lse=True)
    return dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *P.attention_backward(q, k, v, o, dout, lse, plan, hd, scale))))


def _check(lengths, hq, hk, hd, dtype, device, first=0, pad=0, scale=None, seed=0):
    q, k, v, dout = _inputs(lengths, hq, hk, hd, dtype, device, first, pad, seed)
    starts = _starts(lengths, device, first)
    got = _both(q, k, v, dout, starts, hd, scale)
    assert got["o"].dtype is dtype and got["lse"].dtype is torch.float32
    for name, (want, bound) in _oracle(q, k, v, dout, starts, hd, scale or hd ** -0.5, dtype).items():
        _close(name, got[name], want, bound)


RAGGED = [5, 0, 300, 1, 127, 128, 129, 64, 2, 257]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths", [[1], [2], [15], [16], [17], [33], [48], [63], [64], [65], [127], [128], [129], [256], [257], [1, 1, 1], RAGGED], ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_lengths_bf16(device, lengths, hd):
    _check(lengths, 4, 2, hd, torch.bfloat16, device)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[2] * 40, [1, 2, 3, 4, 5, 8, 16] * 3, [15, 9, 2], [32, 17, 1, 25]], ids=["two", "mixed", "three", "32"])
@pytest.mark.parametrize("hq,hk", [(8, 1), (12, 4), (3, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_round_only_the_result(lengths, hq, hk, hd):
    """Up to 32 rows have too few roundings of dS for them to even out: their gradients are off by the rounding of the result and little else."""
    q, k, v, dout = _inputs(lengths, hq, hk, hd, torch.bfloat16, "cuda", pad=5)
    starts = _starts(lengths, "cuda")
    got = _both(q, k, v, dout, starts, hd)
    want = _oracle(q, k, v, dout, starts, hd, hd ** -0.5, torch.bfloat16, exact_ds=True)
    for name in ("dq", "dk"):
        _close(name, got[name], *want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,hq,hk,hd", [([200, 1, 130], 64, 1, 64), ([1000], 12, 4, 64), ([300, 65], 7, 1, 128), ([900, 40], 16, 2, 128), ([64, 65, 128], 10, 2, 64), ([129] * 3, 70, 1, 64)])
def test_heads_of_a_group_on_several_blocks(lengths, hq, hk, hd):
    """Few tiles: a group's heads are dealt out and their sums joined, in one order."""
    _check(lengths, hq, hk, hd, torch.bfloat16, "cuda", first=3, pad=150)
    q, k, v, dout = _inputs(lengths, hq, hk, hd, torch.bfloat16, "cuda", 3, 150)
    starts = _starts(lengths, "cuda", 3)
    one, two = (_both(q, k, v, dout, starts, hd) for _ in range(2))
    assert all(torch.equal(one[n], two[n]) for n in one)


@pytest.mark.gpu
def test_backward_leaves_short_sequences_beside_long_ones():
    """delta's own launch goes over the tiles of longer sequences; scratch of earlier calls, NaN here, reaches no result."""
    lengths = [3, 200, 64, 65, 1, 128, 500, 17]
    q, k, v, dout = _inputs(lengths, 6, 2, 64, torch.bfloat16, "cuda", first=9, pad=300)
    starts = _starts(lengths, "cuda", 9)
    first = _both(q, k, v, dout, starts, 64)
    size = 2 * 6 * q.shape[0] * 4
    for _ in range(4):
        torch.full((size,), 255, dtype=torch.uint8, device="cuda")       # back to the allocator at once
        again = _both(q, k, v, dout, starts, 64)
        assert all(torch.equal(first[n], again[n]) for n in first)
    for name, (want, bound) in _oracle(q, k, v, dout, starts, 64, 64 ** -0.5, torch.bfloat16).items():
        _close(name, first[name], want, bound)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (6, 2), (4, 1), (8, 2), (7, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_heads_bf16(device, hq, hk, hd):
    _check([200, 3, 131], hq, hk, hd, torch.bfloat16, device, first=7, pad=70)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,hd", [(2, 2, 64), (4, 1, 64), (2, 2, 128), (4, 1, 128)])
def test_attention_long_bf16(hq, hk, hd):
    _check([1500, 700, 1], hq, hk, hd, torch.bfloat16, "cuda", pad=3)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk", [(16, 16), (8, 2), (3, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_many_short(hd, hq, hk):
    _check([i % 64 + 1 for i in range(150)] + [300], hq, hk, hd, torch.bfloat16, "cuda", pad=2)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_more_items_than_sms(hd):
    _check([17, 260, 40, 1, 90, 300, 5] * 6, 8, 4, hd, torch.bfloat16, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("hd,hq,hk", [(64, 84, 84), (64, 168, 84), (128, 84, 84)])
def test_attention_more_items_than_are_kept(hd, hq, hk):
    """A CTA's first rounds are kept in shared memory, the others are fetched: the same bits as from calls with fewer heads, which need no others."""
    lengths = [65 + i % 60 for i in range(190)]                      # 190 tiles times 84 heads are more than 96 rounds of 148 CTAs
    q, k, v, dout = _inputs(lengths, hq, hk, hd, torch.bfloat16, "cuda", pad=9, fill=0.0)
    starts = _starts(lengths, "cuda")
    whole = _both(q, k, v, dout, starts, hd)
    for at in range(0, hk, 28):
        mine = lambda t, h: t[:, at * (h // hk) * hd:(at + 28) * (h // hk) * hd]       # noqa: E731
        some = _both(mine(q, hq), mine(k, hk), mine(v, hk), mine(dout, hq), starts, hd)
        for n, h in (("o", hq), ("dq", hq), ("dk", hk), ("dv", hk)):
            assert torch.equal(mine(whole[n], h), some[n]), n


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths", [[1], [31, 33], [129], RAGGED], ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 32), (4, 2, 64), (3, 1, 128), (2, 1, 20), (2, 2, 7), (12, 4, 50), (8, 1, 32), (9, 1, 16), (24, 2, 64)])
def test_attention_fp32(device, lengths, hq, hk, hd):
    _check(lengths, hq, hk, hd, torch.float32, device, first=2, pad=5)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64])
def test_attention_fp32_many(hd):
    _check([400, 200, 1, 128] * 4, 8, 4, hd, torch.float32, "cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_scale(device, dtype):
    _check([140, 20], 2, 2, 64, dtype, device, scale=0.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 1)])
def test_sequences_do_not_reach_one_another(device, dtype, hq, hk):
    """One sequence full of NaN and infinities: the others' results are the same bits as beside zeros."""
    lengths = [3, 40, 20, 130, 129, 1, 60]
    starts = _starts(lengths, device)
    for bad in (1, 3, 5):
        q, k, v, dout = _inputs(lengths, hq, hk, 64, dtype, device)
        lo, hi = int(starts[bad]), int(starts[bad + 1])
        for t in (q, k, v, dout):
            t[lo:hi] = 0
        clean = _both(q, k, v, dout, starts, 64)
        for t, x in zip((q, k, v, dout), (math.nan, math.inf, math.nan, -math.inf)):
            t[lo:hi] = x
        got = _both(q, k, v, dout, starts, 64)
        for name in clean:
            a, b = (d[name].t() if name == "lse" else d[name] for d in (clean, got))
            assert torch.equal(torch.cat([a[:lo], a[hi:]]), torch.cat([b[:lo], b[hi:]])), name


@pytest.mark.parametrize("device", DEVICES)
def test_starts_that_fall_or_leave(device):
    """Starts count as the nearest that rise within the rows."""
    q, k, v, dout = _inputs([50], 2, 1, 64, torch.float32, device)
    got = _both(q, k, v, dout, torch.tensor([-5, 10, 4, 30, 99], dtype=torch.int32, device=device), 64)
    want = _both(q, k, v, dout, torch.tensor([0, 10, 10, 30, 50], dtype=torch.int32, device=device), 64)
    for name in want:
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_to_do(device, dtype):
    for tokens, starts in ((0, [0]), (0, [0, 0]), (5, [0]), (5, [3, 3, 3])):
        q, k, v, dout = (torch.full((tokens, 64), math.nan, dtype=dtype, device=device) for _ in range(4))
        got = _both(q, k, v, dout, torch.tensor(starts, dtype=torch.int32, device=device), 64)
        assert all(bool((got[n] == 0).all()) for n in ("o", "dq", "dk", "dv")) and bool((got["lse"] == -math.inf).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(device, dtype):
    """Rows apart by any distance, columns apart, rows that begin anywhere: the same bits as contiguous operands."""
    lengths, hq, hk, hd = [70, 130], 2, 1, 64
    starts = _starts(lengths, device)
    q, k, v, dout = (t.contiguous() for t in _inputs(lengths, hq, hk, hd, dtype, device))
    want = _both(q, k, v, dout, starts, hd)

    def wide(t, extra, at):
        out = torch.full((t.shape[0], t.shape[1] + extra), math.nan, dtype=dtype, device=device)[:, at:at + t.shape[1]]
        out.copy_(t)
        return out

    for extra, at in ((8, 8), (5, 3), (64, 0)):
        got = _both(*(wide(t, extra, at) for t in (q, k, v, dout)), starts, hd)
        assert all(torch.equal(got[n], want[n]) for n in want)
    got = _both(*(t.t().contiguous().t() for t in (q, k, v, dout)), starts, hd)
    assert all(torch.equal(got[n], want[n]) for n in want)
    row = q[:1].expand(200, hq * hd)
    same = _both(row, k, v, dout, starts, hd)
    assert all(torch.equal(same[n], t) for n, t in _both(row.contiguous(), k, v, dout, starts, hd).items())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_into_a_projections_rows(device, dtype):
    lengths, hq, hk, hd = [40, 200], 4, 2, 64
    q, k, v, dout = _inputs(lengths, hq, hk, hd, dtype, device)
    plan = P.plan(_starts(lengths, device), 240)
    o, lse = P.attention(q, k, v, plan, hd, return_lse=True)
    want = P.attention_backward(q, k, v, o, dout, lse, plan, hd)
    dqkv = torch.full((240, (hq + 2 * hk) * hd), math.nan, dtype=dtype, device=device)
    got = P.attention_backward(q, k, v, o, dout, lse, plan, hd, dqkv=dqkv)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(dqkv, torch.cat(want, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_same_inputs_same_bits(hd):
    lengths = [300, 5, 700, 129, 64] * 3
    q, k, v, dout = _inputs(lengths, 8, 2, hd, torch.bfloat16, "cuda")
    starts = _starts(lengths, "cuda")
    want = _both(q, k, v, dout, starts, hd)
    for _ in range(3):
        got = _both(q, k, v, dout, starts, hd)
        assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_graphs_and_streams(dtype):
    """Two graphs of the whole pass, replayed in turn with other lengths than those they were recorded with, and a call on another stream."""
    hq, hk, hd, tokens = 4, 2, 64, 600
    sets = [[100, 500], [600], [1, 299, 300], [37] * 16]
    q, k, v, dout = _inputs([tokens], hq, hk, hd, dtype, "cuda")
    fit = lambda lengths: torch.tensor(([0] + torch.tensor(lengths).cumsum(0).tolist() + [sum(lengths)] * 16)[:17], dtype=torch.int32, device="cuda")  # noqa: E731
    want = [_both(q, k, v, dout, fit(s), hd) for s in sets]
    starts = [fit(sets[0]), fit(sets[1])]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _both(q, k, v, dout, starts[0], hd)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(other[n], want[0][n]) for n in other)
    for s in starts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_both(q, k, v, dout, s, hd))
        graphs.append(g)
    for a, b in ((0, 1), (2, 3), (3, 0)):
        starts[0].copy_(fit(sets[a]))
        starts[1].copy_(fit(sets[b]))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i, w in ((0, a), (1, b)):
            assert all(torch.equal(outs[i][n], want[w][n]) for n in want[w])


@pytest.mark.gpu
def test_plan_lists():
    """Every tile and pair of every long sequence once, the largest index first, and every short sequence."""
    g = torch.Generator().manual_seed(3)
    for lengths in ([1], [0], RAGGED, torch.randint(0, 5000, (70,), generator=g).tolist(), [10] * 3000, [300000, 1, 200000], torch.randint(0, 400, (2500,), generator=g).tolist()):
        tokens, batch = sum(lengths) + 9, len(lengths)
        p = P.plan(_starts(lengths, "cuda", 2), tokens)
        w = p.words.cpu()
        n, m, classes = w[0].item(), w[1].item(), w[4:7].tolist()
        first = (8 + batch + 1 + 3) // 4 * 4
        starts = p.starts.cpu().tolist()
        most, pairs = tokens // 128 + batch, tokens // 256 + batch
        exact = tokens // 128 < 1024                               # beyond that, bins hold several indices
        lists = [w[at:at + 4 * count].reshape(-1, 4).tolist() for count, at in ((n, first), (m, first + 4 * most), (sum(classes), first + 4 * (most + pairs)))]
        long = [(a, b, s) for s, (a, b) in enumerate(zip(starts, starts[1:])) if b - a > 64]
        for got, rows in zip(lists, (128, 256)):
            assert sorted(map(tuple, got)) == sorted((a, b, i, s) for a, b, s in long for i in range(-(-(b - a) // rows)))
            order = [x[2] for x in got]
            step = 1 if exact else 1 << (tokens // 128 // 1024).bit_length()
            assert all(a // step >= b // step for a, b in zip(order, order[1:]))
        ends = [b - a for a, b, _, _ in lists[2]]
        assert classes == [sum(a < e <= b for e in ends) for a, b in ((32, 64), (16, 32), (0, 16))]
        assert all((-(-a // 16) + 1) // 2 >= (-(-b // 16) + 1) // 2 for a, b in zip(ends, ends[1:]) if a <= 32 or b <= 32)
        assert sorted(map(tuple, lists[2])) == [(a, b, 0, s) for s, (a, b) in enumerate(zip(starts, starts[1:])) if 0 < b - a <= 64]


# ------------------------------------------------------------------------------------------------ rotation
def _rotary_inputs(tokens, cols, axes, dtype, device, far=131072):
    g = torch.Generator().manual_seed(tokens * 7 + cols)
    return torch.randn(tokens, cols, generator=g).to(dtype).to(device), torch.randint(-far, far, (axes, tokens), generator=g, dtype=torch.int32).to(device)


def _rotary_oracle(x, positions, axes, heads, hd, theta, backward):
    n, half = x.shape[0], len(axes)
    v = x.cpu().double()[:, :heads * hd].reshape(n, heads, hd)
    a = positions.cpu().double()[list(axes)].t() * torch.exp(torch.arange(half, dtype=F64) * (-math.log(theta) / half))
    c, s = a.cos()[:, None], (-a.sin() if backward else a.sin())[:, None]
    lo, hi = v[..., :half], v[..., half:2 * half]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s, v[..., 2 * half:]], -1)
    pair = lo.abs() + hi.abs()
    return y.reshape(n, -1), torch.cat([pair, pair, 0 * v[..., 2 * half:]], -1).reshape(n, -1)


ROTARY = [((0,) * 32, 64), ((0,) * 8 + (1,) * 12 + (2,) * 12, 64), (tuple(j % 3 for j in range(64)), 128), ((1, 0, 2) * 5, 64), ((0, 1), 128), ((0,) * 16, 32),
          ((1,) * 7, 19), ((0,) * 128, 256), ((0,) * 24 + (1,) * 8, 64), ((0,), 2)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("axes,hd", ROTARY, ids=[f"{len(a)}of{h}" for a, h in ROTARY])
@pytest.mark.parametrize("backward", [False, True])
def test_rotary(device, dtype, axes, hd, backward):
    for tokens, heads in ((1, 1), (33, 5), (300, 40)):
        x, positions = _rotary_inputs(tokens, (heads + 2) * hd, 3, dtype, device)
        keep = x.clone()
        got = P.rotary(x, positions, axes, heads, hd, THETA, backward)
        want, pair = _rotary_oracle(x, positions, axes, heads, hd, THETA, backward)
        # an angle's turns are rounded to 32 bits within [-1/2, 1/2] (2^-24 turns), its products in 64 bits, sincospif to 2^-22 or so; three roundings of the result's sums
        bound = U[dtype] * want.abs() + pair * (2 * math.pi * 2 ** -24 + 2 ** -21 + 131072 * 2.0 ** -50)
        _close("rotary", got, want, bound)
        assert torch.equal(x, keep)
        inplace = P.rotary(x, positions, axes, heads, hd, THETA, backward, out=x)
        assert torch.equal(inplace, got) and inplace.data_ptr() == x.data_ptr() and torch.equal(x[:, heads * hd:], keep[:, heads * hd:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_layouts(device, dtype):
    axes, heads, hd = (0,) * 16 + (1,) * 16, 3, 64
    x, positions = _rotary_inputs(50, heads * hd + 64, 2, dtype, device)
    want = P.rotary(x[:, :heads * hd].contiguous(), positions, axes, heads, hd, THETA)
    for at in (0, 1, 8, 64):
        y = torch.zeros(50, heads * hd + 64, dtype=dtype, device=device)
        y[:, at:at + heads * hd] = x[:, :heads * hd]
        assert torch.equal(P.rotary(y[:, at:], positions, axes, heads, hd, THETA), want)
        assert torch.equal(P.rotary(y[:, at:], positions, axes, heads, hd, THETA, out=y[:, at:]), want)
    assert torch.equal(P.rotary(x.t().contiguous().t(), positions, axes, heads, hd, THETA), want)
    assert torch.equal(P.rotary(x[:1].expand(50, -1), positions, axes, heads, hd, THETA),
                       P.rotary(x[:1].expand(50, -1).contiguous(), positions, axes, heads, hd, THETA))
    empty = P.rotary(x[:0], positions[:, :0].contiguous(), axes, heads, hd, THETA)
    assert empty.shape == (0, heads * hd)


def test_rotary_is_the_usual_one_with_one_axis():
    from oa_b200.ops import kernels as K
    x, _ = _rotary_inputs(20, 128, 1, torch.float32, "cpu")
    want = K.rope_(x.clone(), 2, 64, 10, pos_offset=5, theta=THETA)
    got = P.rotary(x, (torch.arange(20) % 10 + 5).to(torch.int32)[None], (0,) * 32, 2, 64, THETA)
    assert torch.allclose(got, want, rtol=0, atol=4 * 2 ** -20)      # rope_ works its angles out in 32 bits


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)      # noqa: E731
    plan = P.plan(i32(0, 3, 8), 8)
    q, k = torch.randn(8, 128), torch.randn(8, 64)
    for bad in (torch.tensor([0, 3]), i32(0, 3, 4, 8)[::2], i32(0, 3).reshape(1, 2), i32()):
        with pytest.raises(ValueError, match="starts must be"):
            P.plan(bad, 8)
    for tokens in (-1, (1 << 30) + 1):
        with pytest.raises(ValueError, match="rows; at most"):
            P.plan(i32(0, 1), tokens)
    lse = torch.zeros(2, 8)
    for match, args in (("of one type", (q, k.bfloat16(), k)), ("of one type", (q.half(), k.half(), k.half())), ("of one shape", (q, k, k[:, :32])),
                        ("of one type", (q[0], k, k)), ("multiple of the key-value heads", (q[:, :96], k, k)), ("rows of heads", (q, k[:, :32], k[:, :32])),
                        ("the plan is for 8 rows", (q[:7], k[:7], k[:7])), ("the plan is for 8 rows", (q, k[:7], k[:7]))):
        with pytest.raises(ValueError, match=match):
            P.attention(*args, plan, 64)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale must be positive"):
            P.attention(q, k, k, plan, 64, scale)
        with pytest.raises(ValueError, match="scale must be positive"):
            P.attention_backward(q, k, k, q, q, lse, plan, 64, scale)
    for match, args in (("o and dout", (k, q, lse)), ("o and dout", (q, q.bfloat16(), lse)), ("lse must be", (q, q, lse[:1])), ("lse must be", (q, q, lse.double()))):
        with pytest.raises(ValueError, match=match):
            P.attention_backward(q, k, k, *args, plan, 64)
    for dqkv in (torch.zeros(8, 255), torch.zeros(8, 256, dtype=torch.bfloat16), torch.zeros(256, 8).t()):
        with pytest.raises(ValueError, match="dqkv must be"):
            P.attention_backward(q, k, k, q, q, lse, plan, 64, dqkv=dqkv)


def test_rotary_refusals():
    x, pos = torch.randn(4, 128), torch.zeros(2, 4, dtype=torch.int32)
    ok = dict(pair_axes=(0,) * 32, heads=2, head_dim=64, theta=THETA)
    for match, change in (("x must be", dict(heads=3)), ("x must be", dict(heads=0)), ("pairs of a head", dict(pair_axes=())), ("pairs of a head", dict(pair_axes=(0,) * 33)),
                          ("names axes", dict(pair_axes=(2,))), ("names axes", dict(pair_axes=(-1,))), ("theta must be", dict(theta=0.0)),
                          ("theta must be", dict(theta=math.nan)), ("out must be", dict(out=torch.zeros(4, 127))), ("out must be", dict(out=torch.zeros(4, 128).bfloat16())),
                          ("side by side", dict(out=torch.zeros(128, 4).t())), ("side by side", dict(out=torch.zeros(1, 128).expand(4, 128)))):
        with pytest.raises(ValueError, match=match):
            P.rotary(x, pos, **{**ok, **change})
    for bad in (pos.long(), pos[:, :3], pos[0], torch.zeros(9, 4, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32).t()):
        with pytest.raises(ValueError, match="positions must be"):
            P.rotary(x, bad, **ok)
    with pytest.raises(ValueError, match="x must be"):
        P.rotary(x.half(), pos, **ok)


def test_another_device_than_the_current_one(monkeypatch):
    """Kernels go to the current device's stream: tensors of another one are refused."""
    class Elsewhere:
        is_cuda, device = True, "cuda:1"

        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="the current device is cuda:0"):
        P._together("attention", Elsewhere(), Elsewhere())


@pytest.mark.parametrize("device", DEVICES)
def test_results_in_the_operands_memory(device):
    """Refused where it would be written before it is read; columns beside one another are no overlap."""
    plan = P.plan(torch.tensor([0, 6], dtype=torch.int32, device=device), 6)
    qkv = torch.randn(6, 192, device=device)
    q, k, v = torch.split(qkv, 64, 1)
    o, lse = P.attention(q, k, v, plan, 64, return_lse=True)
    with pytest.raises(ValueError, match="that of an operand"):
        P.attention_backward(q, k, v, o, o, lse, plan, 64, dqkv=qkv)
    pos = torch.zeros(1, 6, dtype=torch.int32, device=device)
    for bad in (qkv.reshape(-1)[64:64 + 5 * 192 + 64].as_strided((6, 64), (192, 1), 32), qkv.reshape(-1).as_strided((6, 64), (64, 1), 0)):
        with pytest.raises(ValueError, match="that of an operand"):
            P.rotary(qkv, pos, (0,) * 32, 1, 64, THETA, out=bad)
    want = P.rotary(qkv[:, :64], pos, (0,) * 32, 1, 64, THETA)
    assert torch.equal(P.rotary(qkv[:, :64], pos, (0,) * 32, 1, 64, THETA, out=qkv[:, 64:128]), want) and torch.equal(qkv[:, 64:128], want)


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    plan = P.plan(torch.tensor([0, 8], dtype=torch.int32, device="cuda"), 8)
    for dtype, hd in ((torch.bfloat16, 32), (torch.bfloat16, 96), (torch.bfloat16, 256), (torch.float32, 192)):
        q = torch.zeros(8, hd, dtype=dtype, device="cuda")
        with pytest.raises(ValueError, match="heads of"):
            P.attention(q, q, q, plan, hd)
    q = torch.zeros(8, 64, device="cuda")
    with pytest.raises(ValueError, match="tensors on"):
        P.attention(q, q.cpu(), q.cpu(), plan, 64)
    with pytest.raises(ValueError, match="tensors on"):
        P.attention(q.cpu(), q.cpu(), q.cpu(), plan, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_beyond_32_bits(dtype):
    """Sequences at the end of tensors of more than 2^31 elements: the bits of small ones."""
    hd, heads, lengths = 128, 16, [200, 30, 64, 300]
    width, n = 3 * heads * hd, sum(lengths)
    tokens = 2 ** 31 // width + n + 50
    q, k, v, dout = _inputs(lengths, heads, heads, hd, dtype, "cuda")
    small = torch.cat([q, k, v], 1)
    far = torch.full((tokens, width), math.nan, dtype=dtype, device="cuda")
    dfar = torch.full((tokens, heads * hd), math.nan, dtype=dtype, device="cuda")
    far[tokens - n:], dfar[tokens - n:] = small, dout
    starts, positions = _starts(lengths, "cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")[None]
    axes = (0,) * (hd // 2)
    P.rotary(far, positions, axes, 2 * heads, hd, THETA, out=far)
    small = torch.cat([P.rotary(small, positions[:, tokens - n:], axes, 2 * heads, hd, THETA), v], 1)
    assert torch.equal(far[tokens - n:], small)
    cols = [heads * hd] * 3
    want = _both(*torch.split(small, cols, 1), dout, starts, hd)
    got = _both(*torch.split(far, cols, 1), dfar, starts + (tokens - n), hd)
    for name, w in want.items():
        g = got[name]
        assert torch.equal(g[:, tokens - n:] if name == "lse" else g[tokens - n:], w), name
        rest = g[:, :tokens - n] if name == "lse" else g[:tokens - n]
        assert all((part == (-math.inf if name == "lse" else 0)).all() for part in rest.split(1 << 16)), name


@pytest.mark.gpu
@pytest.mark.parametrize("hd,hq,tiles,back", [(64, 1, 34001, True), (128, 2, 22001, False)])
def test_waits_for_a_sequence_that_takes_seconds(hd, hq, tiles, back):
    """A ragged sequence behind one of whole tiles that every CTA works on for longer than the 2 s that a wait for one block may take: the ragged one has the bits
    that it has alone, and the long one's last rows are those of the definition."""
    K.check_status()
    n, m = 128 * tiles, 200
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn(n + m, (hq + 2) * hd, generator=g, device="cuda").bfloat16()
    q, k, v = torch.split(qkv, [hq * hd, hd, hd], 1)
    v += 1                                                        # so that the means of millions of them are not 0
    plan, alone = P.plan(_starts([n, m], "cuda"), n + m), P.plan(_starts([m], "cuda"), m)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    o, lse = P.attention(q, k, v, plan, hd, return_lse=True)
    end.record()
    end.synchronize()
    K.check_status()
    assert begin.elapsed_time(end) > 2000
    short = [t[n:].contiguous() for t in (q, k, v)]
    want, want_lse = P.attention(*short, alone, hd, return_lse=True)
    assert torch.equal(o[n:], want) and torch.equal(lse[:, n:], want_lse)
    for i in (n - 1, n - 128, n - 129):
        x = (k[:i + 1].double() @ q[i].double().reshape(hq, hd).t()).t() * hd ** -0.5
        p = torch.softmax(x, -1)
        y = p @ v[:i + 1].double()
        # the result's rounding and the weights'; products added up in 32 bits sixteen keys at a time, 8 additions to a tile that may be cut off (2^-23), and the
        # weights a tile at a time
        bound = 2.0 ** -8 * y.abs() + (2.0 ** -8 + (128 + 17 * tiles) * 2.0 ** -24 + 2.0 ** -15) * (p @ v[:i + 1].double().abs())
        _close("o", o[i].reshape(hq, hd), y.cpu(), bound.cpu())
    if not back:
        return
    dout = torch.randn(n + m, hq * hd, generator=g, device="cuda").bfloat16()
    dqkv = torch.full_like(qkv, math.nan)
    P.attention_backward(q, k, v, o, dout, lse, plan, hd, dqkv=dqkv)
    K.check_status()
    assert bool(dqkv.isfinite().all())
    assert torch.equal(dqkv[n:], torch.cat(P.attention_backward(*short, want, dout[n:].contiguous(), want_lse, alone, hd), 1))


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_given_as_tensors(device):
    """A scale and a theta that are tensors are read at every call, not remembered by which tensor it was."""
    q, k, v, dout = _inputs([9, 3], 2, 1, 64, torch.float32, device)
    plan, pos = P.plan(_starts([9, 3], device), 12), torch.arange(12, dtype=torch.int32, device=device)[None]
    scale, theta = torch.tensor(0.125), torch.tensor(10000.0)
    for s, t in ((0.125, 10000.0), (0.5, 500.0)):
        scale.fill_(s), theta.fill_(t)
        o, lse = P.attention(q, k, v, plan, 64, scale, return_lse=True)
        want, want_lse = P.attention(q, k, v, plan, 64, s, return_lse=True)
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
        for a, b in zip(P.attention_backward(q, k, v, o, dout, lse, plan, 64, scale), P.attention_backward(q, k, v, o, dout, lse, plan, 64, s)):
            assert torch.equal(a, b)
        assert torch.equal(P.rotary(q, pos, (0,) * 32, 2, 64, theta), P.rotary(q, pos, (0,) * 32, 2, 64, t))
    for bad in (0.0, -1.0, math.inf, math.nan):
        scale.fill_(bad), theta.fill_(bad)
        with pytest.raises(ValueError, match="scale must be positive"):
            P.attention(q, k, v, plan, 64, scale)
        with pytest.raises(ValueError, match="theta must be positive"):
            P.rotary(q, pos, (0,) * 32, 2, 64, theta)
    assert torch.equal(P.rotary(q, pos, torch.zeros(32, dtype=torch.int64), 2, 64, 500.0), P.rotary(q, pos, (0,) * 32, 2, 64, 500.0))
    with pytest.raises(ValueError, match="whole numbers"):
        P.rotary(q, pos, tuple(torch.zeros(32, dtype=torch.int64)), 2, 64, 500.0)


@pytest.mark.parametrize("device", DEVICES)
def test_results_carry_no_graph(device):
    """Gradients are calls of their own: what the operators give back of tensors that ask for one has no history, on either path, and can be written in place."""
    q, k, v, dout = (t.detach().clone().requires_grad_(True) for t in _inputs([9, 3], 2, 1, 64, torch.float32, device))
    plan, pos = P.plan(_starts([9, 3], device), 12), torch.arange(12, dtype=torch.int32, device=device)[None]
    o, lse = P.attention(q, k, v, plan, 64, return_lse=True)
    turned = P.rotary(q, pos, (0,) * 32, 2, 64, THETA)
    grads = P.attention_backward(q, k, v, o, dout, lse, plan, 64)
    into = P.rotary(q, pos, (0,) * 32, 2, 64, THETA, out=torch.empty(12, 128, device=device))
    for t in (o, lse, turned, into, *grads):
        assert not t.requires_grad and t.grad_fn is None
    assert torch.equal(into, turned)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("within", [False, True])
def test_inference_mode(device, within):
    """Calls within inference mode, on tensors made there or before, give what they give elsewhere."""
    lengths = [9, 0, 70]
    q, k, v, dout = _inputs(lengths, 2, 1, 64, torch.float32, device)
    starts = _starts(lengths, device)
    want = _both(q, k, v, dout, starts, 64)
    with torch.inference_mode():
        args = [t.clone() for t in (q, k, v, dout, starts)] if within else [q, k, v, dout, starts]
        got = _both(*args, 64)
        assert all(torch.equal(got[n], want[n]) for n in want)
    got = _both(*args, 64)                                           # tensors of inference mode outside it
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,at", [(8, 5), (60, 33), (200, 70), (300, 299)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite_within_a_sequence(device, dtype, n, at, bad):
    """A query or a key that is not finite leaves the results of earlier tokens as they are; a value may reach any token of its sequence and always reaches its own, but
    none of another sequence."""
    q, k, v, _ = _inputs([4, n, 7], 2, 1, 64, dtype, device)
    plan = P.plan(_starts([4, n, 7], device), n + 11)
    want, want_lse = P.attention(q, k, v, plan, 64, return_lse=True)
    assert bool(want.isfinite().all())
    row = 4 + at
    for which in range(3):
        args = [t.clone() for t in (q, k, v)]
        args[which][row] = bad
        got, lse = P.attention(*args, plan, 64, return_lse=True)
        assert not bool(got[row].isfinite().any()) if which == 2 else not bool(got[row].isfinite().all())
        same = [slice(0, 4), slice(4 + n, None)] + ([slice(4, row)] if which < 2 else [])
        assert all(torch.equal(got[s], want[s]) for s in same)
        assert torch.equal(lse if which == 2 else lse[:, :row], want_lse if which == 2 else want_lse[:, :row])
        if which == 0:
            assert torch.equal(got[row + 1:], want[row + 1:])
