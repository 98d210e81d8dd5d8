"""The paged cache's operators against plain statements in 64 bits: tables and slots, release, rotary append, attention behind a shared prompt.

Every check runs on the CPU path and, marked gpu, on the kernels."""
import math

import pytest
import torch

from oa_b200 import _native as N
from oa_b200.ops import paged as P

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------------ plan and release
def _plan_oracle(cached, fresh, tables, free, taken, ps, tokens, position0):
    """One token after the other, with a Python list as the stack."""
    tables = [list(r) for r in tables]
    width, stack = len(tables[0]) if tables else 0, list(free)
    top = taken
    slots, positions, rows, starts, lost = [], [], [], [0], 0
    for b, (c, f) in enumerate(zip(cached, fresh)):
        held = min(-(-c // ps), width)
        for at in range(c, c + f):
            j = at // ps
            if j >= held and j < width:                    # the first token of a page that the request does not hold
                tables[b][j] = stack[top] if top < len(stack) else -1
                top = min(top + 1, len(stack))
                held = j + 1
            page = tables[b][j] if j < width else -1
            slots.append(page * ps + at % ps if page >= 0 else -1)
            lost += page < 0
            positions.append(position0 + at)
            rows.append(b)
        starts.append(starts[-1] + f)
    pad = lambda v: (v + [-1] * tokens)[:tokens]  # noqa: E731
    return (starts, [min(c + f, width * ps) for c, f in zip(cached, fresh)], pad(slots), pad(positions), pad(rows), [top],
            [lost + max(0, starts[-1] - tokens)], tables)


PLANS = [
    # batch, page, width, most new, pages on the stack, room for tokens (more or less than the step has)
    (1, 16, 4, 1, 50, 0), (3, 16, 3, 40, 50, 5), (7, 128, 2, 200, 50, -9), (64, 32, 9, 3, 400, 0), (257, 16, 6, 20, 90, 3), (1100, 64, 3, 2, 3000, -1),
    (5, 16, 2, 90, 1000, 0), (4, 16, 3, 30, 0, 0), (2, 16, 0, 3, 10, 0),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batch,ps,width,most,stack,room", PLANS)
def test_plan(device, batch, ps, width, most, stack, room):
    g = torch.Generator().manual_seed(batch * 31 + ps)
    cached = torch.randint(0, max(1, width * ps), (batch,), generator=g).tolist()
    fresh = torch.randint(0, most + 1, (batch,), generator=g).tolist()
    if batch > 2:
        cached[0], fresh[1], cached[2] = 0, 0, ps * max(width - 1, 0)        # an empty request, one that adds nothing, one that ends at a page's end
    tables = [[b * 1000 + j if j < -(-c // ps) else -7 for j in range(width)] for b, c in enumerate(cached)]
    free = torch.randperm(stack, generator=g).tolist()
    taken = min(2, stack)
    tokens = max(0, sum(fresh) + room)
    want = _plan_oracle(cached, fresh, tables, free, taken, ps, tokens, 11)
    wide = torch.full((batch, width + 3), -9, dtype=torch.int32, device=device)          # a row stride of its own
    t = wide[:, :width]
    t.copy_(_i32(tables, device).reshape(batch, width))
    args = (_i32(cached, device), _i32(fresh, device), t, _i32(free, device), _i32([taken], device), ps, tokens)
    for _ in range(2):                                                                   # the same step again gives the same
        got = P.plan(*args, position0=11)
        for name, a, b in zip(P.PagedStep._fields, got, want):
            assert a.tolist() == b, name
        assert t.tolist() == want[-1]
        assert bool((wide[:, width:] == -9).all())


@pytest.mark.parametrize("device", DEVICES)
def test_plan_of_nothing(device):
    none = _i32([], device)
    got = P.plan(none, none, torch.zeros((0, 4), dtype=torch.int32, device=device), _i32([5, 6], device), _i32([1], device), 16, 3)
    assert got.starts.tolist() == [0] and got.slots.tolist() == [-1] * 3 and got.taken.tolist() == [1] and got.missing.tolist() == [0]


@pytest.mark.parametrize("device", DEVICES)
def test_pages_go_round(device):
    """Requests come and go: no page is held twice, and what is released is taken again."""
    g = torch.Generator().manual_seed(3)
    batch, width, ps, pages = 37, 5, 16, 120
    lens, tables = torch.zeros(batch, dtype=torch.int32, device=device), torch.full((batch, width), -1, dtype=torch.int32, device=device)
    free, taken = torch.randperm(pages, generator=g).to(torch.int32).to(device), _i32([0], device)
    for _ in range(12):
        fresh = torch.minimum(torch.randint(0, 30, (batch,), generator=g), width * ps - lens.cpu().long()).to(torch.int32).to(device)
        step = P.plan(lens, fresh, tables, free, taken, ps, 40 * batch)
        lens, taken = step.lens.clone(), step.taken
        if int(step.missing):
            assert int(taken) == pages
        held = [tables[b, j].item() for b in range(batch) for j in range(-(-int(lens[b]) // ps))]
        live = [i for i in held if i >= 0]
        assert len(set(live)) == len(live) and sorted(live + free[int(taken):].tolist()) == list(range(pages))
        done = torch.rand(batch, generator=g) < 0.4
        taken = P.release(done.to(device), lens, tables, free, taken, ps)
        assert bool((lens.cpu()[done] == 0).all())
        held = [tables[b, j].item() for b in range(batch) for j in range(-(-int(lens[b]) // ps))]
        live = [i for i in held if i >= 0]
        assert sorted(live + free[int(taken):].tolist()) == list(range(pages))


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,qh,kvh,hd,ps", [(1, 4, 4, 32, 16), (5, 6, 2, 64, 16), (33, 3, 1, 128, 64), (700, 8, 8, 16, 128), (2, 64, 8, 64, 32)])
@pytest.mark.parametrize("form", ["plain", "strided", "offset", "unrotated"])
def test_append(device, dtype, tokens, qh, kvh, hd, ps, form):
    g = torch.Generator().manual_seed(tokens + hd)
    theta = 0.0 if form == "unrotated" else 10000.0
    width = (qh + 2 * kvh) * hd
    x = torch.randn(tokens, width, generator=g).to(dtype)
    if form == "strided":
        base = torch.zeros(tokens, width + 16, dtype=dtype)
        base[:, :width] = x
        qkv = base.to(device)[:, :width]
    elif form == "offset":                                        # off 16 bytes: taken by way of a copy
        base = torch.zeros(tokens, width + 1, dtype=dtype)
        base[:, 1:] = x
        qkv = base.to(device)[:, 1:]
    else:
        qkv = x.to(device)
    pages = tokens // ps + 4
    both = torch.randn(pages, 2, kvh, ps, hd, generator=g).to(dtype)               # k and v side by side: a page stride
    pool = both.to(device)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g).to(torch.int32)
    slots = torch.randperm(pages * ps, generator=g)[:tokens].to(torch.int32)
    slots[0] = -1
    if tokens > 4:
        slots[3] = pages * ps                                     # not in the pool
    q = P.append(qkv, positions.to(device), slots.to(device), pool[:, 0], pool[:, 1], theta)
    xd = x.double().reshape(tokens, -1, hd)
    a = positions.double()[:, None] * theta ** (-torch.arange(hd // 2).double() * 2 / hd) if theta > 0 else torch.zeros(tokens, hd // 2).double()
    turn = torch.polar(torch.ones_like(a), a)[:, None] * torch.complex(xd[..., :hd // 2], xd[..., hd // 2:])
    r = torch.cat([turn.real, turn.imag], -1)
    # two products and a sum in fp32, cosine and sine within 2^-22 (position below 2^20 times a turn in 64 bits leaves 2^-33): 2^-20 of
    # what is turned, and the rounding of the result to bf16
    size = math.sqrt(2) * x.float().abs().max().item()
    tol = size * (2 ** -20 + (2 ** -8 if dtype == torch.bfloat16 else 0))
    assert q.shape == (tokens, qh * hd) and q.dtype == dtype
    assert (q.cpu().double() - r[:, :qh].reshape(tokens, -1)).abs().max().item() <= tol
    want_k, want_v = both[:, 0].double().transpose(1, 2).reshape(-1, kvh, hd).clone(), both[:, 1].transpose(1, 2).reshape(-1, kvh, hd).clone()
    ok = (slots >= 0) & (slots < pages * ps)
    want_k[slots[ok].long()] = r[ok, qh:qh + kvh]
    want_v[slots[ok].long()] = x.reshape(tokens, -1, hd)[ok, qh + kvh:]
    got = pool.cpu().transpose(2, 3).reshape(pages, 2, -1, kvh, hd)
    got_k, got_v = got[:, 0].reshape(-1, kvh, hd), got[:, 1].reshape(-1, kvh, hd)
    assert (got_k.double() - want_k).abs().max().item() <= tol
    assert torch.equal(got_v, want_v)                             # values go in as they are, and nothing else is touched
    rest = torch.ones(pages * ps, dtype=torch.bool)
    rest[slots[ok].long()] = False
    assert torch.equal(got_k[rest], both[:, 0].transpose(1, 2).reshape(-1, kvh, hd)[rest])


# ------------------------------------------------------------------------------------------------ attention
def _attention_oracle(q, k, v, tables, lens, starts, prefix_table, prefix_len, scale):
    """Row by row in 64 bits.  Also the bounds' ingredients: per row the largest |v| it sees and the largest sum of |q_d k_d| scale."""
    pages, kvh, ps, hd = k.shape
    tokens, qh = q.shape[0], q.shape[1] // hd
    o, lse = torch.zeros(tokens, qh, hd).double(), torch.full((tokens, qh), -math.inf).double()
    vmax, smax = torch.zeros(tokens, qh).double(), torch.zeros(tokens, qh).double()

    def key_rows(pool, table, n):
        return torch.stack([pool[table[s // ps], :, s % ps] for s in range(n)]).double() if n else torch.zeros(0, kvh, hd).double()

    for b in range(len(lens)):
        lo, hi = starts[b], starts[b + 1]
        for i in range(hi - lo):
            n = max(lens[b] - (hi - lo) + i + 1, 0)
            ks, vs = (torch.cat([key_rows(p, prefix_table, prefix_len), key_rows(p, tables[b], n)]).repeat_interleave(qh // kvh, 1) for p in (k, v))
            if ks.shape[0] == 0:
                continue
            qr = q[lo + i].double().reshape(qh, hd)
            x = torch.einsum("hd,shd->hs", qr, ks) * scale
            lse[lo + i] = torch.logsumexp(x, -1)
            o[lo + i] = torch.einsum("hs,shd->hd", torch.softmax(x, -1), vs)
            vmax[lo + i] = vs.abs().amax((0, 2))
            smax[lo + i] = torch.einsum("hd,shd->hs", qr.abs(), ks.abs()).amax(-1) * abs(scale)
    return o, lse, vmax, smax


def _bounds(dtype, hd, n, vmax, smax, lse):
    """A score is hd products and sums in fp32: off by at most (hd + 2) 2^-23 of the sum of their sizes (2^-23 where the tensor cores cut off
    instead of rounding), and so is its weight, relatively, with 2^-20 for the exponential, its argument and the factors between
    maxima, and n 2^-23 for the sums.  A result is an average of values with such weights, above and below the line.  bf16: weights
    are rounded to 2^-9 before they meet the values, and the result again."""
    rel = (hd + 2) * 2.0 ** -23 * smax + 2.0 ** -20 + n * 2.0 ** -23
    o = (2 * rel + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * vmax
    return o[..., None] + 1e-30, rel + 2.0 ** -22 * (lse.abs().nan_to_num(0, 0, 0) + 1)


def _check_attention(device, dtype, lens, fresh, qh, kvh, hd, ps, prefix_len, *, scale=None, room=0, max_fresh=None, form="plain", q_std=1.5, lse=True):
    g = torch.Generator().manual_seed(sum(lens) + hd + prefix_len + qh)
    batch, width = len(lens), max([-(-n // ps) for n in lens] + [1]) + 1
    pages = batch * width + -(-prefix_len // ps) + 2
    order = torch.randperm(pages, generator=g)
    tables, prefix_table = order[:batch * width].reshape(batch, width), order[batch * width:batch * width + -(-prefix_len // ps)]
    both = torch.randn(pages, 2, kvh, ps, hd, generator=g).to(dtype)
    # whatever no request may see is NaN or infinite: pages of nobody, places beyond a length, beyond the prompt's end
    seen = torch.zeros(pages, ps, dtype=torch.bool)
    for b in range(batch):
        for s in range(lens[b]):
            seen[tables[b, s // ps], s % ps] = True
    for s in range(prefix_len):
        seen[prefix_table[s // ps], s % ps] = True
    waste = torch.tensor([math.nan, math.inf, -math.inf])[torch.randint(0, 3, (pages, ps), generator=g)].to(dtype)
    both = torch.where(seen[:, None, None, :, None], both, waste[:, None, None, :, None])
    k, v = both[:, 0], both[:, 1]
    starts = [0]
    for f in fresh:
        starts.append(starts[-1] + f)
    tokens = starts[-1] + room
    q = (torch.randn(tokens, qh * hd, generator=g) * q_std).to(dtype)
    pool = both.to(device)
    kd, vd = (pool[:, 0], pool[:, 1]) if form != "plain" else (pool[:, 0].contiguous(), pool[:, 1].contiguous())
    qd = q.to(device)
    if form == "strided":                                        # a view of packed rows
        packed = torch.full((tokens, (qh + 2 * kvh) * hd), math.nan, dtype=dtype, device=device)
        packed[:, :qh * hd] = qd
        qd = packed[:, :qh * hd]
    elif form == "offset":
        packed = torch.zeros((tokens, qh * hd + 1), dtype=dtype, device=device)
        packed[:, 1:] = qd
        qd = packed[:, 1:]
    wide = torch.full((batch, width + 2), 1 << 30, dtype=torch.int32, device=device)
    wide[:, :width] = tables.to(torch.int32)
    most = max(fresh + [1]) if max_fresh is None else max_fresh
    got = P.attention(qd, kd, vd, wide[:, :width], _i32(lens, device), _i32(starts, device), most,
                      prefix_table.to(torch.int32).to(device) if prefix_len else None, prefix_len, scale, return_lse=lse)
    got, got_lse = got if lse else (got, None)
    assert got.shape == (tokens, qh * hd) and got.dtype == dtype
    sc = scale if scale is not None else hd ** -0.5
    o, want_lse, vmax, smax = _attention_oracle(q, k, v, tables.tolist(), lens, starts, prefix_table.tolist(), prefix_len, sc)
    bo, bl = _bounds(dtype, hd, prefix_len + max(lens + [0]), vmax, smax, want_lse)
    off = (got.cpu().double().reshape(tokens, qh, hd) - o).abs()
    assert bool((off <= bo).all()), f"worst {float((off / bo).max()):.3f} of the bound"
    if lse:
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(got_lse.cpu()), empty) and bool((got_lse.cpu()[empty] < 0).all())
        assert bool(((got_lse.cpu().double() - want_lse).abs()[~empty] <= bl[~empty]).all())


TYPES = [(torch.float32, 32), (torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 128)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,hd", TYPES)
@pytest.mark.parametrize("qh,kvh,ps", [(4, 4, 16), (8, 1, 32), (6, 2, 128), (5, 5, 64)])
@pytest.mark.parametrize("prefix", [0, 1, 37, 300])
def test_attention_one_token_each(device, dtype, hd, qh, kvh, ps, prefix):
    lens = [1, 16, 17, 63, 128, 129, 200, 2]
    _check_attention(device, dtype, lens, [1] * len(lens), qh, kvh, hd, ps, prefix)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("form", ["plain", "strided", "offset"])
def test_attention_several_tokens_each(device, dtype, hd, form):
    # new tokens alone, behind others, none at all, and rows of no request at the end
    _check_attention(device, dtype, [5, 140, 9, 130, 260, 33], [5, 3, 0, 130, 1, 33], 6, 2, hd, 16, 50, room=3, form=form)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_rows_that_see_nothing(device, dtype, hd):
    # requests of length 0 (their one row has no keys), and more new tokens than keys: the first rows see none
    _check_attention(device, dtype, [0, 3, 0, 40], [1, 5, 0, 2], 4, 2, hd, 16, 0)
    _check_attention(device, dtype, [0, 3, 0, 40], [1, 5, 0, 2], 4, 2, hd, 16, 20)
    _check_attention(device, dtype, [0], [0], 4, 4, hd, 16, 0, room=2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_scales_and_without_lse(device, dtype, hd):
    _check_attention(device, dtype, [70, 150], [1, 2], 4, 2, hd, 32, 129, scale=0.25, lse=False)
    _check_attention(device, dtype, [70, 150], [1, 2], 4, 2, hd, 32, 129, scale=-0.125)
    _check_attention(device, dtype, [70, 150], [1, 2], 4, 2, hd, 32, 129, scale=0.0)
    _check_attention(device, dtype, [70, 150], [1, 2], 4, 2, hd, 32, 129, q_std=12.0)      # one key takes nearly all


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_that_are_no_page_count_as_zeros(device, dtype):
    torch.manual_seed(0)
    k, v = torch.randn(6, 2, 16, 64).to(dtype).to(device), torch.randn(6, 2, 16, 64).to(dtype).to(device)
    q = torch.randn(2, 4 * 64).to(dtype).to(device)
    tables, lens, starts = _i32([[0, -1, 2], [3, 6, 1]], device), _i32([40, 48], device), _i32([0, 1, 2], device)
    got = P.attention(q, k, v, tables, lens, starts, 1)
    zero = torch.zeros(1, 2, 16, 64, dtype=dtype, device=device)
    want = P.attention(q, torch.cat([k, zero]), torch.cat([v, zero]), _i32([[0, 6, 2], [3, 6, 1]], device), lens, starts, 1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_tokens_beyond_max_fresh_are_rows_of_no_request(device):
    torch.manual_seed(0)
    k, v = torch.randn(4, 2, 16, 64).bfloat16().to(device), torch.randn(4, 2, 16, 64).bfloat16().to(device)
    q = torch.randn(5, 4 * 64).bfloat16().to(device)
    args = (k, v, _i32([[0, 1], [2, 3]], device), _i32([20, 9], device), _i32([0, 3, 5], device))
    whole, part = P.attention(q, *args, 3), P.attention(q, *args, 2)
    assert torch.equal(part[[0, 1, 3, 4]], whole[[0, 1, 3, 4]]) and bool((part[2] == 0).all())


@pytest.mark.gpu
def test_attention_past_32_bits():
    """Pages whose elements lie beyond 2^31 (and bytes beyond 2^32): a cache of 4.3 billion elements, of which only a few pages are touched."""
    hd, kvh, ps = 128, 8, 128
    pages = (1 << 32) // (kvh * ps * hd) + 64
    if torch.cuda.mem_get_info()[0] < 2 * pages * kvh * ps * hd * 2 + (4 << 30):
        pytest.skip("not enough memory")
    k, v = (torch.empty(pages, kvh, ps, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(0)
    used = [1, pages - 1, pages // 2 + 3, pages - 5]
    small_k, small_v = (torch.randn(4, kvh, ps, hd, generator=g).bfloat16().cuda() for _ in range(2))
    for i, pg in enumerate(used):
        k[pg], v[pg] = small_k[i], small_v[i]
    q = torch.randn(2, 16 * hd, generator=g).bfloat16().cuda()
    lens, starts = _i32([250, 130], "cuda"), _i32([0, 1, 2], "cuda")
    got = P.attention(q, k, v, _i32([used[:2], used[2:]], "cuda"), lens, starts, 1, _i32([used[1]], "cuda"), 100)
    want = P.attention(q, small_k, small_v, _i32([[0, 1], [2, 3]], "cuda"), lens, starts, 1, _i32([1], "cuda"), 100)
    assert torch.equal(got, want)
    x = torch.randn(3, 3 * kvh * hd, generator=g).bfloat16().cuda()
    slots = _i32([(pages - 2) * ps + 5, (pages - 1) * ps + 127, 7], "cuda")
    P.append(x, _i32([0, 0, 0], "cuda"), slots, k, v, 10000.0)
    at = slots.long()
    assert torch.equal(v[at // ps, :, at % ps], x.reshape(3, 3, kvh, hd)[:, 2]) and torch.equal(k[at // ps, :, at % ps], x.reshape(3, 3, kvh, hd)[:, 1])


@pytest.mark.gpu
def test_on_another_stream():
    torch.manual_seed(1)
    k, v = torch.randn(40, 4, 16, 64).bfloat16().cuda(), torch.randn(40, 4, 16, 64).bfloat16().cuda()
    q, tables = torch.randn(8, 8 * 64).bfloat16().cuda(), torch.randperm(40)[:32].reshape(8, 4).to(torch.int32).cuda()
    lens, starts = _i32([9, 20, 33, 64, 1, 50, 17, 48], "cuda"), _i32(list(range(9)), "cuda")
    want = P.attention(q, k, v, tables, lens, starts, 1, _i32([36, 37, 38], "cuda"), 41, return_lse=True)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in side:
            with torch.cuda.stream(s):
                got.append(P.attention(q, k, v, tables, lens, starts, 1, _i32([36, 37, 38], "cuda"), 41, return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    bf = torch.bfloat16
    plan = (z(3), z(3), z(3, 4), z(9), z(1))
    for bad in [(plan, 24, 5), ((z(3), z(2), *plan[2:]), 16, 5), ((z(3).long(), *plan[1:]), 16, 5), ((z(3), z(3), z(2, 4), z(9), z(1)), 16, 5),
                ((z(3), z(3), z(3, 4).t(), z(9), z(1)), 16, 5), (plan, 16, -1), ((*plan[:4], z(2)), 16, 5), ((*plan[:2], z(3, 4, dtype=torch.int64), *plan[3:]), 16, 5)]:
        with pytest.raises(ValueError):
            P.plan(*bad[0], *bad[1:])
    with pytest.raises(ValueError):
        P.release(z(3), z(3), z(3, 4), z(9), z(1), 16)
    with pytest.raises(ValueError):
        P.release(z(3, dtype=torch.bool), z(3), z(3, 4), z(9), z(1), 8)
    k, v = z(4, 2, 16, 64, dtype=bf), z(4, 2, 16, 64, dtype=bf)
    good = dict(qkv=z(3, 8 * 64, dtype=bf), positions=z(3), slots=z(3), k_pages=k, v_pages=v, theta=1e4)
    for bad in [dict(qkv=z(3, 8 * 64, dtype=torch.float32)), dict(positions=z(2)), dict(slots=z(3).long()), dict(qkv=z(3, 4 * 64, dtype=bf)),
                dict(qkv=z(3, 8 * 64 + 8, dtype=bf)), dict(k_pages=z(4, 2, 20, 64, dtype=bf), v_pages=z(4, 2, 20, 64, dtype=bf)),
                dict(v_pages=z(4, 2, 64, 16, dtype=bf).transpose(2, 3)), dict(v_pages=z(5, 2, 16, 64, dtype=bf))]:
        with pytest.raises(ValueError):
            P.append(**{**good, **bad})
    good = dict(q=z(3, 4 * 64, dtype=bf), k_pages=k, v_pages=v, tables=z(3, 2), lens=z(3), starts=z(4), max_fresh=1)
    for bad in [dict(q=z(3, 3 * 64, dtype=bf)), dict(q=z(3, 4, 64, dtype=bf)), dict(starts=z(3)), dict(lens=z(3).long()), dict(tables=z(2, 2)),
                dict(prefix_len=5), dict(prefix_len=17, prefix_table=z(1)), dict(prefix_len=-1), dict(max_fresh=-1), dict(q=z(3, 4 * 64, dtype=torch.float32)),
                dict(prefix_len=5, prefix_table=z(1).long())]:
        with pytest.raises(ValueError):
            P.attention(**{**good, **bad})


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    z = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="cpu"):
        P.plan(z(3), z(3), z(3, 4), torch.zeros(9, dtype=torch.int32), z(1), 16, 5)
    with pytest.raises(N.OaKernelError):                          # a batch beyond the kernel's prefix sums
        P.plan(z(20000), z(20000), z(20000, 1), z(9), z(1), 16, 5)
    for dtype, hd in ((torch.float16, 64), (torch.bfloat16, 48), (torch.bfloat16, 256)):
        pool = z(4, 2, 16, hd, dtype=dtype)
        with pytest.raises(N.OaKernelError):
            P.attention(z(3, 4 * hd, dtype=dtype), pool, pool, z(3, 2), z(3), z(4), 1)
    pool = z(4, 2, 16, 256, dtype=torch.bfloat16)
    with pytest.raises(N.OaKernelError):
        P.append(z(3, 8 * 256, dtype=torch.bfloat16), z(3), z(3), pool, pool, 1e4)
