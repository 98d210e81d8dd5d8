"""The operators that serve a batch of unequal requests, measured: building page tables and slot maps from request lengths, writing rotated
keys and values to pages, attention over a shared prompt and each request's own pages, and sampling the next tokens.

Where `own` is false, `run` is plain torch in 32 bits; where it is true, the calls that a serving program makes.  `exact` states the
same mathematics in 64 bits, request by request.  Head layouts are those of the models in oa_b200/models (32 heads of 128, 64 query over
8 key-value heads of 64, 4 heads of 32 in fp32) and a generic 32 over 8 of 128.
"""
import math

import torch

DEV = "cuda"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
MASS_BITS = 40          # a sampling weight of 1 is this power of two

own = False


def listed():
    return [
        # one decoding step of 64 conversations: every request adds one token, a few begin a page
        {"name": "plan_decode_b64", "kind": "plan", "batch": 64, "page": 16, "width": 256, "most": 1},
        # admission of 1024 prompts of all lengths at once, an offline batch
        {"name": "plan_prompts_b1024", "kind": "plan", "batch": 1024, "page": 64, "width": 64, "most": 512},
        # the new token of 32 conversations, one layer of the 7B-class model (latency counts)
        {"name": "append_decode_b32", "kind": "append", "tokens": 32, "q_heads": 32, "kv_heads": 32, "hd": 128, "page": 16},
        # prompts of many requests packed together, 64 query heads over 8 key-value heads, positions past 100000
        {"name": "append_prompts_gqa", "kind": "append", "tokens": 16381, "q_heads": 64, "kv_heads": 8, "hd": 64, "page": 64},
        # the fp32 character model: 16 rows behind a short shared prompt (the smallest call)
        {"name": "attend_char_f32", "kind": "attend", "dtype": "f32", "batch": 16, "most": 1, "q_heads": 4, "kv_heads": 4, "hd": 32,
         "prefix": 40, "own": 88, "page": 16},
        # four conversations of the 7B-class model behind a system prompt of 2048 tokens
        {"name": "attend_decode_b4", "kind": "attend", "dtype": "bf16", "batch": 4, "most": 1, "q_heads": 32, "kv_heads": 32, "hd": 128,
         "prefix": 2048, "own": 256, "page": 16},
        # batch-32 decoding of up to 256 tokens behind a prompt of 2048, the benchmark's generation at one layer
        {"name": "attend_decode_b32", "kind": "attend", "dtype": "bf16", "batch": 32, "most": 1, "q_heads": 32, "kv_heads": 32, "hd": 128,
         "prefix": 2048, "own": 256, "page": 64},
        # a busy server: 128 requests with histories of their own behind a long shared document of odd length
        {"name": "attend_decode_b128_gqa", "kind": "attend", "dtype": "bf16", "batch": 128, "most": 1, "q_heads": 64, "kv_heads": 8, "hd": 64,
         "prefix": 8191, "own": 2048, "page": 16},
        # several tokens for each request at once (prompt pieces, drafted tokens), ragged
        {"name": "attend_pieces_gqa", "kind": "attend", "dtype": "bf16", "batch": 24, "most": 24, "q_heads": 32, "kv_heads": 8, "hd": 128,
         "prefix": 1001, "own": 1500, "page": 32},
        # next characters of the character model
        {"name": "sample_char_b16", "kind": "sample", "dtype": "f32", "batch": 16, "vocab": 256},
        # next tokens of 32 conversations at the dense models' vocabulary
        {"name": "sample_b32_v32000", "kind": "sample", "dtype": "bf16", "batch": 32, "vocab": 32000},
        # a large batch at the largest vocabulary of the configurations, logits kept in fp32
        {"name": "sample_b256_v201088", "kind": "sample", "dtype": "f32", "batch": 256, "vocab": 201088},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "plan":
        batch = _log(rng, 1, 2048)
        most = rng.choice([1, _log(rng, 2, max(2, min(2000, 500000 // batch)))])
        return {"kind": kind, "batch": batch, "page": rng.choice([16, 32, 64, 128]), "width": _log(rng, 16, 256), "most": most}
    if kind == "append":
        q, kv, hd = rng.choice([(32, 32, 128), (64, 8, 64), (32, 8, 128), (16, 16, 64), (12, 4, 64)])
        return {"kind": kind, "tokens": _log(rng, 1, 16000 * 80 * 64 // ((q + 2 * kv) * hd)), "q_heads": q, "kv_heads": kv, "hd": hd,
                "page": rng.choice([16, 32, 64, 128])}
    if kind == "attend":
        q, kv, hd = rng.choice([(32, 32, 128), (64, 8, 64), (32, 8, 128), (16, 16, 64), (12, 4, 64), (4, 4, 32)])
        dtype = "f32" if hd == 32 else "bf16"
        batch = _log(rng, 1, 16 if dtype == "f32" else 128)
        prefix = rng.choice([0, _log(rng, 1, 200 if dtype == "f32" else 8192)])
        most = rng.choice([1, 1, rng.randint(2, 24)])
        room = 250e6 / (batch * kv * hd * 4)             # own keys and values at most those of the largest listed case
        length = _log(rng, 24, max(32, min(400 if dtype == "f32" else 2048, room)))
        if most > 1:
            batch = min(batch, 32)
        prefix = min(prefix, int(19e9 / (4 * batch * (most + 1) / 2 * q * hd)) - length)       # and its arithmetic
        prefix = max(0, prefix)
        return {"kind": kind, "dtype": dtype, "batch": batch, "most": most, "q_heads": q, "kv_heads": kv, "hd": hd, "prefix": prefix,
                "own": max(most, length), "page": rng.choice([16, 32, 64, 128])}
    vocab = rng.choice([_log(rng, 64, 1000), 32000, 50257, _log(rng, 1000, 201088)])
    return {"kind": "sample", "dtype": rng.choice(["f32", "bf16"]), "batch": _log(rng, 1, min(256, 40_000_000 // vocab)), "vocab": vocab}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 7919 + salt) & 0x7FFFFFFF)


def _randn(g, *shape, std=1.0, dtype=BF):
    return torch.randn(shape, generator=g, device=DEV, dtype=F32).mul_(std).to(dtype)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


def _fresh(g, batch, most):
    """New tokens of each request: 1 to `most`, all lengths alike, in any order."""
    return (torch.randperm(batch, generator=g, device=DEV) * most // batch + 1).to(torch.int32)


def _exclusive(x):
    return torch.cumsum(x, 0) - x


def _starts(fresh):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(fresh.long(), 0)]).to(torch.int32)


def _tokens(case):
    """Room for the tokens of a plan: what a program allows a step to have."""
    return case["batch"] * case["most"]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "plan":
        b, ps, w, most = case["batch"], case["page"], case["width"], case["most"]
        s["fresh"] = _fresh(g, b, most)
        s["cached"] = _ints(g, 0, max(1, w * ps - most), b) if most == 1 else _ints(g, 0, max(1, min(w * ps - most, 2 * ps)), b)
        have = (s["cached"].long() + ps - 1) // ps
        want = b * (most // ps + 2)
        pages = torch.randperm(int(have.sum()) + want + 8, generator=g, device=DEV).to(torch.int32)
        held = torch.arange(w, device=DEV)[None, :] < have[:, None]
        at = _exclusive(have)[:, None] + torch.arange(w, device=DEV)[None, :]
        s["tables"] = torch.where(held, pages[at.clamp(max=pages.numel() - 1)], -1).to(torch.int32)
        s["free"] = pages[int(have.sum()):].contiguous()
        s["taken"] = torch.full((1,), 3, dtype=torch.int32, device=DEV)
        return s
    if case["kind"] == "append":
        t, hq, hk, hd, ps = case["tokens"], case["q_heads"], case["kv_heads"], case["hd"], case["page"]
        s["qkv"] = _randn(g, t, (hq + 2 * hk) * hd)
        pages = (t + ps - 1) // ps + 16
        s["k_pages"], s["v_pages"] = _randn(g, pages, hk, ps, hd), _randn(g, pages, hk, ps, hd)
        s["slots"] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).repeat_interleave(ps)[:t] * ps \
            + torch.arange(t, device=DEV, dtype=torch.int32) % ps if t > 512 else torch.randperm(pages * ps, generator=g, device=DEV)[:t].to(torch.int32)
        s["slots"] = s["slots"].contiguous()
        s["positions"] = _ints(g, 0, 131072, t)
        return s
    if case["kind"] == "attend":
        dtype = F32 if case["dtype"] == "f32" else BF
        b, most, hq, hk, hd, ps = case["batch"], case["most"], case["q_heads"], case["kv_heads"], case["hd"], case["page"]
        w = -(-case["own"] // ps)
        fresh = _fresh(g, b, most)
        s["starts"] = _starts(fresh)
        s["lens"] = torch.maximum(_ints(g, 1, case["own"] + 1, b), fresh)
        p_pages = -(-case["prefix"] // ps)
        pages = torch.randperm(b * w + p_pages, generator=g, device=DEV).to(torch.int32)
        s["tables"] = pages[:b * w].reshape(b, w).contiguous()
        s["prefix_table"] = pages[b * w:].contiguous()
        s["q"] = _randn(g, int(s["starts"][-1]), hq * hd, std=1.5, dtype=dtype)
        s["k_pages"], s["v_pages"] = (_randn(g, b * w + p_pages, hk, ps, hd, dtype=dtype) for _ in range(2))
        return s
    b, v = case["batch"], case["vocab"]
    x = torch.randn((b, v), generator=g, device=DEV, dtype=F32).mul_(2.5)
    liked = torch.randint(0, v, (b, min(v, 24)), generator=g, device=DEV)
    x.scatter_add_(1, liked, torch.rand(liked.shape, generator=g, device=DEV) * 9)      # a few likely tokens, as a model has
    s["logits"] = x.to(F32 if case["dtype"] == "f32" else BF)
    s["u"] = torch.rand(b, generator=g, device=DEV)
    # five kinds of requests in turn: plain, top-k, top-p, all three, greedy
    row = torch.arange(b, device=DEV) % 5
    pick = lambda *v: torch.tensor(v, device=DEV)[row]  # noqa: E731
    s["temperature"] = pick(1.0, 0.7, 0.9, 1.2, 0.0)
    s["top_k"] = pick(0, 50, 0, 200, 0).to(torch.int32)
    s["top_p"] = pick(1.0, 1.0, 0.9, 0.95, 1.0)
    s["min_p"] = pick(0.0, 0.0, 0.0, 0.02, 0.0)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"plan": _plan, "append": _append, "attend": _attend, "sample": _sample}[state["case"]["kind"]](state)


def _plan(s):
    c = s["case"]
    if own:
        from oa_b200.ops import paged
        p = paged.plan(s["cached"], s["fresh"], s["tables"], s["free"], s["taken"], c["page"], _tokens(c), position0=100)
        return p.starts, p.lens, p.slots, p.positions, p.rows, p.taken, p.missing, s["tables"]
    ps, w, cap = c["page"], c["width"], _tokens(c)
    cached, fresh, free = s["cached"].long(), s["fresh"].long(), s["free"]
    old, new = ((cached + ps - 1) // ps).clamp(max=w), ((cached + fresh + ps - 1) // ps).clamp(max=w)
    need = (new - old).clamp(min=0)
    first = s["taken"].long() + _exclusive(need)
    j = torch.arange(w, device=DEV)[None, :]
    at = first[:, None] + j - old[:, None]
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    s["tables"].copy_(torch.where((j >= old[:, None]) & (j < new[:, None]), page, s["tables"]))
    total = torch.cumsum(fresh, 0)
    t = torch.arange(cap, device=DEV)
    row = torch.searchsorted(total, t, right=True)
    there, row = row < c["batch"], row.clamp(max=c["batch"] - 1)
    at = cached[row] + t - (total - fresh)[row]
    page = s["tables"][row, (at // ps).clamp(max=w - 1)].long()
    fits = there & (at // ps < w) & (page >= 0)
    slots = torch.where(fits, page * ps + at % ps, -1)
    got = torch.minimum(fresh, (old + (free.numel() - first).clamp(min=0).minimum(need)) * ps - cached).clamp(min=0)
    missing = (fresh - got).sum() + (total[-1] - cap).clamp(min=0)
    i32 = torch.int32
    return (torch.cat([total[:1] * 0, total]).to(i32), (cached + fresh).clamp(max=w * ps).to(i32), slots.to(i32), torch.where(there, at + 100, -1).to(i32),
            torch.where(there, row, -1).to(i32), (s["taken"] + need.sum()).clamp(max=free.numel()).to(i32), missing.reshape(1).to(i32), s["tables"])


THETA = 150000.0


def _append(s):
    c = s["case"]
    hq, hk, hd, ps = c["q_heads"], c["kv_heads"], c["hd"], c["page"]
    if own:
        from oa_b200.ops import paged
        return paged.append(s["qkv"], s["positions"], s["slots"], s["k_pages"], s["v_pages"], THETA), s["k_pages"], s["v_pages"]
    x = s["qkv"].float().view(c["tokens"], hq + 2 * hk, hd)
    a = s["positions"].float()[:, None] * torch.pow(THETA, torch.arange(hd // 2, device=DEV).float() * (-2.0 / hd))
    cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]
    lo, hi = x[:, :hq + hk, :hd // 2], x[:, :hq + hk, hd // 2:]
    r = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(BF)
    slots = s["slots"].long()
    s["k_pages"][slots // ps, :, slots % ps] = r[:, hq:]
    s["v_pages"][slots // ps, :, slots % ps] = x[:, hq + hk:].to(BF)
    return r[:, :hq].reshape(c["tokens"], hq * hd), s["k_pages"], s["v_pages"]


def _attend(s):
    c = s["case"]
    if own:
        from oa_b200.ops import paged
        return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["starts"], c["most"], s["prefix_table"], c["prefix"],
                               return_lse=True)
    b, most, hq, hk, hd, ps = c["batch"], c["most"], c["q_heads"], c["kv_heads"], c["hd"], c["page"]
    g, tokens = hq // hk, s["q"].shape[0]
    starts, lens = s["starts"].long(), s["lens"].long()
    fresh = starts[1:] - starts[:-1]
    # requests side by side, each with `most` rows
    row = starts[:-1, None] + torch.arange(most, device=DEV)[None, :]
    live = torch.arange(most, device=DEV)[None, :] < fresh[:, None]
    q = s["q"].float().view(tokens, hk, g, hd)[row.clamp(max=tokens - 1)] / math.sqrt(hd)          # [b, most, hk, g, hd]
    own_len = s["tables"].shape[1] * ps

    def pages(p, table):                                                                            # [..., keys, hk, hd]
        return p[table.long()].float().transpose(-3, -2).flatten(-4, -3)

    k, v = pages(s["k_pages"], s["tables"]), pages(s["v_pages"], s["tables"])
    seen = torch.arange(own_len, device=DEV)[None, None, :] <= (lens - fresh)[:, None, None] + torch.arange(most, device=DEV)[None, :, None]
    x = torch.einsum("bnhgd,bshd->bhgns", q, k).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1)
    if c["prefix"]:
        pk, pv = (pages(s[n], s["prefix_table"])[:c["prefix"]] for n in ("k_pages", "v_pages"))
        y = torch.einsum("bnhgd,shd->bhgns", q, pk)
        top = torch.maximum(top, y.amax(-1))
    x = torch.exp(x - top[..., None])
    mass = x.sum(-1)
    o = torch.einsum("bhgns,bshd->bnhgd", x, v)
    if c["prefix"]:
        y = torch.exp(y - top[..., None])
        mass = mass + y.sum(-1)
        o = o + torch.einsum("bhgns,shd->bnhgd", y, pv)
    o = (o / mass.permute(0, 3, 1, 2)[..., None])[live].reshape(tokens, hq * hd).to(s["q"].dtype)
    return o, (top + torch.log(mass)).permute(0, 3, 1, 2)[live].reshape(tokens, hq)


def _sample(s):
    if own:
        from oa_b200.ops import sampling
        return sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    x = s["logits"].float()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    y = (x - x[:, :1]) * (1.0 / torch.where(greedy, 1.0, s["temperature"]))[:, None]
    w = torch.exp(y)
    mass = (w * float(1 << MASS_BITS)).long()
    keep = torch.arange(vocab, device=DEV)[None, :] < torch.where(s["top_k"] > 0, s["top_k"], vocab).long()[:, None]
    mass = mass * keep
    total = mass.sum(1)
    before = torch.cumsum(mass, 1) - mass
    keep = keep & ((before.double() < (s["top_p"].double() * total.double())[:, None]) | (s["top_p"] >= 1)[:, None])
    keep[:, 0] = True
    keep = keep & (w >= s["min_p"].clamp(max=1)[:, None])
    mass = torch.zeros_like(mass).scatter_(1, order, mass * keep)                                  # back in the vocabulary's order
    total = mass.sum(1)
    at = torch.minimum((s["u"].double() * total.double()).long(), total - 1)
    token = torch.searchsorted(torch.cumsum(mass, 1), at[:, None], right=True)[:, 0]
    token = torch.where(greedy, order[:, 0], token)
    chosen = torch.zeros_like(y).scatter_(1, order, y).gather(1, token[:, None])[:, 0]
    logprob = chosen - torch.log(total.double() / float(1 << MASS_BITS)).float()
    return token.to(torch.int32), torch.where(greedy, 0.0, logprob)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _mean_own(c):
    """Mean length of a request's own part, as prepare() makes them."""
    return (c["own"] + 1) / 2


def work(case):
    c = case
    if c["kind"] == "plan":
        tokens = c["batch"] * (c["most"] + 1) / 2
        return {"bytes": 16 * c["batch"] + 8 * tokens / c["page"] + 12 * _tokens(c), "flops": 4 * tokens}
    if c["kind"] == "append":
        row = (c["q_heads"] + 2 * c["kv_heads"]) * c["hd"]
        return {"bytes": c["tokens"] * (2 * 2 * row + 8), "flops": c["tokens"] * 3 * (c["q_heads"] + c["kv_heads"]) * c["hd"]}
    if c["kind"] == "attend":
        size, tokens = (4 if c["dtype"] == "f32" else 2), c["batch"] * (c["most"] + 1) / 2
        keys = c["prefix"] + c["batch"] * _mean_own(c)
        return {"bytes": size * (2 * tokens * c["q_heads"] * c["hd"] + 2 * keys * c["kv_heads"] * c["hd"]) + 4 * tokens * c["q_heads"],
                "flops": 4 * tokens * c["q_heads"] * c["hd"] * (c["prefix"] + _mean_own(c))}
    return {"bytes": c["batch"] * (c["vocab"] * (4 if c["dtype"] == "f32" else 2) + 28), "flops": 4 * c["batch"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": lambda s: None, "append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _exact_append(s):
    c = s["case"]
    hq, hk, hd, ps = c["q_heads"], c["kv_heads"], c["hd"], c["page"]
    x = s["qkv"].double().view(c["tokens"], hq + 2 * hk, hd)
    turn = torch.polar(torch.ones(c["tokens"], hd // 2, device=DEV, dtype=F64),
                       s["positions"].double()[:, None] * torch.exp(torch.arange(hd // 2, device=DEV, dtype=F64) * (-2.0 / hd * math.log(THETA))))
    z = torch.complex(x[:, :hq + hk, :hd // 2], x[:, :hq + hk, hd // 2:]) * turn[:, None]
    r = torch.cat([z.real, z.imag], -1)
    out = []
    for pool, new in ((s["k_pages"], r[:, hq:]), (s["v_pages"], x[:, hq + hk:])):
        flat = pool.double().transpose(1, 2).reshape(-1, hk, hd)
        flat[s["slots"].long()] = new
        out.append(flat.reshape(pool.shape[0], ps, hk, hd).transpose(1, 2).contiguous())
    return r[:, :hq].reshape(c["tokens"], hq * hd), out[0], out[1]


def _exact_attend(s):
    c = s["case"]
    hq, hk, hd = c["q_heads"], c["kv_heads"], c["hd"]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    flat = [s[n].transpose(1, 2).reshape(-1, hk, hd) for n in ("k_pages", "v_pages")]                # by slot
    step = torch.arange(c["page"], device=DEV)
    shared = (s["prefix_table"].long()[:, None] * c["page"] + step).flatten()[:c["prefix"]]
    o = torch.zeros(s["q"].shape[0], hq, hd, device=DEV, dtype=F64)
    lse = torch.zeros(s["q"].shape[0], hq, device=DEV, dtype=F64)
    for b in range(c["batch"]):
        lo, hi = starts[b], starts[b + 1]
        slots = torch.cat([shared, (s["tables"][b].long()[:, None] * c["page"] + step).flatten()[:lens[b]]])
        k, v = (f[slots].double().repeat_interleave(hq // hk, 1) for f in flat)
        x = torch.einsum("nhd,shd->hns", s["q"][lo:hi].double().view(hi - lo, hq, hd), k) * hd ** -0.5
        late = torch.arange(slots.numel(), device=DEV)[None, :] > slots.numel() - (hi - lo) + torch.arange(hi - lo, device=DEV)[:, None]
        x = x.masked_fill(late[None], -math.inf)
        lse[lo:hi] = torch.logsumexp(x, -1).t()
        o[lo:hi] = torch.einsum("hns,shd->nhd", torch.softmax(x, -1), v)
    return o.reshape(-1, hq * hd), lse


def _exact_sample(s):
    logprobs = []
    for r in range(s["case"]["batch"]):
        t, k, p, least, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t <= 0:
            logprobs.append(torch.zeros((), device=DEV, dtype=F64))
            continue
        x = s["logits"][r].float()
        y = ((x - x.max()) * (1.0 / s["temperature"][r])).double()                                  # its rounding to 32 bits is part of the definition
        w, order = y.exp(), torch.argsort(x, descending=True, stable=True)
        n = min(int(k), x.numel()) if k > 0 else x.numel()
        cum = w[order[:n]].cumsum(0)
        if p < 1:
            n = max(1, int((cum - w[order[:n]] < p * cum[-1]).sum()))
        kept = torch.zeros_like(w)
        kept[order[:n]] = w[order[:n]]
        kept[w < least] = 0
        cum = kept.cumsum(0)
        token = min(int((cum <= u * cum[-1]).sum()), x.numel() - 1)
        logprobs.append(y[token] - cum[-1].log())
    return None, torch.stack(logprobs)
