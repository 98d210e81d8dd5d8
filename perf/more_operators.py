"""The operators of training and scoring on packed sequences, measured: rotary positions with several axes, causal attention with grouped heads over
sequences of different lengths that lie one behind the other, and log-probabilities of given tokens with entropy and the likeliest alternatives.

Where `own` is false, `run` is plain torch in 32 bits (angles in 64); where it is true, the calls that a training or scoring program makes.  `exact`
states the same mathematics in 64 bits, its gradients by differentiation instead of by formula.  Head layouts are those of the configurations in
oa_b200/models (4 heads of 32 in fp32, 16 heads of 64, 32 heads of 128, 64 query over 8 key-value heads of 64) and a generic 32 over 8 of 128;
vocabularies theirs too.
"""
import math
import random

import torch

DEV = "cuda"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
THETA = 150000.0
IGNORED = -100

own = False


def listed():
    return [
        # the newest tokens of 32 conversations, query and key heads of one layer of the 7B-class model (the smallest call; latency counts)
        {"name": "rotary_decode_b32", "kind": "rotary", "dtype": "bf16", "tokens": 32, "heads": 64, "hd": 128, "axes": 3, "woven": False, "part": 1.0,
         "back": False},
        # gradients of the rotated heads of a packed batch of text and images, 64 over 8 heads of 64
        {"name": "rotary_images_back", "kind": "rotary", "dtype": "bf16", "tokens": 16381, "heads": 72, "hd": 64, "axes": 3, "woven": True, "part": 1.0,
         "back": True},
        # the fp32 character model: a training step's attention over 16 texts of up to 128 characters
        {"name": "attend_char_f32_step", "kind": "attend", "dtype": "f32", "step": True, "seqs": 16, "longest": 128, "q_heads": 4, "kv_heads": 4,
         "hd": 32, "pad": 0},
        # documents of up to 2048 tokens packed into a training step of the 350M model, one layer
        {"name": "attend_docs_step", "kind": "attend", "dtype": "bf16", "step": True, "seqs": 16, "longest": 2048, "q_heads": 16, "kv_heads": 16,
         "hd": 64, "pad": 0},
        # one whole prompt of the 7B-class model
        {"name": "attend_prompt_4096", "kind": "attend", "dtype": "bf16", "step": False, "seqs": 1, "longest": 4096, "q_heads": 32, "kv_heads": 32,
         "hd": 128, "pad": 0},
        # prompts of a busy server taken in together, ragged, 64 over 8 heads of 64, the batch padded behind them
        {"name": "attend_prompts_gqa", "kind": "attend", "dtype": "bf16", "step": False, "seqs": 8, "longest": 2000, "q_heads": 64, "kv_heads": 8,
         "hd": 64, "pad": 100},
        # long documents in a training step with grouped heads, odd lengths (the largest of attention)
        {"name": "attend_long_gqa_step", "kind": "attend", "dtype": "bf16", "step": True, "seqs": 6, "longest": 4001, "q_heads": 32, "kv_heads": 8,
         "hd": 128, "pad": 37},
        # a step over many short messages
        {"name": "attend_short_step", "kind": "attend", "dtype": "bf16", "step": True, "seqs": 512, "longest": 48, "q_heads": 16, "kv_heads": 16,
         "hd": 64, "pad": 0},
        # next characters of the character model, with four alternatives
        {"name": "logprob_char_b16", "kind": "logprob", "dtype": "f32", "rows": 16, "vocab": 256, "top": 4, "step": False},
        # the tokens just drawn for 32 conversations, with twenty alternatives, at the largest vocabulary of the configurations
        {"name": "logprob_decode_b32", "kind": "logprob", "dtype": "bf16", "rows": 32, "vocab": 201088, "top": 20, "step": False},
        # scoring a prompt of 4096 tokens with five alternatives
        {"name": "logprob_prompt_4096", "kind": "logprob", "dtype": "bf16", "rows": 4096, "vocab": 32000, "top": 5, "step": False},
        # a policy's training step: log-probabilities and entropy of 16384 tokens, and the gradient of the logits
        {"name": "logprob_policy_step", "kind": "logprob", "dtype": "bf16", "rows": 16384, "vocab": 32000, "top": 0, "step": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attend", "attend", "attend", "logprob", "logprob"])
    if kind == "rotary":
        heads, hd = rng.choice([(64, 128), (72, 64), (40, 128), (32, 64), (16, 64), (8, 32)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "tokens": _log(rng, 1, 16381 * 72 * 64 // (2 * heads * hd)), "heads": heads, "hd": hd,
                "axes": rng.choice([1, 2, 3, 3]), "woven": rng.choice([False, True]), "part": rng.choice([1.0, 1.0, 0.5]), "back": rng.choice([False, True])}
    if kind == "attend":
        q, kv, hd = rng.choice([(32, 32, 128), (64, 8, 64), (32, 8, 128), (16, 16, 64), (12, 4, 64), (4, 4, 32), (8, 2, 64)])
        dtype = "f32" if hd == 32 or (q, hd) == (8, 64) else "bf16"
        longest = _log(rng, 2, 512 if dtype == "f32" else 5000)
        room = 0.7 * _flops({"seqs": 6, "longest": 4001, "q_heads": 32, "hd": 128, "step": True}) / (40 if dtype == "f32" else 1)
        c = {"kind": kind, "dtype": dtype, "step": rng.choice([False, True]), "seqs": 1, "longest": longest, "q_heads": q, "kv_heads": kv, "hd": hd,
             "pad": rng.choice([0, rng.randint(1, 200)])}
        # the work of ragged lengths is a third, their tokens are half
        most = min(600, 3 * room // _flops(c), 2 * min(16000, 11400 * 40 * 128 // ((q + kv) * hd)) // longest)
        return {**c, "seqs": _log(rng, 1, max(1, most))}
    vocab = rng.choice([_log(rng, 64, 1000), 32000, 50257, _log(rng, 1000, 201088)])
    step, dtype = rng.choice([False, True]), rng.choice(["f32", "bf16"])
    top = rng.choice([0, rng.randint(1, 20), 20])
    most = 16384 * 32000 // (2 if dtype == "f32" else 1) // (4 if top else 1)
    return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, min(16384, most // vocab)), "vocab": vocab, "top": top, "step": step}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 7919 + salt) & 0x7FFFFFFF)


def _randn(g, *shape, std=1.0, dtype=BF):
    return torch.randn(shape, generator=g, device=DEV, dtype=F32).mul_(std).to(dtype)


def _dtype(case):
    return F32 if case["dtype"] == "f32" else BF


def _lengths(case):
    """Lengths of the sequences in rising order: all from short to `longest`, evenly."""
    n = case["seqs"]
    return [max(1, (i + 1) * case["longest"] // n) for i in range(n)]


def _pair_axes(case):
    """Which axis turns each pair of a head: time first, then height and width, in sections or woven one by one."""
    pairs, axes = int(case["hd"] // 2 * case["part"]), case["axes"]
    if case["woven"]:
        return tuple(j % axes for j in range(pairs))
    first = pairs if axes == 1 else pairs // 4 if axes == 3 else pairs // 2
    return tuple(0 if j < first else 1 + (j - first) * (axes - 1) // (pairs - first) for j in range(pairs))


def _positions(case, seed):
    """Text with images in it: text moves along all axes together, an image stands at one time and spans height and width."""
    n, axes = case["tokens"], case["axes"]
    rng = random.Random(seed * 31 + 5)
    runs, at, have = [], rng.randint(0, 100000), 0
    while have < n:
        if rng.random() < 0.5 or n < 64:
            m = min(n - have, rng.randint(1, 200))
            runs.append((at + torch.arange(m))[None].expand(3, m))
            at += m
        else:
            h, w = rng.randint(4, 40), rng.randint(4, 40)
            y, x = torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij")
            runs.append(torch.stack([torch.zeros(h * w, dtype=torch.int64), y.flatten(), x.flatten()]) + at)
            at += max(h, w)
        have += runs[-1].shape[1]
    return torch.cat(runs, 1)[:axes, :n].to(torch.int32).to(DEV).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "rotary":
        # the rotated heads are the first of a packed projection's rows
        s["x"] = _randn(g, case["tokens"], (case["heads"] + 8) * case["hd"], dtype=_dtype(case))
        s["positions"] = _positions(case, seed)
        return s
    if case["kind"] == "attend":
        hq, hk, hd = case["q_heads"], case["kv_heads"], case["hd"]
        lengths = _lengths(case)
        random.Random(seed * 17 + 3).shuffle(lengths)
        tokens = sum(lengths) + case["pad"]
        s["lengths"] = lengths
        s["starts"] = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(DEV)
        s["qkv"] = _randn(g, tokens, (hq + 2 * hk) * hd, dtype=_dtype(case))
        s["qkv"][:, :hq * hd] *= 1.5
        if case["step"]:
            s["dout"] = _randn(g, tokens, hq * hd, std=0.02, dtype=_dtype(case))
        if own:
            from oa_b200.ops import packed
            s["plan"] = packed.plan(s["starts"], tokens)
        return s
    rows, v = case["rows"], case["vocab"]
    s["logits"] = torch.empty((rows, v), dtype=_dtype(case), device=DEV)
    for at in range(0, rows, 2048):
        n = min(2048, rows - at)
        x = torch.randn((n, v), generator=g, device=DEV, dtype=F32).mul_(2.5)
        liked = torch.randint(0, v, (n, min(v, 24)), generator=g, device=DEV)
        x.scatter_add_(1, liked, torch.rand(liked.shape, generator=g, device=DEV) * 9)          # a few likely tokens, as a model has
        x[::7, v // 3:v // 2] = -math.inf                                                       # tokens that a grammar forbids
        s["logits"][at:at + n] = x
    targets = torch.randint(0, v, (rows,), generator=g, device=DEV)
    allowed = torch.where((targets >= v // 3) & (targets < v // 2), 0, targets)
    s["targets"] = torch.where(torch.arange(rows, device=DEV) % 11 == 5, IGNORED, allowed).to(torch.int32)      # a prompt's tokens do not count
    if case["step"]:
        s["dlogprobs"], s["dentropy"] = _randn(g, rows, dtype=F32), _randn(g, rows, std=0.01, dtype=F32)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"rotary": _rotary, "attend": _attend, "logprob": _logprob}[state["case"]["kind"]](state)


def _rotary(s):
    c = s["case"]
    heads, hd, axes = c["heads"], c["hd"], _pair_axes(c)
    if own:
        from oa_b200.ops import packed
        return packed.rotary(s["x"], s["positions"], axes, heads, hd, THETA, backward=c["back"])
    half = len(axes)
    x = s["x"][:, :heads * hd].float().view(c["tokens"], heads, hd)
    freq = torch.pow(torch.tensor(THETA, device=DEV, dtype=F64), torch.arange(half, device=DEV, dtype=F64) * (-1.0 / half))
    a = s["positions"].double()[list(axes)].t() * freq
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    if c["back"]:
        sin = -sin
    lo, hi = x[..., :half], x[..., half:2 * half]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 2 * half:]], -1).reshape(c["tokens"], heads * hd).to(s["x"].dtype)


def _split(s):
    c = s["case"]
    return torch.split(s["qkv"], [c["q_heads"] * c["hd"], c["kv_heads"] * c["hd"], c["kv_heads"] * c["hd"]], 1)


def _attend(s):
    c = s["case"]
    hq, hk, hd, tokens = c["q_heads"], c["kv_heads"], c["hd"], s["qkv"].shape[0]
    q, k, v = _split(s)
    if own:
        from oa_b200.ops import packed
        o, lse = packed.attention(q, k, v, s["plan"], hd, return_lse=True)
        return (o, *packed.attention_backward(q, k, v, o, s["dout"], lse, s["plan"], hd)) if c["step"] else (o, lse)
    dtype, scale = q.dtype, hd ** -0.5
    o, lse = torch.zeros_like(q, memory_format=torch.contiguous_format), torch.full((hq, tokens), -math.inf, device=DEV)
    dq, dk, dv = (torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    lo = 0
    for n in s["lengths"]:
        hi = lo + n
        qs = q[lo:hi].float().view(n, hk, hq // hk, hd).permute(1, 2, 0, 3)                     # [kv heads, queries of one, n, hd]
        ks, vs = (t[lo:hi].float().view(n, hk, 1, hd).permute(1, 2, 0, 3) for t in (k, v))
        x = torch.matmul(qs, ks.transpose(-1, -2)) * scale
        x = x.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - top)
        mass = p.sum(-1, keepdim=True)
        p = p / mass
        y = torch.matmul(p, vs)
        o[lo:hi] = y.permute(2, 0, 1, 3).reshape(n, hq * hd).to(dtype)
        lse[:, lo:hi] = (top + torch.log(mass)).reshape(hq, n)
        if c["step"]:
            dy = s["dout"][lo:hi].float().view(n, hk, hq // hk, hd).permute(1, 2, 0, 3)
            ds = p * (torch.matmul(dy, vs.transpose(-1, -2)) - (dy * y).sum(-1, keepdim=True)) * scale
            dq[lo:hi] = torch.matmul(ds, ks).permute(2, 0, 1, 3).reshape(n, hq * hd).to(dtype)
            dk[lo:hi] = torch.matmul(ds.transpose(-1, -2), qs).sum(1).permute(1, 0, 2).reshape(n, hk * hd).to(dtype)
            dv[lo:hi] = torch.matmul(p.transpose(-1, -2), dy).sum(1).permute(1, 0, 2).reshape(n, hk * hd).to(dtype)
        lo = hi
    return (o, dq, dk, dv) if c["step"] else (o, lse)


def _logprob(s):
    c = s["case"]
    if own:
        from oa_b200.ops import logprob
        r = logprob.token_logprobs(s["logits"], s["targets"], top=c["top"])
        out = (r.logprobs, r.entropy) + ((r.top_logprobs, r.top_ids) if c["top"] else ())
        return out + (logprob.token_logprobs_backward(s["logits"], s["targets"], r, s["dlogprobs"], s["dentropy"]),) if c["step"] else out
    x = s["logits"].float()
    y = x - x.amax(1, keepdim=True)
    w = torch.exp(y)
    mass = w.sum(1, keepdim=True)
    y = y - torch.log(mass)                                                                     # log-probabilities
    p = w / mass
    entropy = -torch.where(p > 0, p * y, 0.0).sum(1)
    counts = s["targets"] != IGNORED
    at = torch.where(counts, s["targets"], 0).long()[:, None]
    out = (torch.where(counts, y.gather(1, at)[:, 0], 0.0), entropy)
    if c["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
        out += (y.gather(1, ids), ids.to(torch.int32))
    if not c["step"]:
        return out
    g = torch.where(counts, s["dlogprobs"], 0.0)[:, None]
    d = -p * (g + s["dentropy"][:, None] * (torch.where(p > 0, y, 0.0) + entropy[:, None]))
    return out + (d.scatter_add_(1, at, g).to(s["logits"].dtype),)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _flops(c):
    """Of attention: two products of the pairs that are seen forward, five backward."""
    pairs = sum(n * (n + 1) // 2 for n in _lengths(c))
    return 2 * pairs * c["q_heads"] * c["hd"] * (7 if c["step"] else 2)


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "rotary":
        turned = c["tokens"] * c["heads"] * int(c["hd"] // 2 * c["part"])
        return {"bytes": 2 * size * c["tokens"] * c["heads"] * c["hd"] + 4 * c["tokens"] * c["axes"], "flops": 6 * turned}
    if c["kind"] == "attend":
        tokens, row = sum(_lengths(c)), size * c["hd"]
        q, kv = tokens * row * c["q_heads"], tokens * row * c["kv_heads"]
        # forward q, k, v, o; a step reads dO beside them and writes dQ, dK, dV
        return {"bytes": 2 * q + 2 * kv + ((2 * q + 2 * kv) if c["step"] else 4 * tokens * c["q_heads"]), "flops": _flops(c)}
    n = c["rows"] * c["vocab"]
    return {"bytes": size * n * (2 if c["step"] else 1) + c["rows"] * (12 + 8 * c["top"] + (8 if c["step"] else 0)), "flops": (9 if c["step"] else 4) * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "attend": _exact_attend, "logprob": _exact_logprob}[case["kind"]](s)


def _exact_rotary(s):
    c, axes = s["case"], _pair_axes(s["case"])
    half = len(axes)
    out = s["x"][:, :c["heads"] * c["hd"]].double().view(c["tokens"], c["heads"], c["hd"])
    for j, axis in enumerate(axes):
        turn = torch.polar(torch.ones(c["tokens"], device=DEV, dtype=F64), s["positions"][axis].double() * math.exp(-j / half * math.log(THETA)))
        z = torch.complex(out[..., j], out[..., j + half]) * (turn.conj() if c["back"] else turn)[:, None]
        out[..., j], out[..., j + half] = z.real, z.imag
    return out.reshape(c["tokens"], c["heads"] * c["hd"])


def _exact_attend(s):
    c = s["case"]
    hq, hk, hd, tokens = c["q_heads"], c["kv_heads"], c["hd"], s["qkv"].shape[0]
    outs = [torch.zeros(tokens, h * hd, device=DEV, dtype=F64) for h in (hq, hq, hk, hk)]        # o, dq, dk, dv
    lse = torch.full((hq, tokens), -math.inf, device=DEV, dtype=F64)
    per = max(1, min(hk, int(2e9) // (max(s["lengths"]) ** 2 * (hq // hk) * 8)))                 # key-value heads at a time
    for lo, n in zip([0] + torch.tensor(s["lengths"]).cumsum(0).tolist(), s["lengths"]):
        late = torch.arange(n, device=DEV)[None, :] > torch.arange(n, device=DEV)[:, None]
        for h in range(0, hk, per):
            m = min(per, hk - h)
            cols = [slice(h * hq // hk * hd, (h + m) * hq // hk * hd), slice(h * hd, (h + m) * hd), slice(h * hd, (h + m) * hd)]
            with torch.enable_grad():
                q, k, v = (t[lo:lo + n, w].double().view(n, -1, hd).requires_grad_(c["step"]) for t, w in zip(_split(s), cols))
                kk, vv = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
                x = (torch.einsum("ihd,jhd->hij", q, kk) / math.sqrt(hd)).masked_fill(late[None], -math.inf)
                y = torch.einsum("hij,jhd->ihd", torch.softmax(x, -1), vv)
                lse[h * hq // hk:(h + m) * hq // hk, lo:lo + n] = torch.logsumexp(x.detach(), -1)
                outs[0][lo:lo + n, cols[0]] = y.detach().reshape(n, -1)
                if c["step"]:
                    grads = torch.autograd.grad(y, (q, k, v), s["dout"][lo:lo + n, cols[0]].double().view(n, -1, hd))
                    for o, d, w in zip(outs[1:], grads, cols):
                        o[lo:lo + n, w] = d.reshape(n, -1)
    return tuple(outs) if c["step"] else (outs[0], lse)


def _exact_logprob(s):
    c = s["case"]
    rows, k = c["rows"], c["top"]
    parts = []
    for at in range(0, rows, max(1, int(5e7) // c["vocab"])):
        n = min(max(1, int(5e7) // c["vocab"]), rows - at)
        with torch.enable_grad():
            x = s["logits"][at:at + n].double().requires_grad_(c["step"])
            y = x - torch.logsumexp(x, 1, keepdim=True)
            counts = s["targets"][at:at + n] != IGNORED
            logp = y.gather(1, s["targets"][at:at + n].clamp(min=0).long()[:, None])[:, 0] * counts
            entropy = torch.special.entr(torch.softmax(x, 1)).sum(1) if not c["step"] else \
                -(torch.softmax(x, 1) * y.masked_fill(x == -math.inf, 0.0)).sum(1)
            out = [logp.detach(), entropy.detach()]
            if k:
                out.append(torch.sort(y.detach(), dim=1, descending=True).values[:, :k])
            if c["step"]:
                out.append(torch.autograd.grad((logp * s["dlogprobs"][at:at + n]).sum() + (entropy * s["dentropy"][at:at + n]).sum(), x)[0])
        parts.append(out)
    whole = [torch.cat([p[i] for p in parts]) for i in range(len(parts[0]))]
    if k:
        whole.insert(3, None)                                                                    # which alternatives: whole numbers
    return tuple(whole)
