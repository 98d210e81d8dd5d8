"""Decoding for a batch of requests of unequal length behind a prompt that they share, with the keys and values in pages.

The reference generates for one text at a time by re-running its whole window (Tutorial/Cpp/Ml/Nlp/TutorialNlpCommon.h:145-177).  Here a
step takes whatever new tokens the requests have, one each or whole prompts, in one pass: room in the pages (`paged.plan`), rotation and
append (`paged.append`), attention over the shared prompt and each request's own pages (`paged.attention`), and the next tokens
(`sampling.sample`).  Pages, lengths and tables stay on the device; a step of one token each is a CUDA graph.

    dec = OaBatchDecoder(model, batch=8, max_tokens=512)
    dec.SetPrompt(system_prompt)                      # once: its keys and values are kept once for all requests
    texts = dec.Generate([[1, 2, 3], [4]], new_tokens=64, stop=0)
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from ..core import fn_matrix as F
from ..core.matrix import OaMatrix
from ..ml import autograd as AG
from ..models.gpt import OaGptModel
from ..ops import kernels as K
from ..ops import paged, sampling
from .decoder import block_tail


@dataclass
class OaSampling:
    """How a request's tokens are drawn: see `sampling.sample`.  The default takes the likeliest token."""
    Temperature: float = 0.0
    TopK: int = 0
    TopP: float = 1.0
    MinP: float = 0.0


class OaPagedCache:
    """Keys and values of every layer in pages [2, pages, heads, page_size, head_dim], and what says whose they are (all on the device): the
    requests' tables and lengths, the stack of free pages, and the table of the prompt that they share."""

    def __init__(self, layers: int, batch: int, heads: int, head_dim: int, pages: int, page_size: int, max_tokens: int, max_prompt: int, dtype, device):
        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        self.Layers = [torch.zeros((2, pages, heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(layers)]
        self.PageSize, self.Pages, self.Batch = page_size, pages, batch
        self.Tables, self.Lens = ints(batch, -(-max_tokens // page_size), value=-1), ints(batch)
        self.PromptTable, self.PromptLens = ints(1, max(-(-max_prompt // page_size), 1), value=-1), ints(1)
        self.Free, self.Taken = torch.arange(pages, dtype=torch.int32, device=device), ints(1)
        self.MaxTokens, self.MaxPrompt = max_tokens, max_prompt
        # what the host knows of it: tokens of each request, of the prompt, and pages in use
        self.Held, self.PromptLen, self.Used = [0] * batch, 0, 0

    def Bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.Layers)

    def Room(self, held: Sequence[int], fresh: Sequence[int], limit: int) -> int:
        """The pages that `fresh` more tokens take; raises where there is no room for them."""
        need = 0
        for b, (h, f) in enumerate(zip(held, fresh)):
            if h + f > limit:
                raise ValueError(f"request {b}: {h + f} tokens, {limit} is the most")
            need += -(-(h + f) // self.PageSize) - -(-h // self.PageSize)
        if self.Used + need > self.Pages:
            raise ValueError(f"no room: {need} pages wanted, {self.Pages - self.Used} of {self.Pages} are free")
        return need


class OaBatchDecoder:
    def __init__(self, model: OaGptModel, batch: int, max_tokens: int, max_prompt: int = 0, pages: Optional[int] = None, page_size: int = 64,
                 seed: int = 0, use_graph: bool = True):
        """`max_tokens`: of a request's own, prompt and generated; `max_prompt`: of the shared prompt; `pages`: by default enough for all."""
        c = model.Cfg
        w = model.Embed.Weight.Tensor()
        if batch < 1 or max_tokens < 1:
            raise ValueError("OaBatchDecoder: batch and max_tokens must be positive")
        if model.PosEmbed is not None and max_tokens + max_prompt > c.SeqLen:
            raise ValueError(f"OaBatchDecoder: {max_prompt} + {max_tokens} tokens, but the model has {c.SeqLen} positions")
        if page_size not in paged.PAGE_SIZES:
            raise ValueError(f"OaBatchDecoder: a page holds one of {paged.PAGE_SIZES} tokens, not {page_size}")
        if w.is_cuda and c.DModel // c.NHeads not in paged.HEAD_DIMS:
            raise ValueError(f"OaBatchDecoder: heads of one of {paged.HEAD_DIMS}, not of {c.DModel // c.NHeads}")
        if pages is None:
            pages = batch * -(-max_tokens // page_size) + -(-max_prompt // page_size)
        self.Model, self.Cfg, self.Batch = model, c, batch
        self.Cache = OaPagedCache(c.NLayers, batch, c.NHeads, c.DModel // c.NHeads, pages, page_size, max_tokens, max_prompt, w.dtype, w.device)
        self.Logits: Optional[torch.Tensor] = None        # [batch, vocab] of the newest token of each request in the last step; rows of requests without one mean nothing
        self.LogProbs: Optional[torch.Tensor] = None      # [batch] of the tokens that the last step drew, likewise
        self._random = torch.Generator(device=w.device)
        self._random.manual_seed(seed)
        self._ids = torch.zeros(batch, dtype=torch.int32, device=w.device)
        self._fresh = torch.zeros(batch, dtype=torch.int32, device=w.device)
        self._u = torch.zeros(batch, dtype=torch.float32, device=w.device)
        self._temperature, self._top_p, self._min_p = torch.zeros_like(self._u), torch.ones_like(self._u), torch.zeros_like(self._u)
        self._top_k = torch.zeros_like(self._ids)
        self._may_record = use_graph and w.is_cuda and w.dtype == torch.bfloat16
        self._graph: Optional[torch.cuda.CUDAGraph] = None
        self._steps = 0                                   # of one token each, with what a graph would hold as it is now

    def SetSampling(self, how: Sequence[OaSampling]) -> None:
        """How the tokens of each request are drawn, from the next step on."""
        if len(how) != self.Batch:
            raise ValueError(f"SetSampling: {self.Batch} requests, {len(how)} settings")
        for to, name in ((self._temperature, "Temperature"), (self._top_k, "TopK"), (self._top_p, "TopP"), (self._min_p, "MinP")):
            to.copy_(torch.tensor([getattr(s, name) for s in how], dtype=to.dtype))

    def SetPrompt(self, ids: Sequence[int]) -> None:
        """The prompt that all requests share (none: an empty one), in place of the one before; no request may be under way.  Should it fail once the
        pages of the one before are given back, there is no prompt."""
        c = self.Cache
        if any(c.Held):
            raise ValueError("SetPrompt: requests are under way")
        held = -(-c.PromptLen // c.PageSize)
        c.Used -= held
        try:
            need = c.Room([0], [len(ids)], c.MaxPrompt)
        finally:
            c.Used += held
        c.Taken.copy_(paged.release(torch.ones(1, dtype=torch.bool, device=c.Lens.device), c.PromptLens, c.PromptTable, c.Free, c.Taken, c.PageSize))
        c.PromptLen = 0
        c.Used -= held
        self._graph, self._steps = None, 0
        if not len(ids):
            return
        t = torch.tensor(list(ids), dtype=torch.int32, device=c.Lens.device)
        with AG.OaGradNo():
            step = paged.plan(c.PromptLens, torch.full_like(c.PromptLens, len(ids)), c.PromptTable, c.Free, c.Taken, c.PageSize, len(ids))
            self._layers(t, step, c.PromptTable, len(ids), 0)
            self._keep(step, c.PromptLens)
        c.Used += need
        c.PromptLen = len(ids)

    def Release(self, requests: Sequence[int]) -> None:
        """Forgets these requests; their pages are free for others."""
        c, requests = self.Cache, list(requests)
        done = torch.zeros(self.Batch, dtype=torch.bool)
        done[requests] = True
        c.Taken.copy_(paged.release(done.to(c.Lens.device), c.Lens, c.Tables, c.Free, c.Taken, c.PageSize))
        for b in requests:
            c.Used -= -(-c.Held[b] // c.PageSize)
            c.Held[b] = 0

    def Feed(self, new: Sequence[Sequence[int]]) -> torch.Tensor:
        """New tokens of each request (of some none): the token that comes next, int32 [batch], -1 where there was nothing new."""
        if len(new) != self.Batch or not any(len(n) for n in new):
            raise ValueError(f"Feed: new tokens of {self.Batch} requests expected, at least one in all")
        counts = [len(n) for n in new]
        need = self.Cache.Room(self.Cache.Held, counts, self.Cache.MaxTokens)
        flat = torch.tensor([t for n in new for t in n], dtype=torch.int32, device=self._ids.device)
        return self._take(counts, need, lambda: self._step(flat, max(counts), False))

    def Step(self, ids: torch.Tensor, active: Optional[Sequence[bool]] = None) -> torch.Tensor:
        """One more token ids[b] (on the device) of each active request (default: of all): the tokens that come next, int32 [batch], -1 for the others.
        Where the step is a graph the result is overwritten by the next one."""
        if ids.numel() != self.Batch:
            raise ValueError(f"Step: one token for each of {self.Batch} requests")
        counts = [1] * self.Batch if active is None else [int(bool(a)) for a in active]
        need = self.Cache.Room(self.Cache.Held, counts, self.Cache.MaxTokens)
        self._ids.copy_(ids.reshape(-1))

        def one():
            if self._graph is None and self._may_record and self._steps > 0:  # the step before was eager: buffers that are made once exist
                self._record()
            if self._graph is None:
                return self._step(self._ids, 1, True)
            self._graph.replay()
            return self._static

        out = self._take(counts, need, one)
        self._steps += 1
        return out

    def Generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, stop: Optional[int] = None) -> List[List[int]]:
        """Up to `new_tokens` tokens for each prompt (not empty; at most `batch` of them), `stop` being the last where it comes.  The requests are
        released at the end."""
        n = len(prompts)
        if n > self.Batch or n == 0 or any(len(p) == 0 for p in prompts):
            raise ValueError(f"Generate: between 1 and {self.Batch} prompts, none of them empty")
        if any(self.Cache.Held):
            raise ValueError("Generate: requests are under way")
        self.Cache.Room([0] * n, [len(p) + max(new_tokens - 1, 0) for p in prompts], self.Cache.MaxTokens)
        texts: List[List[int]] = [[] for _ in prompts]
        drawn = []                                        # tokens of the steps, which stay on the device while nothing asks for them
        active = [b < n for b in range(self.Batch)]
        try:
            for i in range(new_tokens):
                out = self.Feed([*prompts, *[[]] * (self.Batch - n)]) if i == 0 else self.Step(out, active)
                drawn.append(out.clone())
                if stop is not None and i + 1 < new_tokens:
                    for b, t in enumerate(drawn[-1].tolist()):
                        active[b] = active[b] and t != stop and t >= 0
                    if not any(active):
                        break
            for row in torch.stack(drawn).tolist() if drawn else []:
                for b in range(n):
                    if row[b] >= 0:
                        texts[b].append(row[b])
        finally:
            self.Release(range(n))
        return texts

    # ---- one step
    def _take(self, counts: Sequence[int], need: int, step) -> torch.Tensor:
        """One step of `counts` new tokens of each request with numbers of its own.  A step that fails moves nothing, and may be made again."""
        c, numbers = self.Cache, self._random.get_state()
        try:
            self._fresh.copy_(torch.tensor(counts, dtype=torch.int32))
            torch.rand(self.Batch, generator=self._random, out=self._u)
            out, logits, logprobs = step()
        except BaseException:
            self._random.set_state(numbers)
            raise
        self.Logits, self.LogProbs = logits, logprobs
        c.Held = [h + f for h, f in zip(c.Held, counts)]
        c.Used += need
        return out

    def _keep(self, step: paged.PagedStep, lens: torch.Tensor) -> None:
        """The step's tokens and pages are the cache's from here on; before, what it wrote lies beyond the lengths and the stack's top."""
        lens.copy_(step.lens)
        self.Cache.Taken.copy_(step.taken)

    def _layers(self, ids: torch.Tensor, step: paged.PagedStep, tables: torch.Tensor, most: int, prompt_len: int) -> torch.Tensor:
        """The rows of the tokens behind the last block; their keys and values go to their pages."""
        m, c = self.Model, self.Cache
        n = ids.numel()
        pos = None
        if m.PosEmbed is not None:
            pos = OaMatrix(m.PosEmbed.Weight.Tensor().index_select(0, step.positions.clamp(min=0)))
        x = F.Embedding(m.Embed.Weight.Data, OaMatrix(ids.reshape(1, n)), pos, n)
        for b, pool in zip(m.Blocks, c.Layers):
            qkv = b.Attention.ProjectQkv(b.LnAttn.Forward(x)).Tensor()
            q = paged.append(qkv, step.positions, step.slots, pool[0], pool[1], b.Attention.RopeTheta)
            attn = paged.attention(q, pool[0], pool[1], tables, step.lens, step.starts, most, c.PromptTable.reshape(-1) if prompt_len else None, prompt_len)
            x = block_tail(b, x, OaMatrix(attn), n <= self.Batch)
        return x.Tensor()

    def _step(self, ids: torch.Tensor, most: int, by_request: bool):
        """(next tokens, logits, log-probabilities).  `by_request`: ids [batch], of which the requests that have a new token take theirs."""
        m, c = self.Model, self.Cache
        with AG.OaGradNo():
            step = paged.plan(c.Lens, self._fresh, c.Tables, c.Free, c.Taken, c.PageSize, ids.numel(), c.PromptLen)
            if by_request:
                ids = ids.index_select(0, step.rows.clamp(min=0)).clamp(min=0)             # rows of no request are some token's, whose result nothing reads
            x = self._layers(ids, step, c.Tables, most, c.PromptLen)
            last = x.index_select(0, (step.starts[1:] - 1).clamp(min=0))
            logits = m.Head.Forward(m.LnFinal.Forward(OaMatrix(last))).Tensor()
            tokens, logprobs = sampling.sample(logits, self._u, self._temperature, self._top_k, self._top_p, self._min_p)
            out = torch.where(self._fresh > 0, tokens, -1)
            self._keep(step, c.Lens)
            return out, logits, logprobs

    def _record(self) -> None:
        """A step of one token each as a graph: it reads the ids, the requests that have one, the random numbers and the settings where they lie."""
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        # a replay begins after everything before it on the stream, so whatever changed the weights has finished by then
        with torch.cuda.graph(g, capture_error_mode="thread_local"), K.weights_at_rest([p.Data.Tensor() for p in self.Model.AllParameterPtrs()]):
            self._static = self._step(self._ids, 1, True)
        self._graph = g
