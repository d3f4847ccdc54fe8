"""A whole decoder on the library's calls: packed int4 linears with their neighbours (kq_linear_fused), keys and values in a
paged 4-bit cache, rotary positions applied on the way into the cache and into the attention over it.

    h = embedding(ids)
    every layer:   q | k | v = linear(rms_norm(h));  append(rotate(k), v);  h += o(attention(rotate(q)))
                   h += down(silu(gate(rms_norm(h))) * up(rms_norm(h)))
    logits = head(rms_norm(h of each sequence's last token))

Prompts of any lengths run at once; single-token steps are recorded once as a CUDA graph and replayed, the sequences'
lengths advancing on the device.  With a pool of pages (`pool_pages`) sequences branch, are cut back and end (fork): what they have in common is
held once, and read once where that is faster.  With `select` single tokens read a budget of pages.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass

from .runtime import CacheBatch, Gpu, KqError, Rope, SharedPrefixes


@dataclass(frozen=True)
class DecoderShape:
    layers: int
    hidden: int
    heads: int
    kv_heads: int
    head_dim: int
    ffn: int
    vocab: int
    eps: float = 1e-5


@dataclass(frozen=True)
class Selection:
    """A single token attends to up to `budget` pages of its sequence: the first `first`, the last `last` and those whose keys promise most."""
    budget: int
    first: int = 1
    last: int = 2


class Decoder:
    """`weights` maps "embedding", "head" and "{layer}.{q,k,v,o,gate,up,down}" to resident weights, `norms` "{layer}.1",
    "{layer}.2" and "final" to f32 tensors [hidden].  Up to `sequences` conversations of up to `longest` tokens.  Calls are made
    with torch on the context's stream (on its default one if the context has its own), which is checked: lengths, ids and what
    a prompt's layers work in are torch's, and nothing else orders the two.

    pool_pages: so many pages for all sequences, taken as they grow (0: each sequence has its own, as many as `longest` needs).
    select: see Selection; prompts read everything."""

    def __init__(self, gpu: Gpu, shape: DecoderShape, weights: dict, norms: dict, rope: Rope, sequences: int, longest: int,
                 page_tokens: int = 64, window: int = 0, pool_pages: int = 0, select: "Selection | None" = None):
        import torch
        self.torch, self.gpu, self.shape, self.weights, self.norms, self.rope, self.window = torch, gpu, shape, weights, norms, rope, window
        self._check_stream()
        width = (longest + page_tokens - 1) // page_tokens
        if longest > rope.positions:
            raise KqError(2, f"the rotation table has {rope.positions} positions, sequences may have {longest}")
        if select is not None and window:
            raise KqError(2, "a token reads a window of its sequence or selected pages, not both")
        count = pool_pages or sequences * width
        self.caches = [gpu.kv_cache(count, page_tokens, shape.kv_heads, shape.head_dim) for _ in range(shape.layers)]
        self.select, self.summaries = select, [gpu.cache_summaries(c) for c in self.caches] if select is not None else []
        self.book, self.shared, self.free = None, None, 0
        if pool_pages:
            self.book = gpu.cache_pages(sequences, longest, pool_pages, page_tokens)
            self.pages, self.lengths, self.free = self.book.table, self.book.lengths, pool_pages
            self.news = torch.zeros(sequences, dtype=torch.int32, device=gpu.device)  # what a step adds to each sequence
            # groups of sequences that begin alike, as many as there may be
            self.shared = SharedPrefixes(torch.full((sequences + 1,), sequences, dtype=torch.int32, device=gpu.device), torch.zeros_like(self.news))
        else:
            self.pages = torch.arange(sequences * width, dtype=torch.int32, device=gpu.device).view(sequences, width)
            self.lengths = torch.zeros(sequences, dtype=torch.int32, device=gpu.device)
        self.ids = torch.zeros(sequences, dtype=torch.int32, device=gpu.device)
        self.longest, self.held = longest, [0] * sequences  # what the host knows of the lengths
        self._ended, self._stepped = [False] * sequences, None  # by a fork; what `news` holds
        self._zero = torch.zeros(max(shape.ffn, shape.vocab, shape.hidden, shape.heads * shape.head_dim), device=gpu.device)
        self._step = None
        self._step_batch = CacheBatch(self.pages, self.lengths)
        self._step_buffers = self._buffers(sequences)

    def _check_stream(self) -> None:
        if int(self.torch.cuda.current_stream(self.gpu.device).cuda_stream) != self.gpu.stream:
            raise KqError(8, "torch's current stream is not the context's: install it with use_stream(), or make the call under the context's")

    @contextmanager
    def _lengths_kept(self):
        """Where a call fails, the sequences are as long as before; rows that it appended lie behind their ends."""
        try:
            yield
        except BaseException:
            if self.book is not None:  # pages that it took go back
                whole = self.torch.arange(len(self.held), dtype=self.torch.int32, device=self.gpu.device)
                self.gpu.pages_fork(self.book, whole, self._numbers(self.held))
            else:
                self.lengths.copy_(self.torch.tensor(self.held, dtype=self.torch.int32))
            raise

    def _numbers(self, values):
        return self.torch.tensor(list(values), dtype=self.torch.int32).to(self.gpu.device)

    def _needed(self, news) -> int:
        """Pages that so many more tokens of each sequence take."""
        page = self.book.page_tokens
        return sum(-(-(n + h) // page) - -(-h // page) for n, h in zip(news, self.held))

    def _take(self, news) -> int:
        """The same, and an error where the pool has not so many."""
        need = self._needed(news)
        if need > self.free:
            raise KqError(3, f"{need} pages needed, {self.free} of the pool's {self.book.pages} are free")
        return need

    def _record(self) -> None:
        self.logits = self.torch.empty((len(self.held), self.shape.vocab), device=self.gpu.device)

        def enqueue():
            if self.book is not None:
                self.gpu.pages_grow(self.book, self.news)
            self._head(self._layers(self._step_buffers, self.ids, self._step_batch, step=True), self.logits)

        # once outside the recording, so that scratch has its size: over idle sequences, which changes no page
        try:
            self.lengths.zero_()
            if self.book is not None:
                self.news.zero_()
                self._stepped = None
            enqueue()
            self.gpu.sync()
            self.gpu.graph_begin()
            try:
                enqueue()
            except BaseException:
                self.gpu.graph_free(self.gpu.graph_end())  # the context records no longer
                raise
            self._step = self.gpu.graph_end()
        finally:
            self.lengths.copy_(self.torch.tensor(self.held, dtype=self.torch.int32))

    def _buffers(self, rows: int):
        s, dev = self.shape, self.gpu.device
        sizes = dict(x=s.hidden, h=s.hidden, q=s.heads * s.head_dim, k=s.kv_heads * s.head_dim, v=s.kv_heads * s.head_dim,
                     a=s.heads * s.head_dim, act=s.ffn)
        return {name: self.torch.empty((rows, n), device=dev) for name, n in sizes.items()}

    def _bias(self, n: int):
        return self._zero[:n]

    def _layers(self, b: dict, ids, batch: CacheBatch, step: bool = False):
        """Enqueues the layers over the rows of `ids`; returns the hidden rows."""
        g, s, W, N = self.gpu, self.shape, self.weights, self.norms
        rows = ids.numel()
        g.embedding(ids, W["embedding"], out=b["x"])
        cur = b["x"]
        for i in range(s.layers):
            names = [f"{i}.q", f"{i}.k", f"{i}.v"]
            g.linear_fused(cur, [W[n] for n in names], [self._bias(W[n].n) for n in names], [b["q"], b["k"], b["v"]],
                           norm_weight=N[f"{i}.1"], eps=s.eps)
            heads = lambda t, n: t.view(rows, n, s.head_dim)  # noqa: E731
            g.cache_append(self.caches[i], heads(b["k"], s.kv_heads), heads(b["v"], s.kv_heads), batch, rope=self.rope)
            q, taken, shared = heads(b["q"], s.heads), None, self.shared
            if self.select is not None:
                g.cache_summarize(self.caches[i], self.summaries[i], batch)
                if step:
                    of = self.select
                    taken, shared = g.cache_select(self.caches[i], self.summaries[i], q, batch, of.budget, of.first, of.last, rope=self.rope, out=self._taken()), None
            g.cache_attention(self.caches[i], q, batch, window=self.window, rope=self.rope, out=heads(b["a"], s.heads), shared=shared, selected=taken)
            g.linear_fused(b["a"], [W[f"{i}.o"]], [self._bias(s.hidden)], [b["h"]], residual=cur)
            cur = b["h"]
            g.linear_fused(cur, [W[f"{i}.gate"], W[f"{i}.up"]], [self._bias(s.ffn)] * 2, [b["act"]], norm_weight=N[f"{i}.2"], eps=s.eps, swiglu=True)
            g.linear_fused(b["act"], [W[f"{i}.down"]], [self._bias(s.hidden)], [b["h"]], residual=cur)
        return cur

    def _taken(self):
        """Where a step's selections go, layer after layer: a recorded step keeps it."""
        if "taken" not in self._step_buffers:
            shape = (len(self.held), self.shape.kv_heads, self.select.budget)
            self._step_buffers["taken"] = self.torch.empty(shape, dtype=self.torch.int32, device=self.gpu.device)
        return self._step_buffers["taken"]

    def _head(self, rows, out=None):
        outs = [out if out is not None else self.torch.empty((rows.shape[0], self.shape.vocab), device=self.gpu.device)]
        self.gpu.linear_fused(rows, [self.weights["head"]], [self._bias(self.shape.vocab)], outs, norm_weight=self.norms["final"], eps=self.shape.eps)
        return outs[0]

    def prompt(self, ids, news):
        """Takes `news[b]` more tokens of each sequence b (0: none), packed in `ids` (CUDA int32); returns the logits of each
        sequence's last row [sequences, vocab] (of the rows in front of it where it has none)."""
        torch = self.torch
        self._check_stream()
        if len(news) != len(self.held) or min(news) < 0 or sum(news) != ids.numel() or ids.numel() == 0:
            raise KqError(2, f"{list(news)} new tokens announced for {len(self.held)} sequences, {ids.numel()} given")
        if ids.dtype != torch.int32 or not ids.is_cuda or not ids.is_contiguous():
            raise KqError(2, "ids must be a contiguous CUDA int32 tensor")
        if any(n + h > self.longest for n, h in zip(news, self.held)):
            raise KqError(2, f"a sequence would grow beyond {self.longest} tokens")
        held = [n + h for n, h in zip(news, self.held)]
        need = self._take(news) if self.book is not None else 0
        starts = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32).to(self.gpu.device)
        with self._lengths_kept():
            if self.book is not None:
                self.gpu.pages_grow(self.book, self._numbers(news))
            else:
                self.lengths.copy_(torch.tensor(held, dtype=torch.int32))
            hidden = self._layers(self._buffers(ids.numel()), ids, CacheBatch(self.pages, self.lengths, starts, tokens=ids.numel(), most=max(news)))
            last = (starts[1:] - 1).clamp(min=0).long()
            logits = self._head(hidden[last].contiguous())
        self.held, self.free = held, self.free - need
        self._ended = [e and n == 0 for e, n in zip(self._ended, news)]
        return logits

    def fork(self, parents, keep=None) -> None:
        """Sequence b goes on as the first keep[b] tokens (all, without keep) of sequence parents[b], as it was before the call; a negative parent
        ends it, itself cuts it back or leaves it.  All at once: beams that are reordered, answers that branch, drafts that are given back.
        Pages are shared; only a last page that is not full is copied.  A step leaves sequences that have ended out.  Where the pool has too few
        pages nothing changes (KQ_ERR_OOM)."""
        if self.book is None:
            raise KqError(8, "sequences share pages of a pool: make the decoder with pool_pages")
        self._check_stream()
        n = len(self.held)
        if len(parents) != n or any(p >= n for p in parents) or (keep is not None and (len(keep) != n or min(keep) < 0)):
            raise KqError(2, f"a parent below {n} and a number of tokens for each of {n} sequences")
        pairs = self.gpu.pages_fork(self.book, self._numbers(max(p, -1) for p in parents),
                                    self._numbers(min(k, self.longest) for k in keep) if keep is not None else None)
        self.gpu.pages_copy(self.book, pairs, self.caches)
        missing = int(self.book.report[0])  # waits for the device
        if missing:
            raise KqError(3, f"{missing} pages too few for the last pages of the new sequences")
        self.held = [0 if p < 0 else min(self.held[p], keep[b] if keep is not None else self.longest) for b, p in enumerate(parents)]
        self._ended = [p < 0 or self._ended[p] for p in parents]
        self.free = self.book.pages - int((self.book.refs > 0).sum())
        self._find_groups()

    def _find_groups(self) -> None:
        """Neighbouring sequences whose rows of the page table begin with the same pages, and with how many."""
        n, page, rows = len(self.held), self.book.page_tokens, self.pages.cpu().numpy()
        whole = [h // page for h in self.held]

        def alike(a, b):
            most = min(whole[a], whole[b])
            differ = (rows[a, :most] != rows[b, :most]).nonzero()[0]
            return int(differ[0]) if len(differ) else most

        first, tokens, b = [], [], 0
        while b < n:
            end, least = b + 1, whole[b]
            while end < n and (common := alike(b, end)) > 0:
                least, end = min(least, common), end + 1
            first.append(b)
            tokens.append(least * page if end - b > 1 else 0)
            b = end
        self.shared.first.copy_(self._numbers(first + [n] * (n + 1 - len(first))))
        self.shared.tokens.copy_(self._numbers(tokens + [0] * (n - len(tokens))))

    def step(self):
        """One token of every sequence (but those that a fork has ended), from self.ids (CUDA int32 [sequences]); returns the logits, a buffer
        that the next step writes again."""
        self._check_stream()
        news = [0 if ended else 1 for ended in self._ended]
        if any(h + n > self.longest for h, n in zip(self.held, news)):
            raise KqError(2, f"a sequence would grow beyond {self.longest} tokens")
        need = self._take(news) if self.book is not None else 0
        with self._lengths_kept():
            if self._step is None:
                self._record()
            if self.book is not None:
                if news != self._stepped:
                    self.news.copy_(self._numbers(news))
                    self._stepped = news
            else:
                self.lengths += 1
            self.gpu.graph_launch(self._step)
        self.held, self.free = [h + n for h, n in zip(self.held, news)], self.free - need
        return self.logits

    def close(self) -> None:
        if self._step is not None:
            self.gpu.graph_free(self._step)
            self._step = None
        for c in self.caches:
            c.free()
        self.caches = []
