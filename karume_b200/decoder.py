"""A whole decoder on the library's calls: packed int4 linears with their neighbours (kq_linear_fused), keys and values in a
paged 4-bit cache, rotary positions applied on the way into the cache and into the attention over it.

    h = embedding(ids)
    every layer:   q | k | v = linear(rms_norm(h));  append(rotate(k), v);  h += o(attention(rotate(q)))
                   h += down(silu(gate(rms_norm(h))) * up(rms_norm(h)))
    logits = head(rms_norm(h of each sequence's last token))

Prompts of any lengths run at once; single-token steps are recorded once as a CUDA graph and replayed, the sequences'
lengths advancing on the device.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass

from .runtime import CacheBatch, Gpu, KqError, Rope


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


class Decoder:
    """`weights` maps "embedding", "head" and "{layer}.{q,k,v,o,gate,up,down}" to resident weights, `norms` "{layer}.1",
    "{layer}.2" and "final" to f32 tensors [hidden].  Up to `sequences` conversations of up to `longest` tokens.  Calls are made
    with torch on the context's stream (on its default one if the context has its own), which is checked: lengths, ids and what
    a prompt's layers work in are torch's, and nothing else orders the two."""

    def __init__(self, gpu: Gpu, shape: DecoderShape, weights: dict, norms: dict, rope: Rope, sequences: int, longest: int,
                 page_tokens: int = 64, window: int = 0):
        import torch
        self.torch, self.gpu, self.shape, self.weights, self.norms, self.rope, self.window = torch, gpu, shape, weights, norms, rope, window
        self._check_stream()
        width = (longest + page_tokens - 1) // page_tokens
        if longest > rope.positions:
            raise KqError(2, f"the rotation table has {rope.positions} positions, sequences may have {longest}")
        self.caches = [gpu.kv_cache(sequences * width, page_tokens, shape.kv_heads, shape.head_dim) for _ in range(shape.layers)]
        self.pages = torch.arange(sequences * width, dtype=torch.int32, device=gpu.device).view(sequences, width)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=gpu.device)
        self.ids = torch.zeros(sequences, dtype=torch.int32, device=gpu.device)
        self.longest, self.held = longest, [0] * sequences  # what the host knows of the lengths
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
            self.lengths.copy_(self.torch.tensor(self.held, dtype=self.torch.int32))
            raise

    def _record(self) -> None:
        self.logits = self.torch.empty((len(self.held), self.shape.vocab), device=self.gpu.device)
        enqueue = lambda: self._head(self._layers(self._step_buffers, self.ids, self._step_batch), self.logits)  # noqa: E731
        # once outside the recording, so that scratch has its size: over idle sequences, which changes no page
        self.lengths.zero_()
        enqueue()
        self.gpu.sync()
        self.gpu.graph_begin()
        try:
            enqueue()
        except BaseException:
            self.gpu.graph_free(self.gpu.graph_end())  # the context records no longer
            raise
        self._step = self.gpu.graph_end()
        self.lengths.copy_(self.torch.tensor(self.held, dtype=self.torch.int32))

    def _buffers(self, rows: int):
        s, dev = self.shape, self.gpu.device
        sizes = dict(x=s.hidden, h=s.hidden, q=s.heads * s.head_dim, k=s.kv_heads * s.head_dim, v=s.kv_heads * s.head_dim,
                     a=s.heads * s.head_dim, act=s.ffn)
        return {name: self.torch.empty((rows, n), device=dev) for name, n in sizes.items()}

    def _bias(self, n: int):
        return self._zero[:n]

    def _layers(self, b: dict, ids, batch: CacheBatch):
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
            g.cache_attention(self.caches[i], heads(b["q"], s.heads), batch, window=self.window, rope=self.rope, out=heads(b["a"], s.heads))
            g.linear_fused(b["a"], [W[f"{i}.o"]], [self._bias(s.hidden)], [b["h"]], residual=cur)
            cur = b["h"]
            g.linear_fused(cur, [W[f"{i}.gate"], W[f"{i}.up"]], [self._bias(s.ffn)] * 2, [b["act"]], norm_weight=N[f"{i}.2"], eps=s.eps, swiglu=True)
            g.linear_fused(b["act"], [W[f"{i}.down"]], [self._bias(s.hidden)], [b["h"]], residual=cur)
        return cur

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
        starts = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32).to(self.gpu.device)
        with self._lengths_kept():
            self.lengths.copy_(torch.tensor(held, dtype=torch.int32))
            hidden = self._layers(self._buffers(ids.numel()), ids, CacheBatch(self.pages, self.lengths, starts, tokens=ids.numel(), most=max(news)))
            last = (starts[1:] - 1).clamp(min=0).long()
            logits = self._head(hidden[last].contiguous())
        self.held = held
        return logits

    def step(self):
        """One token of every sequence, from self.ids (CUDA int32 [sequences]); returns the logits, a buffer that the next
        step writes again."""
        self._check_stream()
        if any(h + 1 > self.longest for h in self.held):
            raise KqError(2, f"a sequence would grow beyond {self.longest} tokens")
        with self._lengths_kept():
            if self._step is None:
                self._record()
            self.lengths += 1
            self.gpu.graph_launch(self._step)
        self.held = [h + 1 for h in self.held]
        return self.logits

    def close(self) -> None:
        if self._step is not None:
            self.gpu.graph_free(self._step)
            self._step = None
        for c in self.caches:
            c.free()
        self.caches = []
