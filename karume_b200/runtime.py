"""Host-side mirror of the reference interface for the quantized `linear` path.

karume's TypeScript runtime reaches this path through three steps, and the classes
here keep their names, argument meaning and failure behaviour so the parity tests read
like the reference's own:

* ``acquire_gpu()``             <- ``acquireGpu()`` (packages/runtime/src/gpu/device.ts:1182-1218)
* ``Gpu.upload_weight(...)``    <- the i4 / i8 branch of ``Session.#build``
                                   (packages/runtime/src/runtime/executor.ts:830-896)
* ``Gpu.linear(x, w, bias)``    <- ``RecipeBuilder.#buildLinear``
                                   (packages/runtime/src/runtime/recipe-builder.ts:1311-1392)

Everything funnels into the C ABI of ``libkq.so``; torch is used only to own device
memory and streams.  Errors are raised, never swallowed, and there is no alternative
execution path (the reference's "fail loudly" rule, CLAUDE.md:51 of its repository).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import (KQ_BF16, KQ_F16, KQ_F32, KQ_SHARD_COLUMN, KQ_SHARD_NONE, KQ_SHARD_ROW,
                   KQ_STORAGE_I4, KQ_STORAGE_I8)

L = _lib.lib


class KqError(RuntimeError):
    """A libkq call returned a non-zero status (code + the library's message)."""

    def __init__(self, code: int, message: str):
        self.code = code
        self.status = _lib.STATUS_NAMES.get(code, str(code))
        super().__init__(f"{self.status}: {message}")


KQ_SHARED_AUTO = (1 << 64) - 1
KQ_PAIRS_END = (1 << 64) - 1

_NP_DTYPES = {np.dtype(np.float32): KQ_F32, np.dtype(np.float16): KQ_F16}


def _torch():
    import torch
    return torch


_fast = None  # the native form of the serving calls (csrc/kq_torch.cpp), loaded with the first context


def _load_fast() -> None:
    """Loads the extension module and hands it the library's entry points; raises if it is not built."""
    global _fast
    if _fast is None:
        _torch()
        from . import _kqtorch
        _kqtorch.bind(*[ctypes.cast(f, ctypes.c_void_p).value
                        for f in (L.kq_linear, L.kq_linear_fused, L.kq_quantize_rows, L.kq_linear_a8, L.kq_embedding, L.kq_rope,
                                  L.kq_cache_append, L.kq_cache_read, L.kq_cache_attention, L.kq_cache_attention_shared, L.kq_cache_attention_selected,
                                  L.kq_cache_summarize, L.kq_cache_select, L.kq_pages_grow, L.kq_pages_fork, L.kq_pages_compact, L.kq_pages_copy)])
        _fast = _kqtorch


def _tensor_dtype_code(t) -> int:
    torch = _torch()
    table = {torch.float32: KQ_F32, torch.float16: KQ_F16, torch.bfloat16: KQ_BF16}
    if t.dtype not in table:
        raise KqError(1, f"activation dtype {t.dtype} is not f32 / f16 / bf16")
    return table[t.dtype]


@dataclass
class Weight:
    """A resident quantized weight (handle + the metadata the host planned with)."""
    gpu: "Gpu"
    handle: int
    storage: str        # "i4" | "i8"  (storage.dtype of the initializer)
    n: int
    k: int
    group_size: int     # 0 for i8

    @property
    def resident_bytes(self) -> int:
        return int(L.kq_weight_resident_bytes(self.gpu._ctx, self.handle))

    def dequant(self):
        """f32 [n, k] expansion computed on the device with the kernels' dequant rule."""
        torch = _torch()
        out = torch.empty((self.n, self.k), dtype=torch.float32, device=self.gpu.device)
        self.gpu._check(L.kq_weight_dequant(self.gpu._ctx, self.handle, out.data_ptr()))
        self.gpu.sync()
        return out

    def free(self) -> None:
        if self.handle:
            self.gpu._check(L.kq_weight_free(self.gpu._ctx, self.handle))
            self.handle = 0


@dataclass
class Rope:
    """Rotation angles: table f32 CUDA [positions, rotary / 2, 2] of (cos, sin) (rope_table makes one); pairs are
    (i, i + rotary / 2) of a head, or (2 i, 2 i + 1) with interleaved."""
    table: object
    interleaved: bool = False

    def __post_init__(self):
        t = self.table
        if t.dtype != _torch().float32 or not t.is_cuda or t.dim() != 3 or t.shape[2] != 2 or not t.is_contiguous():
            raise KqError(2, "the rotation table is a contiguous CUDA f32 tensor [positions, rotary / 2, 2]")
        self.positions, self.rotary = int(t.shape[0]), 2 * int(t.shape[1])
        self.index = t.get_device()
        self.args = (t.data_ptr(), self.positions, self.rotary, 1 if self.interleaved else 0)


class CacheBatch:
    """The sequences of a call: pages i32 CUDA [sequences, width] (page numbers in token order), lengths i32
    [sequences] (the new tokens included) and starts i32 [sequences + 1] (rows of each sequence's new tokens; None: one
    each).  tokens is the number of rows, most a bound of any sequence's new tokens; both are host numbers, the
    tensors are read on the device at each launch and may change between replays of a recorded step."""

    def __init__(self, pages, lengths, starts=None, tokens: int = 0, most: int = 0):
        torch = _torch()
        for name, t, dims in (("pages", pages, 2), ("lengths", lengths, 1), ("starts", starts, 1)):
            if t is not None and (t.dtype != torch.int32 or not t.is_cuda or t.dim() != dims or not t.is_contiguous()):
                raise KqError(2, f"{name} must be a contiguous CUDA int32 tensor of {dims} dimension(s)")
        self.sequences, self.width = (int(n) for n in pages.shape)
        if lengths.numel() != self.sequences or (starts is not None and starts.numel() != self.sequences + 1):
            raise KqError(2, f"{self.sequences} sequences need as many lengths and one more starts")
        if starts is not None and tokens <= 0:
            raise KqError(2, "with starts, tokens says how many rows there are")
        if most < 0:
            raise KqError(2, f"most {most}: a bound of a sequence's new tokens, 0 if not known")
        self.pages, self.lengths, self.starts = pages, lengths, starts
        self.index = pages.get_device()  # -1: the tensors are on several devices
        if any(t is not None and t.get_device() != self.index for t in (lengths, starts)):
            self.index = -1
        self.tokens = int(tokens) if starts is not None else self.sequences
        self.most = min(int(most), self.tokens) if starts is not None else 1
        self.args = (self.sequences, pages.data_ptr(), self.width, lengths.data_ptr(), starts.data_ptr() if starts is not None else 0,
                     self.tokens)


@dataclass
class KvCache:
    """Pages of keys and values in 4 bits: pool uint8 CUDA [pages, kv_heads, page_tokens * (head_dim + 8)] and its handle."""
    gpu: "Gpu"
    handle: int
    pool: object
    pages: int
    page_tokens: int
    kv_heads: int
    head_dim: int

    def __post_init__(self):
        self.page_args = (self.pages, self.kv_heads * self.page_tokens * (self.head_dim + 8), self.pool.data_ptr(), self.pool.get_device())

    def free(self) -> None:
        if self.handle:
            self.gpu._check(L.kq_cache_free(self.gpu._ctx, self.handle))
            self.handle = 0


class SharedPrefixes:
    """Sequences that begin alike: first i32 CUDA [groups + 1] (group g is the sequences first[g] .. first[g + 1] - 1) and tokens i32 [groups],
    how many tokens the sequences of each have in common at their beginning, in the same pages or copies of them.  least: how many bytes
    reading those once has to save for a call to do so (0: always; None: what measured faster)."""

    def __init__(self, first, tokens, least: "int | None" = None):
        torch = _torch()
        for name, t in (("first", first), ("tokens", tokens)):
            if t.dtype != torch.int32 or not t.is_cuda or t.dim() != 1 or not t.is_contiguous():
                raise KqError(2, f"{name} must be a contiguous CUDA int32 tensor of one dimension")
        self.groups = int(tokens.numel())
        if first.numel() != self.groups + 1:
            raise KqError(2, f"{self.groups} groups have {self.groups + 1} boundaries, not {first.numel()}")
        _on_device(first.device.index, tokens=tokens)
        if least is not None and not 0 <= least < KQ_SHARED_AUTO:
            raise KqError(2, f"least {least}: a number of bytes")
        self.first, self.tokens, self.index = first, tokens, first.get_device()
        self.args = (self.groups, first.data_ptr(), tokens.data_ptr(), KQ_SHARED_AUTO if least is None else int(least))


class CacheSummaries:
    """What Gpu.cache_select goes by: codes int8 CUDA [pages, kv_heads, 2, head_dim] and scales f32 [pages, kv_heads, 2] of each page's keys
    (channels' middles and half spreads), kept up by Gpu.cache_summarize.  Gpu.cache_summaries makes them for a cache."""

    def __init__(self, codes, scales):
        torch = _torch()
        if codes.dtype != torch.int8 or scales.dtype != torch.float32 or not (codes.is_cuda and scales.is_cuda) or codes.dim() != 4 or scales.dim() != 3 or \
                tuple(scales.shape) != tuple(codes.shape[:3]) or codes.shape[2] != 2 or not (codes.is_contiguous() and scales.is_contiguous()):
            raise KqError(2, "summaries are contiguous CUDA tensors: codes int8 [pages, kv_heads, 2, head_dim], scales f32 [pages, kv_heads, 2]")
        _on_device(codes.device.index, scales=scales)
        self.codes, self.scales, self.index = codes, scales, codes.get_device()
        self.args = (codes.data_ptr(), scales.data_ptr())

        self.shape = tuple(int(n) for n in codes.shape)

    def check(self, cache: "KvCache", index: int) -> None:
        if self.index != index:
            _on_device(index, codes=self.codes)
        pages, heads, _, dim = self.shape
        if pages < cache.pages or heads != cache.kv_heads or dim != cache.head_dim:
            raise KqError(2, f"summaries {list(self.shape)} are not those of {cache.pages} pages of {cache.kv_heads} heads of {cache.head_dim}")


class CachePages:
    """Which page belongs to whom: table i32 CUDA [sequences, width] (a CacheBatch's pages; -1 behind a sequence's own), lengths i32
    [sequences], refs i32 [pages] (how many entries name a page) and report i32 [4] of the last call: pages that were missing (then, and
    with -1 for a refused call, nothing changed), pages taken or in use, pairs, 0.  Gpu.cache_pages makes an empty one."""

    def __init__(self, table, lengths, refs, page_tokens: int, report=None):
        torch = _torch()
        if report is None:
            report = torch.zeros(4, dtype=torch.int32, device=table.device)
            torch.cuda.current_stream(table.device).synchronize()  # the first call may run on another stream
        for name, t, dims in (("table", table, 2), ("lengths", lengths, 1), ("refs", refs, 1), ("report", report, 1)):
            if t.dtype != torch.int32 or not t.is_cuda or t.dim() != dims or not t.is_contiguous():
                raise KqError(2, f"{name} must be a contiguous CUDA int32 tensor of {dims} dimension(s)")
        self.sequences, self.width = (int(n) for n in table.shape)
        if lengths.numel() != self.sequences or report.numel() != 4:
            raise KqError(2, f"{self.sequences} sequences need as many lengths, a report four numbers")
        _on_device(table.device.index, lengths=lengths, refs=refs, report=report)
        self.table, self.lengths, self.refs, self.report, self.index = table, lengths, refs, report, table.get_device()
        self.pages, self.page_tokens = int(refs.numel()), int(page_tokens)
        self.args = (table.data_ptr(), self.sequences, self.width, lengths.data_ptr(), refs.data_ptr(), self.pages, self.page_tokens, report.data_ptr())
        self.args_for_pairs = (*self.args[:-1], KQ_PAIRS_END)  # of a call, which end by themselves
        self.counted = True  # the report may say how many pairs there are: no grow has written it since


def _on_device(index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t.device.index != index:
            raise KqError(2, f"{name} is on {t.device}, the context's device is cuda:{index}")


def _batch_here(index: int, batch: "CacheBatch", rope: "Rope | None" = None) -> None:
    """Raises where a batch's tensors or the angles are not on the context's device."""
    if batch.index != index:
        raise KqError(2, f"the batch is on {'several devices' if batch.index < 0 else f'cuda:{batch.index}'}, the context's device is cuda:{index}")
    if rope is not None and rope.index != index:
        _on_device(index, table=rope.table)


def _per_sequence(t, book: CachePages, name: str) -> int:
    torch = _torch()
    if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.numel() != book.sequences:
        raise KqError(2, f"{name} must be a contiguous CUDA int32 tensor [{book.sequences}]")
    return t.data_ptr()


_NO_ROPE = (0, 0, 0, 0)


def _rows(t, heads: int, dim: int, name: str):
    """(address, elements between tokens) of a CUDA tensor [tokens, heads, dim] whose tokens may be strided."""
    if not t.is_cuda or t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim or t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim):
        raise KqError(2, f"{name} must be a CUDA tensor [tokens, {heads}, {dim}] with heads and values dense")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else heads * dim


class Gpu:
    """One CUDA device = one libkq context (the reference's GpuContext).

    Calls run on the stream that was torch's current one when the context was made, or that use_stream() installed since.
    Where that is torch's default stream (or with use_torch_stream=False) they run on the library's own, which waits for the default
    stream and which the default stream waits for.  Work on any other stream is in no order with the calls: install it first."""

    def __init__(self, device: int = 0, workspace_bytes: int = 0, use_torch_stream: bool = True):
        torch = _torch()
        if not torch.cuda.is_available():
            raise KqError(4, "no CUDA device: libkq has no CPU path")
        self.index = int(device)
        self.device = torch.device("cuda", self.index)
        ctx = ctypes.c_void_p()
        rc = L.kq_init(self.index, int(workspace_bytes), ctypes.byref(ctx))
        if rc != 0:
            raise KqError(rc, (L.kq_last_error(None) or b"").decode())
        self._ctx = ctx
        self._ctx_addr = ctx.value
        self.stream = 0  # handle of the stream the calls run on; 0: the library's own
        _load_fast()
        if use_torch_stream:
            self.use_stream(torch.cuda.current_stream(self.device))

    # -- plumbing -----------------------------------------------------------
    def _done(self, result):
        """What a native call returned: its result, or the status of a call the library refused."""
        if result.__class__ is int:
            self._check(result)
        return result

    def _check(self, rc: int) -> None:
        if rc != 0:
            raise KqError(rc, (L.kq_last_error(self._ctx) or b"").decode())

    def use_stream(self, stream) -> None:
        handle = int(stream.cuda_stream) if stream is not None else 0
        self._check(L.kq_set_stream(self._ctx, handle))
        self.stream = handle

    def set_overlap(self, enabled: bool) -> None:
        self._check(L.kq_set_overlap(self._ctx, 1 if enabled else 0))

    def sync(self) -> None:
        self._check(L.kq_sync(self._ctx))

    @property
    def launch_count(self) -> int:
        return int(L.kq_launch_count(self._ctx))

    def destroy(self) -> None:
        if self._ctx:
            L.kq_destroy(self._ctx)
            self._ctx = self._ctx_addr = None

    # -- weights ------------------------------------------------------------
    def upload_weight(self, storage: str, payload, scale, shape, group_size: int = 0,
                      shard: int = KQ_SHARD_NONE, rank: int = 0, world: int = 1) -> Weight:
        """payload: raw safetensors bytes (uint8 for i4, int8/uint8 for i8) of a [n, k]
        weight; scale: float32 or float16 array, [n, k/group_size] (i4) or [n] / [n,1] (i8)."""
        code = {"i4": KQ_STORAGE_I4, "i8": KQ_STORAGE_I8}.get(storage)
        if code is None:
            raise KqError(1, f"storage {storage!r}: only 'i4' and 'i8' weights take this path")
        if len(shape) != 2:
            raise KqError(2, f"linear weight must be rank 2 [out, in], got {tuple(shape)}")
        n, k = int(shape[0]), int(shape[1])
        pay = np.ascontiguousarray(np.asarray(payload)).view(np.uint8).reshape(-1)
        sc = np.ascontiguousarray(np.asarray(scale))
        if sc.dtype not in _NP_DTYPES:
            raise KqError(1, f"scale dtype {sc.dtype} is not float32 / float16")
        handle = ctypes.c_uint64(0)
        args = (self._ctx, code, pay.ctypes.data, pay.size, sc.ctypes.data, sc.size * sc.itemsize,
                _NP_DTYPES[sc.dtype], n, k, int(group_size))
        if shard == KQ_SHARD_NONE:
            rc = L.kq_weight_upload(*args, ctypes.byref(handle))
        else:
            rc = L.kq_weight_upload_shard(*args, int(shard), int(rank), int(world), ctypes.byref(handle))
        self._check(rc)
        sn, sk = ctypes.c_uint32(), ctypes.c_uint32()
        self._check(L.kq_weight_shape(self._ctx, handle.value, ctypes.byref(sn), ctypes.byref(sk)))
        return Weight(self, handle.value, storage, sn.value, sk.value, int(group_size))

    def embedding(self, index, weight: Weight, out=None):
        """Rows index[...] (CUDA int32) of a resident weight [vocab, hidden], dequantised to f32."""
        done = _fast.embedding(self._ctx_addr, weight.handle, weight.k, index, out)
        if done is not None:
            return self._done(done)
        torch = _torch()
        if index.dtype != torch.int32 or not index.is_cuda or not index.is_contiguous():
            raise ValueError("index must be a contiguous CUDA int32 tensor")
        if out is None:
            out = torch.empty(tuple(index.shape) + (weight.k,), dtype=torch.float32, device=index.device)
        self._check(L.kq_embedding(self._ctx, weight.handle, index.data_ptr(), index.numel(), out.data_ptr()))
        return out

    # -- integer-dot form ------------------------------------------------------
    def quantize_rows(self, x):
        """Per-row symmetric int8 quantisation of a CUDA f32 tensor [..., dim]:
        returns (q int8 [..., dim], scale f32 [...])."""
        done = _fast.quantize_rows(self._ctx_addr, x)
        if done is not None:
            return self._done(done)
        torch = _torch()
        if x.dtype != torch.float32 or not x.is_cuda or not x.is_contiguous():
            raise ValueError("quantize_rows takes a contiguous CUDA f32 tensor")
        dim = x.shape[-1]
        rows = x.numel() // dim if dim else 0
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        self._check(L.kq_quantize_rows(self._ctx, x.data_ptr(), rows, dim, q.data_ptr(), scale.data_ptr()))
        return q, scale

    def linear_a8(self, xq, xs, weight: Weight, bias, out=None):
        """Integer-dot linear: xq int8 [..., k] and xs f32 [...] from quantize_rows against a
        resident int8 (w8a8) or int4 (w4a8) weight.  Returns f32 [..., n]."""
        done = _fast.linear_a8(self._ctx_addr, weight.handle, weight.n, weight.k, xq, xs, bias, out)
        if done is not None:
            return self._done(done)
        torch = _torch()
        if xq.dtype != torch.int8 or xq.shape[-1] != weight.k or not xq.is_contiguous():
            raise ValueError("xq must be a contiguous int8 tensor [..., k]")
        m = xq.numel() // weight.k if weight.k else 0
        if xs.dtype != torch.float32 or xs.numel() != m:
            raise ValueError("xs must hold one f32 scale per row of xq")
        if bias is None or bias.dtype != torch.float32 or bias.numel() != weight.n:
            raise ValueError("bias must be a CUDA f32 tensor [n] (the op's arity is 3)")
        if out is None:
            out = torch.empty(xq.shape[:-1] + (weight.n,), dtype=torch.float32, device=xq.device)
        self._check(L.kq_linear_a8(self._ctx, weight.handle, xq.data_ptr(), xs.data_ptr(), bias.data_ptr(),
                                   out.data_ptr(), m))
        return out

    # -- the op ---------------------------------------------------------------
    def linear(self, x, weight: Weight, bias, out=None):
        """out[..., n] = x[..., k] @ W[n, k]^T + bias[n]; x is a CUDA tensor (f32/f16/bf16),
        bias a CUDA f32 tensor [n] (required: the op's arity is 3).  Returns f32."""
        done = _fast.linear(self._ctx_addr, weight.handle, weight.n, weight.k, x, bias, out)
        if done is not None:
            return self._done(done)
        torch = _torch()
        if x.shape[-1] != weight.k:
            raise KqError(2, f"linear: x[..., {x.shape[-1]}] does not match W[{weight.n},{weight.k}]")
        if bias is None or tuple(bias.shape) != (weight.n,) or bias.dtype != torch.float32:
            raise KqError(2, f"linear: bias must be f32 [{weight.n}] (arity 3 is fixed)")
        x = x.contiguous()
        m = x.numel() // weight.k if weight.k else int(np.prod(x.shape[:-1]))
        if out is None:
            out = torch.empty(tuple(x.shape[:-1]) + (weight.n,), dtype=torch.float32, device=x.device)
        self._check(L.kq_linear(self._ctx, weight.handle, x.data_ptr(), _tensor_dtype_code(x),
                                bias.data_ptr(), out.data_ptr(), m))
        return out

    def linear_multi(self, x, weights, biases, outs=None):
        """Several weights on the same x in one launch (q/k/v, gate/up)."""
        torch = _torch()
        x = x.contiguous()
        k = weights[0].k
        m = x.numel() // k
        if outs is None:
            outs = [torch.empty(tuple(x.shape[:-1]) + (w.n,), dtype=torch.float32, device=x.device)
                    for w in weights]
        cnt = len(weights)
        arr = ctypes.c_uint64 * cnt
        self._check(L.kq_linear_multi(
            self._ctx, cnt, arr(*[w.handle for w in weights]), x.data_ptr(), _tensor_dtype_code(x),
            arr(*[b.data_ptr() for b in biases]), arr(*[o.data_ptr() for o in outs]), m))
        return outs

    def linear_tc(self, x, weights, biases, outs=None):
        """linear_multi on the tcgen05 tensor cores (kq_linear_tc): 5..16 binary16 rows or 5..8
        f32 / bf16 rows, tiled int4 weights; raises KQ_ERR_UNSUPPORTED for anything else."""
        torch = _torch()
        x = x.contiguous()
        k = weights[0].k
        m = x.numel() // k
        if outs is None:
            outs = [torch.empty(tuple(x.shape[:-1]) + (w.n,), dtype=torch.float32, device=x.device)
                    for w in weights]
        cnt = len(weights)
        arr = ctypes.c_uint64 * cnt
        self._check(L.kq_linear_tc(
            self._ctx, cnt, arr(*[w.handle for w in weights]), x.data_ptr(), _tensor_dtype_code(x),
            arr(*[b.data_ptr() for b in biases]), arr(*[o.data_ptr() for o in outs]), m))
        return outs

    # -- the matmul's neighbours in a decoder layer -------------------------------------------
    def rms_norm(self, x, weight, eps: float, out=None):
        """out = x * rsqrt(mean(x^2, last dim) + eps) * weight, f32 (the reference's rms_norm op)."""
        torch = _torch()
        if x.dtype != torch.float32 or weight.dtype != torch.float32 or weight.numel() != x.shape[-1]:
            raise KqError(2, "rms_norm takes f32 x [..., dim] and an f32 weight [dim]")
        x = x.contiguous()
        dim = x.shape[-1]
        if out is None:
            out = torch.empty_like(x)
        self._check(L.kq_rms_norm(self._ctx, x.data_ptr(), weight.data_ptr(), float(eps), out.data_ptr(),
                                  x.numel() // dim if dim else 0, dim))
        return out

    def silu_mul(self, gate, up, out=None):
        """out = (gate * sigmoid(gate)) * up, f32 elementwise (the reference's SiLU pair followed by mul)."""
        torch = _torch()
        if gate.dtype != torch.float32 or up.dtype != torch.float32 or gate.shape != up.shape:
            raise KqError(2, "silu_mul takes two f32 tensors of one shape")
        if out is None:
            out = torch.empty_like(gate)
        self._check(L.kq_silu_mul(self._ctx, gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel()))
        return out

    def add(self, a, b, out=None):
        torch = _torch()
        if a.dtype != torch.float32 or b.dtype != torch.float32 or a.shape != b.shape:
            raise KqError(2, "add takes two f32 tensors of one shape")
        if out is None:
            out = torch.empty_like(a)
        self._check(L.kq_add(self._ctx, a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel()))
        return out

    def linear_fused(self, x, weights, biases, outs=None, norm_weight=None, eps: float = 0.0, residual=None,
                     swiglu: bool = False, reduce: bool = False):
        """[rms_norm ->] linear(s) [-> silu(gate) * up] [-> sum over ranks] [-> + residual] (kq_linear_fused).
        `weights` / `biases` are lists; with swiglu=True they are (gate, up) and there is one output."""
        if outs is not None:
            done = _fast.linear_fused(self._ctx_addr, [w.handle for w in weights], weights[0].k, x, biases, outs, norm_weight, float(eps),
                                      residual, (1 if swiglu else 0) | (2 if reduce else 0))
            if done is not None:
                return self._done(done)
        torch = _torch()
        x = x.contiguous()
        k = weights[0].k
        if x.shape[-1] != k:
            raise KqError(2, f"linear_fused: x[..., {x.shape[-1]}] does not match k={k}")
        m = x.numel() // k if k else 0
        n_out = 1 if swiglu else len(weights)
        if outs is None:
            outs = [torch.empty(tuple(x.shape[:-1]) + (weights[i].n,), dtype=torch.float32, device=x.device)
                    for i in range(n_out)]
        cnt = len(weights)
        arr = ctypes.c_uint64 * cnt
        out_ptrs = [outs[i].data_ptr() if i < len(outs) else 0 for i in range(cnt)]
        flags = (1 if swiglu else 0) | (2 if reduce else 0)
        self._check(L.kq_linear_fused(
            self._ctx, cnt, arr(*[w.handle for w in weights]), x.data_ptr(), _tensor_dtype_code(x),
            norm_weight.data_ptr() if norm_weight is not None else 0, float(eps),
            arr(*[b.data_ptr() for b in biases]), residual.data_ptr() if residual is not None else 0,
            arr(*out_ptrs), m, flags))
        return outs

    def linear_host(self, x: np.ndarray, weight: Weight, bias) -> np.ndarray:
        """Host-buffer round trip: numpy x in, numpy f32 out (copies inside the call)."""
        x = np.ascontiguousarray(x)
        if x.dtype not in _NP_DTYPES:
            raise KqError(1, f"host activations must be float32 / float16, got {x.dtype}")
        if x.shape[-1] != weight.k:
            raise KqError(2, f"linear: x[..., {x.shape[-1]}] does not match W[{weight.n},{weight.k}]")
        m = x.size // weight.k
        out = np.empty(x.shape[:-1] + (weight.n,), np.float32)
        self._check(L.kq_linear_host(self._ctx, weight.handle, x.ctypes.data, _NP_DTYPES[x.dtype],
                                     bias.data_ptr(), out.ctypes.data, m))
        return out

    # -- the attention half of a decoder layer --------------------------------------------------
    def rope(self, x, positions, rope: Rope, out=None):
        """x [tokens, heads, head_dim] (f32 / f16 / bf16, tokens may be strided) rotated to positions (CUDA int32 [tokens])."""
        done = _fast.rope(self._ctx_addr, x, positions, rope.args, out)
        if done is not None:
            return self._done(done)
        torch = _torch()
        tokens, heads, dim = x.shape
        px, stride = _rows(x, heads, dim, "x")
        if positions.dtype != torch.int32 or not positions.is_cuda or positions.numel() != tokens or not positions.is_contiguous():
            raise KqError(2, f"positions must be a contiguous CUDA int32 tensor [{tokens}]")
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=x.dtype, device=x.device)
        elif out.dtype != x.dtype or out.shape != x.shape:
            raise KqError(2, "out must have x's type and shape")
        po, out_stride = _rows(out, heads, dim, "out")
        self._check(L.kq_rope(self._ctx, px, _tensor_dtype_code(x), tokens, heads, dim, stride, positions.data_ptr(), *rope.args, po, out_stride))
        return out

    def kv_cache(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int, pool=None) -> KvCache:
        """Pages for keys and values in 4 bits; pool: the caller's uint8 CUDA memory of kq_cache_bytes() bytes (None: allocated)."""
        torch = _torch()
        need = int(L.kq_cache_bytes(pages, page_tokens, kv_heads, head_dim))
        if pool is None:
            pool = torch.zeros((pages, kv_heads, need // max(1, pages * kv_heads)), dtype=torch.uint8, device=self.device)
            torch.cuda.current_stream(self.device).synchronize()  # the first append may run on another stream than torch's current one
        if pool.dtype != torch.uint8 or not pool.is_cuda or not pool.is_contiguous() or pool.numel() < need:
            raise KqError(2, f"the pool must be {need} bytes of contiguous CUDA uint8 memory")
        handle = ctypes.c_uint64(0)
        self._check(L.kq_cache_create(self._ctx, pool.data_ptr(), pages, page_tokens, kv_heads, head_dim, ctypes.byref(handle)))
        return KvCache(self, handle.value, pool, pages, page_tokens, kv_heads, head_dim)

    def cache_append(self, cache: KvCache, k, v, batch: CacheBatch, rope: "Rope | None" = None) -> None:
        """Stores the new tokens' keys (rotated on the way) and values [tokens, kv_heads, head_dim] in the cache's pages."""
        done = _fast.cache_append(self._ctx_addr, cache.handle, cache.kv_heads, cache.head_dim, k, v, batch.args,
                                  rope.args if rope is not None else None)
        if done is not None:
            return self._check(done)
        if k.shape[0] != batch.tokens or v.shape[0] != batch.tokens or k.dtype != v.dtype:
            raise KqError(2, f"k and v must be [{batch.tokens}, {cache.kv_heads}, {cache.head_dim}] of one type")
        pk, k_stride = _rows(k, cache.kv_heads, cache.head_dim, "k")
        pv, v_stride = _rows(v, cache.kv_heads, cache.head_dim, "v")
        self._check(L.kq_cache_append(self._ctx, cache.handle, pk, k_stride, pv, v_stride, _tensor_dtype_code(k), *batch.args,
                                      *(rope.args if rope is not None else _NO_ROPE)))

    def cache_read(self, cache: KvCache, batch: CacheBatch):
        """(k, v) f32 [tokens, kv_heads, head_dim]: what the cache holds for the new tokens of `batch`."""
        done = _fast.cache_read(self._ctx_addr, cache.handle, cache.kv_heads, cache.head_dim, self.index, batch.args)
        if done is not None:
            return self._done(done)
        torch = _torch()
        k, v = (torch.empty((batch.tokens, cache.kv_heads, cache.head_dim), dtype=torch.float32, device=self.device) for _ in range(2))
        self._check(L.kq_cache_read(self._ctx, cache.handle, *batch.args, k.data_ptr(), v.data_ptr()))
        return k, v

    def cache_attention(self, cache: KvCache, q, batch: CacheBatch, scale: "float | None" = None, window: int = 0,
                        rope: "Rope | None" = None, out=None, shared: "SharedPrefixes | None" = None, selected=None):
        """Causal attention of q [tokens, heads, head_dim] (f32 / f16 / bf16, rotated on the way) over each sequence's keys
        in the cache, the last `window` of them if given; scale defaults to head_dim^-0.5.  Returns q's type.
        shared: what groups of the sequences have in common is read once.  selected: each row sees the tokens of the pages that
        cache_select chose for it."""
        if scale is None:
            scale = cache.head_dim ** -0.5
        if window < 0:
            raise KqError(2, f"window {window}: a number of keys, 0 for all")
        window = min(int(window), 0xFFFFFFFF)  # the ABI's number has 32 bits; no sequence is longer
        angles = rope.args if rope is not None else None
        if shared is not None or selected is not None:
            _batch_here(self.index, batch, rope)
        if shared is None and selected is None:
            done = _fast.cache_attention(self._ctx_addr, cache.handle, cache.head_dim, q, batch.args, batch.most, scale, window, angles, out)
        elif selected is None:
            done = _fast.cache_attention_shared(self._ctx_addr, cache.handle, cache.head_dim, q, batch.args, batch.most, shared.args, scale, window, angles, out, self.index) \
                if shared.index == self.index else None
        elif window or shared is not None:
            raise KqError(2, "selected pages are all that a row sees: no window, no shared prefixes")
        else:
            done = _fast.cache_attention_selected(self._ctx_addr, cache.handle, cache.kv_heads, cache.head_dim, q, batch.args, selected, scale, angles, out, self.index)
        if done is not None:
            return self._done(done)
        if shared is not None:
            _on_device(self.index, q=q, first=shared.first, out=q if out is None else out)
        if selected is not None:
            _on_device(self.index, q=q, selected=selected, out=q if out is None else out)
        torch = _torch()
        heads, dim = int(q.shape[1]), cache.head_dim
        if q.shape[0] != batch.tokens:
            raise KqError(2, f"q must have {batch.tokens} rows")
        pq, q_stride = _rows(q, heads, dim, "q")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif out.dtype != q.dtype or out.shape != q.shape:
            raise KqError(2, "out must have q's type and shape")
        po, out_stride = _rows(out, heads, dim, "out")
        head = (self._ctx, cache.handle, pq, q_stride, _tensor_dtype_code(q), heads, *batch.args)
        tail = (*(rope.args if rope is not None else _NO_ROPE), po, out_stride)
        if selected is not None:
            if selected.dtype != torch.int32 or not selected.is_cuda or not selected.is_contiguous() or selected.dim() != 3 or \
                    tuple(selected.shape[:2]) != (batch.tokens, cache.kv_heads):
                raise KqError(2, f"selected must be a contiguous CUDA int32 tensor [{batch.tokens}, {cache.kv_heads}, budget]")
            self._check(L.kq_cache_attention_selected(*head, selected.data_ptr(), selected.shape[2], float(scale), *tail))
        elif shared is not None:
            self._check(L.kq_cache_attention_shared(*head, batch.most, *shared.args, float(scale), window, *tail))
        else:
            self._check(L.kq_cache_attention(*head, batch.most, float(scale), window, *tail))
        return out

    # -- pages that a query selects ---------------------------------------------------------------
    def cache_summaries(self, cache: KvCache) -> CacheSummaries:
        """Empty summaries for the pages of a cache."""
        torch = _torch()
        shape = (cache.pages, cache.kv_heads, 2)
        made = CacheSummaries(torch.zeros((*shape, cache.head_dim), dtype=torch.int8, device=self.device), torch.zeros(shape, device=self.device))
        torch.cuda.current_stream(self.device).synchronize()  # the first call may run on another stream than torch's current one
        return made

    def cache_summarize(self, cache: KvCache, summaries: CacheSummaries, batch: CacheBatch) -> None:
        """Brings the summaries of the pages that the batch's new tokens are in up to date (behind cache_append)."""
        summaries.check(cache, self.index)
        _batch_here(self.index, batch)
        done = _fast.cache_summarize(self._ctx_addr, cache.handle, summaries.args, batch.args)
        if done is not None:
            return self._check(done)
        self._check(L.kq_cache_summarize(self._ctx, cache.handle, *summaries.args, *batch.args))

    def cache_select(self, cache: KvCache, summaries: CacheSummaries, q, batch: CacheBatch, budget: int, first: int = 1, last: int = 1,
                     rope: "Rope | None" = None, out=None):
        """Up to `budget` pages for every row of q [tokens, heads, head_dim] and kv head, int32 [tokens, kv_heads, budget]: ascending indices into
        the sequence's pages, -1 behind them; always the first `first` and the last `last` ones, then those whose summaries promise most."""
        summaries.check(cache, self.index)
        _batch_here(self.index, batch, rope)
        done = _fast.cache_select(self._ctx_addr, cache.handle, cache.kv_heads, cache.head_dim, summaries.args, q, batch.args, budget, first, last,
                                  rope.args if rope is not None else None, out, self.index)
        if done is not None:
            return self._done(done)
        _on_device(self.index, q=q, out=q if out is None else out)
        torch = _torch()
        heads, dim = int(q.shape[1]), cache.head_dim
        if q.shape[0] != batch.tokens:
            raise KqError(2, f"q must have {batch.tokens} rows")
        if not (0 < budget <= 1 << 20 and 0 <= first <= budget and 0 <= last <= budget):
            raise KqError(2, f"{budget} pages, the first {first} and the last {last} of them always: 1..2^20, no more than all")
        pq, q_stride = _rows(q, heads, dim, "q")
        shape = (batch.tokens, cache.kv_heads, int(budget))
        if out is None:
            out = torch.empty(shape, dtype=torch.int32, device=q.device)
        elif out.dtype != torch.int32 or not out.is_cuda or not out.is_contiguous() or tuple(out.shape) != shape:
            raise KqError(2, f"out must be a contiguous CUDA int32 tensor {list(shape)}")
        self._check(L.kq_cache_select(self._ctx, cache.handle, *summaries.args, pq, q_stride, _tensor_dtype_code(q), heads, *batch.args, budget, first, last,
                                      *(rope.args if rope is not None else _NO_ROPE), out.data_ptr()))
        return out

    # -- pages that sequences share ---------------------------------------------------------------
    def cache_pages(self, sequences: int, longest: int, pages: int, page_tokens: int) -> CachePages:
        """An empty book of `pages` pages for `sequences` sequences of up to `longest` tokens."""
        torch = _torch()
        width = (int(longest) + page_tokens - 1) // page_tokens
        book = CachePages(torch.full((sequences, width), -1, dtype=torch.int32, device=self.device), *(
            torch.zeros(n, dtype=torch.int32, device=self.device) for n in (sequences, pages)), page_tokens)
        torch.cuda.current_stream(self.device).synchronize()  # the first call may run on another stream than torch's current one
        return book

    def pages_grow(self, book: CachePages, news) -> None:
        """Sequence b gets the pages of its next news[b] tokens (CUDA int32) and is that much longer."""
        book.counted = False
        done = _fast.pages_grow(self._ctx_addr, book.args, news, self.index) if book.index == self.index else None
        if done is not None:
            return self._check(done)
        _on_device(self.index, table=book.table, news=news)
        self._check(L.kq_pages_grow(self._ctx, *book.args, _per_sequence(news, book, "news")))

    def pages_fork(self, book: CachePages, parents, keep=None):
        """Every sequence b becomes the first min(keep[b], length) tokens of parents[b] (CUDA int32; negative: it ends), all at once.
        Returns the pairs [sequences, 2] of pages to copy, for pages_copy."""
        done = _fast.pages_fork(self._ctx_addr, book.args, parents, keep, self.index) if book.index == self.index else None
        if done is not None:
            return self._pairs(book, self._done(done))
        _on_device(self.index, table=book.table, parents=parents, keep=parents if keep is None else keep)
        torch = _torch()
        pairs = torch.empty((book.sequences, 2), dtype=torch.int32, device=self.device)
        self._check(L.kq_pages_fork(self._ctx, *book.args, _per_sequence(parents, book, "parents"),
                                    _per_sequence(keep, book, "keep") if keep is not None else 0, pairs.data_ptr()))
        return self._pairs(book, pairs)

    @staticmethod
    def _pairs(book: CachePages, pairs):
        """Pairs that a call made: pages_copy needs no report for them."""
        pairs.end_by_themselves, book.counted = True, True
        return pairs

    def pages_compact(self, book: CachePages):
        """Moves the pages in use to the lowest numbers; returns the pairs [pages, 2] (from, to), for pages_copy."""
        done = _fast.pages_compact(self._ctx_addr, book.args, self.index) if book.index == self.index else None
        if done is not None:
            return self._pairs(book, self._done(done))
        _on_device(self.index, table=book.table)
        torch = _torch()
        pairs = torch.empty((book.pages, 2), dtype=torch.int32, device=self.device)
        self._check(L.kq_pages_compact(self._ctx, *book.args, pairs.data_ptr()))
        return self._pairs(book, pairs)

    def pages_copy(self, book: CachePages, pairs, pools) -> None:
        """Copies the pages of a fork or compact in every pool: KvCaches, CacheSummaries, or CUDA tensors whose first axis is the pages.  pairs: what the
        call returned, whatever was called since; of other tensors as many as the book's report says, which a pages_grow has overwritten (refused)."""
        of_a_call = getattr(pairs, "end_by_themselves", False)
        if not of_a_call and not book.counted:
            raise KqError(2, "pages_grow has overwritten the number of pairs in the report: give the tensor that pages_fork or pages_compact returned")
        args = book.args_for_pairs if of_a_call else book.args
        given, pools = pools, []
        for pool in given:
            if isinstance(pool, KvCache):
                pools.append(pool.page_args)
            elif isinstance(pool, CacheSummaries):
                pools += pool.codes, pool.scales
            else:
                pools.append(pool)
        done = _fast.pages_copy(self._ctx_addr, args, pairs, pools, self.index) if book.index == self.index else None
        if done is not None:
            return self._check(done)
        _on_device(self.index, table=book.table, pairs=pairs)
        for pool in given:
            _on_device(self.index, pool=pool.pool if isinstance(pool, KvCache) else pool.codes if isinstance(pool, CacheSummaries) else pool)
        torch = _torch()
        if pairs.dtype != torch.int32 or not pairs.is_cuda or not pairs.is_contiguous() or pairs.dim() != 2 or pairs.shape[1] != 2:
            raise KqError(2, "pairs must be a contiguous CUDA int32 tensor [pairs, 2]")
        addresses, sizes = [], []
        for pool in pools:
            if isinstance(pool, tuple):
                pages, each, address, _ = pool
            elif not pool.is_cuda or not pool.is_contiguous() or pool.dim() == 0:
                raise KqError(2, "a pool is a KvCache or a contiguous CUDA tensor [pages, ...]")
            else:
                pages, address = int(pool.shape[0]), pool.data_ptr()
                each = pool.numel() // max(pages, 1) * pool.element_size()
            if pages < book.pages:
                raise KqError(2, f"a pool of {pages} pages for a book of {book.pages}")
            addresses.append(address)
            sizes.append(each)
        n = len(addresses)
        self._check(L.kq_pages_copy(self._ctx, n, (ctypes.c_uint64 * n)(*addresses), (ctypes.c_uint64 * n)(*sizes), book.pages, pairs.data_ptr(),
                                    pairs.shape[0], args[-1]))

    # -- replayable plans -------------------------------------------------------
    def graph_begin(self) -> None:
        self._check(L.kq_graph_begin(self._ctx))

    def graph_end(self) -> int:
        g = ctypes.c_uint64(0)
        self._check(L.kq_graph_end(self._ctx, ctypes.byref(g)))
        return g.value

    def graph_launch(self, g: int) -> None:
        self._check(L.kq_graph_launch(self._ctx, g))

    def graph_free(self, g: int) -> None:
        self._check(L.kq_graph_free(self._ctx, g))

    def plan_begin(self) -> None:
        """Start recording linears (and host copies) into a fused plan; nothing runs until launch."""
        self._check(L.kq_plan_begin(self._ctx))

    def plan_end(self) -> int:
        h = ctypes.c_uint64(0)
        self._check(L.kq_plan_end(self._ctx, ctypes.byref(h)))
        return h.value

    def plan_launch(self, plan: int) -> None:
        self._check(L.kq_plan_launch(self._ctx, plan))

    def plan_profile(self, plan: int) -> np.ndarray:
        """One profiled launch of a fused plan: uint64 [ctas, ops, slots] of GPU-timer stamps (ns);
        see kq_plan_profile for the meaning of the slots."""
        ctas, ops, slots = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint32()
        self._check(L.kq_plan_profile(self._ctx, plan, None, 0, ctypes.byref(ctas), ctypes.byref(ops), ctypes.byref(slots)))
        out = np.zeros((ctas.value, ops.value, slots.value), np.uint64)
        self._check(L.kq_plan_profile(self._ctx, plan, out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint64)), out.size,
                                      ctypes.byref(ctas), ctypes.byref(ops), ctypes.byref(slots)))
        return out

    def plan_free(self, plan: int) -> None:
        self._check(L.kq_plan_free(self._ctx, plan))

    # -- tensor-parallel exchange ---------------------------------------------------------
    def connect_ranks(self, rank: int, world: int, max_bytes: int, process_group=None) -> None:
        """Creates this rank's exchange buffer and connects it to every peer's; the 64-byte
        IPC handles travel through torch.distributed (plumbing only)."""
        torch = _torch()
        import torch.distributed as dist
        handle = (ctypes.c_uint8 * 64)()
        self._check(L.kq_comm_create(self._ctx, rank, world, int(max_bytes), handle))
        on_device = dist.get_backend(process_group) == "nccl"  # a gloo group moves host tensors
        mine = torch.tensor(list(handle), dtype=torch.uint8, device=self.device if on_device else "cpu")
        gathered = [torch.empty_like(mine) for _ in range(world)]
        dist.all_gather(gathered, mine, group=process_group)
        blob = bytes(torch.cat(gathered).cpu().numpy().tobytes())
        buf = (ctypes.c_uint8 * len(blob)).from_buffer_copy(blob)
        self._check(L.kq_comm_connect(self._ctx, buf))
        dist.barrier(group=process_group)

    def all_reduce(self, t) -> None:
        """In-place f32 sum over the connected ranks (one peer-memory kernel, rank-ordered)."""
        torch = _torch()
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise KqError(1, "all_reduce takes a contiguous f32 tensor")
        self._check(L.kq_all_reduce(self._ctx, t.data_ptr(), t.numel()))

    def linear_reduce(self, x, weight: Weight, bias, out=None):
        """Row-parallel linear: every rank passes its K shard; out = sum over ranks + bias, the
        same bits on every rank (one kernel for decode shapes, else linear + all_reduce)."""
        torch = _torch()
        if x.shape[-1] != weight.k:
            raise KqError(2, f"x[..., {x.shape[-1]}] does not match the shard's k={weight.k}")
        m = x.numel() // weight.k if weight.k else 0
        if out is None:
            out = torch.empty(tuple(x.shape[:-1]) + (weight.n,), dtype=torch.float32, device=x.device)
        self._check(L.kq_linear_reduce(self._ctx, weight.handle, x.data_ptr(), _tensor_dtype_code(x), bias.data_ptr(),
                                       out.data_ptr(), m))
        return out

    def timer_start(self) -> None:
        self._check(L.kq_timer_start(self._ctx))

    def timer_stop(self) -> float:
        ms = ctypes.c_float(0)
        self._check(L.kq_timer_stop(self._ctx, ctypes.byref(ms)))
        return float(ms.value)


def acquire_gpu(device: int = 0, **kwargs) -> Gpu:
    return Gpu(device, **kwargs)
