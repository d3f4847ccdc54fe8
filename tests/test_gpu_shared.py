"""Attention of sequences that begin alike against the same formula in 64 bits, each sequence by itself.  As in tests/test_gpu_attend.py,
whatever a query must not see is NaN."""
import math

import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests.test_gpu_attend import KINDS, gpu, one_stream  # noqa: F401
from tests.test_gpu_cache import dev

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Groups:
    """groups: (common tokens, tokens of each member behind them, None for an idle one); a negative number of common tokens: sequences of
    no group, so many tokens each.  Made by forking, so that whole pages are shared and the others are copies."""

    def __init__(self, gpu, groups, page, kv_heads, dim, seed=0, spread=1.0, mean=0.3):
        import karume_b200 as kb
        self.gpu, self.dim, self.page = gpu, dim, page
        first, common, lengths, parents, n = [], [], [], [], 0
        for tokens, members in groups:
            if tokens >= 0:
                first.append(n)
                common.append(tokens)
            parents += [n] * len(members)
            lengths += [0 if m is None else max(tokens, 0) + m for m in members]
            n += len(members)
        # groups are neighbours in `first`: sequences of none, in the middle, are groups with nothing in common
        starts, kept, at = [], [], 0
        for tokens, members in groups:
            if tokens >= 0 or (starts and at < n):
                starts.append(at)
                kept.append(max(tokens, 0))
            at += len(members)
        end = n
        if groups[-1][0] < 0 and starts:
            end = starts.pop()
            kept.pop()
        self.first, self.common = starts + [end], kept
        self.lengths, width = lengths, -(-max(max(lengths), 1) // page)
        pages = sum(-(-n // page) + 1 for n in lengths) + sum(-(-max(t, 0) // page) for t, _ in groups) + 2
        book = gpu.cache_pages(n, width * page, pages, page)
        shape = (pages, kv_heads, page * (dim + 8))
        pool = np.zeros(shape, np.uint8)
        pool[..., page * dim:] = np.tile(np.array([0x00, 0x7E], np.uint8), 4 * page)
        self.cache = gpu.kv_cache(pages, page, kv_heads, dim, pool=dev(pool))
        gen = torch.Generator(device="cuda").manual_seed(seed)
        leads = []
        for tokens, members in groups:
            leads += [max(tokens, 0)] + [0] * (len(members) - 1)
        idle = [m is None for _, members in groups for m in members]

        def grow(news):
            gpu.pages_grow(book, i32(news))
            if sum(news):
                batch = kb.CacheBatch(book.table, book.lengths, i32([0] + news).cumsum(0).to(torch.int32), tokens=sum(news))
                k = torch.randn(sum(news), kv_heads, dim, generator=gen, device="cuda") * spread + mean
                v = torch.randn(sum(news), kv_heads, dim, generator=gen, device="cuda") + mean
                gpu.cache_append(self.cache, k, v, batch)

        grow(leads)
        gpu.pages_copy(book, gpu.pages_fork(book, i32([-1 if gone else p for p, gone in zip(parents, idle)])), [self.cache])
        assert book.report.tolist()[0] == 0
        grow([n - have for n, have in zip(lengths, book.lengths.tolist())])
        assert book.report.tolist()[0] == 0 and book.lengths.tolist() == lengths
        self.book, self.table, self.length = book, book.table, book.lengths
        self.cut = np.concatenate([[0], np.cumsum(lengths)])
        if sum(lengths):
            self.k, self.v = gpu.cache_read(self.cache, kb.CacheBatch(book.table, book.lengths, dev(self.cut.astype(np.int32)), tokens=sum(lengths)))

    def prefixes(self, first=None, common=None):
        import karume_b200 as kb
        return kb.SharedPrefixes(i32(first or self.first), i32(common or self.common), least=0)

    def call(self, kind, news, heads, window=0, rotary=0, interleaved=False, scale=None, strided=False, padding=0, prefixes=None, gpu=None, cache=None, most=0):
        import karume_b200 as kb
        gpu, tokens = gpu or self.gpu, sum(news) + padding
        gen = torch.Generator(device="cuda").manual_seed(heads + tokens)
        q = torch.randn(tokens, heads + (2 if strided else 0), self.dim, generator=gen, device="cuda").to(ref.TYPES[kind])[:, :heads]
        table = kb.rope_table(max(max(self.lengths), 1), rotary) if rotary else None
        starts = None if news == [1] * len(news) and not padding else i32(np.concatenate([[0], np.cumsum(news)]).tolist())
        batch = kb.CacheBatch(self.table, self.length, starts, tokens=tokens, most=most or max(news))
        out = torch.full((tokens, heads + (1 if strided else 0), self.dim), -7.0, dtype=q.dtype, device="cuda")
        got = gpu.cache_attention(cache or self.cache, q, batch, scale=scale, window=window, rope=kb.Rope(dev(table), interleaved) if rotary else None,
                                  out=out[:, :heads] if strided else None, shared=prefixes or self.prefixes())
        gpu.sync()
        if strided:
            assert bool((out[:, heads:] == -7).all())
        return q, got, table

    def check(self, kind, news, heads, window=0, rotary=0, interleaved=False, scale=None, padding=0, **more):
        q, got, table = self.call(kind, news, heads, window, rotary, interleaved, scale, padding=padding, **more)
        again = self.call(kind, news, heads, window, rotary, interleaved, scale, padding=padding, **more)[1]
        assert torch.equal(got, again)
        at, off, norm = 0, 0.0, 0.0
        for b, n in enumerate(news):
            length, qb, mine = self.lengths[b], q[at:at + n].float(), got[at:at + n].double()
            at += n
            early = max(n - length, 0)
            assert bool((mine[:early] == 0).all())
            qb, mine = qb[early:], mine[early:]
            if len(qb) == 0:
                continue
            if rotary:
                qb = torch.from_numpy(ref.rotate(qb.cpu().numpy(), table, np.arange(length - len(qb), length), interleaved)).cuda()
            part = slice(self.cut[b], self.cut[b + 1])
            want, reach, largest = ref.attend(qb.double(), self.k[part].double(), self.v[part].double(), scale or self.dim ** -0.5, window)
            d = (mine - want).abs()
            allowed = ref.allowed(kind, want, reach, largest)
            assert bool((d <= allowed).all()), (kind, b, float((d / allowed).max()))
            off, norm = off + float((d * d).sum()), norm + float((want * want).sum())
        assert bool((got[at:] == 0).all())
        if norm:
            assert math.sqrt(off / norm) <= {"f32": 1e-5, "f16": 2e-3, "bf16": 5e-3}[kind], math.sqrt(off / norm)

    def free(self):
        self.cache.free()


@KINDS
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 4, 4, 16), (128, 8, 2, 64), (256, 4, 2, 32), (128, 24, 1, 128), (64, 6, 2, 256), (128, 32, 8, 64)])
def test_groups_of_many_kinds(gpu, kind, dim, heads, kv_heads, page):  # noqa: F811
    g = Groups(gpu, [(300, [1, 40, 7]), (5 * page, [3, None, 1, page]), (-1, [50, 1]), (1, [9, 9]), (page + 1, [2 * page])], page, kv_heads, dim, seed=dim + heads)
    n = len(g.lengths)
    g.check(kind, [1] * n, heads, rotary=dim)
    g.check(kind, [1] * n, heads, window=60)
    g.check(kind, [1, 5, 3, 2, 2, 1, 9, 4, 1, 3, 0, 4], heads, rotary=dim // 2, interleaved=True, padding=3, strided=True)
    g.check(kind, [1, 5, 3, 2, 2, 1, 9, 4, 1, 3, 0, 4], heads, window=7, scale=0.2)
    g.free()


@KINDS
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_behind_a_long_beginning(gpu, kind, dim):  # noqa: F811
    """So many rows that the common keys are the tensor cores' of whole blocks of rows; new tokens few and many; keys that several blocks share."""
    members = [1, 30, 5, 77, 12, 64, 3, 3, 100, 41, 8, 1, 2, 190, 16, 9, 33, 5, 6, 21]
    g = Groups(gpu, [(5003, members)], 64, 2, dim, seed=dim)
    g.check(kind, [1] * 20, 16, rotary=dim)
    g.check(kind, [1] * 20, 16, window=120)
    g.check(kind, [1] * 20, 16, window=4000)
    g.check(kind, [min(m, 12) for m in members], 8, rotary=dim, padding=1)
    g.check(kind, [min(m, 100) for m in members], 6, window=2500)
    g.check(kind, members, 4, rotary=dim // 2)
    g.free()


@KINDS
def test_so_many_groups_that_they_come_in_turns(gpu, kind):  # noqa: F811
    g = Groups(gpu, [(20 + i % 50, [1 + i % 3] * (1 + i % 2)) for i in range(300)], 16, 1, 64, seed=1)
    g.check(kind, [1] * len(g.lengths), 4, rotary=64)
    g.check(kind, [1] * len(g.lengths), 40)  # the other kernel
    g.free()


@KINDS
def test_large_and_small_groups_in_one_call(gpu, kind):  # noqa: F811
    """Few rows a group on the average, so that each group goes to the kernel for its rows; and boundaries for more groups than there are."""
    g = Groups(gpu, [(700, [3] * 30), (90, [5]), (-1, [40]), (400, [2, 90]), (33, [1]), (64, [7]), (640, [9] * 12), (20, [1]), (21, [2]), (22, [3]), (23, [4]),
                     (24, [5]), (25, [6])], 16, 2, 64, seed=11)
    n = len(g.lengths)
    g.check(kind, [1] * n, 8, rotary=64)
    g.check(kind, [1] * n, 8, window=300)
    g.check(kind, [min(2, m + 1) for m in range(n)], 12, padding=2)
    more = g.prefixes(first=g.first + [n] * (n - len(g.common)), common=g.common + [0] * (n - len(g.common)))
    g.check(kind, [1] * n, 8, rotary=64, prefixes=more)
    g.free()


@KINDS
@pytest.mark.parametrize("rows", ["few", "many"])
def test_beginnings_that_reach_into_the_new_tokens(gpu, kind, rows):  # noqa: F811
    """More tokens said to be common than are in front of a sequence's new ones: those count as its own."""
    heads = 4 if rows == "few" else 64
    g = Groups(gpu, [(200, [5, 30, 1, 9])], 16, 1, 64, seed=2)
    g.check(kind, [5, 40, 100, 9], heads)  # some of the common tokens are new
    g.check(kind, [5, 40, 100, 9], heads, window=50)
    g.check(kind, [205, 230, 201, 209], heads, rotary=64)
    g.check(kind, [300, 1, 1, 250], heads)  # rows in front of the first token
    for common in (200, 1 << 30, 0x7FFFFFFF, 17, 0, -5):
        if common <= 200:
            g.check(kind, [1] * 4, heads, prefixes=g.prefixes(common=[common]))
        else:  # said of sequences that are not alike so far: tokens are looked up for the first one, which has its own, and others NaN behind its end
            got = g.call(kind, [1] * 4, heads, prefixes=g.prefixes(common=[common]))[1]
            want = g.call(kind, [1] * 4, heads)[1]
            assert bool(torch.isfinite(got[0]).all()) and float((got[0] - want[0]).float().norm() / want[0].float().norm()) < 1e-2
    g.free()


def test_groups_that_are_none(gpu):  # noqa: F811
    """Boundaries out of order and outside the batch: results say nothing, but every call comes back and the next one is right."""
    g = Groups(gpu, [(100, [5, 30, 1]), (70, [2, 2])], 16, 2, 64, seed=3)
    for first in ([3, 0, 5], [-7, 3, 99], [5, 5, 5], [0, 1 << 30, 5], [4, 2, 1], [0, 0, 0], [-(1 << 31), 0x7FFFFFFF, 0]):
        for heads in (4, 64):
            for news in ([1] * 5, [3, 0, 1, 7, 2]):
                g.call("f32", news, heads, prefixes=g.prefixes(first=first))
                g.call("bf16", news, heads, window=9, prefixes=g.prefixes(first=first))
    g.check("f32", [1] * 5, 4)
    g.check("f32", [3, 0, 1, 7, 2], 64)
    # groups that leave out the first and the last sequences
    g.check("f32", [1] * 5, 4, prefixes=g.prefixes(first=[1, 3], common=[100]))
    g.check("bf16", [4, 2, 1, 1, 1], 64, prefixes=g.prefixes(first=[1, 3], common=[100]))
    g.free()


@KINDS
def test_scores_and_values_far_apart(gpu, kind):  # noqa: F811
    """The common keys count for nothing, or for all: weights that are many powers of two apart in the two sums."""
    for mean, spread in ((30.0, 1.0), (-30.0, 1.0), (0.0, 6.0)):
        g = Groups(gpu, [(500, [20, 1, 64, 300])], 64, 1, 128, seed=4, mean=mean, spread=spread)
        for heads in (4, 40):
            g.check(kind, [1] * 4, heads, scale=0.05)
        g.free()


def test_pages_that_are_none_reach_who_sees_them(gpu):  # noqa: F811
    g = Groups(gpu, [(100, [5, 30, 20])], 16, 1, 64, seed=5)
    table = g.table.clone()
    for heads in (4, 64):
        for kind in ("f32", "bf16"):
            want = g.call(kind, [1] * 3, heads, window=40)[1]
            g.table[0, 2] = -1  # tokens 32 .. 47: nobody's with a window of 40 (keys 66, 91, 81 and up)
            assert torch.equal(g.call(kind, [1] * 3, heads, window=40)[1], want)
            assert bool(torch.isnan(g.call(kind, [1] * 3, heads)[1]).all())
            assert bool(torch.isnan(g.call(kind, [1] * 3, heads, window=70)[1][0]).all()) and bool(torch.isfinite(g.call(kind, [1] * 3, heads, window=70)[1][1:]).all())
            g.table.copy_(table)
            g.table[1, 7] = 1 << 30  # its own tokens 112 .. 127
            got = g.call(kind, [1] * 3, heads)[1]
            assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[[0, 2]]).all())
            g.table.copy_(table)
    g.free()


def test_little_scratch(gpu):  # noqa: F811
    """Too little for the sums of the common keys: every sequence reads all of its own."""
    import karume_b200 as kb
    g = Groups(gpu, [(300, [5, 30, 1, 9]), (64, [70, 3])], 16, 2, 64, seed=6)
    for size in (4096, 20000, 70000, 1 << 20, 8 << 20):
        small = kb.Gpu(0, workspace_bytes=size)
        cache = small.kv_cache(g.cache.pages, 16, 2, 64, pool=g.cache.pool)
        for kind in ("f32", "f16"):
            g.check(kind, [1] * 6, 8, rotary=64, gpu=small, cache=cache)
            g.check(kind, [5, 9, 1, 2, 40, 3], 20, gpu=small, cache=cache)
        small.destroy()
    g.free()


def test_what_reading_once_has_to_save(gpu):  # noqa: F811
    """Less saved than asked for: every sequence reads its own; by what the device arrays say, in a recorded call too.  (Where the work is cut
    differs from a call without groups: sums of f32, each relative to 2^-24 of some hundreds.)"""
    import karume_b200 as kb
    g = Groups(gpu, [(300, [5, 30, 1, 9]), (64, [70, 3])], 16, 2, 64, seed=9)
    saved = (3 * 300 + 64) * 2 * 72
    for heads in (8, 80):
        q, batch = torch.randn(6, heads, 64, device="cuda"), kb.CacheBatch(g.table, g.length)
        alone, once = (gpu.cache_attention(g.cache, q, batch, shared=s) for s in (None, g.prefixes()))
        gpu.sync()
        assert not torch.equal(alone, once)
        far = {}
        for least in (None, saved, 1, 1 << 40):
            far[least] = gpu.cache_attention(g.cache, q, batch, shared=kb.SharedPrefixes(g.prefixes().first, g.prefixes().tokens, least=least))
        gpu.sync()
        assert torch.equal(far[saved], once) and torch.equal(far[1], once) and torch.equal(far[None], far[1 << 40]) and not torch.equal(far[None], once)
        assert float((far[None] - alone).norm() / alone.norm()) < 1e-6
        prefixes, out = kb.SharedPrefixes(g.prefixes().first, g.prefixes().tokens, least=saved), torch.zeros_like(q)
        gpu.sync()
        gpu.graph_begin()
        gpu.cache_attention(g.cache, q, batch, shared=prefixes, out=out)
        graph = gpu.graph_end()
        for common, want in (([300, 64], once), ([299, 64], None), ([0, 64], None), ([300, 64], once)):
            prefixes.tokens.copy_(i32(common))
            gpu.graph_launch(graph)
            gpu.sync()
            g.check("f32", [1] * 6, heads, prefixes=prefixes)
            assert want is None or torch.equal(out, want)
        # below what is asked for, the sums are those of whole sequences but for where the work is cut
        prefixes.tokens.copy_(i32([299, 64]))
        gpu.graph_launch(graph)
        gpu.sync()
        assert float((out - alone).norm() / alone.norm()) < 1e-6
        gpu.graph_free(graph)
    g.free()


def test_recorded_calls_follow_the_lengths_and_share_scratch(gpu):  # noqa: F811
    import karume_b200 as kb
    g = Groups(gpu, [(300, [50, 30, 10, 90]), (128, [70, 13])], 16, 2, 64, seed=7)
    prefixes, length = g.prefixes(), g.length.clone()
    calls = []
    for kind, heads, new in (("f32", 8, 1), ("bf16", 64, 1), ("f16", 8, 6)):
        q = torch.randn(6 * new, heads, 64, device="cuda").to(ref.TYPES[kind])
        batch = kb.CacheBatch(g.table, length, i32([i * new for i in range(7)]) if new > 1 else None, tokens=6 * new, most=new)
        out = torch.zeros_like(q)
        gpu.sync()
        gpu.graph_begin()
        gpu.cache_attention(g.cache, q, batch, shared=prefixes, out=out)
        calls.append((q, batch, out, gpu.graph_end()))
    for lengths, common in ((g.lengths, g.common), ([310, 330, 306, 390, 135, 141], [300, 128]), ([310, 0, 306, 390, 135, 141], [150, 7]), (g.lengths, [0, 128])):
        length.copy_(i32(lengths))
        prefixes.tokens.copy_(i32(common))
        for _, _, _, graph in calls:  # one behind the other, nothing between
            gpu.graph_launch(graph)
        gpu.sync()
        for q, batch, out, _ in calls:
            recorded = out.clone()
            assert torch.equal(recorded, gpu.cache_attention(g.cache, q, batch, shared=prefixes))
    for _, _, _, graph in calls:
        gpu.graph_free(graph)
    g.free()


def test_refusals(gpu):  # noqa: F811
    import karume_b200 as kb
    g = Groups(gpu, [(30, [5, 3])], 16, 2, 64, seed=8)
    q, batch, good = torch.randn(2, 4, 64, device="cuda"), kb.CacheBatch(g.table, g.length), g.prefixes()
    for call in (lambda: kb.SharedPrefixes(i32([0, 2]), i32([3, 4])), lambda: kb.SharedPrefixes(i32([0, 2]).long(), i32([3])),
                 lambda: kb.SharedPrefixes(i32([0, 2]).cpu(), i32([3])), lambda: kb.SharedPrefixes(i32([0, 1, 2, 3])[::2], i32([3])),
                 lambda: kb.SharedPrefixes(i32([[0, 2]]), i32([3])),
                 lambda: gpu.cache_attention(g.cache, q, batch, shared=kb.SharedPrefixes(i32([0, 1, 2, 2]), i32([3, 3, 3]))),
                 lambda: gpu.cache_attention(g.cache, q[:1], batch, shared=good), lambda: gpu.cache_attention(g.cache, q[:, :3], batch, shared=good),
                 lambda: gpu.cache_attention(g.cache, q, batch, shared=good, window=-1), lambda: gpu.cache_attention(g.cache, q, batch, shared=good, scale=0.0)):
        with pytest.raises(kb.KqError):
            call()
    nothing = gpu.cache_attention(g.cache, q, batch, shared=kb.SharedPrefixes(i32([0]), i32([])))
    gpu.sync()
    assert torch.equal(nothing, gpu.cache_attention(g.cache, q, batch))
    tail = (1.0, 0, 0, 0, 0, 0, q.data_ptr(), 256)
    for groups, first, common in ((1, 0, good.tokens.data_ptr()), (1, good.first.data_ptr(), 0), (1, good.first.data_ptr() + 2, good.tokens.data_ptr())):
        assert kb.lib.kq_cache_attention_shared(gpu._ctx, g.cache.handle, q.data_ptr(), 256, 0, 4, *batch.args, 1, groups, first, common, 0, *tail) == 1
    for least in (-1, (1 << 64) - 1, 1 << 70):
        with pytest.raises(kb.KqError):
            kb.SharedPrefixes(good.first, good.tokens, least=least)
    g.free()


def test_calls_on_other_streams(gpu):  # noqa: F811
    """The whole chain on the library's own stream beside torch's default one, on a side stream, and on two contexts at once: the same results."""
    import karume_b200 as kb
    g = Groups(gpu, [(300, [5, 30, 1, 9])], 16, 2, 64, seed=10)
    table, length, pool, pages = g.table.clone(), g.length.clone(), g.cache.pool.clone(), g.cache.pages
    q0, prefixes = torch.randn(4, 8, 64, device="cuda"), g.prefixes()
    refs = g.book.refs.clone()
    torch.cuda.synchronize()

    def chain(on):
        """Everything that a step of branching sequences does, from fresh copies; torch and the library in turn."""
        book = kb.CachePages(table.clone(), length.clone(), refs.clone(), 16)
        mine = pool.clone()
        cache = on.kv_cache(pages, 16, 2, 64, pool=mine)
        pairs = on.pages_fork(book, i32([0, 1, 1, 3]), i32([301, 320, 307, 306]))
        on.pages_copy(book, pairs, [cache])
        on.pages_grow(book, i32([1, 1, 1, 1]))
        batch = kb.CacheBatch(book.table, book.lengths)
        k = q0[:, :2].contiguous() * 2
        on.cache_append(cache, k, k, batch)
        made = on.cache_summaries(cache)
        on.cache_summarize(cache, made, kb.CacheBatch(book.table, book.lengths, i32([0, 302, 623, 931, 1238]), tokens=1238))
        taken = on.cache_select(cache, made, q0, batch, 6)
        out = [on.cache_attention(cache, q0, batch, shared=prefixes), on.cache_attention(cache, q0.bfloat16(), batch, selected=taken), taken, book.table, book.refs, mine, pairs]
        return [t + 0 for t in out]

    want = chain(gpu)
    gpu.sync()
    before = torch.cuda.current_stream()
    side = torch.cuda.Stream()
    contexts = []
    for stream in (torch.cuda.default_stream(), side):
        torch.cuda.set_stream(stream)
        on = kb.Gpu(0)
        contexts.append((on, stream))
        got = chain(on)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), stream
    both = []
    for _ in range(20):  # enqueued on both, neither waits for the other
        for on, stream in contexts:
            torch.cuda.set_stream(stream)
            both.append(chain(on))
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    assert all(torch.equal(a, b) for got in both for a, b in zip(got, want))
    for on, _ in contexts:
        on.destroy()
    g.free()
