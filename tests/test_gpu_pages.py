"""Books of pages (growing, forking, cutting back, compacting) against the plain statement of tests/pages_reference.py: the same whole
numbers, whatever the calls; and the copies of pages that they ask for."""
import ctypes
import random

import numpy as np
import pytest
import torch

from tests.pages_reference import Book
from tests.test_gpu_cache import gpu, one_stream  # noqa: F401

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def same(book, want, what):
    torch.cuda.synchronize()
    assert book.report.tolist() == want.report, what
    assert book.lengths.tolist() == want.lengths, what
    assert book.refs.tolist() == want.refs, what
    assert book.table.tolist() == want.table, what


# one CTA has small books, a cluster the others; tables wider than a chunk of entries, more pages than a step of the cluster's scan
SIZES = [(1, 1, 1, 16), (3, 4, 9, 16), (8, 40, 200, 32), (70, 12, 600, 64), (5, 300, 1100, 16), (300, 33, 5000, 64), (1500, 9, 9000, 128), (40, 900, 70000, 256)]


@pytest.mark.parametrize("sequences,width,pages,page", SIZES)
def test_any_calls(gpu, sequences, width, pages, page):  # noqa: F811
    rng = random.Random(pages)
    book, want = gpu.cache_pages(sequences, width * page, pages, page), Book(sequences, width, pages, page)
    room, refused = width * page, set()
    for step in range(24):
        what = rng.choice(["grow", "grow", "fork", "fork", "fork", "compact"]) if step else "grow"
        if what == "grow":
            usual = max(1, min(room, 2 * pages * page // sequences) // 4)
            news = [rng.choice([0, 1, rng.randint(-5, usual)]) for _ in range(sequences)]
            news = [min(n, room - have) for n, have in zip(news, want.lengths)]
            if step % 7 == 3:
                news[rng.randrange(sequences)] += rng.choice([room, 0x7FFFFFFF - max(want.lengths) - max(news)])
            gpu.pages_grow(book, i32(news))
            want.grow(news)
        elif what == "fork":
            kind = rng.random()
            if kind < 0.3:  # all from a few
                parents = [rng.randrange(min(4, sequences)) for _ in range(sequences)]
            elif kind < 0.6:  # another order
                parents = rng.sample(range(sequences), sequences)
            else:
                parents = [rng.choice([b, b, rng.randrange(sequences), -1 - rng.randrange(3)]) for b in range(sequences)]
            if step % 11 == 5:
                parents[rng.randrange(sequences)] = sequences + rng.choice([0, 1 << 30])
            keep = None if rng.random() < 0.3 else [rng.choice([0x7FFFFFFF, rng.randint(-2, room)]) for _ in range(sequences)]
            pairs = gpu.pages_fork(book, i32(parents), i32(keep) if keep else None)
            assert pairs.tolist() == want.fork(parents, keep), (step, what)
        else:
            pairs = gpu.pages_compact(book)
            assert pairs.tolist() == want.compact(), (step, what)
        refused.add(want.report[0])
        same(book, want, (step, what))
        want.check()
    assert refused != {0} or sequences > 300


def test_too_few_pages_changes_nothing(gpu):  # noqa: F811
    """More last pages to continue in than there are free pages: names that were moved come back."""
    for sequences, pages in ((6, 9), (60, 9000)):
        book, want = gpu.cache_pages(sequences, 200 * 16, pages, 16), Book(sequences, 200, pages, 16)
        news = [4 * 16 + 5] + [0] * (sequences - 1)  # four of nine pages are left, for five copies
        if sequences == 60:
            news = [144 * 16 + 5] * 30 + [0] * 30
            want.refs[:] = [1 if i >= 30 * 145 + 20 else 0 for i in range(pages)]  # somebody else's pages
            book.refs.copy_(i32(want.refs))
        gpu.pages_grow(book, i32(news))
        want.grow(news)
        same(book, want, "grow")
        parents = [0] * sequences if sequences == 6 else list(range(30)) * 2
        pairs = gpu.pages_fork(book, i32(parents))
        assert pairs.tolist() == want.fork(parents) and want.report[0] > 0
        same(book, want, "fork")
        keep = [3 if b % 2 else 1 << 20 for b in range(sequences)]  # ... but room for half of them, when those give theirs back
        parents = list(range(sequences))
        pairs = gpu.pages_fork(book, i32(parents), i32(keep))
        assert pairs.tolist() == want.fork(parents, keep) and want.report[0] == 0
        same(book, want, "cut")


def test_what_sequences_hold_behind_forks_and_moves(gpu):  # noqa: F811
    """Tokens appended to shared books stay their sequences' own, in every layer."""
    import karume_b200 as kb
    rng = random.Random(1)
    sequences, page, pages, heads, dim, layers = 6, 16, 60, 2, 64, 3
    book = gpu.cache_pages(sequences, 12 * page, pages, page)
    caches = [gpu.kv_cache(pages, page, heads, dim) for _ in range(layers)]
    said = [[[] for _ in range(sequences)] for _ in range(layers)]  # what each sequence was given
    gen = torch.Generator(device="cuda").manual_seed(0)
    compared = 0
    for step in range(14):
        news = [rng.choice([0, 1, rng.randint(0, 23)]) for _ in range(sequences)]
        gpu.pages_grow(book, i32(news))
        if book.report.tolist()[0] == 0 and sum(news):
            batch = kb.CacheBatch(book.table, book.lengths, i32([0] + news).cumsum(0).to(torch.int32), tokens=sum(news))
            for layer, cache in enumerate(caches):
                k, v = (torch.randn(sum(news), heads, dim, generator=gen, device="cuda") for _ in range(2))
                gpu.cache_append(cache, k, v, batch)
                k, v = gpu.cache_read(cache, batch)
                at = 0
                for b, n in enumerate(news):
                    said[layer][b] = said[layer][b] + [(k[i], v[i]) for i in range(at, at + n)]
                    at += n
        parents = [rng.choice([b, b, rng.randrange(sequences), -1]) for b in range(sequences)]
        keep = [rng.choice([1000, rng.randint(0, 150)]) for _ in range(sequences)]
        pairs = gpu.pages_fork(book, i32(parents), i32(keep))
        gpu.pages_copy(book, pairs, caches)
        if book.report.tolist()[0] == 0:
            said = [[[] if p < 0 else list(one[p][:k]) for p, k in zip(parents, keep)] for one in said]
        if step % 3 == 2:
            gpu.pages_copy(book, gpu.pages_compact(book), caches)
        lengths = book.lengths.tolist()
        assert lengths == [len(s) for s in said[0]]
        if sum(lengths):
            batch = kb.CacheBatch(book.table, book.lengths, i32([0] + lengths).cumsum(0).to(torch.int32), tokens=sum(lengths))
            for layer, cache in enumerate(caches):
                k, v = gpu.cache_read(cache, batch)
                rows = [t for one in said[layer] for t in one]
                assert torch.equal(k, torch.stack([t[0] for t in rows])) and torch.equal(v, torch.stack([t[1] for t in rows]))
                compared += len(rows)
    assert compared > 500
    for c in caches:
        c.free()


@pytest.mark.parametrize("page_bytes", [4, 8, 16, 44, 272, 4096, 16384, 16388, 16400, 50004, 69632, 70000])
@pytest.mark.parametrize("pools", [1, 3, 130])
def test_copies(gpu, page_bytes, pools):  # noqa: F811
    rng = np.random.default_rng(page_bytes)
    pages = 40
    book = gpu.cache_pages(1, 16, pages, 16)
    tensors = [torch.from_numpy(rng.integers(0, 256, (pages, page_bytes), dtype=np.uint8)).cuda() for _ in range(pools)]
    tensors[-1] = torch.from_numpy(rng.integers(0, 1 << 30, (pages + 2, 3, 4), dtype=np.int32)).cuda()  # 48 bytes a page, and more pages
    order = rng.permutation(pages).tolist()
    pairs = [[order[i], order[i + 20]] for i in range(17)] + [[-1, 3], [order[18], pages], [pages + 5, order[38]], [1 << 30, -1], [order[19], order[19]]]
    for count in (len(pairs), 11, 0, -4):
        want = [t.clone() for t in tensors]
        for w in want:
            for a, b in pairs[:max(count, 0)]:
                if 0 <= a < pages and 0 <= b < pages:
                    w[b] = w[a]
        book.report.copy_(i32([0, 0, count, 0]))
        gpu.pages_copy(book, i32(pairs), tensors)
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for t, w in zip(tensors, want))


def test_copies_without_a_report_and_of_nothing(gpu):  # noqa: F811
    import karume_b200 as kb
    t = torch.arange(8 * 4, dtype=torch.int32, device="cuda").view(8, 4)
    pairs, addresses, sizes = i32([[0, 7], [2, 5]]), (ctypes.c_uint64 * 1)(t.data_ptr()), (ctypes.c_uint64 * 1)(16)
    assert kb.lib.kq_pages_copy(gpu._ctx, 1, addresses, sizes, 8, pairs.data_ptr(), 2, 0) == 0
    assert kb.lib.kq_pages_copy(gpu._ctx, 1, addresses, sizes, 8, pairs.data_ptr(), 0, 0) == 0
    assert kb.lib.kq_pages_copy(gpu._ctx, 0, None, None, 8, pairs.data_ptr(), 2, 0) == 0
    gpu.sync()
    assert t[:, 0].tolist() == [0, 4, 8, 12, 16, 8, 24, 0]


def test_copies_of_pools_that_begin_between_sixteen_bytes(gpu):  # noqa: F811
    rng = np.random.default_rng(3)
    for first, wide in ((1, 4), (3, 1000), (2, 9001)):
        whole = torch.from_numpy(rng.integers(0, 1 << 30, first + 9 * wide + 5, dtype=np.int32)).cuda()
        want, book = whole.clone(), gpu.cache_pages(1, 16, 9, 16)
        want[first:first + 9 * wide].view(9, wide)[[8, 0]] = want[first:first + 9 * wide].view(9, wide)[[1, 5]]
        book.report.copy_(i32([0, 0, 2, 0]))
        gpu.pages_copy(book, i32([[1, 8], [5, 0]]), [whole[first:first + 9 * wide].view(9, wide)])
        gpu.sync()
        assert torch.equal(whole, want), (first, wide)


@pytest.mark.parametrize("heads", [1, 2, 3])
def test_summaries_move_with_their_pages(gpu, heads):  # noqa: F811
    import karume_b200 as kb
    page, dim = 16, 64
    book, cache = gpu.cache_pages(3, 6 * page, 20, page), gpu.kv_cache(20, page, heads, dim)
    made = gpu.cache_summaries(cache)
    gpu.pages_grow(book, i32([70, 40, 33]))
    gen = torch.Generator(device="cuda").manual_seed(heads)
    k, v = (torch.randn(143, heads, dim, generator=gen, device="cuda") for _ in range(2))
    batch = kb.CacheBatch(book.table, book.lengths, i32([0, 70, 110, 143]), tokens=143)
    gpu.cache_append(cache, k, v, batch)
    gpu.cache_summarize(cache, made, batch)
    gpu.pages_fork(book, i32([-1, 1, 2]))
    gpu.pages_copy(book, gpu.pages_compact(book), [cache, made])
    assert book.report.tolist()[2] == 5  # two sequences' pages 5 .. 10 are 0 .. 5 now, of which one was free to stay
    again = gpu.cache_summaries(cache)
    gpu.cache_summarize(cache, again, kb.CacheBatch(book.table, book.lengths, i32([0, 0, 40, 73]), tokens=73))
    gpu.sync()
    assert torch.equal(made.codes[:6], again.codes[:6]) and torch.equal(made.scales[:6], again.scales[:6]) and bool((again.scales[:6] > 0).all())
    cache.free()


def test_copies_of_pages_beyond_4_gib(gpu):  # noqa: F811
    t = torch.zeros(9, 1 << 30, dtype=torch.uint8, device="cuda")
    t[7, ::4096], t[7, -1] = 7, 9
    book = gpu.cache_pages(1, 16, 9, 16)
    book.report.copy_(i32([0, 1, 1, 0]))
    gpu.pages_copy(book, i32([[7, 8]]), [t])
    gpu.sync()
    assert torch.equal(t[8], t[7]) and int(t[6].max()) == 0


def test_recorded_steps_take_pages_as_they_run(gpu):  # noqa: F811
    sequences, page = 5, 16
    book, want = gpu.cache_pages(sequences, 8 * page, 30, page), Book(sequences, 8, 30, page)
    news, parents, pool = i32([1, 0, 5, 2, 16]), i32([0, 0, 2, -1, 2]), torch.arange(30 * 4, dtype=torch.int32, device="cuda").view(30, 4)
    gpu.sync()
    gpu.graph_begin()
    gpu.pages_grow(book, news)
    grow = gpu.graph_end()
    gpu.graph_begin()
    pairs = gpu.pages_fork(book, parents)
    gpu.pages_copy(book, pairs, [pool])
    fork = gpu.graph_end()
    kept = pool.tolist()
    for _ in range(6):
        gpu.graph_launch(grow)
        want.grow(news.tolist())
        gpu.graph_launch(fork)
        asked = want.fork(parents.tolist())
        assert pairs.tolist() == asked
        for a, b in asked[:want.report[2]]:
            kept[b] = kept[a]
        same(book, want, "replayed")
        assert pool.tolist() == kept
    gpu.graph_free(grow)
    gpu.graph_free(fork)


def test_numbers_that_are_no_pages(gpu):  # noqa: F811
    """A table or counts that a host filled wrongly: numbers outside the pool are nobody's, and nothing outside the arrays is touched."""
    book = gpu.cache_pages(4, 64, 12, 16)
    book.table.copy_(i32([[0, 1, 99, -5], [2, 1 << 30, 3, -(1 << 31)], [4, 5, -1, -1], [-1, -1, -1, -1]]))
    book.lengths.copy_(i32([60, 1 << 30, 20, -7]))
    book.refs.copy_(i32([1] * 6 + [-3, 0, 0, 0, 0, 0]))
    pairs = gpu.pages_fork(book, i32([1, 0, 3, 2]), i32([55, 50, 9, 30]))
    assert book.lengths.tolist() == [55, 50, 0, 20] and book.report.tolist()[0] == 0
    assert book.table.tolist()[0][:3] == [2, 1 << 30, 3] and book.table.tolist()[3][0] == 4
    assert pairs.shape == (4, 2)
    gpu.pages_compact(book)
    gpu.pages_grow(book, i32([0, 1, 3, 0]))
    assert book.report.tolist()[0] == 0 and book.lengths.tolist() == [55, 51, 3, 20]
    # counts that know fewer pages than the table names
    book.refs.zero_()
    book.refs[11] = 2
    gpu.pages_compact(book)
    assert book.report.tolist() == [0, 1, 1, 0] and book.refs.tolist() == [2] + [0] * 11


def test_refusals(gpu):  # noqa: F811
    import karume_b200 as kb
    book = gpu.cache_pages(3, 64, 8, 16)
    good = i32([0, 0, 0])
    for call in (lambda: gpu.pages_grow(book, good.long()), lambda: gpu.pages_grow(book, good[:2]), lambda: gpu.pages_grow(book, good.cpu()),
                 lambda: gpu.pages_fork(book, i32([0] * 6)[::2]), lambda: gpu.pages_fork(book, good, good[:1]),
                 lambda: gpu.pages_copy(book, good, []), lambda: gpu.pages_copy(book, i32([[0, 1]]), [torch.zeros(7, 16, device="cuda")]),
                 lambda: gpu.pages_copy(book, i32([[0, 1]]), [torch.zeros(8, 6, dtype=torch.uint8, device="cuda")]),
                 lambda: gpu.pages_copy(book, i32([[0, 1]]), [torch.zeros(8, 32, device="cuda")[:, :16]]),
                 lambda: kb.CachePages(book.table.long(), book.lengths, book.refs, 16), lambda: kb.CachePages(book.table, good[:2], book.refs, 16),
                 lambda: gpu.pages_grow(kb.CachePages(book.table, book.lengths, book.refs, 24), good),
                 lambda: gpu.pages_grow(kb.CachePages(book.table, book.lengths, book.refs, 8), good),
                 lambda: gpu.pages_grow(kb.CachePages(book.table, book.lengths, book.refs[:0], 16), good)):
        with pytest.raises(kb.KqError):
            call()
    a = list(book.args)
    for at, value in ((0, 0), (0, a[0] + 2), (1, 0), (1, (1 << 24) + 1), (2, 0), (2, (1 << 27) + 1), (3, 0), (4, 2), (5, 0), (5, (1 << 30) + 1), (6, 512), (7, 0)):
        bad = a[:at] + [value] + a[at + 1:]
        assert kb.lib.kq_pages_grow(gpu._ctx, *bad, good.data_ptr()) in (1, 2)
        assert kb.lib.kq_pages_fork(gpu._ctx, *bad, good.data_ptr(), 0, good.data_ptr()) in (1, 2)
        assert kb.lib.kq_pages_compact(gpu._ctx, *bad, good.data_ptr()) in (1, 2)
    assert kb.lib.kq_pages_grow(gpu._ctx, *a, 0) == 1 and kb.lib.kq_pages_fork(gpu._ctx, *a, 0, 0, good.data_ptr()) == 1
    assert kb.lib.kq_pages_fork(gpu._ctx, *a, good.data_ptr(), 0, 0) == 1 and kb.lib.kq_pages_compact(gpu._ctx, *a, 2) == 1
    assert kb.lib.kq_pages_grow(None, *a, good.data_ptr()) == 1
    gpu.plan_begin()
    try:
        assert kb.lib.kq_pages_grow(gpu._ctx, *a, good.data_ptr()) == 8
    finally:
        try:
            gpu.plan_end()
        except kb.KqError:
            pass
    small = kb.Gpu(0, workspace_bytes=1 << 16)
    big = small.cache_pages(2, 16, 70000, 16)
    with pytest.raises(kb.KqError) as e:
        small.pages_grow(big, i32([1, 1]))
    assert e.value.status == "KQ_ERR_UNSUPPORTED" and "scratch" in str(e.value)
    small.destroy()
