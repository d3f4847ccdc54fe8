"""Copies of pages that are made when the book has been called again, and lists of pairs that end by themselves."""
import ctypes

import pytest
import torch

from tests.pages_reference import Book
from tests.test_gpu_attend import gpu, one_stream  # noqa: F401

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def pool_of(pages, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 1 << 30, (pages, 4), generator=gen, device="cuda", dtype=torch.int32)


def copied(pool, pairs):
    want = pool.clone()
    for a, b in pairs:
        if a >= 0:
            want[b] = pool[a]
    return want


@pytest.mark.parametrize("later", ["grow", "fork", "fork and grow", "refused fork"])
def test_pairs_outlive_the_next_calls(gpu, later):  # noqa: F811
    book, want, pool = gpu.cache_pages(6, 8 * 16, 60, 16), Book(6, 8, 60, 16), pool_of(60)
    gpu.pages_grow(book, i32([40, 0, 0, 25, 0, 7]))
    want.grow([40, 0, 0, 25, 0, 7])
    pairs, asked = gpu.pages_fork(book, i32([0, 0, 0, 3, 3, 5])), want.fork([0, 0, 0, 3, 3, 5])
    assert pairs.tolist() == asked and want.report[2] == 3
    more = None
    if later == "refused fork":
        gpu.pages_fork(book, i32([6] * 6))
    elif "fork" in later:
        more, also = gpu.pages_fork(book, i32([0, 1, 2, 3, 4, 1])), want.fork([0, 1, 2, 3, 4, 1])
        assert more.tolist() == also and want.report[2] == 1
    if "grow" in later:
        gpu.pages_grow(book, i32([1] * 6))
    expected = copied(pool, asked)
    gpu.pages_copy(book, pairs, [pool])
    gpu.sync()
    assert torch.equal(pool, expected)
    if more is not None:
        expected = copied(pool, also)
        gpu.pages_copy(book, more, [pool])
        gpu.sync()
        assert torch.equal(pool, expected)


def test_pairs_of_a_compaction_outlive_a_grow(gpu):  # noqa: F811
    book, want, pool = gpu.cache_pages(40, 64 * 16, 3000, 16), Book(40, 64, 3000, 16), pool_of(3000, 1)
    parents = [-1 if i % 3 == 0 else i for i in range(40)]
    gpu.pages_grow(book, i32([1000] * 40))
    gpu.pages_fork(book, i32(parents))
    want.grow([1000] * 40)
    want.fork(parents)
    pairs, asked = gpu.pages_compact(book), want.compact()
    assert pairs.tolist() == asked and want.report[2] > 300
    gpu.pages_grow(book, i32([0] * 40))
    expected = copied(pool, asked)
    gpu.pages_copy(book, pairs, [pool])
    gpu.sync()
    assert torch.equal(pool, expected)


def test_recorded_copies_behind_a_recorded_grow(gpu):  # noqa: F811
    """Three recordings, replayed in another order than they were made in."""
    book, pool = gpu.cache_pages(4, 8 * 16, 40, 16), pool_of(40, 2)
    gpu.pages_grow(book, i32([20, 0, 0, 0]))
    parents, ones = i32([0, 0, 0, 0]), i32([1, 1, 1, 1])
    gpu.sync()
    graphs = []
    gpu.graph_begin()
    pairs = gpu.pages_fork(book, parents)
    graphs.append(gpu.graph_end())
    gpu.graph_begin()
    gpu.pages_copy(book, pairs, [pool])
    graphs.append(gpu.graph_end())
    gpu.graph_begin()
    gpu.pages_grow(book, ones)
    graphs.append(gpu.graph_end())
    fork, copy, grow = graphs
    for _ in range(3):
        gpu.graph_launch(fork)
        gpu.graph_launch(grow)
        gpu.sync()
        assert int((pairs[:, 0] >= 0).sum()) == 3
        expected = copied(pool, pairs.tolist())
        gpu.graph_launch(copy)
        gpu.sync()
        assert torch.equal(pool, expected)
    for g in graphs:
        gpu.graph_free(g)


@pytest.mark.parametrize("most", [1, 31, 32, 33, 1023, 1024, 1025, 5000])
def test_lists_of_any_length_end_by_themselves(gpu, most):  # noqa: F811
    import karume_b200 as kb
    pages = 2 * most
    addresses, sizes = (ctypes.c_uint64 * 1)(), (ctypes.c_uint64 * 1)(16)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(most)).tolist()
    for count in sorted({0, 1, 2, most // 33, most // 2, most - 2, most - 1, most} & set(range(most + 1))):
        pool = pool_of(pages, most)
        addresses[0] = pool.data_ptr()
        listed = [[order[2 * i], order[2 * i + 1]] for i in range(count)] + [[-1, -1]] * (most - count)
        expected, pairs = pool.clone(), i32(listed)
        expected[pairs[:count, 1].long()] = pool[pairs[:count, 0].long()]
        assert kb.lib.kq_pages_copy(gpu._ctx, 1, addresses, sizes, pages, pairs.data_ptr(), most, (1 << 64) - 1) == 0
        gpu.sync()
        assert torch.equal(pool, expected), count


def test_a_number_that_a_grow_has_overwritten_is_refused(gpu):  # noqa: F811
    import karume_b200 as kb
    book, pool = gpu.cache_pages(2, 64, 12, 16), pool_of(12, 3)
    kept = pool.clone()
    gpu.pages_grow(book, i32([5, 0]))
    pairs = gpu.pages_fork(book, i32([0, 0]))
    gpu.pages_copy(book, pairs.clone(), [pool])  # by the report, which is the fork's still
    kept[1] = kept[0]
    gpu.pages_grow(book, i32([1, 1]))
    with pytest.raises(kb.KqError, match="overwritten"):
        gpu.pages_copy(book, pairs.clone(), [pool])
    with pytest.raises(kb.KqError, match="overwritten"):
        gpu.pages_copy(book, pairs[:1], [pool])
    gpu.sync()
    assert torch.equal(pool, kept)


def test_an_empty_book_and_pools_without_pages_are_refused(gpu):  # noqa: F811
    import karume_b200 as kb
    book = kb.CachePages(torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), i32([0, 0]), i32([]), 16)
    for pool in (torch.empty(0, 4, device="cuda"), torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")):
        with pytest.raises(kb.KqError):
            gpu.pages_copy(book, i32([[0, 1]]), [pool])
    for call in (lambda: gpu.pages_grow(book, i32([1, 0])), lambda: gpu.pages_fork(book, i32([0, 0])), lambda: gpu.pages_compact(book)):
        with pytest.raises(kb.KqError):
            call()
    assert book.table.tolist() == [[-1] * 4] * 2 and book.lengths.tolist() == [0, 0]
