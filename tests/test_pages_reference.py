"""The plain statement of the books of pages (tests/pages_reference.py) keeps the rules that it states."""
import random

import pytest

from tests.pages_reference import Book


@pytest.mark.parametrize("seed", range(20))
def test_rules_hold_over_any_calls(seed):
    rng = random.Random(seed)
    book = Book(rng.randint(1, 9), rng.randint(1, 6), rng.randint(1, 30), 16)
    content = {}  # page -> what its tokens are
    n_seq = len(book.table)
    said = [[] for _ in range(n_seq)]  # the tokens that each sequence should hold
    clock = 0
    for _ in range(60):
        what = rng.choice(["grow", "grow", "fork", "fork", "compact"])
        if what == "grow":
            news, before = [rng.choice([0, 1, rng.randint(-3, 40)]) for _ in range(n_seq)], list(book.lengths)
            book.grow(news)
            if book.report[0] == 0:
                for b in range(n_seq):
                    for i in range(before[b], book.lengths[b]):
                        clock += 1
                        said[b].append(clock)
                        content.setdefault(book.table[b][i // 16], {})[i % 16] = clock
            else:
                assert book.lengths == before
        elif what == "fork":
            parents = [rng.choice([b, b, rng.randint(-1, n_seq - 1)]) for b in range(n_seq)]
            keep = [rng.choice([1000, rng.randint(-1, 70)]) for _ in range(n_seq)]
            pairs = book.fork(parents, keep)
            if book.report[0] == 0:
                said = [[] if p < 0 else list(said[p][:max(k, 0)]) for p, k in zip(parents, keep)]
        else:
            pairs = book.compact()
        if what != "grow":
            for a, b in pairs[:book.report[2]]:
                content[b] = dict(content.get(a, {}))
        book.check()
        assert [len(s) for s in said] == book.lengths
        for b in range(n_seq):
            assert [content[book.table[b][i // 16]][i % 16] for i in range(book.lengths[b])] == said[b]
