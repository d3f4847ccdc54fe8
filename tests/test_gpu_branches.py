"""A decoder whose sequences share a pool of pages: branching, cutting back and ending, a pool that runs out, steps that read selected pages."""
import os
import sys

import numpy as np
import pytest
import torch

from tests.test_gpu_generate import ROOT, gpu  # noqa: F401

pytestmark = pytest.mark.gpu


def make(gpu, sequences=4, longest=512, layers=2, **more):  # noqa: F811
    """examples/generate.py's decoder, with weights around zero, so that what a sequence says depends on what it has seen."""
    import karume_b200 as kb
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    from bench_workload import synth_weight
    from generate import around_zero, small_decoder
    from karume_b200.decoder import Decoder
    d = small_decoder(gpu, layers=layers, sequences=sequences, longest=longest, make=lambda *of: around_zero(*synth_weight(*of)))
    made = Decoder(gpu, d.shape, d.weights, d.norms, d.rope, sequences, longest, page_tokens=more.pop("page_tokens", 16), **more)
    d.close()
    assert kb
    return made


def tokens(n, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 1024, n).astype(np.int32)).cuda()


def check(d):
    """What host and device know is the same, and what is free too."""
    assert d.lengths.tolist() == d.held
    refs = d.book.refs.cpu()
    assert int((refs == 0).sum()) == d.free
    named = d.pages[d.pages >= 0].cpu().long()
    assert torch.equal(torch.bincount(named, minlength=len(refs)).int(), refs)


def test_a_pool_gives_what_pages_of_their_own_give(gpu):  # noqa: F811
    own, pooled = make(gpu), make(gpu, pool_pages=64)
    news = [50, 3, 17, 130]
    for ids, n in ((tokens(200), news), (tokens(20, 1), [5, 0, 14, 1])):
        assert torch.equal(own.prompt(ids, n), pooled.prompt(ids, n))
        check(pooled)
    for i in range(20):
        for d in (own, pooled):
            d.ids.copy_(tokens(4, 10 + i))
        assert torch.equal(own.step(), pooled.step())
    gpu.sync()
    check(pooled)
    for d in (own, pooled):
        d.close()


def test_answers_branch_and_are_cut_back(gpu):  # noqa: F811
    d = make(gpu, pool_pages=40)
    d.prompt(tokens(75), [75, 0, 0, 0])
    d.fork([0, 0, 0, 0])
    check(d)
    assert d.held == [75] * 4 and d.free == 40 - 4 - 4  # four pages are everybody's, the fifth everyone's own
    assert d.shared.first.tolist() == [0, 4, 4, 4, 4] and d.shared.tokens.tolist() == [64, 0, 0, 0]

    def say(many):
        got = []
        for i in range(many):
            d.ids.copy_(tokens(4, 20 + i))
            got.append(d.step() + 0)
        gpu.sync()
        return got

    first = say(12)
    check(d)
    d.fork([0, 1, 2, 3], [75, 80, 75, 75])
    check(d)
    assert d.held == [75, 80, 75, 75]
    again = say(12)  # the same tokens on the same sequences, whatever pages they have now
    assert all(torch.equal(a[b], c[b]) for a, c in zip(first, again) for b in (0, 2, 3))
    # the same ids in all: the same logits but for where kernels cut their sums, which a code of the cache may turn over
    d.fork([2, 2, 2, -1])
    assert d.held == [87, 87, 87, 0] and d._ended == [False, False, False, True]
    d.fork([2, 2, 2, -1], [70, 70, 70, 0])
    for i in range(5):
        d.ids.fill_(40 + i)
        logits = d.step()
        for b in (1, 2):
            assert float((logits[b] - logits[0]).norm() / logits[0].norm()) < 2e-2
    assert d.held == [75, 75, 75, 0]  # what has ended stays so
    check(d)
    logits = d.prompt(tokens(6, 3), [0, 0, 0, 6])  # ... until it is given a prompt
    assert d.held == [75, 75, 75, 6] and bool(torch.isfinite(logits).all())
    d.ids.fill_(9)
    d.step()
    assert d.held == [76, 76, 76, 7]
    check(d)
    # beams in another order, one dropped and one doubled
    before = d.pages.tolist()
    d.fork([3, 2, 2, 0])
    assert d.held == [7, 76, 76, 76] and d.pages.tolist()[0] == before[3] and d.pages.tolist()[3][:4] == before[0][:4]
    check(d)
    d.close()


def test_a_branch_goes_on_as_its_parent_would(gpu):  # noqa: F811
    """Against the parent itself, in another decoder, alone: what a branch reads through shared and copied pages is what the parent wrote."""
    one, many = make(gpu, sequences=1, pool_pages=32), make(gpu, sequences=4, pool_pages=64)
    ids = tokens(100, 5)
    want = [one.prompt(ids, [100])]
    many.prompt(ids, [0, 100, 0, 0])
    many.fork([1, 1, -1, 1], [90, 100, 0, 100])
    for d in (one, many):
        d.ids.fill_(7)
    for i in range(6):
        want.append(one.step() + 0)
        got = many.step()
        for b in (1, 3):
            assert float((got[b] - want[-1][0]).norm() / want[-1].norm()) < 2e-2, (i, b)
        assert float((got[0] - want[-1][0]).norm() / want[-1].norm()) > 5e-2  # ten tokens fewer
        for d in (one, many):
            d.ids.fill_(100 + i)
    gpu.sync()
    for d in (one, many):
        d.close()


def test_steps_that_read_common_pages_once(gpu):  # noqa: F811
    """What branches have in common is read once whatever it saves: the same logits but for roundings, which a code of the cache may turn over."""
    import karume_b200 as kb
    each, once = make(gpu, sequences=8, pool_pages=80), make(gpu, sequences=8, pool_pages=80)
    once.shared = kb.SharedPrefixes(once.shared.first, once.shared.tokens, least=0)
    for i in range(16):
        if i in (0, 6):
            for d in (each, once):
                d.prompt(tokens(170, i), [100, 0, 0, 0, 70, 0, 0, 0])
                d.fork([0, 0, 0, 0, 4, 4, 4, 7], [400, 400, 400, 90 + i, 400, 400, 64, 400])
        got = []
        for d in (each, once):
            d.ids.copy_(tokens(8, 60 + i))
            got.append(d.step() + 0)
        gpu.sync()
        assert bool(torch.isfinite(got[1]).all())
        assert float((got[1] - got[0]).norm() / got[0].norm()) < 2e-2, i
    assert once.shared.first.tolist()[:4] == [0, 4, 7, 8] and once.shared.tokens.tolist()[:3] == [96, 64, 0]
    check(once)
    for d in (each, once):
        d.close()


def test_a_pool_that_runs_out(gpu, monkeypatch):  # noqa: F811
    import karume_b200 as kb
    d = make(gpu, pool_pages=8)
    with pytest.raises(kb.KqError) as e:
        d.prompt(tokens(150), [150, 0, 0, 0])
    assert e.value.status == "KQ_ERR_OOM" and d.held == [0] * 4
    d.prompt(tokens(100), [60, 40, 0, 0])  # four and three pages
    check(d)
    with pytest.raises(kb.KqError) as e:
        d.fork([0, 1, 0, 0])  # two last pages to copy, one free
    assert e.value.status == "KQ_ERR_OOM" and d.held == [60, 40, 0, 0]
    check(d)
    d.fork([0, 1, 0, -1])
    assert d.held == [60, 40, 60, 0] and d.free == 0
    for _ in range(4):
        d.step()
    assert d.held == [64, 44, 64, 0]
    with pytest.raises(kb.KqError) as e:
        d.step()  # two more pages
    assert e.value.status == "KQ_ERR_OOM" and d.held == [64, 44, 64, 0]
    check(d)
    d.fork([0, -1, 2, -1])
    assert d.free == 8 - 5
    d.step()
    assert d.held == [65, 0, 65, 0] and d.free == 1
    check(d)
    # a call that fails behind its pages gives them back
    real = d._head
    monkeypatch.setattr(d, "_head", lambda *a: (_ for _ in ()).throw(RuntimeError("no head")))
    with pytest.raises(RuntimeError, match="no head"):
        d.prompt(tokens(10), [0, 10, 0, 0])
    monkeypatch.setattr(d, "_head", real)
    check(d)
    for bad in (([0, 1, 2], None), ([0, 1, 2, 4], None), ([0, 1, 2, 3], [1, 1, 1]), ([0, 1, 2, 3], [1, 1, 1, -1])):
        with pytest.raises(kb.KqError) as e:
            d.fork(*bad)
        assert e.value.status == "KQ_ERR_SHAPE"
    check(d)
    d.close()
    own = make(gpu)
    with pytest.raises(kb.KqError) as e:
        own.fork([0, 1, 2, 3])
    assert e.value.status == "KQ_ERR_STATE"
    own.close()


def test_recording_that_fails_leaves_the_book_as_it_was(gpu, monkeypatch):  # noqa: F811
    d = make(gpu, pool_pages=40)
    d.prompt(tokens(60), [50, 3, 7, 0])
    real, calls = d._head, []

    def head(*args):
        calls.append(args)
        if len(calls) > 1:
            raise RuntimeError("no head")
        return real(*args)

    monkeypatch.setattr(d, "_head", head)
    with pytest.raises(RuntimeError, match="no head"):
        d.step()
    monkeypatch.setattr(d, "_head", real)
    check(d)
    d.step()
    gpu.sync()
    assert d.held == [51, 4, 8, 1]
    check(d)
    d.close()


def test_steps_over_selected_pages(gpu):  # noqa: F811
    import karume_b200 as kb
    from karume_b200.decoder import Selection
    whole, all_pages, some = make(gpu, pool_pages=80), make(gpu, pool_pages=80, select=Selection(32)), make(gpu, pool_pages=80, select=Selection(4, 1, 1))
    ids, news = tokens(400), [300, 20, 64, 16]
    first = [d.prompt(ids, news) for d in (whole, all_pages, some)]
    assert torch.equal(first[0], first[1]) and torch.equal(first[0], first[2])
    differ = 0.0
    for i in range(20):
        if i == 10:  # branches and cut ones keep their summaries
            for d in (whole, all_pages, some):
                d.fork([0, 1, 0, 3], [300, 21, 290, 3])
        got = []
        for d in (whole, all_pages, some):
            d.ids.copy_(tokens(4, 50 + i))
            got.append(d.step() + 0)
        gpu.sync()
        assert torch.equal(got[0], got[1]), i
        assert torch.equal(got[0][1], got[2][1]) and torch.equal(got[0][3], got[2][3])  # no more pages than the budget
        differ = max(differ, float((got[0][0] - got[2][0]).norm() / got[0][0].norm()))
    assert differ > 1e-3
    for d in (whole, all_pages, some):
        d.close()
    with pytest.raises(kb.KqError):
        make(gpu, window=64, select=Selection(4))
    own = make(gpu, select=Selection(4, 1, 1))  # without a pool as well
    own.prompt(ids, news)
    assert bool(torch.isfinite(own.step()).all())
    own.close()
