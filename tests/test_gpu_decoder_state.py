"""What a decoder holds behind a call that failed: what it held in front of it."""
import os
import sys

import numpy as np
import pytest
import torch

from tests.test_gpu_generate import ROOT, gpu  # noqa: F401

pytestmark = pytest.mark.gpu


def small(gpu):  # noqa: F811
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    from generate import small_decoder
    return small_decoder(gpu, layers=2)


def tokens(n, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 1024, n).astype(np.int32)).cuda()


def test_a_prompt_that_is_refused(gpu):  # noqa: F811
    import karume_b200 as kb
    d = small(gpu)
    for ids, news in ((tokens(4), [-1, 3, 2]), (tokens(4), [1, 1, 1]), (tokens(2), [1, 1]), (tokens(600), [600, 0, 0]), (tokens(3).long(), [1, 1, 1]),
                      (tokens(3).cpu(), [1, 1, 1]), (tokens(0), [0, 0, 0])):
        with pytest.raises(kb.KqError) as e:
            d.prompt(ids, news)
        assert e.value.status == "KQ_ERR_SHAPE" and d.held == d.lengths.tolist() == [0, 0, 0]
    d.close()


def test_calls_that_fail_leave_the_sequences_as_they_were(gpu, monkeypatch):  # noqa: F811
    """The head's weight is missing: behind all layers, in a prompt, outside and inside the recording of a step."""
    a, b = small(gpu), small(gpu)
    ids, more = tokens(60), tokens(3, 1)
    want = [a.prompt(ids, [50, 3, 7]) + 0]
    a.ids.copy_(more)
    want += [a.step() + 0, a.step() + 0]
    got = []

    def without_head(call, after=0):
        calls = []
        real = b._head

        def head(*args):
            calls.append(args)
            if len(calls) > after:
                raise RuntimeError("no head")
            return real(*args)

        monkeypatch.setattr(b, "_head", head)
        before = list(b.held)
        with pytest.raises(RuntimeError, match="no head"):
            call()
        monkeypatch.setattr(b, "_head", real)
        assert b.held == before == b.lengths.tolist()

    without_head(lambda: b.prompt(ids, [50, 3, 7]))
    got.append(b.prompt(ids, [50, 3, 7]) + 0)
    b.ids.copy_(more)
    without_head(b.step)
    without_head(b.step, after=1)
    got += [b.step() + 0, b.step() + 0]
    gpu.sync()
    assert a.held == b.held == [52, 5, 9] and all(torch.equal(x, y) for x, y in zip(got, want))
    a.close()
    b.close()
