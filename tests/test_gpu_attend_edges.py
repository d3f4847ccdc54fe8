"""Attention over the packed cache where one step of a kernel depends on another: scores that climb inside a tile, values at
the ends of what a row can hold, rows that are far apart, long sums."""
import math

import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests.test_gpu_attend import KINDS, Filled, gpu, one_stream  # noqa: F401
from tests.test_gpu_cache import dev

pytestmark = pytest.mark.gpu


@KINDS
@pytest.mark.parametrize("dim,period", [(128, 128), (64, 128), (128, 96), (128, 400)])
def test_scores_that_climb_inside_a_tile(gpu, kind, dim, period):  # noqa: F811
    """The largest score rises by many powers of two from each few keys to the next, so that what is already summed, and what
    of the same tile is already weighed, is scaled again and again; for other rows it falls."""
    def climb(f):
        n = f.k.shape[0]
        sign = torch.where(torch.arange(dim, device="cuda") * 7 % 5 < 2, 1.0, -1.0)  # two values a row: held exactly
        at = torch.arange(n, device="cuda") % period
        # q has spread 2: q . sign / dim has 2 / sqrt(dim), the score of key j then 0.4 j (8 powers of two in 14 keys)
        f.k[:] = (0.2 * at)[:, None, None] * sign

    f = Filled(gpu, [400], 64, 1, dim, seed=12, rows=climb)
    f.check(kind, [400], 4, q_spread=2.0)
    f.check(kind, [100], 4, q_spread=2.0, window=150)
    f.check(kind, [1], 4, q_spread=2.0)
    f.free()
