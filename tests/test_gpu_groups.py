"""Groups of sequences that begin alike, as hosts may hand them over: boundaries and starts out of order, members that are idle or shorter than what
their group is said to have in common."""
import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests.test_gpu_attend import KINDS, gpu, one_stream  # noqa: F401
from tests.test_gpu_shared import Groups, i32

pytestmark = pytest.mark.gpu


@KINDS
@pytest.mark.parametrize("heads", [4, 64])
def test_boundaries_out_of_order_have_nothing_in_common(gpu, kind, heads):  # noqa: F811
    """Groups that overlap, or take turns at the same sequences (and two in order, partly outside the batch): every row is what its own keys give."""
    g = Groups(gpu, [(100, [5 + i % 7 for i in range(64)])], 16, 2, 64, seed=21)
    for i, first in enumerate(([0, 63] * 32 + [64], [64, 0, 64], [0, 40, 20, 64], [0x7FFFFFFF, -(1 << 31)], [-7, 63, 99], [3, 3, 3, 64])):
        prefixes = g.prefixes(first=first, common=[100] * (len(first) - 1))
        g.check(kind, [1 + j * i % 3 for j in range(64)], heads, window=50 * (i % 2), rotary=64 * (i // 2 % 2), prefixes=prefixes)
    g.free()


@pytest.mark.parametrize("heads", [4, 64])
def test_starts_out_of_order_come_back(gpu, heads):  # noqa: F811
    """Rows that several groups would share: results say nothing, as without groups, but the call comes back and the next one is right."""
    import karume_b200 as kb
    g = Groups(gpu, [(100, [5 + i % 7 for i in range(32)])], 16, 2, 64, seed=22)
    q, pairs = torch.randn(96, heads, 64, device="cuda"), g.prefixes(first=list(range(0, 33, 2)), common=[100] * 16)
    for starts in ([0, 50] * 16 + [96], [96] + [0, 90] * 16, [3 * i for i in range(32)] + [7], [-4, 200] * 16 + [96]):
        for kind in ("f32", "bf16"):
            gpu.cache_attention(g.cache, q.to(ref.TYPES[kind]), kb.CacheBatch(g.table, g.length, i32(starts), tokens=96), shared=pairs)
    gpu.sync()
    g.check("f32", [1] * 32, heads)
    g.check("bf16", [3] * 32, heads, prefixes=pairs)
    g.free()


def cut_back(g, keep):
    """Some sequences of g end (None) or keep only their first tokens; whole numbers of the others' pages stay shared."""
    import karume_b200 as kb
    parents = [-1 if k is None else b for b, k in enumerate(keep)]
    g.gpu.pages_copy(g.book, g.gpu.pages_fork(g.book, i32(parents), i32([0 if k is None else k for k in keep])), [g.cache])
    g.lengths = [0 if k is None else min(k, n) for k, n in zip(keep, g.lengths)]
    assert g.book.report.tolist()[0] == 0 and g.book.lengths.tolist() == g.lengths
    g.cut = np.concatenate([[0], np.cumsum(g.lengths)])
    if sum(g.lengths):
        g.k, g.v = g.gpu.cache_read(g.cache, kb.CacheBatch(g.book.table, g.book.lengths, i32(g.cut.tolist()), tokens=sum(g.lengths)))


@KINDS
@pytest.mark.parametrize("dim,heads", [(64, 4), (64, 64), (128, 24), (256, 16)])
def test_leading_members_that_ended(gpu, kind, dim, heads):  # noqa: F811
    """The first member of a group, several of them, all of them: the others read what they have in common as before."""
    g = Groups(gpu, [(300, [None, 5, 40, 7]), (170, [None] * 35 + [9, 30]), (64, [None, None, 1, 17]), (90, [None, None]), (33, [2, None])], 16, 2, dim, seed=31)
    n = len(g.lengths)
    g.check(kind, [1] * n, heads, rotary=dim)
    g.check(kind, [0 if length == 0 else 1 + b % 3 for b, length in enumerate(g.lengths)], heads, window=100)
    g.check(kind, [1 + b % 2 for b in range(n)], heads, window=20)  # idle ones with rows
    g.free()


@KINDS
@pytest.mark.parametrize("heads", [4, 64])
def test_members_with_less_than_what_is_common(gpu, kind, heads):  # noqa: F811
    """The group's numbers stay as they were when its members are cut back: the first one, all but one, all of them, to the middle of a page and its end."""
    for keep in ([100, 999, 999, 999], [100, 17, 999, 31], [96, 33, 7, 250], [1, None, 999, 150], [None, 3, 299, 301], [None, 200, 100, None], [304, 288, 16, 999]):
        g = Groups(gpu, [(300, [5, 30, 1, 9]), (50, [7, 7])], 16, 2, 64, seed=32)
        cut_back(g, keep + [999, 20])
        g.check(kind, [1] * 6, heads, rotary=64)
        g.check(kind, [1] * 6, heads, window=64)
        g.check(kind, [0 if n == 0 else min(n, 1 + 4 * b) for b, n in enumerate(g.lengths)], heads, padding=1)
        g.free()


@pytest.mark.parametrize("heads", [8, 80])
def test_a_recorded_step_whose_leading_beam_ends(gpu, heads):  # noqa: F811
    import karume_b200 as kb
    g = Groups(gpu, [(300, [50, 30, 10, 90])], 16, 2, 64, seed=33)
    q, prefixes = torch.randn(4, heads, 64, device="cuda"), g.prefixes()
    out, batch = torch.zeros_like(q), kb.CacheBatch(g.table, g.length)
    gpu.sync()
    gpu.graph_begin()
    gpu.cache_attention(g.cache, q, batch, shared=prefixes, out=out)
    graph = gpu.graph_end()
    for keep in ([999] * 4, [None, 999, 999, 999], [None, 120, 999, 999], [None, None, None, 200]):
        cut_back(g, keep)
        gpu.graph_launch(graph)
        gpu.sync()
        q_again = q.clone()
        want = gpu.cache_attention(g.cache, q_again, batch, shared=kb.SharedPrefixes(i32([0, 0]), i32([0])))
        gpu.sync()
        live = [b for b, k in enumerate(keep) if k is not None]
        assert bool((out[[b for b in range(4) if b not in live]] == 0).all())
        # two orders of the same f32 sums: each within 2^-24 of some hundreds of terms
        assert float((out[live] - want[live]).norm() / want[live].norm()) < 1e-6, keep
        g.check("f32", [1] * 4, heads, prefixes=prefixes)
    gpu.graph_free(graph)
    g.free()
