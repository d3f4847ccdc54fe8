"""Groups of sequences that begin alike, as hosts may hand them over: boundaries and starts out of order, members that are idle or shorter than what
their group is said to have in common."""
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
