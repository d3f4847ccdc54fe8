"""Summaries of so many sequences and heads that a grid has not a block for each."""
import pytest
import torch

from tests.test_gpu_attend import gpu, one_stream  # noqa: F401

pytestmark = pytest.mark.gpu


def test_more_tokens_times_heads_than_a_grid_has_blocks(gpu):  # noqa: F811
    """2^24 sequences of 300 heads, of which four, the last one among them, have a token each."""
    import karume_b200 as kb
    sequences, heads, dim, page = 1 << 24, 300, 64, 16
    cache = gpu.kv_cache(5, page, heads, dim)
    here = torch.tensor([0, 7_000_001, sequences - 2, sequences - 1], device="cuda")
    pages = torch.full((sequences, 1), -1, dtype=torch.int32, device="cuda")
    pages[here, 0] = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    lengths[here] = 1
    few = kb.CacheBatch(pages[here].clone(), lengths[here].clone())
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(4, heads, dim, generator=gen, device="cuda")
    gpu.cache_append(cache, k, k, few)
    want, got = gpu.cache_summaries(cache), gpu.cache_summaries(cache)
    gpu.cache_summarize(cache, want, few)
    gpu.cache_summarize(cache, got, kb.CacheBatch(pages, lengths))
    gpu.sync()
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales) and bool((want.scales[1:] > 0).all())
    cache.free()
