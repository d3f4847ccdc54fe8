"""The library beside torch's default stream: calls see what torch enqueued in front of them, and torch sees what they give, with
no synchronisation in between."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LONG = 40_000_000  # clocks that the default stream is kept busy: some 20 ms


@pytest.fixture(autouse=True)
def default_stream():
    before = torch.cuda.current_stream()
    torch.cuda.set_stream(torch.cuda.default_stream())
    yield
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)


@pytest.fixture(params=[True, False], ids=["torch's stream", "own stream"])
def gpu(request):
    import karume_b200 as kb
    g = kb.acquire_gpu(0, use_torch_stream=request.param)
    yield g
    g.destroy()


def cached(gpu, tokens=300):
    import karume_b200 as kb
    torch.manual_seed(tokens)
    cache = gpu.kv_cache((tokens + 63) // 64, 64, 2, 128)
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")[None]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    whole = kb.CacheBatch(pages, i32(tokens), i32(0, tokens), tokens=tokens)
    gpu.cache_append(cache, torch.randn(tokens, 2, 128, device="cuda"), torch.randn(tokens, 2, 128, device="cuda"), whole)
    torch.cuda.synchronize()
    gpu.sync()
    return cache, kb.CacheBatch(pages, i32(tokens)), kb.CacheBatch(pages, i32(tokens), i32(0, 100), tokens=100)


def test_what_torch_is_still_making_is_waited_for(gpu):
    import karume_b200 as kb
    cache, one, many = cached(gpu)
    rope = kb.Rope(torch.from_numpy(kb.rope_table(300, 128)).cuda())
    for batch in (one, many):
        source = torch.randn(batch.tokens, 8, 128, device="cuda")
        position = torch.arange(batch.tokens, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        want = gpu.cache_attention(cache, source, batch), gpu.rope(source, position, rope)
        gpu.sync()
        q = torch.zeros_like(source)
        torch.cuda.synchronize()
        torch.cuda._sleep(LONG)
        q.copy_(source)
        got = gpu.cache_attention(cache, q, batch), gpu.rope(q, position, rope)
        seen = [t + 0 for t in got]  # torch reads at once
        q.zero_()                    # and writes again
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(seen, want))
    cache.free()


def test_torch_waits_for_what_a_call_is_still_making(gpu):
    """Long work of the library in front of the call that counts: torch's copy of its result, and what it writes over its inputs, come behind."""
    cache, _, many = cached(gpu, tokens=4000)
    q, k = torch.randn(100, 8, 128, device="cuda"), torch.randn(100, 2, 128, device="cuda")
    torch.cuda.synchronize()
    want = gpu.cache_attention(cache, q, many)
    gpu.sync()
    out, scratch = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    for _ in range(300):
        gpu.cache_attention(cache, q, many, out=scratch)
    gpu.cache_attention(cache, q, many, out=out)
    seen = out + 0
    q.zero_()
    gpu.cache_append(cache, k, k, many)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(seen, want)
    cache.free()


def test_a_recording_beside_the_default_stream(gpu):
    """torch may go on while a graph is recorded; replays keep the order with it."""
    cache, one, _ = cached(gpu)
    source, q, out = (torch.randn(1, 8, 128, device="cuda") for _ in range(3))
    torch.cuda.synchronize()
    want = gpu.cache_attention(cache, source, one)
    gpu.sync()
    gpu.graph_begin()
    gpu.cache_attention(cache, q, one, out=out)
    other = torch.zeros(1 << 20, device="cuda") + 3
    graph = gpu.graph_end()
    assert float(other.sum()) == 3 << 20
    for _ in range(2):
        q.zero_()
        out.zero_()
        torch.cuda._sleep(LONG)
        q.copy_(source)
        gpu.graph_launch(graph)
        seen = out + 0
        torch.cuda.synchronize()
        assert torch.equal(seen, want) and torch.equal(out, want)
    gpu.graph_free(graph)
    cache.free()


def test_linears_beside_the_default_stream(gpu):
    rng = np.random.default_rng(0)
    n, k = 256, 512
    w = gpu.upload_weight("i4", rng.integers(0, 256, n * k // 2, dtype=np.uint8), rng.random((n, k // 32), np.float32), (n, k), 32)
    bias = torch.zeros(n, device="cuda")
    for rows in (1, 40):
        source = torch.randn(rows, k, device="cuda")
        torch.cuda.synchronize()
        want = gpu.linear(source, w, bias)
        gpu.sync()
        x = torch.zeros_like(source)
        torch.cuda.synchronize()
        torch.cuda._sleep(LONG)
        x.copy_(source)
        seen = gpu.linear(x, w, bias) + 0
        torch.cuda.synchronize()
        assert torch.equal(seen, want)
    w.free()


def test_a_pool_made_on_another_stream_is_there_before_its_first_row(gpu):
    import karume_b200 as kb
    k = torch.randn(1, 2, 128, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kb.CacheBatch(i32([0]), i32(1))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(LONG)
        cache = gpu.kv_cache(1, 64, 2, 128)
    gpu.cache_append(cache, k, k, batch)
    torch.cuda.synchronize()
    held, _ = gpu.cache_read(cache, batch)
    gpu.sync()
    assert float((held - k).abs().max()) < 0.5  # a step of these rows is about a third
    cache.free()


def test_a_decoder_on_the_default_stream_and_refused_on_another(gpu):
    import os
    import sys
    import karume_b200 as kb
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    from generate import small_decoder
    rng = np.random.default_rng(3)
    ids = torch.from_numpy(rng.integers(0, 1024, 90).astype(np.int32)).cuda()
    ones = [torch.from_numpy(rng.integers(0, 1024, 3).astype(np.int32)).cuda() for _ in range(3)]

    def logits_of(d, busy):
        got = []
        if busy:
            torch.cuda._sleep(LONG)
        got.append(d.prompt(ids + 0, [70, 3, 17]) + 0)
        for more in ones:
            if busy:
                torch.cuda._sleep(LONG // 4)
            d.ids.copy_(more)
            got.append(d.step() + 0)
        torch.cuda.synchronize()
        assert d.lengths.tolist() == d.held == [73, 6, 20]
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apart = kb.acquire_gpu(0)
        d = small_decoder(apart, layers=2)
        want = logits_of(d, False)
        d.close()
    apart.destroy()
    d = small_decoder(gpu, layers=2)
    assert all(torch.equal(a, b) for a, b in zip(logits_of(d, True), want))
    with torch.cuda.stream(side):
        for call in (lambda: d.prompt(ids, [70, 3, 17]), d.step, lambda: small_decoder(gpu, layers=1)):
            with pytest.raises(kb.KqError) as e:
                call()
            assert e.value.status == "KQ_ERR_STATE"
    assert d.held == [73, 6, 20]
    d.close()
