"""Attention over the paged 4-bit cache against the same formula in 64 bits on the values that the cache stands for.
Whatever a query must not see - slots behind a sequence's end, pages that are nobody's - is NaN here."""
import math

import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests.test_gpu_cache import dev, make_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def one_stream():
    """torch and the library on one stream: what torch makes is there when a kernel reads it."""
    before = torch.cuda.current_stream()
    torch.cuda.set_stream(torch.cuda.Stream())
    yield
    torch.cuda.set_stream(before)


@pytest.fixture(scope="module")
def gpu(one_stream):
    import karume_b200 as kb
    g = kb.acquire_gpu(0)
    yield g
    g.destroy()


class Filled:
    """A cache with lengths[b] random tokens a sequence, everything else NaN, and the rotated queries' reference."""

    def __init__(self, gpu, lengths, page, kv_heads, dim, seed=0, spread=1.0, value=1.0, rows=None):
        import karume_b200 as kb
        rng = np.random.default_rng([seed, dim, page])
        self.gpu, self.lengths, self.dim = gpu, lengths, dim
        pages, starts, total = make_batch(rng, lengths, lengths, page)
        pool = np.zeros((total, kv_heads, page * (dim + 8)), np.uint8)
        pool[..., page * dim:] = np.tile(np.array([0x00, 0x7E], np.uint8), 4 * page)  # every scale and offset NaN
        pool[..., :page * dim] = rng.integers(0, 256, (total, kv_heads, page * dim), dtype=np.uint8)
        self.cache = gpu.kv_cache(total, page, kv_heads, dim, pool=dev(pool))
        self.pages, self.length = dev(pages), dev(np.array(lengths, np.int32))
        tokens = sum(lengths)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.k = torch.randn(tokens, kv_heads, dim, generator=gen, device="cuda") * spread + 0.3
        self.v = torch.randn(tokens, kv_heads, dim, generator=gen, device="cuda") * value
        if rows:
            rows(self)
        if tokens:
            batch = kb.CacheBatch(self.pages, self.length, dev(starts), tokens=tokens)
            gpu.cache_append(self.cache, self.k, self.v, batch)
            self.k, self.v = gpu.cache_read(self.cache, batch)
        self.cut = np.concatenate([[0], np.cumsum(lengths)])

    def check(self, kind, news, heads, window=0, rotary=0, interleaved=False, scale=None, most=0, strided=False, q_spread=1.0, padding=0):
        import karume_b200 as kb
        gpu, dim, tokens = self.gpu, self.dim, sum(news) + padding
        gen = torch.Generator(device="cuda").manual_seed(heads + tokens)
        wide = torch.randn(tokens, heads + (2 if strided else 0), dim, generator=gen, device="cuda") * q_spread
        q = wide.to(ref.TYPES[kind])[:, :heads]
        table = kb.rope_table(max(max(self.lengths), 1), rotary) if rotary else None
        rope = kb.Rope(dev(table), interleaved) if rotary else None
        starts = None if news == [1] * len(news) and not padding else dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32))
        batch = kb.CacheBatch(self.pages, self.length, starts, tokens=tokens, most=most)
        out = torch.full((tokens, heads + (1 if strided else 0), dim), -7.0, dtype=q.dtype, device="cuda")
        got = gpu.cache_attention(self.cache, q, batch, scale=scale, window=window, rope=rope, out=out[:, :heads] if strided else None)
        again = gpu.cache_attention(self.cache, q, batch, scale=scale, window=window, rope=rope)
        gpu.sync()
        assert torch.equal(got.view(torch.uint8) if got.is_contiguous() else got.nan_to_num(), again.view(torch.uint8) if got.is_contiguous() else again.nan_to_num())
        if strided:
            assert bool((out[:, heads:] == -7).all())
        at = 0
        for b, n in enumerate(news):
            length = self.lengths[b]
            qb = q[at:at + n].float()
            mine = got[at:at + n].double()
            at += n
            early = max(n - length, 0)  # queries in front of the sequence's first token
            assert bool((mine[:early] == 0).all())
            qb, mine = qb[early:], mine[early:]
            if len(qb) == 0:
                continue
            if rotary:
                position = np.arange(length - len(qb), length)
                qb = torch.from_numpy(ref.rotate(qb.cpu().numpy(), table, position, interleaved)).cuda()
            part = slice(self.cut[b], self.cut[b + 1])
            want, reach, largest = ref.attend(qb.double(), self.k[part].double(), self.v[part].double(), scale or dim ** -0.5, window)
            assert torch.equal(torch.isnan(mine), torch.isnan(want)), (kind, b)
            off = (mine - want).abs().nan_to_num()
            allowed = ref.allowed(kind, want, reach, largest).nan_to_num(posinf=math.inf)
            assert bool((off <= allowed).all()), (kind, b, float((off / allowed).max()))
            fine = ~torch.isnan(want)
            norm = float(want[fine].norm())
            if norm and q_spread == 1.0:
                rel = float((mine - want)[fine].norm()) / norm
                grain = 2.0 ** -25 * fine.sum().item() ** 0.5 / norm if kind == "f16" else 0.0  # half the spacing of binary16's smallest numbers
                assert rel <= {"f32": 1e-5, "f16": 2e-3, "bf16": 5e-3}[kind] + grain, (kind, b, rel)
        if padding:
            assert bool((got[at:] == 0).all())  # rows that belong to no sequence

    def free(self):
        self.cache.free()


KINDS = pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])


@KINDS
@pytest.mark.parametrize("dim,kv_heads,heads,page", [(64, 2, 4, 16), (128, 2, 12, 64), (128, 1, 1, 32), (128, 3, 24, 128), (256, 2, 8, 16), (64, 1, 40, 256), (256, 1, 7, 64)])
def test_single_tokens(gpu, kind, dim, kv_heads, heads, page):
    f = Filled(gpu, [1, 0, 15, 16, 17, 63, 64, 65, 300, 1025], page, kv_heads, dim, seed=heads)
    f.check(kind, [1] * 10, heads)
    f.check(kind, [1] * 10, heads, rotary=dim, window=33)
    f.check(kind, [1] * 10, heads, rotary=dim // 4, interleaved=True, strided=True, scale=0.31)
    f.free()


@KINDS
@pytest.mark.parametrize("dim,kv_heads,heads,page", [(128, 2, 8, 64), (64, 2, 12, 16), (256, 1, 2, 32)])
def test_drafts_and_mixed_batches(gpu, kind, dim, kv_heads, heads, page):
    lengths = [5, 200, 0, 64, 777, 3]
    f = Filled(gpu, lengths, page, kv_heads, dim, seed=3)
    f.check(kind, [5, 1, 0, 3, 8, 2], heads, rotary=dim, most=8)
    f.check(kind, [5, 1, 2, 3, 8, 7], heads, rotary=dim)             # more new tokens than there are
    f.check(kind, [5, 1, 0, 3, 90, 2], heads, window=17, padding=3)   # a prompt among them, rows of nobody behind
    f.check(kind, [1, 100, 0, 64, 777, 0], heads, rotary=dim // 2, interleaved=True, most=777)
    f.free()


@KINDS
@pytest.mark.parametrize("dim,kv_heads,heads,page,new,length", [
    (128, 1, 4, 64, 128, 128), (128, 2, 8, 64, 129, 400), (64, 1, 6, 16, 1000, 1000), (128, 1, 1, 32, 257, 1300), (256, 1, 2, 64, 300, 333),
    (128, 1, 12, 128, 85, 86), (64, 2, 2, 256, 513, 2000)])
def test_prompts(gpu, kind, dim, kv_heads, heads, page, new, length):
    f = Filled(gpu, [length], page, kv_heads, dim, seed=new)
    f.check(kind, [new], heads, rotary=dim, strided=True)
    f.check(kind, [new], heads, window=1)
    f.check(kind, [new], heads, window=70)
    f.free()


@KINDS
def test_long_axis_is_split_and_joined(gpu, kind):
    f = Filled(gpu, [70001, 3], 64, 2, 128, seed=9)
    f.check(kind, [1, 1], 8)
    f.check(kind, [40, 2], 8, rotary=128)
    f.check(kind, [1, 1], 8, window=50000)
    f.free()


@KINDS
def test_sharp_and_flat_scores(gpu, kind):
    """One key that takes all the weight wherever it stands, scores far from zero, and equal scores."""
    def one_hot(f):
        f.k[f.k.shape[0] // 2] *= 40

    for rows, spread, q_spread in ((one_hot, 0.2, 1.0), (None, 6.0, 8.0), (None, 0.0, 1.0)):
        f = Filled(gpu, [500, 130], 32, 1, 128, seed=5, spread=spread, rows=rows)
        f.check(kind, [1, 1], 4, q_spread=q_spread)
        f.check(kind, [200, 130], 4, q_spread=q_spread)
        f.free()


@KINDS
@pytest.mark.parametrize("value", [1e-4, 3000.0])
def test_small_and_large_values(gpu, kind, value):
    """Values whose binary16 scales are tiny or large, and rows of very different size side by side."""
    def uneven(f):
        f.v[::3] *= 1e-2
        f.v[5::7] = 0

    f = Filled(gpu, [300, 90], 16, 2, 64, seed=6, value=value, rows=uneven)
    f.check(kind, [1, 1], 4)
    f.check(kind, [150, 90], 4)
    f.free()


@KINDS
def test_a_row_held_as_nan_reaches_only_those_who_see_it(gpu, kind):
    def poison(f):
        f.k[100], f.v[260] = math.nan, math.inf

    f = Filled(gpu, [400], 64, 1, 128, seed=7, rows=poison)
    f.check(kind, [400], 2, window=50)
    f.check(kind, [1], 2, window=120)
    f.check(kind, [1], 2, window=200)
    f.free()


def test_missing_pages_read_as_nan_to_those_who_see_them(gpu):
    import karume_b200 as kb
    f = Filled(gpu, [200, 100], 64, 1, 64)
    pages = f.pages.clone()
    pages[0, 1] = 99
    for kind in ("f32", "f16"):
        q = torch.randn(2, 2, 64, device="cuda").to(ref.TYPES[kind])
        got = gpu.cache_attention(f.cache, q, kb.CacheBatch(pages, f.length))
        far = gpu.cache_attention(f.cache, q, kb.CacheBatch(pages, f.length), window=60)
        many = torch.randn(300, 2, 64, device="cuda").to(ref.TYPES[kind])
        starts = dev(np.array([0, 200, 300], np.int32))
        prompt = gpu.cache_attention(f.cache, many, kb.CacheBatch(pages, f.length, starts, tokens=300))
        gpu.sync()
        assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all() and torch.isfinite(far).all()
        assert torch.isfinite(prompt[:64]).all() and torch.isnan(prompt[64:200]).all() and torch.isfinite(prompt[200:]).all()
    beyond = kb.CacheBatch(f.pages, torch.full((2,), 1000, dtype=torch.int32, device="cuda"))
    got = gpu.cache_attention(f.cache, torch.ones(2, 2, 64, device="cuda"), beyond)
    gpu.sync()
    assert torch.isnan(got).all()
    f.free()


def test_a_recorded_step_follows_the_lengths(gpu):
    """Append and attention in a graph: replays read the lengths and pages of their time."""
    import karume_b200 as kb
    torch.manual_seed(0)
    cache = gpu.kv_cache(8, 16, 2, 128)
    pages = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    k, v, q = (torch.zeros(2, n, 128, device="cuda") for n in (2, 2, 4))
    out = torch.zeros_like(q)
    batch, rope = kb.CacheBatch(pages, lengths), kb.Rope(dev(kb.rope_table(64, 128)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gpu.use_stream(stream)
        gpu.cache_attention(cache, q, batch, rope=rope, out=out)  # what a kernel sets up once is set up outside
        gpu.sync()
        gpu.graph_begin()
        gpu.cache_append(cache, k, v, batch, rope=rope)
        gpu.cache_attention(cache, q, batch, rope=rope, out=out)
        step = gpu.graph_end()
        replayed = []
        for i in range(40):
            for t in (k, v, q):
                t.normal_()
            lengths += torch.tensor([1, i % 2], dtype=torch.int32, device="cuda")
            gpu.graph_launch(step)
            direct = gpu.cache_attention(cache, q, batch, rope=rope)
            replayed.append((out.clone(), direct))
        gpu.sync()
        gpu.graph_free(step)
    torch.cuda.synchronize()
    gpu.use_stream(torch.cuda.current_stream())
    assert all(torch.equal(a, b) for a, b in replayed) and lengths.tolist() == [40, 20]
    assert all(bool(torch.isfinite(a).all()) for a, _ in replayed)
    cache.free()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_sequences(gpu, kind):
    """More sequences than a block has threads, a few of them prompts, some idle; `most` says too little and is still only a hint."""
    rng = np.random.default_rng(2)
    lengths = rng.integers(0, 40, 700).tolist()
    lengths[5], lengths[300], lengths[699] = 500, 130, 77
    f = Filled(gpu, lengths, 16, 1, 64, seed=8)
    f.check(kind, [1] * 700, 2)
    news = [0 if i % 7 == 3 else min(1, n) for i, n in enumerate(lengths)]
    news[5], news[300], news[699] = 400, 130, 20
    f.check(kind, news, 2, rotary=64, most=400)
    f.check(kind, news, 2, most=2)
    f.check(kind, news, 2, padding=2)
    f.free()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_little_scratch(kind):
    """Too little for parts: fewer CTAs share a run, or none."""
    import karume_b200 as kb
    for scratch in (1 << 12, 1 << 18):
        g = kb.acquire_gpu(0, workspace_bytes=scratch)
        f = Filled(g, [3000, 100], 64, 1, 128, seed=4)
        f.check(kind, [1, 1], 4)
        f.check(kind, [90, 3], 4, rotary=128)
        f.free()
        g.destroy()


def test_offsets_beyond_32_bits(gpu):
    """Pages more than 4 GiB into the pool, and an output whose rows are far apart."""
    import karume_b200 as kb
    page, dim, heads = 256, 128, 2
    block = page * (dim + 8)
    count = (5 << 30) // (block * heads)
    pool = torch.zeros(count, heads, block, dtype=torch.uint8, device="cuda")
    cache = gpu.kv_cache(count, page, heads, dim, pool=pool)
    pages = torch.tensor([[count - 1, 0, count - 2]], dtype=torch.int32, device="cuda")
    n = 700
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(n, heads, dim, generator=gen, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    lengths, starts = dev(np.array([n], np.int32)), dev(np.array([0, n], np.int32))
    whole = kb.CacheBatch(pages, lengths, starts, tokens=n)
    gpu.cache_append(cache, k, v, whole)
    k, v = gpu.cache_read(cache, whole)
    for kind, new in (("f32", 1), ("bf16", 1), ("f32", 100), ("bf16", 100)):
        q = torch.randn(new, 4, dim, generator=gen, device="cuda").to(ref.TYPES[kind])
        stride = (3 << 30) // q.element_size() if new == 1 else 4 * dim
        torch.cuda.synchronize()
        got = gpu.cache_attention(cache, q, kb.CacheBatch(pages, lengths, dev(np.array([0, new], np.int32)), tokens=new))
        gpu.sync()
        want, reach, largest = ref.attend(q.double(), k.double(), v.double(), dim ** -0.5, 0)
        assert bool(((got.double() - want).abs() <= ref.allowed(kind, want, reach, largest)).all()), (kind, new, stride)
    wide = torch.zeros(3, 1 << 31, dtype=torch.int8, device="cuda").view(torch.float16)  # rows 2 GiB apart
    q = torch.randn(3, 4, dim, generator=gen, device="cuda").half()
    out = wide[:, :4 * dim].unflatten(1, (4, dim))
    torch.cuda.synchronize()
    batch = kb.CacheBatch(pages, lengths, dev(np.array([0, 3], np.int32)), tokens=3)
    gpu.cache_attention(cache, q, batch, out=out)
    near = gpu.cache_attention(cache, q, batch)
    gpu.sync()
    assert torch.equal(out, near)
    cache.free()
