"""Summaries of pages, the selection by them, attention over what was selected."""
import math

import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests import select_reference as sel
from tests.test_gpu_attend import KINDS, Filled, gpu, one_stream  # noqa: F401
from tests.test_gpu_cache import dev, make_batch

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def as_numpy(t):
    return t.cpu().numpy()


# ---- summaries ------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (128, 64, 2), (256, 256, 1), (128, 16, 8), (64, 128, 1)])
def test_summaries_of_the_pages_that_new_tokens_are_in(gpu, dim, page, heads):  # noqa: F811
    import karume_b200 as kb
    lengths = [1, 5 * page + 3, 0, 2 * page, page - 1, 3 * page + page // 2]
    f = Filled(gpu, lengths, page, heads, dim, seed=dim + page)
    made = gpu.cache_summaries(f.cache)
    k, pages = as_numpy(f.k), as_numpy(f.pages)
    for news in ([1] * 6, [1, 2 * page + 4, 0, page, page - 1, page // 2 + 1], [0, 0, 0, 2 * page, 0, 0], [2, 5 * page + 3, 4, 1, 1, 3 * page + page // 2]):
        made.codes.fill_(77)
        made.scales.fill_(-3.0)
        starts = None if news == [1] * 6 else i32(np.concatenate([[0], np.cumsum(news)]).tolist())
        # (rows behind the last sequence belong to nobody)
        gpu.cache_summarize(f.cache, made, kb.CacheBatch(f.pages, f.length, starts, tokens=sum(news) + 3 if starts is not None else 0))
        gpu.sync()
        want_codes, want_scales = np.full(tuple(made.codes.shape), 77), np.full(tuple(made.scales.shape), -3.0, np.float32)
        for b, (n, length) in enumerate(zip(news, lengths)):
            first = max(length - n, 0)
            for i in range(first // page, -(-length // page)) if min(n, length) else ():
                rows = k[f.cut[b] + i * page:f.cut[b] + min((i + 1) * page, length)]
                for h in range(heads):
                    want_codes[pages[b, i], h], want_scales[pages[b, i], h] = sel.summary(rows[:, h])
        assert np.array_equal(as_numpy(made.codes), want_codes), news
        assert np.array_equal(as_numpy(made.scales), want_scales), news
    f.free()


def test_summaries_of_pages_with_what_is_not_finite(gpu):  # noqa: F811
    """A NaN key, infinite ones of a pool that a host filled; values do not matter; and constant, tiny and large keys."""
    import karume_b200 as kb
    page, dim = 16, 64

    def rows(f):
        f.k[20, 0, 3] = math.nan
        f.v[40, 0, 3] = math.nan
        f.k[48:64] = 0.0
        f.k[64:80] = 1e-6
        f.k[80:96] = torch.linspace(-65504, 65504, 16, device="cuda")[:, None, None]

    f = Filled(gpu, [100], page, 1, dim, seed=3, rows=rows)
    params = f.cache.pool[f.pages[0, 6].item(), 0, page * dim:].view(torch.float16).view(2, page, 2)
    params[0, 1, 0] = math.inf
    k = as_numpy(f.k).copy()
    k[97] = math.inf
    made = gpu.cache_summaries(f.cache)
    gpu.cache_summarize(f.cache, made, kb.CacheBatch(f.pages, f.length, i32([0, 100]), tokens=100))
    gpu.sync()
    for i, p in enumerate(as_numpy(f.pages)[0]):
        codes, scales = sel.summary(k[i * page:min((i + 1) * page, 100), 0])
        assert np.array_equal(as_numpy(made.codes)[p, 0], codes) and np.array_equal(as_numpy(made.scales)[p, 0], scales, equal_nan=True), i
    assert np.isnan(as_numpy(made.scales)[as_numpy(f.pages)[0, [1, 6]]]).all() and np.isfinite(as_numpy(made.scales)[as_numpy(f.pages)[0, [0, 2, 3, 4, 5]]]).all()
    f.free()


# ---- selections -----------------------------------------------------------------------------


class Summarised:
    """Summaries at random, without the cache behind them: selecting reads nothing else."""

    def __init__(self, gpu, lengths, page, kv_heads, dim, seed, equal=0):
        import karume_b200 as kb
        rng = np.random.default_rng(seed)
        self.gpu, self.lengths, self.page, self.dim, self.kv_heads = gpu, lengths, page, dim, kv_heads
        pages, _, total = make_batch(rng, lengths, lengths, page)
        self.pages = pages
        codes = rng.integers(-127, 128, (total, kv_heads, 2, dim)).astype(np.int8)
        codes[:, :, 1] = np.abs(codes[:, :, 1]) // 8
        scales = np.exp(rng.normal(0, 0.3, (total, kv_heads, 2))).astype(np.float32) * 0.01
        if equal:  # pages that cannot be told apart
            codes, scales = codes[np.arange(total) % equal], scales[np.arange(total) % equal]
        self.codes, self.scales = codes, scales
        self.cache = gpu.kv_cache(total, page, kv_heads, dim)
        self.made = kb.CacheSummaries(dev(codes), dev(scales))

    def check(self, kind, news, heads, budget, first=1, last=1, rotary=0, interleaved=False, padding=0, strided=False, change=None, gpu=None):
        import karume_b200 as kb
        gpu, dim, h, tokens = gpu or self.gpu, self.dim, self.kv_heads, sum(news) + padding
        gen = torch.Generator(device="cuda").manual_seed(heads + tokens + budget)
        wide = torch.randn(tokens, heads + (3 if strided else 0), dim, generator=gen, device="cuda").to(ref.TYPES[kind])
        q = wide[:, :heads]
        if change is not None:
            change(q)
        table = kb.rope_table(max(self.lengths) + 1, rotary) if rotary else None
        starts = None if news == [1] * len(news) and not padding else i32(np.concatenate([[0], np.cumsum(news)]).tolist())
        batch = kb.CacheBatch(dev(self.pages), i32(self.lengths), starts, tokens=tokens)
        cache = self.cache if gpu is self.gpu else gpu.kv_cache(self.cache.pages, self.page, h, dim, pool=self.cache.pool)
        got = gpu.cache_select(cache, self.made, q, batch, budget, first=first, last=last, rope=kb.Rope(dev(table), interleaved) if rotary else None)
        again = gpu.cache_select(cache, self.made, q, batch, budget, first=first, last=last, rope=kb.Rope(dev(table), interleaved) if rotary else None,
                                 out=torch.full_like(got, 5))
        gpu.sync()
        assert torch.equal(got, again)
        got, at = as_numpy(got), 0
        for b, (n, length) in enumerate(zip(news, self.lengths)):
            qb, mine = q[at:at + n].float().cpu().numpy(), got[at:at + n]
            at += n
            position = np.arange(length - n, length)
            if rotary and n:
                qb = ref.rotate(qb, table, np.maximum(position, 0), interleaved)
            for t in range(n):
                count = position[t] // self.page + 1 if position[t] >= 0 else 0
                for g in range(h):
                    rows = slice(g * heads // h, (g + 1) * heads // h)
                    p = self.pages[b, :count]
                    ok = (p >= 0) & (p < len(self.codes))
                    score = np.full(count, np.nan, np.float32)
                    if ok.any():
                        score[ok] = sel.scores(qb[t, rows], self.codes[p[ok], g], self.scales[p[ok], g])
                    assert mine[t, g].tolist() == sel.select(score, budget, first, last), (kind, b, t, g)
        assert (got[at:] == -1).all()


@KINDS
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (256, 5, 1), (128, 32, 2), (64, 9, 1)])
def test_selections(gpu, kind, dim, heads, kv_heads):  # noqa: F811
    s = Summarised(gpu, [700, 16, 2100, 0, 33, 1], 16, kv_heads, dim, seed=dim + heads)
    s.check(kind, [1] * 6, heads, 8, first=1, last=2)
    s.check(kind, [1] * 6, heads, 40, first=0, last=1, rotary=dim)
    s.check(kind, [3, 5, 2, 0, 2, 1], heads, 20, first=2, last=3, rotary=dim // 2, interleaved=True, padding=2, strided=True)
    s.check(kind, [1] * 6, heads, 1, first=0, last=1)
    s.check(kind, [0, 0, 1, 0, 0, 0], heads, 131, first=100, last=31, rotary=dim)


@pytest.mark.parametrize("lengths,page,budget", [([16 * 9000 - 5, 100], 16, 128), ([64 * 1500, 64 * 900 + 1], 64, 200), ([32 * 1030], 32, 1029), ([16 * 8200], 16, 8199),
                                                 ([16 * 300], 16, 4000)])
def test_selections_of_long_sequences(gpu, lengths, page, budget):  # noqa: F811
    s = Summarised(gpu, lengths, page, 2, 64, seed=budget)
    s.check("f32", [1] * len(lengths), 6, budget, first=2, last=3, rotary=64)


def test_ties_go_to_the_lower_page(gpu):  # noqa: F811
    for equal, budget in ((1, 17), (3, 30), (7, 11)):
        s = Summarised(gpu, [16 * 60 + 4, 16 * 1200], 16, 2, 64, seed=equal, equal=equal)
        s.check("f32", [1, 1], 4, budget, first=0, last=2)
    # scores of zero have no sign
    s = Summarised(gpu, [16 * 50], 16, 1, 64, seed=9)
    s.check("f32", [1], 4, 9, first=0, last=1, change=lambda q: q.zero_())
    s.codes[:] = 0
    s.codes[::2, :, 0] = -1
    s.made.codes.copy_(dev(s.codes))
    s.check("f32", [1], 1, 9, first=0, last=1, change=lambda q: q.copy_(torch.where(torch.arange(64, device="cuda") % 2 == 0, 1.0, -1.0).expand_as(q)))


def test_what_is_not_a_number_is_taken(gpu):  # noqa: F811
    s = Summarised(gpu, [16 * 100, 16 * 40, 16 * 70], 16, 2, 64, seed=5)
    s.scales[s.pages[0, 13], 1] = np.nan
    s.scales[s.pages[0, 70], 0, 1] = np.nan
    s.scales[s.pages[0, 71], 0] = np.inf
    s.made.scales.copy_(dev(s.scales))
    s.pages[1, 5], s.pages[1, 9], s.pages[1, 20] = -1, len(s.codes), 1 << 30
    s.check("f32", [1, 1, 1], 4, 6, first=1, last=1)

    def bad(q):
        q[2, 1, 5] = math.nan
        q[0, 3, 0] = math.inf

    s.check("f32", [1, 1, 1], 4, 6, first=1, last=1, change=bad)


def test_selections_with_little_scratch_and_recorded(gpu):  # noqa: F811
    import karume_b200 as kb
    s = Summarised(gpu, [16 * 100, 16 * 40, 16 * 70, 16 * 90], 16, 2, 64, seed=6)
    small = kb.Gpu(0, workspace_bytes=4096)  # the keys of five rows
    s.check("f32", [1] * 4, 4, 6, gpu=small)
    s.check("f32", [9, 4, 1, 7], 4, 6, gpu=small)
    with pytest.raises(kb.KqError) as e:
        tiny = kb.Gpu(0, workspace_bytes=512)
        s.check("f32", [1] * 4, 4, 6, gpu=tiny)
    assert e.value.status == "KQ_ERR_UNSUPPORTED"
    q, length = torch.randn(4, 4, 64, device="cuda"), i32(s.lengths)
    batch, out = kb.CacheBatch(dev(s.pages), length), torch.zeros(4, 2, 6, dtype=torch.int32, device="cuda")
    gpu.sync()
    gpu.graph_begin()
    gpu.cache_select(s.cache, s.made, q, batch, 6, out=out)
    g = gpu.graph_end()
    for lengths in (s.lengths, [16 * 50, 1, 0, 16 * 90 - 3]):
        length.copy_(i32(lengths))
        gpu.graph_launch(g)
        gpu.sync()
        recorded = out.clone()
        assert torch.equal(recorded, gpu.cache_select(s.cache, s.made, q, batch, 6))
    gpu.graph_free(g)


# ---- attention over selected pages -------------------------------------------------------------


def check_selected(f, kind, news, heads, taken, rotary=0, strided=False, padding=0, scale=None):
    """f: a Filled cache; taken: function of the number of pages -> ascending indices, the last page among them, for each row and kv head."""
    import karume_b200 as kb
    gpu, dim, tokens = f.gpu, f.dim, sum(news) + padding
    kv_heads, page = f.cache.kv_heads, f.cache.page_tokens
    gen = torch.Generator(device="cuda").manual_seed(heads + tokens)
    q = torch.randn(tokens, heads + (1 if strided else 0), dim, generator=gen, device="cuda").to(ref.TYPES[kind])[:, :heads]
    table = kb.rope_table(max(max(f.lengths), 1), rotary) if rotary else None
    starts = None if news == [1] * len(news) and not padding else i32(np.concatenate([[0], np.cumsum(news)]).tolist())
    lists, where = [], []
    for b, n in enumerate(news):
        for t in range(n):
            position = f.lengths[b] - n + t
            lists.append([taken(position // page + 1, h) if position >= 0 else [] for h in range(kv_heads)])
            where.append((b, position))
    budget = max([len(one) for row in lists for one in row] + [1])
    selected = i32([[one + [-1] * (budget - len(one)) for one in row] for row in lists] + [[[-1] * budget] * kv_heads] * padding)
    batch = kb.CacheBatch(f.pages, f.length, starts, tokens=tokens)
    out = torch.full((tokens, heads + 1, dim), -7.0, dtype=q.dtype, device="cuda") if strided else None
    rope = kb.Rope(dev(table)) if rotary else None
    got = gpu.cache_attention(f.cache, q, batch, rope=rope, selected=selected, scale=scale, out=out[:, :heads] if strided else None)
    gpu.sync()
    if strided:
        assert bool((out[:, heads:] == -7).all())
    off = norm = 0.0
    for row, (b, position) in enumerate(where):
        if position < 0:
            assert bool((got[row] == 0).all())
            continue
        qr = q[row:row + 1].float()
        if rotary:
            qr = torch.from_numpy(ref.rotate(qr.cpu().numpy(), table, np.array([position]), False)).cuda()
        for h in range(kv_heads):
            keys = [i for j in lists[row][h] for i in range(j * page, min((j + 1) * page, position + 1))]
            at = torch.tensor(keys, device="cuda") + int(f.cut[b])
            mine = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            want, reach, largest = ref.attend(qr[:, mine].double(), f.k[at, h:h + 1].double(), f.v[at, h:h + 1].double(), scale or dim ** -0.5, 0)
            d = (got[row, mine].double() - want[0]).abs()
            assert bool((d <= ref.allowed(kind, want, reach, largest)[0]).all()), (kind, row, h)
            off, norm = off + float((d * d).sum()), norm + float((want * want).sum())
    assert bool((got[len(where):] == 0).all())
    if norm:
        assert math.sqrt(off / norm) <= {"f32": 1e-5, "f16": 2e-3, "bf16": 5e-3}[kind]


def some_of(seed, budget):
    rng = np.random.default_rng(seed)

    def taken(count, head):
        if count <= budget:
            return list(range(count))
        return sorted(rng.choice(count - 1, budget - 1, replace=False).tolist()) + [count - 1]

    return taken


@KINDS
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 4, 4, 16), (128, 8, 2, 64), (256, 4, 1, 32), (128, 24, 1, 128), (64, 40, 1, 256), (128, 9, 3, 16)])
def test_attention_over_selected_pages(gpu, kind, dim, heads, kv_heads, page):  # noqa: F811
    f = Filled(gpu, [5 * page + 3, 1, 0, 12 * page, page, 9 * page + page - 1], page, kv_heads, dim, seed=dim + page)
    check_selected(f, kind, [1] * 6, heads, some_of(0, 4), rotary=dim)
    check_selected(f, kind, [1] * 6, heads, some_of(1, 1))
    check_selected(f, kind, [3, 2, 1, 5, 0, 2], heads, some_of(2, 7), rotary=dim // 2, strided=True, padding=2, scale=0.2)
    f.free()


@KINDS
def test_long_selections_that_many_blocks_share(gpu, kind):  # noqa: F811
    f = Filled(gpu, [70001], 64, 2, 128, seed=1)
    check_selected(f, kind, [1], 12, some_of(3, 1000))
    check_selected(f, kind, [1], 12, some_of(3, 5000))
    check_selected(f, kind, [200], 2, some_of(4, 3))  # more rows than a block keeps the numbers of
    f.free()


def test_all_pages_are_the_whole(gpu):  # noqa: F811
    import karume_b200 as kb
    f = Filled(gpu, [1000, 30, 513], 64, 2, 128, seed=2)
    q, batch = torch.randn(3, 8, 128, device="cuda"), kb.CacheBatch(f.pages, f.length)
    made = gpu.cache_summaries(f.cache)
    gpu.cache_summarize(f.cache, made, kb.CacheBatch(f.pages, f.length, i32([0, 1000, 1030, 1543]), tokens=1543))
    every = gpu.cache_select(f.cache, made, q, batch, 16)
    assert every[0, 0].tolist() == list(range(16)) and every[1, 1].tolist() == [0] + [-1] * 15
    got, want = gpu.cache_attention(f.cache, q, batch, selected=every), gpu.cache_attention(f.cache, q, batch)
    gpu.sync()
    assert torch.equal(got, want)
    f.free()


def test_indices_that_are_no_pages_read_as_nan(gpu):  # noqa: F811
    import karume_b200 as kb
    f = Filled(gpu, [16 * 10, 16 * 10], 16, 1, 64, seed=4)
    q, batch = torch.randn(2, 2, 64, device="cuda"), kb.CacheBatch(f.pages, f.length)
    for bad in (-1, f.pages.shape[1], 1 << 30, -(1 << 31)):
        got = gpu.cache_attention(f.cache, q, batch, selected=i32([[[0, bad, 9]], [[3, 5, 9]]]))
        gpu.sync()
        assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    f.free()


def test_a_step_recorded_with_its_selection(gpu):  # noqa: F811
    """append, summarise, select, attend: replayed while the sequences grow, as when each is called."""
    import karume_b200 as kb
    steps, page, dim = 40, 16, 64
    f = Filled(gpu, [100, 16, 203], page, 2, dim, seed=5)
    free = f.cache.pool.shape[0]
    pool = torch.cat([f.cache.pool, torch.zeros((30, *f.cache.pool.shape[1:]), dtype=torch.uint8, device="cuda")])
    cache = gpu.kv_cache(free + 30, page, 2, dim, pool=pool)
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    table[:, :f.pages.shape[1]] = f.pages
    for b, n in enumerate((100, 16, 203)):
        held = -(-n // page)
        table[b, held:held + 4] = torch.arange(free + 10 * b, free + 10 * b + 4, device="cuda")
    length = f.length.clone()
    made = gpu.cache_summaries(cache)
    gpu.cache_summarize(cache, made, kb.CacheBatch(table, length, i32([0, 100, 116, 319]), tokens=319))
    q, k, v = (torch.zeros(3, n, dim, device="cuda") for n in (4, 2, 2))
    taken, out = torch.zeros(3, 2, 5, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, dim, device="cuda")
    rope, batch = kb.Rope(dev(kb.rope_table(400, dim))), kb.CacheBatch(table, length)

    def step():
        gpu.cache_append(cache, k, v, batch, rope=rope)
        gpu.cache_summarize(cache, made, batch)
        gpu.cache_select(cache, made, q, batch, 5, first=1, last=2, rope=rope, out=taken)
        gpu.cache_attention(cache, q, batch, rope=rope, selected=taken, out=out)

    gpu.sync()
    gpu.graph_begin()
    step()
    g = gpu.graph_end()
    before = pool.clone(), made.codes.clone(), made.scales.clone()
    runs = []
    for run in (lambda: gpu.graph_launch(g), step):
        for t, b in zip((pool, made.codes, made.scales), before):
            t.copy_(b)
        length.copy_(f.length)
        gen, got = torch.Generator(device="cuda").manual_seed(0), []
        for _ in range(steps):
            length += 1
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
            run()
            got.append((taken.clone(), out.clone()))
        gpu.sync()
        runs.append(got)
    assert all(torch.equal(a, c) and torch.equal(b, d) for (a, b), (c, d) in zip(*runs))
    assert len({tuple(t[0].flatten().tolist()) for t in runs[0]}) > 3
    gpu.graph_free(g)
    f.free()


def test_refusals(gpu):  # noqa: F811
    import karume_b200 as kb
    f = Filled(gpu, [40, 20], 16, 2, 64, seed=6)
    made, batch = gpu.cache_summaries(f.cache), kb.CacheBatch(f.pages, f.length)
    q, good = torch.randn(2, 4, 64, device="cuda"), i32([[[0, 2]] * 2, [[0, 1]] * 2])
    for call in (lambda: gpu.cache_select(f.cache, made, q, batch, 0), lambda: gpu.cache_select(f.cache, made, q, batch, 3, first=2, last=2),
                 lambda: gpu.cache_select(f.cache, made, q, batch, 3, last=0), lambda: gpu.cache_select(f.cache, made, q, batch, 3, first=-1),
                 lambda: gpu.cache_select(f.cache, made, q, batch, (1 << 20) + 1), lambda: gpu.cache_select(f.cache, made, q[:1], batch, 3),
                 lambda: gpu.cache_select(f.cache, made, q[:, :3], batch, 3), lambda: gpu.cache_select(f.cache, made, q, batch, 2, out=good[:, :1]),
                 lambda: gpu.cache_select(f.cache, made, q, batch, 2, out=good.long()), lambda: gpu.cache_select(f.cache, made, q.double(), batch, 2),
                 lambda: gpu.cache_select(f.cache, made, q, batch, 1 << 70),
                 lambda: gpu.cache_attention(f.cache, q, batch, selected=good, window=5), lambda: gpu.cache_attention(f.cache, q, batch, selected=good.long()),
                 lambda: gpu.cache_attention(f.cache, q, batch, selected=good[:1]), lambda: gpu.cache_attention(f.cache, q, batch, selected=good[:, :, :0]),
                 lambda: gpu.cache_attention(f.cache, q, batch, selected=good.transpose(1, 2)),
                 lambda: gpu.cache_attention(f.cache, q, batch, selected=good, shared=kb.SharedPrefixes(i32([0, 2]), i32([3]))),
                 lambda: kb.CacheSummaries(made.codes.float(), made.scales), lambda: kb.CacheSummaries(made.codes, made.scales[:, :1]),
                 lambda: kb.CacheSummaries(made.codes[:, :, :1], made.scales[:, :, :1]),
                 lambda: gpu.cache_summarize(f.cache, kb.CacheSummaries(made.codes[:2], made.scales[:2]), batch),
                 lambda: gpu.cache_summarize(f.cache, kb.CacheSummaries(torch.zeros(50, 2, 2, 128, dtype=torch.int8, device="cuda"), torch.zeros(50, 2, 2, device="cuda")), batch)):
        with pytest.raises(kb.KqError):
            call()
    cache, a = f.cache.handle, batch.args
    codes, scales = made.args
    for bad in ((codes + 4, scales), (0, scales), (codes, scales + 4), (codes, 0)):
        assert kb.lib.kq_cache_summarize(gpu._ctx, cache, *bad, *a) == 1
        assert kb.lib.kq_cache_select(gpu._ctx, cache, *bad, q.data_ptr(), 256, 0, 4, *a, 2, 1, 1, 0, 0, 0, 0, good.data_ptr()) == 1
    assert kb.lib.kq_cache_summarize(gpu._ctx, 12345, codes, scales, *a) == 1
    assert kb.lib.kq_cache_select(gpu._ctx, cache, codes, scales, q.data_ptr(), 256, 0, 4, *a, 2, 1, 1, 0, 0, 0, 0, 0) == 1
    assert kb.lib.kq_cache_attention_selected(gpu._ctx, cache, q.data_ptr(), 256, 0, 4, *a, 0, 2, 1.0, 0, 0, 0, 0, q.data_ptr(), 256) == 1
    gpu.plan_begin()
    try:
        assert kb.lib.kq_cache_summarize(gpu._ctx, cache, codes, scales, *a) == 8
    finally:
        with pytest.raises(kb.KqError):
            gpu.plan_end()
    f.free()


def test_pages_beyond_4_gib(gpu):  # noqa: F811
    """Pages, and their summaries, more than 4 GiB into the pool: selected, shared and summarised as those in front."""
    import karume_b200 as kb
    page, dim, heads = 256, 128, 2
    block = page * (dim + 8)
    count = (5 << 30) // (block * heads)
    cache = gpu.kv_cache(count, page, heads, dim, pool=torch.zeros(count, heads, block, dtype=torch.uint8, device="cuda"))
    near = gpu.kv_cache(8, page, heads, dim)
    far_rows, near_rows = i32([[count - 1, count - 3, count - 2], [count - 1, count - 4, count - 5]]), i32([[7, 5, 6], [7, 4, 3]])
    k, v = (torch.randn(1300, heads, dim, device="cuda") for _ in range(2))
    lengths, q = i32([700, 600]), torch.randn(2, 8, dim, device="cuda")
    out = []
    for c, rows in ((cache, far_rows), (near, near_rows)):
        both, one = kb.CacheBatch(rows, lengths, i32([0, 700, 1300]), tokens=1300), kb.CacheBatch(rows, lengths)
        gpu.cache_append(c, k, v, both)
        gpu.cache_append(c, k[:700], v[:700], kb.CacheBatch(rows[:1], lengths[:1], i32([0, 700]), tokens=700))  # the first page is the first one's
        made = gpu.cache_summaries(c)
        gpu.cache_summarize(c, made, both)
        taken = gpu.cache_select(c, made, q, one, 2, first=0, last=1)
        out.append([taken, made.codes[rows.long()], made.scales[rows.long()], gpu.cache_attention(c, q, one, selected=taken),
                    gpu.cache_attention(c, q.half(), one, shared=kb.SharedPrefixes(i32([0, 2]), i32([256]), least=0))])
        gpu.sync()
    assert all(torch.equal(a, b) for a, b in zip(*out))
    cache.free()
    near.free()


def test_summaries_beyond_4_gib(gpu):  # noqa: F811
    """Selecting reads nothing of the pool, so that it may be a small one: 9000 pages of 1024 heads of 256."""
    import ctypes
    import karume_b200 as kb
    pages, heads, dim, page = 9000, 1024, 256, 16
    handle, small = ctypes.c_uint64(0), torch.zeros(4096, dtype=torch.uint8, device="cuda")
    assert kb.lib.kq_cache_create(gpu._ctx, small.data_ptr(), pages, page, heads, dim, ctypes.byref(handle)) == 0
    cache = kb.KvCache(gpu, handle.value, small, pages, page, heads, dim)
    codes, scales = torch.zeros(pages, heads, 2, dim, dtype=torch.int8, device="cuda"), torch.zeros(pages, heads, 2, device="cuda")
    table = torch.arange(pages - 60, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    gen = torch.Generator(device="cuda").manual_seed(0)
    of = table[0].long()
    codes[of] = torch.randint(-127, 128, (60, heads, 2, dim), generator=gen, device="cuda").to(torch.int8)
    codes[of, :, 1] = codes[of, :, 1].abs()
    scales[of] = torch.rand(60, heads, 2, generator=gen, device="cuda")
    q = torch.randn(1, heads, dim, generator=gen, device="cuda")
    got = gpu.cache_select(cache, kb.CacheSummaries(codes, scales), q, kb.CacheBatch(table, i32([60 * page - 3])), 7, first=1, last=2)
    gpu.sync()
    for h in (0, 1, 511, 1022, 1023):
        score = sel.scores(as_numpy(q)[0, h:h + 1], as_numpy(codes[of, h]), as_numpy(scales[of, h]))
        assert got[0, h].tolist() == sel.select(score, 7, 1, 2), h
    cache.free()
