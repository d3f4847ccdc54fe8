"""Rotary positions, appending to the paged 4-bit cache and reading it back, against the plain statements of
tests/cache_reference.py: the same bits, since every rounding is part of the definition."""
import numpy as np
import pytest
import torch

from tests import cache_reference as ref

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


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def same(got, want):
    """Equal bits, any NaN equal to any other."""
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, want))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 3, 80, 20), (5, 2, 96, 6), (33, 4, 256, 64), (3, 5, 31, 30)])
def test_rope(gpu, kind, interleaved, tokens, heads, dim, rotary):
    import karume_b200 as kb
    rng = np.random.default_rng(tokens * dim + rotary)
    table = kb.rope_table(300, rotary)
    x = torch.from_numpy(rng.standard_normal((tokens, heads, dim)).astype(np.float32)).to(ref.TYPES[kind])
    positions = rng.integers(0, 300, tokens).astype(np.int32)
    want = torch.from_numpy(ref.rotate(x.float().numpy(), table, positions, interleaved)).to(x.dtype)
    got = gpu.rope(x.cuda(), dev(positions), kb.Rope(dev(table), interleaved))
    gpu.sync()
    same(got, want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset,stride", [(0, 64), (1, 65), (2, 70), (4, 68), (8, 72)])
def test_rope_of_strided_rows_in_place_at_any_alignment(gpu, interleaved, offset, stride):
    import karume_b200 as kb
    rng = np.random.default_rng(offset)
    for kind in ("f32", "bf16"):
        store = torch.from_numpy(rng.standard_normal(4 * stride + 80).astype(np.float32)).to(ref.TYPES[kind])
        table, positions = kb.rope_table(9, 24), np.array([8, 0, 3, 5], np.int32)
        rows = store.as_strided((4, 2, 32), (stride, 32, 1), offset)
        want = store.clone()
        want.as_strided((4, 2, 32), (stride, 32, 1), offset).copy_(
            torch.from_numpy(ref.rotate(rows.float().numpy(), table, positions, interleaved)).to(store.dtype))
        there = store.cuda()
        view = there.as_strided((4, 2, 32), (stride, 32, 1), offset)
        assert gpu.rope(view, dev(positions), kb.Rope(dev(table), interleaved), out=view) is view
        gpu.sync()
        same(there, want)


def test_rope_position_outside_the_table_is_nan(gpu):
    import karume_b200 as kb
    x = torch.ones(4, 2, 16, device="cuda")
    for interleaved in (False, True):
        got = gpu.rope(x, dev(np.array([0, 5, -1, 4], np.int32)), kb.Rope(dev(kb.rope_table(5, 8)), interleaved))
        gpu.sync()
        assert torch.isfinite(got[[0, 3]]).all() and torch.isnan(got[1:3, :, :8]).all() and (got[..., 8:] == 1).all()


def test_rope_table_scalings():
    """Host arithmetic: the ends of each scaling are what it promises."""
    import karume_b200 as kb
    plain, one = kb.rope_frequencies(64)
    assert one == 1.0 and plain[0] == 1.0
    linear, _ = kb.rope_frequencies(64, scaling=dict(kind="linear", factor=8))
    assert np.array_equal(linear, plain / 8)
    raised, _ = kb.rope_frequencies(64, scaling=dict(kind="base", factor=8))
    assert raised[0] == 1.0 and np.isclose(raised[-1], plain[-1] / 8, rtol=1e-12)
    for over, amplitude in (("turns", 1.0), ("index", 1 + 0.1 * np.log(4))):
        ramp, a = kb.rope_frequencies(64, scaling=dict(kind="ramp", factor=4, trained=2048, slow=1, fast=32, over=over))
        turns = 2048 * plain / (2 * np.pi)
        assert a == amplitude and np.array_equal(ramp[turns >= 40], plain[turns >= 40])
        assert np.allclose(ramp[turns <= 0.7], plain[turns <= 0.7] / 4, rtol=1e-12) and np.all(np.diff(ramp) < 0)
    table = kb.rope_table(100001, 8, base=500000.0)
    angle = 100000.0 * 500000.0 ** -0.25
    assert np.allclose(table[100000, 1], [np.cos(angle), np.sin(angle)], atol=1e-7)
    for bad in (dict(kind="linear", factor=0.5), dict(kind="other", factor=2), dict(kind="ramp", factor=2, trained=8, slow=2, fast=1)):
        with pytest.raises(ValueError):
            kb.rope_frequencies(64, scaling=bad)


def make_batch(rng, news, lengths, page, spare=2):
    """(pages i32 [sequences, width], starts, number of pages): scattered pages, unused entries out of range."""
    counts = [(n + page - 1) // page for n in lengths]
    width = max(1, max(counts))
    total = sum(counts) + spare
    order = rng.permutation(total)[:sum(counts)].astype(np.int32)
    pages = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, c in enumerate(counts):
        pages[b, :c] = order[at:at + c]
        at += c
    return pages, np.concatenate([[0], np.cumsum(news)]).astype(np.int32), total


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (128, 128, True), (128, 40, False), (256, 12, True), (64, 0, False), (128, 6, False)])
@pytest.mark.parametrize("page,news,lengths", [(16, [1, 1, 1], [1, 17, 40]), (64, [5, 0, 130, 1], [70, 9, 130, 1]), (32, [33], [64])])
def test_append_and_read(gpu, kind, dim, rotary, interleaved, page, news, lengths):
    import karume_b200 as kb
    rng = np.random.default_rng(dim + rotary + page)
    heads, tokens = 3, sum(news)
    pages, starts, total = make_batch(rng, news, lengths, page)
    pool = np.full((total, heads, page * (dim + 8)), 0xA5, np.uint8)
    qkv = rng.standard_normal((tokens, 2 * heads + 1, dim)).astype(np.float32) * 3
    qkv[0, 1] = 0.25         # a constant row
    qkv[-1, 2, 3] = 1000     # an outlier
    x = torch.from_numpy(qkv).to(ref.TYPES[kind])
    there = x.cuda()
    table = kb.rope_table(max(lengths), rotary) if rotary else None
    rope = kb.Rope(dev(table), interleaved) if rotary else None
    one_each = news == [1] * len(news)
    batch = kb.CacheBatch(dev(pages), dev(np.array(lengths, np.int32)), None if one_each else dev(starts), tokens=tokens)
    cache = gpu.kv_cache(total, page, heads, dim, pool=dev(pool))
    gpu.cache_append(cache, there[:, 1:1 + heads], there[:, 1 + heads:], batch, rope=rope)
    got_k, got_v = gpu.cache_read(cache, batch)
    gpu.sync()
    position = np.concatenate([np.arange(length - n, length) for n, length in zip(news, lengths)])
    seq = np.repeat(np.arange(len(news)), news)
    k, v = x.float().numpy()[:, 1:1 + heads], x.float().numpy()[:, 1 + heads:]
    if rotary:
        k = ref.rotate(k, table, position, interleaved)
    want = pool.copy()
    for which, rows, got in ((0, k, got_k), (1, v, got_v)):
        codes, scale, offset = ref.quantise(rows)
        same(got, torch.from_numpy(ref.stands_for(codes, scale, offset)))
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        params = np.stack([scale, offset], -1).view(np.uint8).reshape(tokens, heads, 4)
        # a held value is within half a step of the row's (and the roundings of scale and offset to binary16)
        step, top = scale.astype(np.float32)[..., None], np.abs(rows).max(-1, keepdims=True)
        assert np.all(np.abs(ref.stands_for(codes, scale, offset) - rows) <= 0.5 * step + 2.0 ** -9 * (top + step) * 2)
        for t in range(tokens):
            block = pages[seq[t], position[t] // page]
            slot = position[t] % page + which * page
            want[block, :, slot * dim // 2:(slot + 1) * dim // 2] = packed[t]
            want[block, :, page * dim + 4 * slot:page * dim + 4 * slot + 4] = params[t]
    assert np.array_equal(cache.pool.cpu().numpy(), want)  # and nothing else was touched
    cache.free()


def test_rows_that_four_bits_cannot_hold(gpu):
    """NaN, infinities and values beyond binary16 make their own row NaN, no other."""
    import karume_b200 as kb
    rng = np.random.default_rng(1)
    k = rng.standard_normal((6, 1, 64)).astype(np.float32)
    v = rng.standard_normal((6, 1, 64)).astype(np.float32)
    k[0, 0, 5], k[1, 0, 63], k[2, 0, 0], v[3, 0, 7], v[4, 0, 8] = np.nan, np.inf, -np.inf, 1e30, -70000
    k[5], v[5] = 6e-8, -65504.0
    batch = kb.CacheBatch(dev(np.zeros((1, 1), np.int32)), dev(np.array([6], np.int32)), dev(np.array([0, 6], np.int32)), tokens=6)
    cache = gpu.kv_cache(1, 16, 1, 64)
    gpu.cache_append(cache, dev(k), dev(v), batch)
    got = gpu.cache_read(cache, batch)
    gpu.sync()
    for rows, held in zip((k, v), got):
        same(held, torch.from_numpy(ref.stands_for(*ref.quantise(rows))))
    assert torch.isnan(got[0][:3]).all() and torch.isnan(got[1][3:5]).all() and torch.isfinite(got[0][3:]).all()
    cache.free()


def test_pages_and_positions_that_are_not_there(gpu):
    """A page number outside the pool, a token beyond the table and more new tokens than the sequence is long: nothing is
    written, what is read is NaN; an idle sequence is left alone."""
    import karume_b200 as kb
    pages = np.array([[0, -1], [7, 1], [2, 2], [1, 1]], np.int32)  # the pool has three pages
    lengths = np.array([20, 20, 35, 0], np.int32)
    k = torch.ones(4, 2, 64, device="cuda") * torch.arange(64, device="cuda")
    cache = gpu.kv_cache(3, 16, 2, 64)
    batch = kb.CacheBatch(dev(pages), dev(lengths))
    gpu.cache_append(cache, k, k, batch)
    got, _ = gpu.cache_read(cache, batch)
    gpu.sync()
    assert torch.isnan(got[[0, 2, 3]]).all() and torch.isfinite(got[1]).all()  # sequence 1's token 19 is on page 1
    assert int((cache.pool[[0, 2]] != 0).sum()) == 0
    late = kb.CacheBatch(dev(pages[2:3]), dev(np.array([2], np.int32)), dev(np.array([0, 4], np.int32)), tokens=4)
    gpu.cache_append(cache, k, k, late)
    got, _ = gpu.cache_read(cache, late)
    gpu.sync()
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2:]).all()
    cache.free()


def test_refusals(gpu):
    import karume_b200 as kb
    x, positions, rope = torch.zeros(2, 4, 64, device="cuda"), dev(np.zeros(2, np.int32)), kb.Rope(dev(kb.rope_table(8, 64)))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = gpu.kv_cache(2, 16, 2, 64)
    batch = kb.CacheBatch(i32(2, 1), i32(2))
    L = kb.lib

    def refused(status, call, *args, **kw):
        with pytest.raises(kb.KqError) as e:
            call(*args, **kw)
        assert e.value.status == status, e.value

    refused("KQ_ERR_SHAPE", gpu.rope, x, positions, kb.Rope(dev(kb.rope_table(8, 80))))
    refused("KQ_ERR_SHAPE", gpu.rope, x, positions.long(), rope)
    refused("KQ_ERR_BAD_ARG", gpu.rope, x.double(), positions, rope)
    refused("KQ_ERR_SHAPE", gpu.rope, x.transpose(1, 2), positions, rope)
    refused("KQ_ERR_SHAPE", gpu.kv_cache, 2, 24, 2, 64)
    refused("KQ_ERR_SHAPE", gpu.kv_cache, 2, 16, 2, 80)
    refused("KQ_ERR_SHAPE", gpu.kv_cache, 0, 16, 2, 64)
    refused("KQ_ERR_SHAPE", gpu.kv_cache, 2, 16, 2, 64, pool=torch.zeros(100, dtype=torch.uint8, device="cuda"))
    k = torch.zeros(2, 2, 64, device="cuda")
    refused("KQ_ERR_SHAPE", gpu.cache_append, cache, k[:1], k, batch)
    refused("KQ_ERR_SHAPE", gpu.cache_append, cache, x, x, batch)
    refused("KQ_ERR_BAD_ARG", gpu.cache_append, cache, k.double(), k.double(), batch)
    refused("KQ_ERR_SHAPE", gpu.cache_append, cache, k, k, batch, rope=kb.Rope(dev(kb.rope_table(8, 80))))
    shifted = torch.zeros(2 * 2 * 64 + 1, device="cuda")[1:].view(2, 2, 64)
    refused("KQ_ERR_BAD_ARG", gpu.cache_append, cache, shifted, k, batch)
    refused("KQ_ERR_SHAPE", gpu.cache_attention, cache, torch.zeros(2, 3, 64, device="cuda"), batch)
    refused("KQ_ERR_SHAPE", gpu.cache_attention, cache, torch.zeros(3, 4, 64, device="cuda"), batch)
    refused("KQ_ERR_BAD_ARG", gpu.cache_attention, cache, x, batch, scale=float("nan"))
    refused("KQ_ERR_BAD_ARG", gpu.cache_attention, cache, x, batch, scale=0.0)
    refused("KQ_ERR_BAD_ARG", gpu.cache_attention, cache, x.double(), batch)
    refused("KQ_ERR_SHAPE", kb.CacheBatch, i32(2, 1).long(), i32(2))
    refused("KQ_ERR_SHAPE", kb.CacheBatch, i32(2, 1), i32(3))
    refused("KQ_ERR_SHAPE", kb.CacheBatch, i32(2, 1), i32(2), i32(3))
    refused("KQ_ERR_SHAPE", kb.Rope, torch.zeros(8, 32, device="cuda"))
    gpu.plan_begin()
    for call in (lambda: gpu.rope(x, positions, rope), lambda: gpu.cache_append(cache, k, k, batch), lambda: gpu.cache_read(cache, batch),
                 lambda: gpu.cache_attention(cache, x, batch)):
        refused("KQ_ERR_STATE", call)
    with pytest.raises(kb.KqError):
        gpu.plan_end()  # nothing was recorded
    assert L.kq_cache_bytes(3, 16, 2, 64) == 3 * 2 * 16 * 72 and L.kq_cache_bytes(3, 17, 2, 64) == 0
    handle = cache.handle
    cache.free()
    assert L.kq_cache_free(gpu._ctx, handle) == 1
    cache.handle = handle
    refused("KQ_ERR_BAD_ARG", gpu.cache_append, cache, k, k, batch)
    refused("KQ_ERR_BAD_ARG", gpu.cache_read, cache, batch)
    refused("KQ_ERR_BAD_ARG", gpu.cache_attention, cache, x, batch)
    gpu.sync()
