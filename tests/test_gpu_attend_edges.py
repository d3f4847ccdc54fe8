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


def check_within_range(f, kind, new, heads, window=0, q_spread=1.0):
    """Filled.check for one sequence whose results may leave binary16: both sides end at its largest number there."""
    import karume_b200 as kb
    gen = torch.Generator(device="cuda").manual_seed(heads + new)
    q = (torch.randn(new, heads, f.dim, generator=gen, device="cuda") * q_spread).to(ref.TYPES[kind])
    batch = kb.CacheBatch(f.pages, f.length, dev(np.array([0, new], np.int32)), tokens=new)
    got = f.gpu.cache_attention(f.cache, q, batch, window=window)
    f.gpu.sync()
    want, reach, largest = ref.attend(q.double(), f.k.double(), f.v.double(), f.dim ** -0.5, window)
    allowed, got = ref.allowed(kind, want, reach, largest), got.double()
    assert not bool(torch.isnan(got).any())
    if kind == "f16":
        got, want = got.clamp(-65504, 65504), want.clamp(-65504, 65504)
    off = (got - want).abs()
    assert bool((off <= allowed).all()), (kind, new, window, float((off / allowed).max()))


@KINDS
@pytest.mark.parametrize("which", ["keys", "values", "both"])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_stand_for_more_than_binary16(gpu, kind, which, dim):  # noqa: F811
    """A row's offset and scale are binary16, what it stands for reaches beyond: rows up to 1e5 and 9e5 among ordinary ones, for who
    sees them and who does not."""
    def large(f):
        rng = np.random.default_rng(dim)
        for at, low, high in ((150, -3e4, 1e5), (151, -65000.0, 66000.0), (300, -65504.0, 9e5), (301, -65504.0, 65530.0)):
            for rows, wanted in ((f.k, which != "values"), (f.v, which != "keys")):
                if wanted:
                    row = rng.uniform(low, high, rows.shape[1:]).astype(np.float32)
                    row[:, 3], row[:, dim - 2] = low, high
                    rows[at] = torch.from_numpy(row).cuda()

    f = Filled(gpu, [400], 64, 1, dim, seed=13, spread=0.3, rows=large)
    assert float(f.v.abs().max()) > 8e5 or which == "keys"
    q_spread = 0.999 if which == "values" else 1e-5
    for new, window in ((400, 0), (100, 120), (1, 0)):
        check_within_range(f, kind, new, 4, window, q_spread)
    f.free()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_rows_of_infinities_reach_only_those_who_see_them(gpu, kind):  # noqa: F811
    """A pool that a host filled itself may hold infinite scales and offsets: to who sees them nothing is promised, to others they
    are nothing."""
    import karume_b200 as kb
    n, dim, page = 200, 128, 64
    f = Filled(gpu, [n], page, 1, dim, seed=14)
    pool, bad = f.cache.pool, 120
    at = f.pages[0, bad // page].item()
    params = pool[at, 0, page * dim:].view(torch.float16).view(2, page, 2)
    clean = params[:, bad % page].clone()
    q = torch.randn(n, 4, dim, device="cuda").to(ref.TYPES[kind])
    batch = kb.CacheBatch(f.pages, f.length, dev(np.array([0, n], np.int32)), tokens=n)
    want = gpu.cache_attention(f.cache, q, batch, window=50)
    gpu.sync()
    for scale, offset in ((math.inf, 0.0), (1.0, -math.inf), (-math.inf, math.inf)):
        params[:, bad % page] = torch.tensor([scale, offset], dtype=torch.float16, device="cuda")
        got = gpu.cache_attention(f.cache, q, batch, window=50)
        gpu.sync()
        assert torch.equal(got[:bad], want[:bad]) and torch.equal(got[bad + 50:], want[bad + 50:])
        assert not bool(torch.isfinite(got[bad:bad + 50]).all(-1).any())
    params[:, bad % page] = clean
    f.free()


@KINDS
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_with_one_large_value(gpu, kind, dim):  # noqa: F811
    """A value far from a key's others makes code times scale as large in every dim. A rotated query that is rounded to binary16
    must meet the offset as it was rounded: here all dims round the same way (an amplitude a little above one, as scalings for long
    contexts have it), 2^-11 of the score and not of dim times as much."""
    import karume_b200 as kb
    n = 300

    def outliers(f):
        at = torch.arange(n, device="cuda")
        f.k.zero_()
        f.k[at, 0, (5 * at) % dim] = -0.8 * dim * torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(dim), device="cuda")

    f = Filled(gpu, [n], 64, 1, dim, seed=15, rows=outliers)
    table = torch.zeros(n, dim // 2, 2, device="cuda")
    table[..., 0] = 1 + 0.45 * 2.0 ** -10  # no angle
    for new in (1, 5, 100):
        q = torch.ones(new, 4, dim, device="cuda", dtype=ref.TYPES[kind])
        batch = kb.CacheBatch(f.pages, f.length, dev(np.array([0, new], np.int32)), tokens=new)
        got = gpu.cache_attention(f.cache, q, batch, rope=kb.Rope(table))
        gpu.sync()
        want, reach, largest = ref.attend(q.double() * table[0, 0, 0].double(), f.k.double(), f.v.double(), dim ** -0.5, 0)
        off, allowed = (got.double() - want).abs(), ref.allowed(kind, want, reach, largest)
        assert bool((off <= allowed).all()), (kind, new, float((off / allowed).max()))
        # keys whose weights count have scores within a few of the largest: 2^-11 of that, and the bounds that Filled.check has
        assert float(off.norm() / want.norm()) <= {"f32": 1e-5, "f16": 2e-3, "bf16": 5e-3}[kind], (kind, new, float(off.norm() / want.norm()))
    f.free()


def test_windows_beyond_32_bits_and_below_zero(gpu):  # noqa: F811
    """A window is a number of keys: one that no sequence reaches hides nothing, whatever its low bits."""
    import karume_b200 as kb
    f = Filled(gpu, [300], 64, 1, 64, seed=16)
    q = torch.randn(1, 4, 64, device="cuda")
    one, many = kb.CacheBatch(f.pages, f.length), kb.CacheBatch(f.pages, f.length, dev(np.array([0, 40], np.int32)), tokens=40, most=(1 << 32) + 1)
    for batch, rows in ((one, q), (many, torch.randn(40, 4, 64, device="cuda"))):
        want = gpu.cache_attention(f.cache, rows, batch)
        for window in ((1 << 32) + 5, 1 << 32, (1 << 32) - 1, 1 << 31, 1 << 70):
            got = gpu.cache_attention(f.cache, rows, batch, window=window)
            gpu.sync()
            assert torch.equal(got, want), window
        narrow = gpu.cache_attention(f.cache, rows, batch, window=np.int64(5))
        gpu.sync()
        assert not torch.equal(narrow, want)
        with pytest.raises(kb.KqError) as e:
            gpu.cache_attention(f.cache, rows, batch, window=-1)
        assert e.value.status == "KQ_ERR_SHAPE"
    with pytest.raises(kb.KqError):
        kb.CacheBatch(f.pages, f.length, many.starts, tokens=40, most=-1)
    f.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [3, 80])
def test_query_rows_more_than_4_gib_apart(gpu, kind, new):  # noqa: F811
    import karume_b200 as kb
    f = Filled(gpu, [100], 16, 1, 64, seed=17)
    stride = (5 << 30) // (new - 1)  # bytes: the last row begins 5 GiB behind the first
    stride -= stride % 16
    store = torch.zeros(new * stride // 4, device="cuda").view(ref.TYPES[kind])
    each = stride // store.element_size()
    near = torch.randn(new, 4, 64, device="cuda").to(ref.TYPES[kind])
    far = store.as_strided((new, 4, 64), (each, 64, 1))
    far.copy_(near)
    batch = kb.CacheBatch(f.pages, f.length, dev(np.array([0, new], np.int32)), tokens=new)
    for rotary in (0, 64, 20):
        rope = kb.Rope(dev(kb.rope_table(100, rotary))) if rotary else None
        got, want = gpu.cache_attention(f.cache, far, batch, rope=rope), gpu.cache_attention(f.cache, near, batch, rope=rope)
        gpu.sync()
        assert torch.equal(got, want)
    f.free()


@KINDS
@pytest.mark.parametrize("dim,mean", [(64, 0.0), (64, 3.0), (128, 3.0)])
def test_long_sums_that_no_other_block_shares(gpu, kind, dim, mean):  # noqa: F811
    """So many blocks of rows that each walks over all 70001 keys by itself, 16-bit sums in one chain of the tensor core's accumulators.
    It cuts a sum at its last bit at every sixteen keys: 2^-23 of it each, all one way where the values have one sign. On top 16-bit
    results have three roundings of binary16 (2.1e-4 each of the norm) and that of their type."""
    import karume_b200 as kb
    n, new, heads, last = 70001, 9600, 8, 40

    def one_sign(f):
        f.v += mean

    f = Filled(gpu, [n], 64, heads, dim, seed=18, spread=0.3, rows=one_sign)
    q = torch.randn(new, heads, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(dim)).to(ref.TYPES[kind])
    got = gpu.cache_attention(f.cache, q, kb.CacheBatch(f.pages, f.length, dev(np.array([0, new], np.int32)), tokens=new))
    gpu.sync()
    want, reach, largest = ref.attend(q[-last:].double(), f.k.double(), f.v.double(), dim ** -0.5, 0)
    off = (got[-last:].double() - want).abs()
    assert bool((off <= ref.allowed(kind, want, reach, largest)).all())
    chain = 0.0 if kind == "f32" else n / 16 * 2.0 ** -23
    bound = {"f32": 1e-5, "f16": 6e-4, "bf16": 2e-3}[kind] + chain
    assert float(off.norm() / want.norm()) <= bound, (kind, float(off.norm() / want.norm()), bound)
    f.free()
