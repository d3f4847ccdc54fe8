"""Serving many conversations from one paged 4-bit cache: pages that sequences share (forked, truncated, grown, compacted, copied),
attention for groups of sequences with a common prefix, attention over the pages that a cheap score selects for each query.

The cache: a page holds `page` tokens; for each kv head its block is
    [K codes: page x dim / 2 bytes][V codes: likewise][K (scale, offset): page x 2 binary16][V (scale, offset): likewise]
with element 2 i in the low nibble of byte i; a code stands for code * scale + offset.

Pages: `table` [sequences, width] names the pages of each sequence in order (-1 behind them), `lengths` [sequences] its tokens,
`refs` [pages] how many rows of the table name a page.  Sequence b of length n has ceil(n / page) pages; one that is not full has one name.
  fork(parents, keep)  all at once, from what was there before: b becomes the first min(keep[b], length) tokens of sequence parents[b]
                       (negative: none).  Whole pages are shared.  A last page that is not full and that nobody names any more goes to
                       the lowest b that continues in it; every other one gets a free page and a pair (its page, the free page).
  grow(news)           room for news[b] more tokens of b.
  compact()            pages in use move to the lowest numbers: the r-th of those at or beyond the number of pages in use to the r-th
                       free one below it, as pairs (from, to).
  copy(pairs)          the pages' content, in every layer's pool.
Free pages (refs 0) are taken lowest first, in the order of sequences and of their pages.

Shared prefixes: sequences first[g] .. first[g + 1] - 1 have the same first shared[g] tokens.  Attention is that over the whole of each
sequence: query i of the n new ones of a sequence of length L has position p = L - n + i and sees the keys max(0, p - window + 1) .. p.

Selection: a page's summary for a kv head is, over its tokens' keys, c = (max + min) / 2 and r = (max - min) / 2 of each channel, both held as
8-bit codes with a scale, as rows of activations are: scale = max(max |x| / 127, tiny), code = rint(x / scale).  A rotated query held likewise (codes
a, scale s_a) scores s_a ((a . c) s_c + (|a| . r) s_r), a bound of its products with the page's keys; the largest of the heads that share the kv head counts.
Every (query, kv head) takes the first `first` pages, the last `last` ones and, up to `budget` in all, those with the largest scores, ties to
the lower page; it attends to their tokens up to its position.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 1.1754943508222875e-38
# (query heads, kv heads, head dim): the 8B-shaped decoder, the 1.5B-class one and the small test decoder of this
# repository, then one key head for all queries, one for each, and wide heads.
HEADS = [(32, 8, 128), (12, 2, 128), (8, 4, 64), (16, 1, 128), (8, 8, 64), (8, 4, 256)]


def listed():
    return [
        # Beam search on two short prompts: each beam continues one of the four.  The smallest call: what it takes is latency.
        dict(name="fork_beams", kind="fork", prompts=2, children=3, longest=403, page=16, kv_heads=4, dim=64, layers=4, cut=0),
        # Sixteen answers to each of four long prompts, in every layer's pool of an 8B-shaped decoder.
        dict(name="fork_answers", kind="fork", prompts=4, children=15, longest=8190, page=64, kv_heads=8, dim=128, layers=32, cut=0),
        # 256 conversations give back the drafted tokens that were not accepted, and make room for the next ones.
        dict(name="fork_drafts", kind="fork", prompts=256, children=0, longest=32768, page=64, kv_heads=2, dim=128, layers=1, cut=40),
        # A small pool after a third of its conversations ended.
        dict(name="compact_small", kind="compact", sequences=12, longest=2000, page=32, kv_heads=2, dim=128, layers=2),
        # A server's pool, eight layers at a time.
        dict(name="compact_server", kind="compact", sequences=96, longest=8192, page=64, kv_heads=8, dim=128, layers=8),
        # Two answers to one question of a thousand tokens: the smallest group.
        dict(name="shared_pair", kind="shared", x="f32", groups=1, members=2, new=1, prefix=1000, longest=100, heads=32, kv_heads=8, dim=128, page=64,
             window=0, rotary=128),
        # Sixteen conversations behind one system prompt, f32 as the projections give it.
        dict(name="shared_batch", kind="shared", x="f32", groups=1, members=16, new=1, prefix=4096, longest=500, heads=12, kv_heads=2, dim=128, page=64,
             window=0, rotary=128),
        # A full server whose 64 conversations are about one long document.
        dict(name="shared_server", kind="shared", x="bf16", groups=1, members=64, new=1, prefix=32768, longest=1024, heads=32, kv_heads=8, dim=128, page=64,
             window=0, rotary=128),
        # Drafts of five tokens in four groups of eight, prefixes that end inside a page, a window, small heads and pages.
        dict(name="shared_drafts", kind="shared", x="f16", groups=4, members=8, new=5, prefix=3001, longest=700, heads=8, kv_heads=4, dim=64, page=16,
             window=2048, rotary=64),
        # One conversation that reads 32 of its pages at each token.
        dict(name="select_one", kind="select", x="f32", sequences=1, new=1, longest=8190, budget=32, first=1, last=2, heads=32, kv_heads=8, dim=128, page=64,
             rotary=128),
        # One very long document on a small decoder, f16.
        dict(name="select_long", kind="select", x="f16", sequences=1, new=1, longest=200003, budget=128, first=1, last=4, heads=12, kv_heads=2, dim=128, page=64,
             rotary=128),
        # A server of 64 long conversations, bf16, 64 pages a token: the largest set of scores and of selected pages.
        dict(name="select_server", kind="select", x="bf16", sequences=64, new=1, longest=32768, budget=64, first=1, last=2, heads=32, kv_heads=8, dim=128, page=64,
             rotary=128),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["fork", "compact", "shared", "select"], [2, 1, 4, 3])[0]
    heads, kv_heads, dim = rng.choice(HEADS[:3] * 2 + HEADS[3:])
    page = rng.choice([16, 32, 64, 64, 128])
    x = rng.choice(["f32", "f32", "f16", "bf16"])
    rotary = rng.choice([dim, dim, dim // 2, 0])
    while True:
        if kind == "fork":
            children = rng.choice([0, _spread(rng, 1, 16)])
            case = dict(kind=kind, prompts=_spread(rng, 1, 256 if children == 0 else 16), children=children, longest=_spread(rng, 20, 32768), page=page,
                        kv_heads=kv_heads, dim=dim, layers=_spread(rng, 1, 32), cut=_spread(rng, 1, 200) if children == 0 else rng.choice([0, 0, 17]))
        elif kind == "compact":
            case = dict(kind=kind, sequences=_spread(rng, 3, 96), longest=_spread(rng, 50, 8192), page=page, kv_heads=kv_heads, dim=dim, layers=_spread(rng, 1, 8))
        elif kind == "shared":
            case = dict(kind=kind, x=x, groups=_spread(rng, 1, 8), members=_spread(rng, 1, 64), new=rng.choice([1, 1, 1, rng.randint(2, 8), _spread(rng, 9, 300)]),
                        prefix=_spread(rng, 16, 32768), longest=_spread(rng, 1, 2048), heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                        window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]), rotary=rotary)
        else:
            first, last = rng.randint(0, 2), rng.randint(1, 4)
            case = dict(kind=kind, x=x, sequences=_spread(rng, 1, 64), new=rng.choice([1, 1, 1, rng.randint(2, 6)]), longest=_spread(rng, 20, 200000),
                        budget=max(first + last, _spread(rng, 4, 256)), first=first, last=last, heads=heads, kv_heads=kv_heads, dim=dim, page=page, rotary=rotary)
        most = [work(c) for c in listed() if c["kind"] == kind]
        need = work(case)
        if need["bytes"] > max(w["bytes"] for w in most) or need["flops"] > max(w["flops"] for w in most):
            continue
        # what is held: pools of at most 2 GB, and scores of a plain form of at most 2^30
        if _held(case) <= (2 << 30) and case.get("members", 1) * case.get("groups", 1) * case.get("new", 1) * (case.get("prefix", 0) + case["longest"]) * heads <= 1 << 30:
            return case


def _share(count):
    """1 / 4 to all of something, spread evenly over `count`."""
    return [1.0 if b == 0 else 0.25 + 0.75 * math.modf(b * 0.6180339887498949)[0] for b in range(count)]


def _page_bytes(case):
    return case["kv_heads"] * case["page"] * (case["dim"] + 8)


def _fork_lengths(case):
    """(length, kept, new) of each sequence: a prompt and behind it its children; or (no children) all cut back and grown again."""
    lengths, keep, news = [], [], []
    for i, s in enumerate(_share(case["prompts"])):
        n = max(1, round(s * case["longest"]))
        if case["children"] == 0:
            kept = max(0, n - 1 - (i * 7) % max(case["cut"], 1))
            lengths, keep, news = lengths + [n], keep + [kept], news + [n - kept]
        else:
            kept = max(1, n - case["cut"])
            lengths += [n] + [0] * case["children"]
            keep += [n] + [kept] * case["children"]
            news += [0] + [1] * case["children"]
    return lengths, keep, news


def _pages_of(n, page):
    return (n + page - 1) // page


def _compact_lengths(case):
    return [0 if b % 3 == 1 else max(1, round(s * case["longest"])) for b, s in enumerate(_share(case["sequences"]))]


def _shared_lengths(case):
    """(prefix of each group, new and length of each sequence)."""
    prefix = [max(1, round(s * case["prefix"])) for s in _share(case["groups"])]
    new, lengths = [], []
    for b, s in enumerate(_share(case["groups"] * case["members"])):
        n = max(1, round(s * case["new"]))
        new.append(n)
        lengths.append(prefix[b // case["members"]] + n - 1 + max(1, round(s * case["longest"])))
    return prefix, new, lengths


def _select_lengths(case):
    """(new, length) of each sequence."""
    new = [max(1, round(s * case["new"])) for s in _share(case["sequences"])]
    return new, [max(n, round(s * case["longest"])) for n, s in zip(new, _share(case["sequences"]))]


def _held(case):
    page = case["page"]
    if case["kind"] == "fork":
        lengths, keep, news = _fork_lengths(case)
        return case["layers"] * _page_bytes(case) * _fork_pool(case)
    if case["kind"] == "compact":
        return case["layers"] * _page_bytes(case) * sum(_pages_of(max(1, round(s * case["longest"])), page) for s in _share(case["sequences"]))
    if case["kind"] == "shared":
        return _page_bytes(case) * (case["groups"] * (case["prefix"] // page) + case["groups"] * case["members"] * _pages_of(case["longest"] + case["new"] + page, page))
    return _page_bytes(case) * sum(_pages_of(n, page) for n in _select_lengths(case)[1])


def _fork_pool(case):
    lengths, keep, news = _fork_lengths(case)
    page = case["page"]
    return sum(_pages_of(n, page) for n in lengths) + sum(2 + _pages_of(m, page) for m in news) + 5


# ---- what a user's program holds -----------------------------------------------------------


class _State:
    held = None  # the framework's view of the tensors, made at the first call


def _i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _angles(positions, rotary):
    """(cos, sin) of position * 10000^(-2 i / rotary), f32."""
    f = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _pool(case, pages, gen):
    """A pool in which every page has been used: keys with channels of different spread and mean that drift from page to page, values around zero."""
    h, d, p = case["kv_heads"], case["dim"], case["page"]
    pool = torch.empty(pages, h, p * (d + 8), device="cuda", dtype=torch.uint8)
    gain = torch.exp(0.3 * torch.randn(h, 1, d, generator=gen, device="cuda"))
    mean = 0.5 * torch.randn(h, 1, d, generator=gen, device="cuda")
    step = max(1, (1 << 26) // (h * d * p))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        drift = 0.5 * torch.randn(n, h, 1, d, generator=gen, device="cuda")
        for which in (0, 1):
            x = torch.randn(n, h, p, d, generator=gen, device="cuda")
            codes, params = _quantise(torch.addcmul(mean + drift, x, gain) if which == 0 else x)
            pool[at:at + n, :, which * p * d // 2:(which + 1) * p * d // 2] = codes.flatten(-2)
            pool[at:at + n, :, p * d + 4 * which * p:p * d + 4 * (which + 1) * p] = params.flatten(-2)
    return pool


def _table(counts, width, order):
    """Rows of the page numbers in `order`, counts[b] of them in row b, -1 behind them."""
    table = torch.full((len(counts), width), -1, device="cuda", dtype=torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table[used] = order[:sum(counts)].to(torch.int32)
    return table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.case, page = case, case["page"]
    if case["kind"] in ("fork", "compact"):
        if case["kind"] == "fork":
            lengths, keep, news = _fork_lengths(case)
            pages, live = _fork_pool(case), lengths
            width = max(_pages_of(max(n, k + m), page) for n, k, m in zip(lengths, keep, news))
            per = case["children"] + 1
            s.parents = _i32([b - b % per for b in range(len(lengths))])
            s.keep, s.news = _i32(keep), _i32(news)
        else:  # page numbers as when the conversations that ended were there too
            live = _compact_lengths(case)
            lengths = [max(1, round(v * case["longest"])) for v in _share(case["sequences"])]
            pages = sum(_pages_of(n, page) for n in lengths)
            width = max(_pages_of(n, page) for n in lengths)
        order = torch.randperm(pages, generator=gen, device="cuda")
        s.table = _table([_pages_of(n, page) for n in lengths], width, order)
        s.table[_i32(live) == 0] = -1
        s.lengths = _i32(live)
        s.refs = torch.zeros(pages + 1, device="cuda", dtype=torch.int32)
        s.refs.scatter_add_(0, torch.where(s.table < 0, pages, s.table).flatten().long(), torch.ones_like(s.table).flatten())
        s.refs = s.refs[:pages].clone()
        s.report = torch.zeros(4, device="cuda", dtype=torch.int32)
        s.pools = torch.randint(0, 256, (case["layers"], pages, _page_bytes(case)), generator=gen, device="cuda", dtype=torch.uint8)
        if case["kind"] == "compact":
            s.before = s.table.clone(), s.refs.clone()
        return s
    h, d, dtype = case["kv_heads"], case["dim"], TORCH_DTYPE[case["x"]]
    if case["kind"] == "shared":
        prefix, news, lengths = _shared_lengths(case)
        whole = [prefix[b // case["members"]] // page for b in range(len(lengths))]
        width = max(_pages_of(n, page) for n in lengths)
        own_pages = [_pages_of(n, page) - w for n, w in zip(lengths, whole)]
        total = sum(own_pages) + sum(n // page for n in prefix) + 1  # page 0 is nobody's
        order = 1 + torch.randperm(total - 1, generator=gen, device="cuda").to(torch.int32)
        s.pool = _pool(case, total, gen)
        s.pages = torch.zeros(len(lengths), width, device="cuda", dtype=torch.int32)
        at = 0
        for g, n in enumerate(prefix):
            s.pages[g * case["members"]:(g + 1) * case["members"], :n // page] = order[at:at + n // page]
            at += n // page
        for b, n in enumerate(own_pages):
            s.pages[b, whole[b]:whole[b] + n] = order[at:at + n]
            at += n
        for g, n in enumerate(prefix):  # a prefix's last page that is not full: the members' copies of it
            if n % page:
                copies = s.pages[g * case["members"]:(g + 1) * case["members"], n // page].long()
                s.pool[copies] = s.pool[copies[0]].clone()
        s.first, s.shared = _i32([g * case["members"] for g in range(case["groups"] + 1)]), _i32(prefix)
    else:
        news, lengths = _select_lengths(case)
        counts = [_pages_of(n, page) for n in lengths]
        s.pool = _pool(case, sum(counts) + 1, gen)
        s.pages = _table(counts, max(counts), 1 + torch.randperm(sum(counts), generator=gen, device="cuda")).clamp(min=0)
        s.codes = torch.zeros(len(s.pool), h, 2, d, device="cuda", dtype=torch.int8)
        s.scales = torch.zeros(len(s.pool), h, 2, device="cuda")
        step = max(1, (1 << 26) // (h * page * d))
        for at in range(0, len(s.pool), step):  # every page's summary, as earlier calls left them
            keys = _values(*(v[at:at + step] for v in _views(s.pool, page, d)[0::2]))
            s.codes[at:at + step], s.scales[at:at + step] = _summary(keys.amin(2), keys.amax(2))
    s.lengths = _i32(lengths)
    s.starts = _i32([0] + news).cumsum(0).to(torch.int32) if case["new"] > 1 else None
    s.tokens, s.most = sum(news), max(news)
    s.angles = _angles(max(lengths), case["rotary"]) if case["rotary"] else None
    s.q = torch.randn(s.tokens, case["heads"], d, generator=gen, device="cuda").to(dtype)
    return s


# ---- the plain form ------------------------------------------------------------------------


def _add_names(refs, table, counted, by):
    """refs plus `by` for every page that `table` names where `counted`."""
    there = counted & (table >= 0) & (table < len(refs))
    refs.scatter_add_(0, torch.where(there, table, 0).flatten().long(), (there * by).flatten().to(torch.int32))


def _plain_fork(s):
    """Returns the pairs; table, lengths and refs are written."""
    table, lengths, refs, page = s.table, s.lengths, s.refs, s.case["page"]
    n_seq, width = table.shape
    seq, index = torch.arange(n_seq, device="cuda"), torch.arange(width, device="cuda")[None]
    parent = s.parents.long().clamp(min=0)
    n = torch.where(s.parents >= 0, torch.minimum(s.keep, lengths[parent]), 0)
    changed = ((s.parents != seq) | (n < lengths))[:, None]
    rows = table[parent]
    _add_names(refs, table, changed & (index < (lengths[:, None] + page - 1) // page), -1)
    _add_names(refs, rows, changed & (index < n[:, None] // page), 1)
    tail = changed[:, 0] & (n % page > 0)
    at = (n // page).clamp(max=width - 1).long()[:, None]
    last = rows.gather(1, at)[:, 0].long().clamp(min=0)
    free = tail & (refs[last] == 0)
    lowest = torch.full((len(refs),), n_seq, device="cuda").scatter_reduce_(0, last, torch.where(free, seq, n_seq), "amin")
    takes = free & (lowest[last] == seq)
    refs.scatter_add_(0, last, takes.to(torch.int32))
    copies = tail & ~takes
    rank = (copies.cumsum(0) - 1).clamp(min=0)
    fresh = torch.argsort((refs != 0).to(torch.int8), stable=True)[:n_seq][rank.clamp(max=len(refs) - 1)]
    refs.scatter_add_(0, fresh, copies.to(torch.int32))
    pairs = torch.full((n_seq + 1, 2), -1, device="cuda", dtype=torch.int32)
    pairs[torch.where(copies, rank, n_seq)] = torch.stack([last, fresh], 1).to(torch.int32)
    rows = rows.scatter(1, at, torch.where(copies[:, None], fresh[:, None].to(torch.int32), rows.gather(1, at)))
    table.copy_(torch.where(index < (n[:, None] + page - 1) // page, rows, -1))
    lengths.copy_(n)
    count = copies.sum().to(torch.int32)
    s.report.copy_(torch.stack([count * 0, count, count, count * 0]))
    return pairs[:n_seq]


def _plain_grow(s):
    table, lengths, refs, page = s.table, s.lengths, s.refs, s.case["page"]
    index = torch.arange(table.shape[1], device="cuda")[None]
    held, wanted = (lengths[:, None] + page - 1) // page, ((lengths + s.news)[:, None] + page - 1) // page
    takes = (index >= held) & (index < wanted)
    rank = takes.flatten().cumsum(0).view(takes.shape) - 1
    fresh = torch.argsort((refs != 0).to(torch.int8), stable=True)[rank.clamp(0, len(refs) - 1)]
    table.copy_(torch.where(takes, fresh.to(torch.int32), table))
    refs.scatter_add_(0, fresh.flatten(), takes.flatten().to(torch.int32))
    lengths += s.news
    count = takes.sum().to(torch.int32)
    s.report.copy_(torch.stack([count * 0, count, count * 0, count * 0]))


def _plain_copy(pools, pairs):
    pairs = pairs[pairs[:, 0] >= 0].long()
    pools[:, pairs[:, 1]] = pools[:, pairs[:, 0]]


def _plain_compact(s):
    table, refs = s.table, s.refs
    page = torch.arange(len(refs), device="cuda")
    used = refs > 0
    count = used.sum()
    moves, holes = used & (page >= count), ~used & (page < count)
    n = moves.sum()
    source, target = (torch.argsort((~m).to(torch.int8), stable=True) for m in (moves, holes))
    moved = page < n
    to = page.scatter(0, source, torch.where(moved, target, source))
    table.copy_(torch.where(table >= 0, to[table.long().clamp(min=0)].to(torch.int32), -1))
    names = refs[source]
    refs.copy_(torch.where(moves, 0, refs))
    refs.scatter_add_(0, target, torch.where(moved, names, 0).to(torch.int32))
    s.report.copy_(torch.stack([count * 0, count, n, count * 0]).to(torch.int32))
    return torch.where(moved[:, None], torch.stack([source, target], 1), -1).to(torch.int32)


def _rotate(x, rows):
    """x [tokens, heads, dim] in f32; rows [tokens, rotary / 2, 2]: pairs i and i + rotary / 2."""
    c, s = rows[:, None, :, 0], rows[:, None, :, 1]
    r = 2 * c.shape[-1]
    x0, x1 = x[..., :r // 2], x[..., r // 2:r]
    return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s, x[..., r:]], -1)


def _quantise(x):
    """f32 rows [..., dim] -> 4-bit codes [..., dim / 2] and (scale, offset) as bytes [..., 4]."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    offset = low.half()
    scale = ((high - offset.float()) * torch.tensor(1 / 15, device=x.device)).half().clamp(min=0)
    code = torch.round((x - offset.float()) * (1 / scale.float())).clamp(0, 15)
    code = torch.where(scale > 0, code, 0).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([scale, offset], -1).view(torch.uint8)


def _views(pool, page, dim):
    """The pool's K codes, V codes [pages, heads, page, dim / 2], K and V (scale, offset) bytes [pages, heads, page, 4]."""
    half = page * dim // 2
    return (pool[..., :half].unflatten(-1, (page, dim // 2)), pool[..., half:2 * half].unflatten(-1, (page, dim // 2)),
            pool[..., 2 * half:2 * half + 4 * page].unflatten(-1, (page, 4)), pool[..., 2 * half + 4 * page:].unflatten(-1, (page, 4)))


def _values(codes, params):
    """What codes [..., dim / 2] with (scale, offset) bytes [..., 4] stand for, f32."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.contiguous().view(torch.float16).float()
    return code * p[..., :1] + p[..., 1:]


def _eight_bits(x):
    """f32 rows [..., dim] -> 8-bit codes (as f32) and a scale [...]."""
    scale = (x.abs().amax(-1) * torch.tensor(1 / 127, device=x.device)).clamp(min=TINY)
    return torch.round(x / scale[..., None]).clamp(-127, 127), scale


def _summary(low, high):
    """Channels' least and largest keys [..., dim] -> codes int8 [..., 2, dim], scales f32 [..., 2]."""
    codes, scales = _eight_bits(torch.stack([(high + low) * 0.5, (high - low) * 0.5], -2))
    return codes.to(torch.int8), scales


def _new_tokens(s):
    """(sequence, position) of each new token."""
    if s.starts is None:
        return torch.arange(len(s.lengths), device="cuda"), s.lengths.long() - 1
    at = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(s.starts.long(), at, right=True) - 1
    return seq, s.lengths.long()[seq] - s.starts.long()[seq + 1] + at


def _softmax_of(score, sees, value):
    """Weights of `score` [.., rows, keys] where it `sees`, times `value` [.., keys, dim]; zeros where nothing is seen."""
    score = score.masked_fill_(~sees, -math.inf)
    weight = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, value) / torch.where(total > 0, total, 1)


def _plain_shared(s):
    case = s.case
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    group, n, members, width = case["heads"] // h, s.most, case["members"], s.pages.shape[1]
    seq, pos = _new_tokens(s)
    q = s.q.float()
    if s.angles is not None:
        q = _rotate(q, s.angles[pos])
    first = s.starts.long()[:-1] if s.starts is not None else torch.arange(len(s.lengths), device="cuda")
    row = torch.arange(s.tokens, device="cuda") - first[seq]
    padded = torch.zeros(len(s.lengths), n, case["heads"], d, device="cuda")
    padded[seq, row] = q
    at = torch.full((len(s.lengths), n), -1, device="cuda")
    at[seq, row] = pos
    rows = padded.view(-1, n, h, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [sequences, kv heads, group x n, dim]
    kc, vc, kp, vp = (t[s.pages.long()].transpose(1, 2).flatten(2, 3) for t in _views(s.pool, page, d))  # [sequences, heads, width * page, ..]
    key = torch.arange(width * page, device="cuda")
    sees = key <= at[..., None]
    if case["window"]:
        sees &= key > at[..., None] - case["window"]
    score = torch.matmul(rows, _values(kc, kp).transpose(-1, -2)) * d ** -0.5
    out = _softmax_of(score, sees[:, None, None].expand(-1, h, group, -1, -1).flatten(2, 3), _values(vc, vp))
    return out.view(-1, h, group, n, d).permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, row].to(s.q.dtype)


def _plain_select(s):
    case = s.case
    h, d, page, budget, width = case["kv_heads"], case["dim"], case["page"], case["budget"], s.pages.shape[1]
    group = case["heads"] // h
    seq, pos = _new_tokens(s)
    kc, vc, kp, vp = _views(s.pool, page, d)
    # the summaries of the pages that the new tokens are in
    index = pos // page
    written = s.pages.long()[seq, index]
    keys = _values(kc[written], kp[written])  # [tokens, kv heads, page, dim]
    there = ((index * page)[:, None] + torch.arange(page, device="cuda") < s.lengths[seq][:, None])[:, None, :, None]
    s.codes[written], s.scales[written] = _summary(torch.where(there, keys, math.inf).amin(2), torch.where(there, keys, -math.inf).amax(2))
    # the scores of all pages; whole numbers below 2^24, exact in f32
    q = s.q.float()
    if s.angles is not None:
        q = _rotate(q, s.angles[pos])
    code, scale = _eight_bits(q.view(-1, h, group, d))
    both = s.codes[s.pages.long()].transpose(1, 2)[seq].float()  # [tokens, kv heads, width, 2, dim]
    by = s.scales[s.pages.long()].transpose(1, 2)[seq][:, :, None]  # [tokens, kv heads, 1, width, 2]
    mid = torch.matmul(code, both[..., 0, :].transpose(-1, -2)) * by[..., 0]
    score = ((mid + torch.matmul(code.abs(), both[..., 1, :].transpose(-1, -2)) * by[..., 1]) * scale[..., None]).amax(2)
    # the pages that are taken, ascending
    at = torch.arange(width, device="cuda")
    count = index[:, None, None] + 1
    score = torch.where((at < case["first"]) | (at >= count - case["last"]), math.inf, score)
    score = torch.where(at < count, score, -math.inf)
    taken = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    taken = torch.where(taken < count, taken, width).sort(-1).values
    taken = torch.nn.functional.pad(taken, (0, budget - taken.shape[-1]), value=width)
    # attention over them
    head = torch.arange(h, device="cuda")[:, None]
    held = s.pages.long()[seq[:, None, None], taken.clamp(max=width - 1)]
    key = (taken[..., None] * page + torch.arange(page, device="cuda")).flatten(-2)
    sees = ((key <= pos[:, None, None]) & (taken < width)[..., None].expand(-1, -1, -1, page).flatten(-2))[:, :, None]
    score = torch.matmul(q.view(-1, h, group, d), _values(kc[held, head], kp[held, head]).flatten(2, 3).transpose(-1, -2)) * d ** -0.5
    out = _softmax_of(score, sees, _values(vc[held, head], vp[held, head]).flatten(2, 3))
    return {"codes": s.codes, "scales": s.scales, "pages": torch.where(taken < width, taken, -1).to(torch.int32),
            "out": out.flatten(1, 2).to(s.q.dtype)}


# ---- the framework's calls -----------------------------------------------------------------

_gpu_kept = None


def _gpu():
    """The process's one context, on torch's stream."""
    global _gpu_kept
    if _gpu_kept is None:
        import karume_b200 as kb
        _gpu_kept = kb.acquire_gpu(0)
    return _gpu_kept


def _hold(s):
    """What a program makes once for its tensors: no data passes."""
    import karume_b200 as kb
    case = s.case
    if case["kind"] in ("fork", "compact"):
        s.held = kb.CachePages(s.table, s.lengths, s.refs, case["page"], report=s.report)
        s.layers = [pool for pool in s.pools]
        return
    s.rope = kb.Rope(s.angles) if s.angles is not None else None
    s.batch = kb.CacheBatch(s.pages, s.lengths, s.starts, tokens=s.tokens, most=s.most)
    s.held = _gpu().kv_cache(len(s.pool), case["page"], case["kv_heads"], case["dim"], pool=s.pool)
    if case["kind"] == "shared":
        s.prefixes = kb.SharedPrefixes(s.first, s.shared)
    else:
        s.summaries = kb.CacheSummaries(s.codes, s.scales)


def run(s):
    case = s.case
    if own and s.held is None:
        _hold(s)
    if case["kind"] == "fork":
        if own:
            g = _gpu()
            pairs = g.pages_fork(s.held, s.parents, s.keep)
            g.pages_copy(s.held, pairs, s.layers)
            g.pages_grow(s.held, s.news)
        else:
            pairs = _plain_fork(s)
            _plain_copy(s.pools, pairs)
            _plain_grow(s)
        return {"table": s.table, "lengths": s.lengths, "refs": s.refs, "pairs": pairs, "report": s.report, "pools": s.pools}
    if case["kind"] == "compact":
        s.table.copy_(s.before[0])  # the pages where they were, so that every pass moves the same ones
        s.refs.copy_(s.before[1])
        if own:
            g = _gpu()
            pairs = g.pages_compact(s.held)
            g.pages_copy(s.held, pairs, s.layers)
        else:
            pairs = _plain_compact(s)
            _plain_copy(s.pools, pairs)
        return {"table": s.table, "refs": s.refs, "pairs": pairs, "report": s.report, "pools": s.pools}
    if case["kind"] == "shared":
        if own:
            return _gpu().cache_attention(s.held, s.q, s.batch, window=case["window"], rope=s.rope, shared=s.prefixes)
        return _plain_shared(s)
    if own:
        g = _gpu()
        g.cache_summarize(s.held, s.summaries, s.batch)
        taken = g.cache_select(s.held, s.summaries, s.q, s.batch, case["budget"], first=case["first"], last=case["last"], rope=s.rope)
        return {"codes": s.codes, "scales": s.scales, "pages": taken, "out": g.cache_attention(s.held, s.q, s.batch, rope=s.rope, selected=taken)}
    return _plain_select(s)


# ---- what a call cannot do without -----------------------------------------------------------


def work(case):
    page = case["page"]
    if case["kind"] == "fork":  # the pages' names of the sequences that change, in and out; the pages that are copied, in and out
        lengths, keep, news = _fork_lengths(case)
        per = case["children"] + 1
        names = copied = 0
        for b, (n, k, m) in enumerate(zip(lengths, keep, news)):
            if case["children"] == 0:
                names += 2 * (_pages_of(n, page) - k // page)
            elif b % per:
                names += 2 * _pages_of(k + m, page)
                copied += 1 if k % page else 0
        return {"bytes": 4 * names + 2 * copied * case["layers"] * _page_bytes(case), "flops": 0}
    if case["kind"] == "compact":  # the counts, the names; the pages that move (those in use beyond as many as are in use), in and out
        all_pages = sum(_pages_of(max(1, round(s * case["longest"])), page) for s in _share(case["sequences"]))
        used = sum(_pages_of(n, page) for n in _compact_lengths(case))
        moved = used * (all_pages - used) // all_pages  # numbers are spread at random
        return {"bytes": 8 * (all_pages + used) + 2 * moved * case["layers"] * _page_bytes(case), "flops": 0}
    each, d, h = BYTES[case["x"]], case["dim"], case["kv_heads"]
    if case["kind"] == "shared":
        prefix, news, lengths = _shared_lengths(case)
        w = case["window"] or 1 << 31
        keys = pairs = 0
        for b, (n, length) in enumerate(zip(news, lengths)):
            before = prefix[b // case["members"]]
            seen = [(max(0, p - w + 1), p) for p in range(length - n, length)]
            pairs += sum(p - f + 1 for f, p in seen)
            keys += length - max(before, seen[0][0])
        for g, n in enumerate(prefix):  # once, from the first key that one of its members sees
            least = min(max(0, lengths[b] - news[b] - w + 1) for b in range(g * case["members"], (g + 1) * case["members"]))
            keys += max(0, n - least)
        tokens = sum(news)
        return {"bytes": keys * h * (d + 8) + tokens * (2 * each * case["heads"] * d + 4 * case["rotary"]), "flops": 4 * pairs * case["heads"] * d}
    news, lengths = _select_lengths(case)
    scored = keys = written = 0
    for n, length in zip(news, lengths):
        written += _pages_of(length, page) - (length - n) // page
        scored += _pages_of(length, page)  # once for a sequence's new tokens
        keys += min(length, case["budget"] * page)  # likewise: what one of them takes
    tokens, pairs = sum(news), sum(n * min(length, case["budget"] * page) for n, length in zip(news, lengths))
    held = 2 * d + 8
    return {"bytes": h * (written * (page * (d // 2 + 4) + held) + scored * held + keys * (d + 8)) + tokens * (2 * each * case["heads"] * d + 4 * case["rotary"] + 4 * h * case["budget"]),
            "flops": 4 * pairs * case["heads"] * d + 4 * case["heads"] * d * sum(n * _pages_of(length, page) for n, length in zip(news, lengths))}


# ---- the definition in 64 bits -----------------------------------------------------------------


def _held_in_64_bits(raw, par, count, d):
    """`count` rows of codes with their (scale, offset) bytes."""
    par = par.reshape(-1, 4)[:count].contiguous().view(torch.float16).double()
    raw = raw.reshape(-1, d // 2)[:count]
    x = torch.empty(count, d, device="cuda", dtype=torch.float64)
    x[:, 0::2], x[:, 1::2] = (raw % 16).double(), (raw // 16).double()
    return x * par[:, :1] + par[:, 1:]


def _turned_in_64_bits(x, positions, rotary):
    x = x.double().clone()
    if rotary:
        i = torch.arange(rotary // 2, device="cuda")
        z = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), positions.double()[:, None] * 10000.0 ** (-2.0 * i.double() / rotary))
        w = torch.complex(x[..., :rotary // 2], x[..., rotary // 2:rotary]) * z[:, None]
        x[..., :rotary // 2], x[..., rotary // 2:rotary] = w.real, w.imag
    return x


def exact(case, seed):
    """The attention's outputs; what the others give are whole numbers and codes whose every rounding is part of the definition.  Which pages are
    selected follows from the codes, so those are taken from the plain form."""
    if case["kind"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    h, d, page, group = case["kv_heads"], case["dim"], case["page"], case["heads"] // case["kv_heads"]
    half = page * d // 2
    if case["kind"] == "shared":
        news, lengths = _shared_lengths(case)[1:]
        if work(case)["flops"] > 2e12:
            return None
        out = torch.zeros(s.tokens, case["heads"], d, device="cuda", dtype=torch.float64)
        at = 0
        for b, (n, length) in enumerate(zip(news, lengths)):
            blocks = s.pool[s.pages[b, :_pages_of(length, page)].long()].transpose(0, 1)  # [h, pages, bytes]
            q = _turned_in_64_bits(s.q[at:at + n], torch.arange(length - n, length, device="cuda"), case["rotary"])
            position = torch.arange(length - n, length, device="cuda").repeat_interleave(group)[:, None]
            key = torch.arange(length, device="cuda")[None]
            hidden = (key > position) | ((key <= position - case["window"]) if case["window"] else False)
            for head in range(h):
                k, v = (_held_in_64_bits(blocks[head, :, i * half:(i + 1) * half], blocks[head, :, 2 * half + 4 * page * i:2 * half + 4 * page * (i + 1)], length, d)
                        for i in (0, 1))
                rows = q[:, head * group:(head + 1) * group].reshape(-1, d)
                p = torch.softmax((rows @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out[at:at + n, head * group:(head + 1) * group] = (p @ v).view(n, group, d)
            at += n
        return out
    taken = _plain_select(s)["pages"]
    seq, pos = _new_tokens(s)
    if s.tokens * h > 2048:
        return None
    q = _turned_in_64_bits(s.q, pos, case["rotary"])
    out = torch.zeros(s.tokens, case["heads"], d, device="cuda", dtype=torch.float64)
    order, places, table = taken.tolist(), pos.tolist(), s.pages.long()
    for t, b in enumerate(seq.tolist()):
        for head in range(h):
            mine = [i for i in order[t][head] if i >= 0]
            blocks = s.pool[table[b, mine], head]
            k, v = (_held_in_64_bits(blocks[:, i * half:(i + 1) * half], blocks[:, 2 * half + 4 * page * i:2 * half + 4 * page * (i + 1)], len(mine) * page, d)
                    for i in (0, 1))
            where = (torch.tensor(mine, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
            p = torch.softmax((q[t, head * group:(head + 1) * group] @ k.T / math.sqrt(d)).masked_fill(where > places[t], -math.inf), -1)
            out[t, head * group:(head + 1) * group] = p @ v
    return {"codes": None, "scales": None, "pages": None, "out": out}
