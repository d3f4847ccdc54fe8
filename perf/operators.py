"""The attention half of a decoder layer: rotary positions, appending to a paged cache held in 4 bits, attention over it.

What a program holds: a pool of pages (uint8), the pages of each sequence, the sequences' lengths and the table of rotation
angles.  Sequence b has lengths[b] tokens, of which the last starts[b + 1] - starts[b] are new in this call (one each where
there is no `starts`).

Rotation: pairs (x0, x1) of a head's first `rotary` values, i and i + rotary / 2 (half layout) or 2 i and 2 i + 1
(interleaved), become (x0 c - x1 s, x1 c + x0 s) with (c, s) = table[position, i], in f32.

Cache: a page holds `page` tokens; for each kv head its block is
    [K codes: page x dim / 2 bytes][V codes: likewise][K (scale, offset): page x 2 binary16][V (scale, offset): likewise]
with element 2 i in the low nibble of byte i.  A row x (one token, one head; keys after their rotation) is held as
    offset = f16(min x), scale = f16((max x - offset) / 15), code = clamp(rint((x - offset) / scale), 0, 15)
and stands for code * scale + offset.

Attention: query i of the n new ones of a sequence of length L has position p = L - n + i and sees the keys
max(0, p - window + 1) .. p (all up to p where window is 0); out = softmax(q . k / sqrt(dim)) v, zeros where it sees none.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# (query heads, kv heads, head dim): the 8B-shaped decoder, the 1.5B-class one and the small test decoder of this
# repository, then one key head for all queries, one for each, and wide heads.
HEADS = [(32, 8, 128), (12, 2, 128), (8, 4, 64), (16, 1, 128), (8, 8, 64), (8, 4, 256)]


def listed():
    return [
        # One token's queries, rotated by themselves (a host with its own attention): the smallest call.
        dict(name="rope_token", kind="rope", x="f32", tokens=1, heads=32, dim=128, rotary=128, interleaved=False, positions=8192),
        # The queries of a long prompt in bf16, half of each head rotated, pairs interleaved.
        dict(name="rope_prompt", kind="rope", x="bf16", tokens=8191, heads=32, dim=128, rotary=64, interleaved=True, positions=131072),
        # One token of one conversation: its key and value go into the cache.
        dict(name="append_token", kind="append", x="f32", sequences=1, new=1, longest=4096, heads=32, kv_heads=8, dim=128, page=64,
             rotary=128, interleaved=False),
        # A step of 64 conversations of many lengths; keys and values are columns of the fused projection's output.
        dict(name="append_batch", kind="append", x="f32", sequences=64, new=1, longest=8192, heads=32, kv_heads=8, dim=128, page=64,
             rotary=128, interleaved=False),
        # Five prompts of different lengths at once in bf16, on small pages.
        dict(name="append_prompts", kind="append", x="bf16", sequences=5, new=2047, longest=3001, heads=12, kv_heads=2, dim=128, page=16,
             rotary=128, interleaved=True),
        # One token of one conversation over 4096: what every chat user waits for.
        dict(name="attend_token", kind="attend", x="f32", sequences=1, new=1, longest=4096, heads=32, kv_heads=8, dim=128, page=64,
             window=0, rotary=128),
        # Sixteen conversations of many lengths, one slot idle, f32 as the projections give it.
        dict(name="attend_batch", kind="attend", x="f32", sequences=16, new=1, longest=8190, heads=32, kv_heads=8, dim=128, page=64,
             window=0, rotary=128),
        # One very long document on a small decoder: few rows, a long axis.
        dict(name="attend_long", kind="attend", x="f16", sequences=1, new=1, longest=200003, heads=12, kv_heads=2, dim=128, page=128,
             window=0, rotary=0),
        # A full server: 64 conversations of up to 16384 tokens in bf16, the largest cache a step reads.
        dict(name="attend_server", kind="attend", x="bf16", sequences=64, new=1, longest=16384, heads=32, kv_heads=8, dim=128, page=64,
             window=0, rotary=128),
        # Verifying drafts of five tokens on eight sequences, a window of 1024, small heads and pages.
        dict(name="attend_draft", kind="attend", x="f32", sequences=8, new=5, longest=3001, heads=8, kv_heads=4, dim=64, page=16,
             window=1024, rotary=64),
        # Three prompts, part of them cached before, in f32.
        dict(name="attend_prompts_f32", kind="attend", x="f32", sequences=3, new=777, longest=1501, heads=12, kv_heads=2, dim=128,
             page=32, window=0, rotary=128),
        # A long prompt in bf16: the largest contraction.
        dict(name="attend_prompt_bf16", kind="attend", x="bf16", sequences=1, new=4096, longest=5000, heads=32, kv_heads=8, dim=128,
             page=64, window=0, rotary=128),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["rope", "append", "attend"], [1, 2, 5])[0]
    heads, kv_heads, dim = rng.choice(HEADS[:3] * 2 + HEADS[3:])
    x = rng.choice(["f32", "f32", "f16", "bf16"])
    rotary = rng.choice([dim, dim, dim // 2, dim // 4])
    interleaved = rng.random() < 0.4
    if kind == "rope":
        return dict(kind=kind, x=x, tokens=_spread(rng, 1, 8192), heads=heads, dim=dim, rotary=rotary, interleaved=interleaved,
                    positions=_spread(rng, 8192, 131072))
    page = rng.choice([16, 32, 64, 128])
    while True:
        sequences = _spread(rng, 1, 64)
        new = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 4096)])
        longest = new - 1 + _spread(rng, 1, 200000 if new == 1 else 8192)
        case = dict(kind=kind, x=x, sequences=sequences, new=new, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    rotary=rotary)
        case.update(dict(interleaved=interleaved) if kind == "append" else dict(window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)])))
        news, lengths = _lengths(case)
        # at most the largest listed case: its cached values, its scores
        if sum(lengths) * kv_heads * dim <= 64 * 10300 * 1024 and sequences * new * longest * heads <= 4096 * 5000 * 32 and \
                sum(news) * heads * dim <= 8192 * 32 * 128:
            return case


def _lengths(case):
    """(new, lengths) of each sequence: 1 / 4 to all of the longest, spread evenly; every sixteenth slot of a batch is idle."""
    share = [1.0 if b == 0 else 0.25 + 0.75 * math.modf(b * 0.6180339887498949)[0] for b in range(case["sequences"])]
    if case["new"] == 1:
        return [1] * len(share), [0 if b % 16 == 9 and case["kind"] == "attend" else max(1, round(s * case["longest"])) for b, s in enumerate(share)]
    news = [max(1, round(s * case["new"])) for s in share]
    return news, [max(n, round(s * case["longest"])) for n, s in zip(news, share)]


# ---- what a user's program holds -----------------------------------------------------------


class _State:
    cache = None  # the framework's view of the pool, made at the first call


def _table(positions, rotary):
    """(cos, sin) of position * 10000^(-2 i / rotary), f32."""
    f = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _pool(case, pages, gen):
    """A pool in which every page has been used: keys with channels of different spread and mean, values around zero."""
    h, d, p = case["kv_heads"], case["dim"], case["page"]
    pool = torch.empty(pages, h, p * (d + 8), device="cuda", dtype=torch.uint8)
    gain = torch.exp(0.3 * torch.randn(h, 1, d, generator=gen, device="cuda"))
    mean = 0.5 * torch.randn(h, 1, d, generator=gen, device="cuda")
    step = max(1, (1 << 26) // (h * d * p))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        for which in (0, 1):
            x = torch.randn(n, h, p, d, generator=gen, device="cuda")
            codes, params = _quantise(torch.addcmul(mean, x, gain) if which == 0 else x)
            pool[at:at + n, :, which * p * d // 2:(which + 1) * p * d // 2] = codes.flatten(-2)
            pool[at:at + n, :, p * d + 4 * which * p:p * d + 4 * (which + 1) * p] = params.flatten(-2)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.case, dtype = case, TORCH_DTYPE[case["x"]]
    if case["kind"] == "rope":
        s.x = torch.randn(case["tokens"], case["heads"], case["dim"], generator=gen, device="cuda").to(dtype)
        s.positions = torch.randint(case["positions"], (case["tokens"],), generator=gen, device="cuda", dtype=torch.int32)
        s.table = _table(case["positions"], case["rotary"])
        return s
    news, lengths = _lengths(case)
    h, d, p = case["kv_heads"], case["dim"], case["page"]
    width = (case["longest"] + p - 1) // p
    counts = [(n + p - 1) // p for n in lengths]
    total = sum(counts) + 1  # page 0 is nobody's
    order = (1 + torch.randperm(total - 1, generator=gen, device="cuda")).to(torch.int32)
    table = torch.zeros(case["sequences"], width, device="cuda", dtype=torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table[used] = order
    s.pages, s.lengths = table, torch.tensor(lengths, device="cuda", dtype=torch.int32)
    s.starts = None
    if case["new"] > 1:
        s.starts = torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32)
    s.tokens, s.most = sum(news), max(news)
    s.table = _table(case["longest"], case["rotary"]) if case["rotary"] else None
    if case["kind"] == "append":
        s.pool = torch.zeros(total, h, p * (d + 8), device="cuda", dtype=torch.uint8)
        qkv = torch.randn(s.tokens, case["heads"] + 2 * h, d, generator=gen, device="cuda").to(dtype)
        s.k, s.v = qkv[:, -2 * h:-h], qkv[:, -h:]
    else:
        s.pool = _pool(case, total, gen)
        s.q = torch.randn(s.tokens, case["heads"], d, generator=gen, device="cuda").to(dtype)
    return s


# ---- the plain form ------------------------------------------------------------------------


def _rotate(x, rows, interleaved):
    """x [tokens, heads, dim] in f32; rows [tokens, rotary / 2, 2]."""
    c, s = rows[:, None, :, 0], rows[:, None, :, 1]
    r = 2 * c.shape[-1]
    x0, x1 = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y0, y1 = x0 * c - x1 * s, x1 * c + x0 * s
    y = torch.stack([y0, y1], -1).flatten(-2) if interleaved else torch.cat([y0, y1], -1)
    return torch.cat([y, x[..., r:]], -1)


def _quantise(x):
    """f32 rows [..., dim] -> codes [..., dim / 2] and (scale, offset) as bytes [..., 4]."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    offset = low.half()
    scale = ((high - offset.float()) * torch.tensor(1 / 15, device=x.device)).half().clamp(min=0)
    lost = ~(torch.isfinite(offset) & torch.isfinite(scale))
    code = torch.round((x - offset.float()) * (1 / scale.float())).clamp(0, 15)
    code = torch.where((scale > 0) & ~lost, code, 0).to(torch.uint8)
    params = torch.where(lost, math.nan, torch.cat([scale, offset], -1)).half()
    return code[..., 0::2] | (code[..., 1::2] << 4), params.view(torch.uint8)


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


def _new_tokens(s):
    """(sequence, position) of each new token."""
    if s.starts is None:
        return torch.arange(len(s.lengths), device="cuda"), s.lengths.long() - 1
    at = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(s.starts.long(), at, right=True) - 1
    return seq, s.lengths.long()[seq] - s.starts.long()[seq + 1] + at


def _plain_append(s):
    case = s.case
    seq, pos = _new_tokens(s)
    page, slot = s.pages.long()[seq, pos // case["page"]], pos % case["page"]
    kc, vc, kp, vp = _views(s.pool, case["page"], case["dim"])
    k = _rotate(s.k.float(), s.table[pos], case["interleaved"])
    kc[page, :, slot], kp[page, :, slot] = _quantise(k)
    vc[page, :, slot], vp[page, :, slot] = _quantise(s.v.float())
    return {"k": _values(kc[page, :, slot], kp[page, :, slot]), "v": _values(vc[page, :, slot], vp[page, :, slot])}


def _plain_attend(s):
    case = s.case
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    group, n, width = case["heads"] // h, s.most, s.pages.shape[1]
    seq, pos = _new_tokens(s)
    q = s.q.float()
    if s.table is not None:
        q = _rotate(q, s.table[pos.clamp(min=0)], False)
    first = s.starts.long()[:-1] if s.starts is not None else torch.arange(len(s.lengths), device="cuda")
    row = torch.arange(s.tokens, device="cuda") - first[seq]
    padded = torch.zeros(len(s.lengths), n, case["heads"], d, device="cuda")
    padded[seq, row] = q
    at = torch.full((len(s.lengths), n), -1, device="cuda")
    at[seq, row] = pos
    kc, vc, kp, vp = (t[s.pages.long()].transpose(1, 2).flatten(2, 3) for t in _views(s.pool, page, d))  # [sequences, heads, width * page, ..]
    score = torch.matmul(padded.view(-1, n, h, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3), _values(kc, kp).transpose(-1, -2))
    score = score.view(-1, h, group, n, width * page) * d ** -0.5
    key = torch.arange(width * page, device="cuda")
    sees = key <= at[..., None]
    if case["window"]:
        sees &= key > at[..., None] - case["window"]
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    value = torch.where(sees.any(1)[:, None, :, None], _values(vc, vp), 0)
    out = torch.matmul(weight.flatten(2, 3), value).view(-1, h, group, n, d) / torch.where(total > 0, total, 1)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, row].to(s.q.dtype)


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
    """What a program makes once for a pool and a batch of sequences: no data passes."""
    import karume_b200 as kb
    case = s.case
    s.rope = kb.Rope(s.table, case.get("interleaved", False)) if s.table is not None else None
    if case["kind"] != "rope":
        s.batch = kb.CacheBatch(s.pages, s.lengths, s.starts, tokens=s.tokens, most=s.most)
        s.cache = _gpu().kv_cache(len(s.pool), case["page"], case["kv_heads"], case["dim"], pool=s.pool)
    else:
        s.cache = True


def run(s):
    kind = s.case["kind"]
    if own:
        g = _gpu()
        if s.cache is None:
            _hold(s)
        if kind == "rope":
            return g.rope(s.x, s.positions, s.rope)
        if kind == "append":
            g.cache_append(s.cache, s.k, s.v, s.batch, rope=s.rope)
            k, v = g.cache_read(s.cache, s.batch)
            return {"k": k, "v": v}
        return g.cache_attention(s.cache, s.q, s.batch, window=s.case["window"], rope=s.rope)
    if kind == "rope":
        return _rotate(s.x.float(), s.table[s.positions.long()], s.case["interleaved"]).to(s.x.dtype)
    return _plain_append(s) if kind == "append" else _plain_attend(s)


# ---- what a call cannot do without -----------------------------------------------------------


def _seen(case):
    """(keys that some query sees, pairs of a query and a key it sees) over all sequences."""
    keys = pairs = 0
    w = case["window"]
    for n, length in zip(*_lengths(case)):
        n = min(n, length)
        if n:
            first = length - n  # position of the first query
            keys += length - max(0, first - w + 1) if w else length
            full = n * length - n * (n - 1) // 2
            pairs += full if not w else sum(min(w, p + 1) for p in range(first, length))
    return keys, pairs


def work(case):
    each = BYTES[case["x"]]
    if case["kind"] == "rope":
        n = case["tokens"]
        return {"bytes": 2 * each * n * case["heads"] * case["dim"] + 4 * n * (case["rotary"] + 1), "flops": 3 * n * case["heads"] * case["rotary"]}
    news, lengths = _lengths(case)
    h, d, tokens = case["kv_heads"], case["dim"], sum(news)
    if case["kind"] == "append":  # rows in, the packed rows out, and the values they stand for
        row = 2 * h * (each * d + d // 2 + 4 + 4 * d) + 4 * case["rotary"]
        return {"bytes": tokens * row, "flops": tokens * h * (3 * case["rotary"] + 2 * 6 * d)}
    keys, pairs = _seen(case)
    return {"bytes": keys * h * (d + 8) + tokens * (2 * each * case["heads"] * d + 4 * case["rotary"]), "flops": 4 * pairs * case["heads"] * d}


# ---- the definition in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64

    def turn(x, positions, interleaved):
        r = case["rotary"]
        if not r:
            return x.to(f64)
        i = torch.arange(r // 2, device="cuda")
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        z = torch.polar(torch.ones((), device="cuda", dtype=f64), positions.to(f64)[:, None] * 10000.0 ** (-2.0 * i.to(f64) / r))
        x = x.to(f64).clone()
        w = torch.complex(x[..., first], x[..., second]) * z[:, None]
        x[..., first], x[..., second] = w.real, w.imag
        return x

    if case["kind"] == "rope":
        return turn(s.x, s.positions, case["interleaved"])
    news, lengths = _lengths(case)
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    half = page * d // 2
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(length - n, length, device="cuda") for n, length in zip(news, lengths)])

        def held(x):
            low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            low = low.to(torch.float16).to(f64)
            step = ((high - low) / 15).to(torch.float16).to(f64)
            return torch.clamp(torch.round((x - low) / step), 0, 15) * step + low

        return {"k": held(turn(s.k, positions, case["interleaved"])), "v": held(s.v.to(f64))}
    if _seen(case)[1] * case["heads"] * d > 2e12:
        return None
    out = torch.zeros(s.tokens, case["heads"], d, device="cuda", dtype=f64)
    at = 0
    for b, (n, length) in enumerate(zip(news, lengths)):
        if length == 0:
            at += n
            continue
        blocks = s.pool[s.pages[b, :(length + page - 1) // page].long()].transpose(0, 1)  # [h, pages, bytes]
        q = turn(s.q[at:at + n], torch.arange(length - n, length, device="cuda"), False)
        for head in range(h):
            held = []
            for which in (0, 1):
                raw = blocks[head, :, which * half:(which + 1) * half].reshape(-1, d // 2)[:length]
                par = blocks[head, :, 2 * half + 4 * page * which:2 * half + 4 * page * (which + 1)].reshape(-1, 4)[:length]
                par = par.contiguous().view(torch.float16).to(f64)
                x = torch.empty(length, d, device="cuda", dtype=f64)
                x[:, 0::2], x[:, 1::2] = (raw % 16).to(f64), (raw // 16).to(f64)
                held.append(x * par[:, :1] + par[:, 1:])
            group = case["heads"] // h
            rows = q[:, head * group:(head + 1) * group].reshape(-1, d)
            position = torch.arange(length - n, length, device="cuda").repeat_interleave(group)[:, None]
            key = torch.arange(length, device="cuda")[None]
            hidden = key > position
            if case["window"]:
                hidden |= key <= position - case["window"]
            p = torch.softmax((rows @ held[0].T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            out[at:at + n, head * group:(head + 1) * group] = (p @ held[1]).view(n, group, d)
        at += n
    return out
