"""Plain statements of rotary positions, the 4-bit cache rows and attention, for the tests of those kernels."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rotate(x, table, positions, interleaved):
    """f32 [tokens, heads, dim] on the CPU, the products and sums rounded one by one; table f32 [positions, rotary / 2, 2]."""
    rows = table[positions]
    c, s = rows[:, None, :, 0], rows[:, None, :, 1]
    r = 2 * c.shape[-1]
    y = x.copy()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x0, x1 = x[..., first], x[..., second]
    y[..., first] = x0 * c - x1 * s
    y[..., second] = x1 * c + x0 * s
    return y


def quantise(x):
    """f32 rows [..., dim] -> codes uint8 [..., dim], scale and offset binary16 [...]; NaN pairs for rows it cannot hold."""
    with np.errstate(all="ignore"):
        low, high = x.min(-1), x.max(-1)
        offset = low.astype(np.float16)
        scale = np.maximum(((high - offset.astype(np.float32)) * np.float32(1 / 15)).astype(np.float16), np.float16(0))
        lost = ~np.isfinite(offset) | ~np.isfinite(scale) | np.isnan(x).any(-1)
        inv = np.float32(1) / scale.astype(np.float32)
        codes = np.clip(np.rint((x - offset.astype(np.float32)[..., None]) * inv[..., None]), 0, 15)
        codes = np.where(((scale > 0) & ~lost)[..., None], codes, 0).astype(np.uint8)
        scale, offset = (np.where(lost, np.float16(np.nan), t) for t in (scale, offset))
    return codes, scale, offset


def stands_for(codes, scale, offset):
    return (codes.astype(np.float32) * scale.astype(np.float32)[..., None] + offset.astype(np.float32)[..., None]).astype(np.float32)


def attend(q, k, v, scale, window):
    """One sequence in 64 bits: q f64 [new, heads, dim] (rotated), k and v f64 [length, kv_heads, dim].  Returns the output and,
    per output row, the largest sum_d |q_d k_jd| * scale and the largest |v_j| a query sees (zero where it sees none)."""
    new, heads, dim = q.shape
    length, kv_heads, _ = k.shape
    out = torch.zeros_like(q)
    reach = torch.zeros(new, heads, dtype=torch.float64, device=q.device)
    largest = torch.zeros_like(reach)
    position = torch.arange(length - new, length, device=q.device)[:, None]
    key = torch.arange(length, device=q.device)[None]
    sees = key <= position
    if window:
        sees &= key > position - window
    some = sees.any(1)
    for h in range(heads):
        g = h // (heads // kv_heads)
        if length == 0 or not bool(some.any()):
            continue
        score = (q[:, h] @ k[:, g].T * scale).masked_fill(~sees, -torch.inf)
        weight = torch.softmax(score[some], -1)
        # a value that is not seen does not count, whatever it is
        value = torch.where(sees.any(0)[:, None], v[:, g], 0)
        if bool(torch.isnan(value).any()) or bool(torch.isnan(score).any()):
            for i in torch.nonzero(some).flatten().tolist():
                w = torch.softmax(score[i, sees[i]], -1)
                out[i, h] = w @ v[sees[i], g]
        else:
            out[some, h] = weight @ value
        reach[:, h] = (q[:, h].abs() @ k[:, g].abs().T * scale).masked_fill(~sees, 0).amax(-1)
        largest[:, h] = torch.where(sees, v[:, g].abs().amax(-1)[None], 0).amax(-1)
    return out, reach, largest


def allowed(kind, out, reach, largest):
    """What the kernels may be off by, per output value.

    A score s = scale q.k off by d changes the output by at most 2 d max|v|; weights off by a relative e, by 2 e max|v|.
    f32 queries: the operands keep 21 bits at least (two binary16 parts), sums are f32: d = 2^-20 reach, e = 2^-20.
    16-bit queries: keys, weights and values are rounded to binary16, 2^-11 each: d = 2^-11 reach, e = 2^-10; one rounding
    of the output to its type on top."""
    bits, type_bits = {"f32": (-20, -23), "f16": (-11, -11), "bf16": (-11, -8)}[kind]
    e = 2.0 ** bits
    return (2 * e * reach * largest + 6 * e * largest)[..., None] + out.abs() * 2.0 ** type_bits + 1e-30
