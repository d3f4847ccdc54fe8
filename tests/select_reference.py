"""Plain statements of page summaries, scores and selections, every operation rounded to f32 as the definition has it."""
import numpy as np

F = np.float32
TINY = F(1.17549435e-38)


def eight_bits(x):
    """f32 rows [..., dim] -> 8-bit codes (whole numbers) and scales [...]; NaN scales and codes 0 for rows that are not finite."""
    with np.errstate(all="ignore"):
        scale = np.maximum(np.abs(x).max(-1) * F(1 / 127), TINY).astype(F)
        codes = np.clip(np.rint(x / scale[..., None]), -127, 127)
    lost = ~np.isfinite(x).all(-1)
    return np.where(lost[..., None], 0, codes).astype(np.int64), np.where(lost, F(np.nan), scale).astype(F)


def summary(keys):
    """Keys f32 [tokens, dim] of a page and head -> codes [2, dim], scales [2]."""
    if not np.isfinite(keys).all():
        return np.zeros((2, keys.shape[1]), np.int64), np.full(2, np.nan, F)
    low, high = keys.min(0), keys.max(0)
    codes, scales = zip(*(eight_bits(x) for x in (((high + low) * F(0.5)).astype(F), ((high - low) * F(0.5)).astype(F))))
    return np.stack(codes), np.array(scales, F)


def scores(q, codes, scales):
    """q f32 [heads of a kv head, dim] (rotated); codes [pages, 2, dim], scales [pages, 2]: f32 [pages]."""
    a, s = eight_bits(q)
    with np.errstate(all="ignore"):
        c = (codes[:, 0].astype(np.int64) @ a.T).astype(F) * scales[:, :1]
        r = (codes[:, 1].astype(np.int64) @ np.abs(a).T).astype(F) * scales[:, 1:]
        each = ((c + r).astype(F) * s).astype(F)
    best = each.max(1)
    return np.where(np.isnan(each).any(1), F(np.nan), best)


def select(score, budget, first, last):
    """Indices of the pages of `score`, ascending, -1 behind them."""
    n = len(score)
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    value = np.where(np.isnan(score), np.inf, score).astype(np.float64)
    kind = np.isnan(score).astype(int)  # what is not a number above infinities
    at = np.arange(n)
    kind[(at < first) | (at >= n - last)] = 2
    value[kind == 2] = 0
    order = np.lexsort((at, -value, -kind))
    return sorted(order[:budget].tolist())
