"""How far a key's product with a query may be above its page's score: the summaries' codes are rounded to the nearest."""
import numpy as np

from tests.select_reference import eight_bits, scores, summary


def test_keys_are_above_their_pages_score_by_the_codes_rounding_at_most():
    rng = np.random.default_rng(5)
    above = 0
    for _ in range(300):
        dim, tokens = int(rng.choice([64, 128, 256])), int(rng.integers(1, 40))
        gain, mean = np.exp(rng.normal(size=dim) * rng.choice([0, 0.5, 2])), rng.normal(size=dim) * rng.choice([0, 1, 5])
        keys = (rng.normal(size=(tokens, dim)) * gain + mean).astype(np.float32)
        q = rng.normal(size=(1, dim)).astype(np.float32)
        codes, scales = summary(keys)
        a, s = (v[0].astype(np.float64) for v in eight_bits(q))
        score = float(scores(q, codes[None], scales[None])[0])
        products = s * (keys.astype(np.float64) @ a)
        # half a step of each code; middles and spreads are f32 (two roundings of 2^-24 of up to twice the largest key), three more of the score
        rounding = s * np.abs(a).sum() * (float(scales.sum()) / 2 + 4 * 2.0**-24 * float(np.abs(keys).max())) + 3 * 2.0**-24 * s * np.abs(a).sum() * 127 * float(scales.sum())
        assert products.max() <= score + rounding
        above += products.max() > score
    assert above > 0  # so the score is no bound
