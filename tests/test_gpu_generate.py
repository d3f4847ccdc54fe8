"""A whole decoder (karume_b200/decoder.py) against the same layers in 64 bits, with keys and values as the 4-bit cache holds
them: prompts of several lengths at once, further tokens of some, single-token steps replayed from a recorded graph."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import cache_reference as ref

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def gpu():
    import karume_b200 as kb
    before = torch.cuda.current_stream()
    torch.cuda.set_stream(torch.cuda.Stream())
    g = kb.acquire_gpu(0)
    yield g
    g.destroy()
    torch.cuda.set_stream(before)


class Plain:
    """One sequence of the decoder, f64 throughout; rotation, quantisation and the cached values as the cache defines them
    (f32 steps on the f64 projections rounded to f32)."""

    def __init__(self, d):
        self.d, self.w = d, {n: w.dequant().double() for n, w in d.weights.items()}
        self.k, self.v = [[] for _ in range(d.shape.layers)], [[] for _ in range(d.shape.layers)]
        self.table, self.near = d.rope.table.cpu().numpy(), 0.0

    def norm(self, x):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.d.shape.eps)

    def held(self, rows):
        rows = rows.float().cpu().numpy()
        codes, scale, offset = ref.quantise(rows)
        return torch.from_numpy(ref.stands_for(codes, scale, offset)).cuda().double()

    def take(self, ids):
        s = self.d.shape
        h = self.w["embedding"][ids.long()]
        at = len(self.k[0])
        positions = np.arange(at, at + len(ids))
        for i in range(s.layers):
            x = self.norm(h)
            q, k, v = ((x @ self.w[f"{i}.{n}"].T).view(len(ids), -1, s.head_dim) for n in "qkv")
            turn = lambda t: torch.from_numpy(ref.rotate(t.float().cpu().numpy(), self.table, positions, False)).cuda().double()  # noqa: E731
            self.k[i] += list(self.held(turn(k)))
            self.v[i] += list(self.held(v))
            out, _, _ = ref.attend(turn(q), torch.stack(self.k[i]), torch.stack(self.v[i]), s.head_dim ** -0.5, self.d.window)
            h = h + out.reshape(len(ids), -1) @ self.w[f"{i}.o"].T
            x = self.norm(h)
            gate, up = x @ self.w[f"{i}.gate"].T, x @ self.w[f"{i}.up"].T
            h = h + (gate * torch.sigmoid(gate) * up) @ self.w[f"{i}.down"].T
        return self.norm(h[-1]) @ self.w["head"].T


@pytest.mark.parametrize("heads,kv_heads,head_dim,window", [(8, 2, 64, 0), (4, 1, 128, 0), (6, 3, 64, 50)])
def test_prompts_and_recorded_steps(gpu, heads, kv_heads, head_dim, window):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    from generate import small_decoder
    d = small_decoder(gpu, layers=2, sequences=3, longest=400, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window)
    rng = np.random.default_rng(heads)
    plain = [Plain(d) for _ in range(3)]

    def close(got, want, what):
        # a projection off by f32 rounding may move a key or value across a rounding of its code, one step of about a fifteenth
        # of the row's range in one of a head's dims: a part in a hundred of what attention adds there, less behind the layers
        off = float((got.double() - want).norm() / want.norm())
        assert off < 1e-2, (what, off)
        return off

    offs = []
    for news in ([3, 150, 70], [0, 40, 1]):
        ids = [torch.from_numpy(rng.integers(0, 1024, n).astype(np.int32)).cuda() for n in news]
        logits = d.prompt(torch.cat(ids), news)
        gpu.sync()
        for b, n in enumerate(news):
            if n:
                offs.append(close(logits[b], plain[b].take(ids[b]), ("prompt", news, b)))
    for i in range(6):
        ids = torch.from_numpy(rng.integers(0, 1024, 3).astype(np.int32)).cuda()
        d.ids.copy_(ids)
        logits = d.step().clone()
        gpu.sync()
        for b in range(3):
            offs.append(close(logits[b], plain[b].take(ids[b:b + 1]), ("step", i, b)))
    assert float(np.median(offs)) < 1e-3, sorted(offs)
    assert d.lengths.tolist() == d.held == [9, 196, 77]
    import karume_b200 as kb
    with pytest.raises(kb.KqError):
        d.prompt(ids, [400, 0, 0])
    d.close()


def test_the_example_runs(gpu):
    done = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "generate.py"), "--layers", "2", "--tokens", "5"], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert len(done.stdout.splitlines()) == 3
