"""Generates tokens with a small random decoder: prompts of different lengths at once, then recorded single-token steps.

    python examples/generate.py [--layers 4] [--tokens 32]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import karume_b200 as kb  # noqa: E402
from bench_workload import synth_weight  # noqa: E402
from karume_b200.decoder import Decoder, DecoderShape  # noqa: E402


def around_zero(payload, scale):
    """The codes 0 (-8) become 8 (0): otherwise every output shares a direction, and one token wins whatever the prompt."""
    codes = np.frombuffer(payload, np.uint8)
    low, high = codes & 15, codes >> 4
    return (np.where(low == 0, 8, low) | np.where(high == 0, 8, high) << 4).astype(np.uint8), scale


def small_decoder(gpu, layers=4, sequences=3, longest=512, seed=0, heads=8, kv_heads=2, head_dim=64, window=0, make=synth_weight):
    shape = DecoderShape(layers=layers, hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim, ffn=2 * heads * head_dim, vocab=1024)
    q, kv = shape.heads * shape.head_dim, shape.kv_heads * shape.head_dim
    sizes = {"embedding": (shape.vocab, shape.hidden), "head": (shape.vocab, shape.hidden)}
    for i in range(layers):
        sizes.update({f"{i}.q": (q, shape.hidden), f"{i}.k": (kv, shape.hidden), f"{i}.v": (kv, shape.hidden), f"{i}.o": (shape.hidden, q),
                      f"{i}.gate": (shape.ffn, shape.hidden), f"{i}.up": (shape.ffn, shape.hidden), f"{i}.down": (shape.hidden, shape.ffn)})
    weights = {name: gpu.upload_weight("i4", *make(seed, name, n, k), (n, k), 32) for name, (n, k) in sizes.items()}
    norms = {name: torch.ones(shape.hidden, device=gpu.device) for name in [f"{i}.{j}" for i in range(layers) for j in (1, 2)] + ["final"]}
    rope = kb.Rope(torch.from_numpy(kb.rope_table(longest, head_dim)).to(gpu.device))
    return Decoder(gpu, shape, weights, norms, rope, sequences, longest, window=window)


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    args = ap.parse_args()
    torch.cuda.set_stream(torch.cuda.Stream())  # the library and torch on one stream, which can be recorded
    gpu = kb.acquire_gpu(0)
    decoder = small_decoder(gpu, layers=args.layers, make=lambda *of: around_zero(*synth_weight(*of)))
    news = [5, 70, 200]
    prompts = torch.from_numpy(np.random.default_rng(1).integers(0, 1024, sum(news)).astype(np.int32)).cuda()
    logits = decoder.prompt(prompts, news)
    made = []
    for _ in range(args.tokens):
        decoder.ids.copy_(logits.argmax(-1))
        made.append(decoder.ids.clone())
        logits = decoder.step()
    gpu.sync()
    for b, row in enumerate(torch.stack(made, 1).tolist()):
        print(f"sequence {b} ({news[b]} tokens of prompt):", " ".join(map(str, row)))
    decoder.close()
    gpu.destroy()


if __name__ == "__main__":
    main()
