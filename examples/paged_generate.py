"""Serves a few requests together over a paged KV cache: paged append with the
rotation, attention of chunks and single tokens, and sampling from given
uniforms, on one GPU.

    python examples/paged_generate.py [model.hypno]

Without a file it makes a small synthetic model.
"""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402

from hypno_b200 import synth  # noqa: E402
from hypno_b200.paged_model import PagedGenerator, PagedModel  # noqa: E402

SMALL = dict(hidden=512, layers=4, heads=8, kv_heads=2, inter=1408, vocab=8000, theta=10000.0, max_pos=1024)


def main(argv):
    if len(argv) > 1:
        image = np.memmap(argv[1], dtype=np.uint8, mode="r")
    else:
        image = synth.build_image(SMALL, seed=1)
    model = PagedModel(image, n_pages=256, page_size=16)
    gen = PagedGenerator(model, max_seqs=8, budget=128)
    g = np.random.default_rng(0)
    for i in range(12):  # prompts of different lengths, greedy and sampled
        prompt = g.integers(0, model.vocab, size=int(g.integers(1, 300)))
        gen.submit(prompt, max_tokens=24, temperature=0.0 if i % 3 == 0 else 0.8, top_k=50, top_p=0.95, min_p=0.02, seed=i)
    steps, began = 0, time.perf_counter()
    while not gen.idle:
        gen.step()
        steps += 1
    took = time.perf_counter() - began
    for i, tokens in sorted(gen.finished.items()):
        print(f"request {i}: {tokens[:8]} ... ({len(tokens)} tokens)")
    print(f"{sum(map(len, gen.finished.values()))} tokens in {steps} steps, {took:.2f} s; {len(gen.pages.free)} of {model.n_pages} pages free")
    model.close()
    return gen.finished


if __name__ == "__main__":
    main(sys.argv)
