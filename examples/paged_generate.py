"""Serves a few requests together over a paged KV cache: paged append with the
rotation, attention of chunks and single tokens, and sampling from given
uniforms, on one GPU.

    python examples/paged_generate.py [model.hypno] [--cache f16|f32|q4] [--keep-pages N]

Without a file it makes a small synthetic model.  --cache q4 holds keys and values
in 4 bits; --keep-pages lets a generated token read N pages of its sequence alone,
those that score highest for it.
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from hypno_b200 import synth  # noqa: E402
from hypno_b200.paged_model import PagedGenerator, PagedModel  # noqa: E402

SMALL = dict(hidden=512, layers=4, heads=8, kv_heads=2, inter=1408, vocab=8000, theta=10000.0, max_pos=1024)


def main(argv):
    ap = argparse.ArgumentParser()
    ap.add_argument("model", nargs="?")
    ap.add_argument("--cache", choices=("f16", "f32", "q4"), default="f16")
    ap.add_argument("--keep-pages", type=int)
    args = ap.parse_args(argv[1:])
    if args.model:
        image = np.memmap(args.model, dtype=np.uint8, mode="r")
    else:
        image = synth.build_image(SMALL, seed=1)
    cache = {"f16": torch.float16, "f32": torch.float32, "q4": "q4"}[args.cache]
    model = PagedModel(image, n_pages=256, page_size=16, cache_dtype=cache, keep_pages=args.keep_pages)
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
