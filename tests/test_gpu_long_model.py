"""A model over a cache in 4 bits, and with generated tokens that read a part of
their pages: PagedModel and PagedGenerator with these operators."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from hypno_b200 import paged, paged_model, sampling, synth
from hypno_b200.paged_model import PagedGenerator, PagedModel

from . import _long as long
from . import _paged as ref
from . import test_gpu_paged_model as base

pytestmark = pytest.mark.gpu
CFG = base.CFG


@pytest.fixture(scope="module")
def image(cuda_device):
    return synth.build_image(CFG, seed=5, std=0.08)


class Recorded:
    """What a model's layers give the operators and get from them."""

    def __init__(self, monkeypatch):
        self.stored, self.read, real_append, real_attention = [], [], paged.append, paged.attention

        def append(kv, batch, k, v, **more):
            turned = real_append(kv, batch, k, v, **more)
            self.stored.append((k.clone(), v.clone(), batch.kv_len.clone(), [t.clone() for t in kv.values()]))
            return turned

        def attention(kv, batch, q, out=None, pages=None):
            got = real_attention(kv, batch, q, out=out, pages=pages)
            self.read.append((kv, batch, q.clone(), got.clone(), pages))
            return got

        monkeypatch.setattr(paged, "append", append)
        monkeypatch.setattr(paged, "attention", attention)


def test_layers_over_4_bits(cuda_device, image, monkeypatch):
    """What is stored is the quantized key and value of each row, what is read the attention over these."""
    m = PagedModel(image, n_pages=8, page_size=16, cache_dtype="q4")
    seen = Recorded(monkeypatch)
    ids = synth.prompt_ids(CFG["vocab"], 40, seed=3).astype(np.int64)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.tensor([[5, 2, 7]], **i32)
    H, KH, D = m.heads, m.kv_heads, m.dim
    for start, n in ((0, 17), (17, 1), (18, 22)):
        batch = paged.PagedBatch(table, torch.tensor([0, n], **i32), torch.tensor([start + n], **i32), n, start + n)
        got = m.logits(torch.from_numpy(ids[start:start + n]).to(cuda_device), batch, torch.arange(n, device=cuda_device))
        assert bool(torch.isfinite(got).all())
        assert len(seen.stored) == len(seen.read) == CFG["layers"]
        for (k, v, _, values), (_, _, q, out, pages) in zip(seen.stored, seen.read):
            assert pages is None
            p = np.arange(start, start + n)
            at = table[0].cpu().numpy()[p // 16], slice(None), p % 16
            turned = long.rotate32(k.cpu().numpy(), m.rope.cpu().numpy()[p], "adjacent")
            for t, x in zip(values, (turned, v.cpu().numpy())):
                assert np.array_equal(t.cpu().numpy()[at].astype(np.float32), long.quantize(x)[2])
            c = type("Held", (), dict(heads=H, kv_heads=KH, dim=D, page=16, rows=n, q=q.cpu().numpy(), k=values[0].cpu().numpy(), v=values[1].cpu().numpy(),
                                      table=table.cpu().numpy(), where=lambda s: [(0, int(x)) for x in p], page_of=ref.Case.page_of))()
            want, _, A, M = ref.attention(c)
            assert np.all(np.abs(out.cpu().numpy() - want) <= ref.tolerance(c, A, M, False))
        seen.stored.clear(), seen.read.clear()
    m.close()


def forward(image, ids, first_generated, page):
    """base.forward with the tokens from first_generated on reading their first page and last two."""
    n = len(ids)
    real, mask = np.tril, np.tril(np.ones((n, n), bool))
    for p in range(first_generated, n):
        pages = np.arange(n) // page
        mask[p] &= (pages == 0) | (pages >= p // page - 1)
    try:
        base.np.tril = lambda x: mask
        return base.forward(image, ids)
    finally:
        base.np.tril = real


@pytest.mark.parametrize("cache", [torch.float16, torch.float32])
def test_logits_of_tokens_that_read_three_pages(cuda_device, image, cache):
    """keep_pages of 3 leaves the first page and the last two, whatever they score; a prompt beside them reads all."""
    ids, other = (synth.prompt_ids(CFG["vocab"], n, seed=3 + n).astype(np.int64) for n in (60, 50))
    want, beside = forward(image, ids, 40, 4), base.forward(image, other)
    m = PagedModel(image, n_pages=40, page_size=4, cache_dtype=cache, keep_pages=3)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(cuda_device)[:30].view(2, 15)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda_device)  # noqa: E731
    batch = paged.PagedBatch(table[:1], torch.tensor([0, 40], **i32), torch.tensor([40], **i32), 40, 40)
    got = m.logits(dev(ids[:40]), batch, torch.arange(40, device=cuda_device)).cpu().numpy()
    bar = lambda w: 1e-3 * max(1.0, np.abs(w).max())  # noqa: E731  (the framework's for logits)
    assert np.max(np.abs(got - want[:40])) <= bar(want)
    fed = 0
    for p in range(40, 60):
        take = [1, 5, 2][p % 3] if fed < 50 else 0
        take = min(take, 50 - fed)
        if take:
            batch = paged.PagedBatch(table, torch.tensor([0, 1, 1 + take], **i32), torch.tensor([p + 1, fed + take], **i32), take, 60)
            got = m.logits(dev(np.concatenate([ids[p:p + 1], other[fed:fed + take]])), batch, torch.arange(1 + take, device=cuda_device), lone=1).cpu().numpy()
            assert np.max(np.abs(got[1:] - beside[fed:fed + take])) <= bar(beside)
            fed += take
        else:
            batch = paged.PagedBatch(table[:1], torch.tensor([0, 1], **i32), torch.tensor([p + 1], **i32), 1, 60)
            got = m.logits(dev(ids[p:p + 1]), batch, torch.arange(1, device=cuda_device), lone=1).cpu().numpy()
        assert np.max(np.abs(got[0] - want[p])) <= bar(want)
    with pytest.raises(ValueError):
        m.logits(dev(ids[:1]), batch, torch.arange(1, device=cuda_device), lone=3)
    m.close()


@pytest.mark.parametrize("cache", [torch.float16, "q4"])
def test_a_captured_pass(cuda_device, image, cache):
    """Two sequences that read a part of their pages, beside a chunk, in a graph."""
    m = PagedModel(image, n_pages=64, page_size=4, cache_dtype=cache, keep_pages=5)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.randperm(64, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(cuda_device)[:60].view(3, 20)
    fill = paged.PagedBatch(table, torch.tensor([0, 60, 130, 140], **i32), torch.tensor([60, 70, 10], **i32), 70, 70)
    prompt = torch.from_numpy(synth.prompt_ids(CFG["vocab"], 140, seed=9).astype(np.int64)).to(cuda_device)
    m.logits(prompt, fill, torch.tensor([59], device=cuda_device))
    batch = paged.PagedBatch(table, torch.tensor([0, 1, 2, 6], **i32), torch.tensor([61, 71, 14], **i32), 4, 80)
    ids, last = torch.tensor([5, 6, 7, 8, 9, 10], device=cuda_device), torch.arange(6, device=cuda_device)
    first = m.logits(ids, batch, last, lone=2)
    dense = m.logits(ids, batch, last)
    assert not torch.equal(first[:2], dense[:2])           # fewer pages: other logits
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m.logits(ids, batch, last, lone=2)
    g.replay()
    assert torch.equal(out, first)
    ids.copy_(torch.tensor([50, 60, 70, 80, 90, 100])), batch.kv_len.add_(1)
    g.replay()
    got = out.clone()
    assert torch.equal(got, m.logits(ids, batch, last, lone=2)) and not torch.equal(got, first)
    m.check()
    del g, out
    m.close()


@pytest.mark.parametrize("cache,keep", [("q4", None), (torch.float16, 4), ("q4", 4)])
def test_tokens_do_not_depend_on_the_schedule(cuda_device, image, cache, keep):
    def tokens(max_seqs, budget):
        m = PagedModel(image, n_pages=160, page_size=4, cache_dtype=cache, keep_pages=keep)
        gen = PagedGenerator(m, max_seqs=max_seqs, budget=budget)
        g = np.random.default_rng(1)
        for i in range(6):
            gen.submit(g.integers(0, CFG["vocab"], size=int(g.integers(1, 90))), 12, temperature=[0.0, 0.7][i % 2], top_k=30, top_p=0.9, seed=i)
        out = gen.run()
        assert len(gen.pages.free) == 160
        m.close()
        return out

    want = tokens(1, 1000)
    assert all(len(v) == 12 for v in want.values())
    for other in ((6, 1000), (4, 13)):
        got = tokens(*other)
        # a draw or a greedy pick may turn where two tokens lie within the logits' rounding
        assert sum(got[k] != want[k] for k in want) <= 1


def test_pages_for_all_is_the_dense_pass(cuda_device, image):
    ids = synth.prompt_ids(CFG["vocab"], 40, seed=3).astype(np.int64)
    args = ids, np.array([[5, 2, 7]]), [0, 40], [40], [(0.3, 0.9, 0, 1.0, 0.0)]
    one = [3], np.array([[5, 2, 7]]), [0, 1], [41], [(0.3, 0.9, 0, 1.0, 0.0)]
    tokens = []
    for keep in (None, 3, 100):
        m = PagedModel(image, n_pages=8, page_size=16, keep_pages=keep)
        tokens.append([int(m.step(*args)[0]), int(m.step(*one)[0])])
        with pytest.raises(ValueError):
            m.step(*args, lone=1)
        with pytest.raises(ValueError):
            m.step(*one, lone=2)
        m.close()
    assert tokens[0] == tokens[1] == tokens[2]


def test_what_a_model_refuses(cuda_device, image):
    for more in (dict(cache_dtype="q8"), dict(cache_dtype=torch.bfloat16), dict(keep_pages=2), dict(keep_pages=0)):
        with pytest.raises(ValueError):
            PagedModel(image, n_pages=4, **more)


def test_another_device_than_the_current_one(cuda_device, image, monkeypatch):
    far = ref.Elsewhere(monkeypatch, paged, sampling, paged_model)
    m = PagedModel(image, n_pages=40, page_size=4, cache_dtype="q4", device="cuda:0", keep_pages=3)
    table = np.arange(40).reshape(2, 20)
    m.step([3] * 90, table, [0, 60, 90], [60, 30], [(0.3, 0.0, 0, 1.0, 0.0)] * 2)
    tokens = m.step([3, 4], table, [0, 1, 2], [61, 31], [(0.3, 0.0, 0, 1.0, 0.0)] * 2)
    m.close()
    assert tokens.shape == (2,) and far.device == 7
    there = {"hc_rope_table_host", "hc_paged_attention_workspace", "hc_paged_list_attention_workspace", "hc_page_select_workspace", "hc_q4_matrix_free"}
    assert {n for n, d in far.calls if d != 0} <= there
    assert {n for n, d in far.calls if d == 0} >= {"hc_paged_append_dev", "hc_page_bounds_update_dev", "hc_page_select_dev", "hc_paged_list_attention_dev"}


@pytest.mark.parametrize("flags", [["--cache", "q4"], ["--keep-pages", "4"], ["--cache", "q4", "--keep-pages", "5"]])
def test_example_runs(cuda_device, capsys, flags):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_generate.py")
    spec = importlib.util.spec_from_file_location("paged_generate", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = mod.main([path, *flags])
    assert len(out) == 12 and all(len(v) == 24 for v in out.values())
    assert "256 of 256 pages free" in capsys.readouterr().out
