"""The paged path end to end: a synthetic Q4_0 model through PagedModel against
its forward pass in 64 bits on the host, and PagedGenerator's tokens whatever
the schedule."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from hypno_b200 import hypno_file as hf
from hypno_b200 import ops, paged, synth
from hypno_b200.paged_model import PagedGenerator, PagedModel

from . import _paged as ref

pytestmark = pytest.mark.gpu
CFG = dict(hidden=256, layers=2, heads=8, kv_heads=2, inter=384, vocab=700, theta=10000.0, max_pos=256)


@pytest.fixture(scope="module")
def image(cuda_device):
    return synth.build_image(CFG, seed=5, std=0.08)


def forward(image, ids):
    """Logits after every token, in 64 bits."""
    man = hf.Manifest(image)

    def w(name):
        shape, dt, _, _ = man.tensors[name]
        raw, _ = man.tensor_bytes(name)
        v = ops.dequantize_q4_0(bytes(raw)) if dt == hf.DT_Q4_0 else np.frombuffer(raw, np.float32)
        return v[:int(np.prod(shape))].reshape(shape).astype(np.float64)

    H, KH, D, n = CFG["heads"], CFG["kv_heads"], CFG["hidden"] // CFG["heads"], len(ids)
    norm = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * g  # noqa: E731
    a = np.arange(n)[:, None] * CFG["theta"] ** (-2 * np.arange(D // 2) / D)
    cs, sn = np.cos(a)[:, None], np.sin(a)[:, None]

    def turn(x):
        y = x.copy()
        y[..., 0::2], y[..., 1::2] = x[..., 0::2] * cs - x[..., 1::2] * sn, x[..., 0::2] * sn + x[..., 1::2] * cs
        return y

    x = w("model.embed_tokens.weight")[ids]
    for i in range(CFG["layers"]):
        p = f"model.layers.{i}."
        h = norm(x, w(p + "input_layernorm.weight"))
        q, k, v = (h @ w(p + f"self_attn.{c}_proj.weight").T for c in "qkv")
        q, k, v = turn(q.reshape(n, H, D)), turn(k.reshape(n, KH, D)), v.reshape(n, KH, D)
        k, v = (np.repeat(t.astype(np.float16).astype(np.float64), H // KH, 1) for t in (k, v))
        s = np.einsum("ihd,jhd->hij", q, k) / np.sqrt(D)
        s = np.where(np.tril(np.ones((n, n), bool)), s, -np.inf)
        e = np.exp(s - s.max(-1, keepdims=True))
        x = x + np.einsum("hij,jhd->ihd", e / e.sum(-1, keepdims=True), v).reshape(n, -1) @ w(p + "self_attn.o_proj.weight").T
        h = norm(x, w(p + "post_attention_layernorm.weight"))
        g = h @ w(p + "mlp.gate_proj.weight").T
        x = x + (g / (1 + np.exp(-g)) * (h @ w(p + "mlp.up_proj.weight").T)) @ w(p + "mlp.down_proj.weight").T
    return norm(x, w("model.norm.weight")) @ w("model.embed_tokens.weight").T


@pytest.mark.parametrize("sizes", [(40,), (17, 1, 1, 21), (1,) * 40])
def test_logits(cuda_device, image, sizes):
    """A prompt in one piece, in chunks, and token by token."""
    ids = synth.prompt_ids(CFG["vocab"], 40, seed=3).astype(np.int64)
    want = forward(image, ids)
    m = PagedModel(image, n_pages=8, page_size=16)
    t = paged.PageTable(8, 16, 1, 16)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    at = 0
    for n in sizes:
        length = t.grow(0, n)
        batch = paged.PagedBatch(torch.from_numpy(t.table[:, :3].copy()).to(cuda_device), torch.tensor([0, n], **i32), torch.tensor([length], **i32), n, length)
        got = m.logits(torch.from_numpy(ids[at:at + n]).to(cuda_device), batch, torch.arange(n, device=cuda_device)).cpu().numpy()
        # the framework's bar for logits (an FP16 cache rounds keys either way within it)
        assert np.max(np.abs(got - want[at:at + n])) <= 1e-3 * max(1.0, np.abs(want).max())
        at += n
    m.close()


@pytest.mark.parametrize("sizes", [(40,), (17, 1, 1, 21)])
def test_logits_over_an_fp32_cache(cuda_device, image, sizes):
    ids = synth.prompt_ids(CFG["vocab"], 40, seed=4).astype(np.int64)
    want = forward(image, ids)
    m = PagedModel(image, n_pages=8, page_size=16, cache_dtype=torch.float32)
    t = paged.PageTable(8, 16, 1, 16)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    at = 0
    for n in sizes:
        length = t.grow(0, n)
        batch = paged.PagedBatch(torch.from_numpy(t.table[:, :3].copy()).to(cuda_device), torch.tensor([0, n], **i32), torch.tensor([length], **i32), n, length)
        got = m.logits(torch.from_numpy(ids[at:at + n]).to(cuda_device), batch, torch.arange(n, device=cuda_device)).cpu().numpy()
        assert np.max(np.abs(got - want[at:at + n])) <= 1e-3 * max(1.0, np.abs(want).max())
        at += n
    m.close()


def test_a_captured_pass(cuda_device, image):
    """A pass of the model in a graph, replayed with other tokens in the same pages."""
    m = PagedModel(image, n_pages=6, page_size=16)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    batch = paged.PagedBatch(torch.tensor([[1], [4]], **i32), torch.tensor([0, 4, 7], **i32), torch.tensor([4, 3], **i32), 4, 4)
    ids, last = torch.tensor([5, 6, 7, 8, 9, 10, 11], device=cuda_device), torch.tensor([3, 6], device=cuda_device)
    first = m.logits(ids, batch, last)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m.logits(ids, batch, last)
    g.replay()
    assert torch.equal(out, first)
    ids.copy_(torch.tensor([50, 60, 70, 80, 90, 100, 110]))
    g.replay()
    got = out.clone()
    assert torch.equal(got, m.logits(ids, batch, last)) and not torch.equal(got, first)
    m.check()
    del g, out
    m.close()


def test_tokens_do_not_depend_on_the_schedule(cuda_device, image):
    def tokens(max_seqs, budget):
        m = PagedModel(image, n_pages=40, page_size=16)
        gen = PagedGenerator(m, max_seqs=max_seqs, budget=budget)
        g = np.random.default_rng(1)
        for i in range(6):
            gen.submit(g.integers(0, CFG["vocab"], size=int(g.integers(1, 90))), 12, temperature=[0.0, 0.7][i % 2], top_k=30, top_p=0.9, seed=i)
        out = gen.run()
        assert len(gen.pages.free) == 40
        m.close()
        return out

    want = tokens(1, 1000)
    assert all(len(v) == 12 for v in want.values())
    for other in ((6, 1000), (4, 13)):
        got = tokens(*other)
        # a draw or a greedy pick may turn where two tokens lie within the logits' rounding
        assert sum(got[k] != want[k] for k in want) <= 1


WIDE = dict(CFG, hidden=1024, heads=8, inter=2816)


def passes(device, first_page, n, tokens, steps, seed):
    """Arguments of `steps` calls of PagedModel.logits: n sequences, `tokens` new ones each a call,
    in pages of their own from first_page on; and the pages behind the last."""
    per = -(-tokens * steps // 16)
    table = torch.arange(first_page, first_page + n * per, dtype=torch.int32, device=device).view(n, per)
    g = torch.Generator(device=device).manual_seed(seed)
    out = []
    for i in range(1, steps + 1):
        batch = paged.PagedBatch(table, torch.arange(0, tokens * n + 1, tokens, dtype=torch.int32, device=device),
                                 torch.full((n,), tokens * i, dtype=torch.int32, device=device), tokens, tokens * i)
        ids = torch.randint(0, CFG["vocab"], (tokens * n,), generator=g, device=device)
        out.append((ids, batch, torch.arange(tokens * n, device=device)))
    return out, first_page + n * per


SHAPES = [(3, 40, 6), (13, 2, 30), (1, 90, 2), (2, 1, 60)]  # sequences, tokens, calls: products of every tile size, and single rows


def alone(m, todo):
    """The logits of each list of calls, one call at a time."""
    out = []
    for calls in todo:
        out.append([])
        for c in calls:
            out[-1].append(m.logits(*c))
            torch.cuda.synchronize()
    return out


def same(got, want):
    return all(len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b)) for a, b in zip(got, want))


def test_models_on_streams_of_their_own(cuda_device):
    """Four models, each on its own stream with nothing that waits between them."""
    image = synth.build_image(WIDE, seed=1, std=0.05)
    todo = [passes(cuda_device, 0, *shape, seed=i)[0] for i, shape in enumerate(SHAPES)]
    m = PagedModel(image, n_pages=60, page_size=16)
    want = [alone(m, [calls])[0] for calls in todo]
    m.close()
    models, streams = [PagedModel(image, n_pages=60, page_size=16) for _ in todo], [torch.cuda.Stream() for _ in todo]
    torch.cuda.synchronize()
    got = [[] for _ in todo]
    for i in range(max(map(len, todo))):
        for k, calls in enumerate(todo):
            if i < len(calls):
                with torch.cuda.stream(streams[k]):
                    got[k].append(models[k].logits(*calls[i]))
    torch.cuda.synchronize()
    assert same(got, want)
    for m in models:
        m.check()
        m.close()


@pytest.mark.parametrize("threads", [False, True])
def test_one_model_on_several_streams(cuda_device, threads):
    """Requests of one model, each on its own stream, in turn from one thread or from a thread each."""
    import threading
    todo, at = [], 0
    for i, shape in enumerate(SHAPES):
        calls, at = passes(cuda_device, at, *shape, seed=i)
        todo.append(calls)
    m = PagedModel(synth.build_image(WIDE, seed=1, std=0.05), n_pages=at, page_size=16)
    want = alone(m, todo)
    streams, got, errors = [torch.cuda.Stream() for _ in todo], [[] for _ in todo], []
    torch.cuda.synchronize()

    def run(k, calls):
        try:
            with torch.cuda.stream(streams[k]):
                for c in calls:
                    got[k].append(m.logits(*c))
        except Exception as e:  # (of a thread: for the assertion below)
            errors.append(e)

    if threads:
        each = [threading.Thread(target=run, args=(k, calls)) for k, calls in enumerate(todo)]
        for t in each:
            t.start()
        for t in each:
            t.join()
    else:
        for i in range(max(map(len, todo))):
            for k, calls in enumerate(todo):
                run(k, calls[i:i + 1])
    torch.cuda.synchronize()
    assert not errors and same(got, want)
    m.check()
    m.close()


def test_ids_outside_the_vocabulary_on_the_device(cuda_device, image):
    """They make their row NaN, and the rows of their sequence that see it; earlier
    ones stay within the framework's bar for logits, other sequences keep their bits."""
    m = PagedModel(image, n_pages=6, page_size=16)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    batch = paged.PagedBatch(torch.tensor([[1], [4]], **i32), torch.tensor([0, 4, 7], **i32), torch.tensor([4, 3], **i32), 4, 4)
    last = torch.arange(7, device=cuda_device)
    want = m.logits(torch.tensor([5, 6, 7, 8, 9, 10, 11], device=cuda_device), batch, last)
    for bad in (-1, CFG["vocab"], 2 ** 40):
        got = m.logits(torch.tensor([5, 6, bad, 8, 9, 10, 11], device=cuda_device), batch, last)
        assert bool(torch.isnan(got[2:4]).all()) and torch.equal(got[4:], want[4:])
        # (rows of a tile with such a value add its products in another order)
        assert bool(((got[:2] - want[:2]).abs() <= 1e-3 * want.abs().max().clamp_min(1.0)).all())
    m.close()


def test_an_aborted_product_is_reported(cuda_device, image, monkeypatch):
    """step() raises what the check of its products says, instead of returning tokens."""
    from hypno_b200 import paged_model
    from hypno_b200._lib import HypnoCudaError
    m = PagedModel(image, n_pages=4, page_size=16)
    args = [3, 4], np.array([[1]]), [0, 2], [2], [(0.3, 0.0, 0, 1.0, 0.0)]
    assert m.step(*args).shape == (1,)
    real = paged_model.call

    def call(name, *a):
        if name == "hc_q4_workspace_check":
            raise HypnoCudaError(-7, "a bounded pipeline wait timed out")
        return real(name, *a)

    monkeypatch.setattr(paged_model, "call", call)
    with pytest.raises(HypnoCudaError):
        m.step(*args)
    m.close()


def test_another_device_than_the_current_one(cuda_device, image, monkeypatch):
    from hypno_b200 import paged_model, sampling
    far = ref.Elsewhere(monkeypatch, paged, sampling, paged_model)
    m = PagedModel(image, n_pages=4, page_size=16, device="cuda:0")
    tokens = m.step([3, 4, 5], np.array([[1], [2]]), [0, 2, 3], [2, 1], [(0.3, 0.0, 0, 1.0, 0.0)] * 2)
    m.close()
    assert tokens.shape == (2,) and far.device == 7
    there = {"hc_rope_table_host", "hc_paged_attention_workspace", "hc_q4_matrix_free"}  # host work and a release need no device
    assert {n for n, d in far.calls if d != 0} <= there
    assert {n for n, d in far.calls if d == 0} >= {"hc_q4_matrix_upload", "hc_paged_append_dev", "hc_paged_attention_dev", "hc_sample_uniform_dev"}
    m = PagedModel(image, n_pages=4, device=torch.device("cuda"))
    assert m.device == torch.device("cuda:0")
    m.close()


def test_example_runs(cuda_device, capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_generate.py")
    spec = importlib.util.spec_from_file_location("paged_generate", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = mod.main([path])
    assert len(out) == 12 and all(len(v) == 24 for v in out.values())
    assert "256 of 256 pages free" in capsys.readouterr().out
