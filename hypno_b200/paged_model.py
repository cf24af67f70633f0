"""A .hypno model decoded over a paged KV cache, and continuous batching on it.

    PagedModel      the forward pass of a ragged batch of new tokens (chunks of
                    prompts and single tokens together): Q4_0 products of the C
                    ABI, paged append and attention, logits of each sequence's
                    last row
    PagedGenerator  requests of any length served together: prompts enter in
                    chunks beside the running requests' single tokens, pages are
                    taken as sequences grow and given back when they end, tokens
                    are drawn on the device from the request's own uniforms

The forward pass is transformer.rs:281-528 with the exact softmax instead of the
reference's polynomial (hypno_b200.engine keeps that one).
"""
import ctypes
import threading
from collections import deque

import numpy as np
import torch

from . import hypno_file as hf
from . import paged, sampling
from ._lib import call, check, load, on_device, raw_stream

__all__ = ["PagedModel", "PagedGenerator"]


class _Linear:
    """One weight matrix on the device: Q4_0 in the backend's layout, or FP32."""

    def __init__(self, man, name, device, workspace):
        self.workspace = workspace
        (self.n, self.k), dt, _, _ = man.tensors[name]
        raw = np.frombuffer(man.tensor_bytes(name)[0], np.uint8)
        self.q4 = self.dense = None
        if dt == hf.DT_Q4_0:
            self.q4 = ctypes.c_void_p()
            with on_device(device.index):
                call("hc_q4_matrix_upload", raw.ctypes.data, raw.size, self.n, self.k, ctypes.byref(self.q4))
        elif dt == hf.DT_FP32:
            self.dense = torch.from_numpy(raw.view(np.float32).reshape(self.n, self.k).copy()).to(device)
        else:
            raise ValueError(f"{name}: dtype {dt} is not supported here")

    def __call__(self, x):
        """x times the matrix, with the matrix's device current."""
        if self.dense is not None:
            return x @ self.dense.T
        x = x.contiguous()
        y = torch.empty((x.shape[0], self.n), dtype=torch.float32, device=x.device)
        check(load().hc_q4_matmul_ws_dev(self.q4, x.data_ptr(), x.shape[0], y.data_ptr(), self.workspace, raw_stream(x.get_device())))
        return y

    def close(self):
        if self.q4:
            load().hc_q4_matrix_free(self.q4)
            self.q4 = None


class PagedModel:
    """A .hypno image (bytes or a uint8 array) on a CUDA device, current or not,
    with one page pool per layer: of cache_dtype torch.float16 or torch.float32, or
    "q4" for 4 bits (paged.PagedKV4; heads of a multiple of 32 elements).

    keep_pages: the pages that a generated token reads per KV head, the first, the
    last two and those with the largest scores (paged.select_pages), at least 3;
    None: all.  Prompts read all of theirs."""

    def __init__(self, image, n_pages, page_size=16, cache_dtype=torch.float16, device="cuda", keep_pages=None):
        if cache_dtype not in (torch.float16, torch.float32, "q4"):
            raise ValueError(f"cache_dtype must be torch.float16, torch.float32 or 'q4', not {cache_dtype!r}")
        if keep_pages is not None and keep_pages < 3:
            raise ValueError(f"keep_pages must be at least 3, not {keep_pages}")
        self.keep_pages = keep_pages
        man = hf.Manifest(np.frombuffer(image, np.uint8) if isinstance(image, (bytes, bytearray)) else image)
        meta = man.metadata
        dim = int(meta["hidden_size"]) // int(meta["num_attention_heads"])
        if cache_dtype == "q4" and (dim % 32 or dim > 256) or keep_pages is not None and (dim % 4 or dim > 256):
            raise ValueError(f"heads of {dim} elements: 4 bits take a multiple of 32, keep_pages of 4, at most 256")
        self.device = torch.device("cuda", torch.cuda.current_device()) if str(device) == "cuda" else torch.device(device)
        self.workspace = ctypes.c_void_p()  # of this model's products
        with on_device(self.device.index):
            call("hc_q4_workspace_new", ctypes.byref(self.workspace))
        self.heads, self.kv_heads = int(meta["num_attention_heads"]), int(meta["num_key_value_heads"])
        self.hidden, self.layers = int(meta["hidden_size"]), int(meta["num_hidden_layers"])
        self.dim, self.vocab = self.hidden // self.heads, int(meta["vocab_size"])
        self.max_pos, self.eps = int(meta["max_position_embeddings"]), float(meta["rms_norm_eps"])
        self.n_pages, self.page_size = n_pages, page_size
        self.rope = paged.rope_table(self.max_pos, self.dim, float(meta["rope_theta"]), self.device)

        def vector(name):
            return torch.from_numpy(np.frombuffer(man.tensor_bytes(name)[0], np.float32).copy()).to(self.device)

        name = "model.embed_tokens.weight"
        raw, dt = man.tensor_bytes(name)
        if dt == hf.DT_Q4_0:
            q = torch.from_numpy(np.frombuffer(raw, np.uint8).copy()).to(self.device)
            self.embed = torch.empty((self.vocab, self.hidden), dtype=torch.float32, device=self.device)
            with on_device(self.device.index):
                call("hc_q4_0_dequantize_dev", q.data_ptr(), q.numel(), self.embed.data_ptr(), raw_stream(self.device.index))
            torch.cuda.synchronize(self.device)
        else:
            self.embed = vector(name).view(self.vocab, self.hidden)
        self.lm_head = _Linear(man, "lm_head.weight" if "lm_head.weight" in man.tensors else name, self.device, self.workspace)
        self.norm = vector("model.norm.weight")
        self.blocks, self.caches = [], []
        for i in range(self.layers):
            p = f"model.layers.{i}."
            block = {k: _Linear(man, p + n + ".weight", self.device, self.workspace) for k, n in
                     (("q", "self_attn.q_proj"), ("k", "self_attn.k_proj"), ("v", "self_attn.v_proj"), ("o", "self_attn.o_proj"),
                      ("gate", "mlp.gate_proj"), ("up", "mlp.up_proj"), ("down", "mlp.down_proj"))}
            block["in"], block["post"] = vector(p + "input_layernorm.weight"), vector(p + "post_attention_layernorm.weight")
            self.blocks.append(block)
            if cache_dtype == "q4":
                self.caches.append(paged.PagedKV4.alloc(n_pages, page_size, self.kv_heads, self.dim, self.device))
            else:
                self.caches.append(paged.PagedKV.alloc(n_pages, page_size, self.kv_heads, self.dim, cache_dtype, self.device))
        self.bounds = [None if keep_pages is None else paged.PageBounds.alloc(kv) for kv in self.caches]
        # the model's passes follow one another, the first one what was made here
        self.lock, self.done = threading.Lock(), torch.cuda.Event()
        with on_device(self.device.index):
            self.done.record(torch.cuda.current_stream())

    def _normed(self, x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * w

    def logits(self, ids, batch, last, lone=0):
        """Runs the packed rows' token ids (int64 on the device) through the
        layers, storing their keys and values, and returns the logits of the
        rows `last`.  The first `lone` sequences have one row each, which reads
        the pages that keep_pages leaves it.  An id outside the vocabulary gives NaN
        for its row and the rows of its sequence that see it (step() and
        PagedGenerator refuse it).
        Passes of one model on different streams, or from different
        threads, are made to follow one another on the device (they share its
        workspace and pools); other models run beside them.  A pass captured in a
        graph is not: its replays must not overlap the model's other passes."""
        known = (ids >= 0) & (ids < self.vocab)
        if not 0 <= lone <= batch.block_table.shape[0]:
            raise ValueError(f"{lone} sequences of one row among {batch.block_table.shape[0]}")
        return self._pass(torch.where(known, ids, 0), batch, last, lone, ~known[:, None])

    def _pass(self, ids, batch, last, lone=0, unknown=None):
        with self.lock, on_device(self.device.index):
            stream = torch.cuda.current_stream()
            if torch.cuda.is_current_stream_capturing():
                return self._layers(ids, batch, last, lone, unknown)
            stream.wait_event(self.done)
            try:
                return self._layers(ids, batch, last, lone, unknown)
            finally:
                self.done.record(stream)

    def _attend(self, kv, bounds, batch, parts, q):
        if bounds is not None:
            paged.update_bounds(bounds, kv, batch)
        if parts is None:
            return paged.attention(kv, batch, q)
        lone, few, rest = parts
        out = torch.empty_like(q)
        pages = paged.select_pages(bounds, few, q[:lone], self.keep_pages)
        paged.attention(kv, few, q[:lone], out=out[:lone], pages=pages)
        if rest is not None:
            paged.attention(kv, rest, q, out=out)
        return out

    def _layers(self, ids, batch, last, lone, unknown):
        n = ids.shape[0]
        parts = None
        if self.keep_pages is not None and lone and batch.block_table.shape[1] > self.keep_pages:
            table, starts, lengths = batch.block_table, batch.q_start, batch.kv_len
            few = paged.PagedBatch(table[:lone], starts[:lone + 1], lengths[:lone], 1, batch.max_kv_len)
            rest = None if lone == table.shape[0] else paged.PagedBatch(table[lone:], starts[lone:], lengths[lone:], batch.max_q_len, batch.max_kv_len)
            parts = lone, few, rest
        x = self.embed[ids]
        if unknown is not None:
            x.masked_fill_(unknown, float("nan"))
        for b, kv, bounds in zip(self.blocks, self.caches, self.bounds):
            h = self._normed(x, b["in"])
            q, k, v = b["q"](h).view(n, -1, self.dim), b["k"](h).view(n, -1, self.dim), b["v"](h).view(n, -1, self.dim)
            q = paged.append(kv, batch, k, v, q=q, rope=self.rope)
            x = x + b["o"](self._attend(kv, bounds, batch, parts, q).view(n, -1))
            h = self._normed(x, b["post"])
            x = x + b["down"](torch.nn.functional.silu(b["gate"](h)) * b["up"](h))
        return self.lm_head(self._normed(x[last], self.norm))

    def check(self):
        """Waits for the current stream; raises HypnoCudaError if a product on it
        gave up a bounded wait since the last check (its output is not written)."""
        with on_device(self.device.index):
            call("hc_q4_workspace_check", self.workspace, raw_stream(self.device.index))

    def step(self, ids, table, q_start, kv_len, settings, lone=None):
        """One step of a serving loop from host arrays: ids of the packed rows,
        the sequences' pages, row starts and lengths, and per sequence
        (u, temperature, top_k, top_p, min_p); returns the token drawn after
        each sequence's last row.  lone: how many of the first sequences have a
        single row that reads the pages keep_pages leaves it (None: all with one
        row, up to the first with more)."""
        _check_ids(ids, self.vocab)
        dev = self.device
        start, length = np.asarray(q_start, np.int32), np.asarray(kv_len, np.int32)
        if start.ndim != 1 or start.size < 2 or start[0] != 0 or start[-1] != len(ids) or np.diff(start).min() < 1:
            raise ValueError(f"row starts {start.tolist()} of {len(ids)} rows: they begin at 0, each sequence has a row, and the last ends")
        if length.shape != (start.size - 1,) or len(settings) != start.size - 1:
            raise ValueError(f"{start.size - 1} sequences with {length.size} lengths and {len(settings)} settings")
        single = int(np.argmin(np.append(np.diff(start) == 1, False)))  # leading sequences of one row
        if lone is None:
            lone = single
        elif not 0 <= lone <= single:
            raise ValueError(f"{lone} sequences of one row, the first {single} have one")
        t = lambda a, d: torch.from_numpy(np.ascontiguousarray(a, d)).to(dev)  # noqa: E731
        batch = paged.PagedBatch(t(table, np.int32), t(start, np.int32), t(length, np.int32), int(np.diff(start).max()), int(length.max()))
        logits = self._pass(t(ids, np.int64), batch, t(start[1:] - 1, np.int64), lone)
        u, temp, k, p, m = (t([s[i] for s in settings], np.int32 if i == 2 else np.float32) for i in range(5))
        tokens = sampling.sample(logits, u, temp, k, p, m)[0].cpu().numpy()
        self.check()
        return tokens

    def close(self):
        for b in self.blocks:
            for w in b.values():
                if isinstance(w, _Linear):
                    w.close()
        self.lm_head.close()
        with on_device(self.device.index):
            load().hc_q4_workspace_free(self.workspace)
        self.workspace = ctypes.c_void_p()


def _check_ids(ids, vocab):
    """Refuses token ids outside the vocabulary."""
    a = np.asarray(ids)
    if a.dtype.kind not in "iu":
        raise TypeError(f"token ids must be integers, not {a.dtype}")
    if a.size and not 0 <= int(a.min()) <= int(a.max()) < vocab:
        raise ValueError(f"token ids from {int(a.min())} to {int(a.max())}, the vocabulary has {vocab}")


class _Request:
    def __init__(self, rid, prompt, max_tokens, settings, seed):
        self.id, self.prompt, self.max_tokens, self.settings = rid, [int(t) for t in prompt], max_tokens, settings
        self.rng = np.random.Generator(np.random.PCG64(seed))
        self.fed = 0          # tokens whose keys are in the cache
        self.tokens = []
        self.seq = -1


class PagedGenerator:
    """Continuous batching over a model with `step(ids, table, q_start, kv_len,
    settings)`, `n_pages`, `page_size`, `max_pos` and, where it has one, `vocab`
    (PagedModel).  A request is admitted when the pool can hold it to
    its last token; a step feeds every running request its next token and fills
    up to `budget` rows with chunks of the prompts still entering."""

    def __init__(self, model, max_seqs=8, budget=256, eos_id=None):
        if budget < 1 or max_seqs < 1:
            raise ValueError("budget and max_seqs must be positive")
        self.model, self.budget, self.eos_id = model, budget, eos_id
        self.pages = paged.PageTable(model.n_pages, model.page_size, max_seqs, -(-model.max_pos // model.page_size))
        self.slots = list(range(max_seqs - 1, -1, -1))
        self.waiting, self.running, self.finished = deque(), [], {}
        self.promised = 0     # pages that running requests may still come to hold, with those they hold
        self.next_id = 0

    def _need(self, r):
        return -(-(len(r.prompt) + r.max_tokens) // self.model.page_size)

    def submit(self, prompt, max_tokens, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seed=0):
        """Queues a request; returns its id."""
        r = _Request(self.next_id, prompt, int(max_tokens), (float(temperature), int(top_k), float(top_p), float(min_p)), seed)
        vocab = getattr(self.model, "vocab", None)
        if vocab is not None:
            _check_ids(r.prompt, vocab)
        if not r.prompt or r.max_tokens < 1:
            raise ValueError("a request needs a prompt and at least one token to make")
        if len(r.prompt) + r.max_tokens > self.model.max_pos or self._need(r) > self.model.n_pages:
            raise ValueError(f"{len(r.prompt)} + {r.max_tokens} tokens exceed the model's positions or the pool")
        self.next_id += 1
        self.waiting.append(r)
        return r.id

    @property
    def idle(self):
        return not self.waiting and not self.running

    def step(self):
        """One step; returns the (request id, token) pairs it made."""
        while self.waiting and self.slots and self.promised + self._need(self.waiting[0]) <= self.model.n_pages:
            r = self.waiting.popleft()
            r.seq = self.slots.pop()
            self.promised += self._need(r)
            self.running.append(r)
        # single tokens first, then chunks of prompts while the budget lasts
        rows, room = [], self.budget
        for r in sorted(self.running, key=lambda r: r.fed < len(r.prompt)):
            left = len(r.prompt) + len(r.tokens) - r.fed
            take = min(left, max(room, 0)) if r.fed < len(r.prompt) else left
            if take > 0:
                rows.append((r, take))
                room -= take
        if not rows:
            return []
        ids, start, length = [], [0], []
        for r, take in rows:
            ids += (r.prompt + r.tokens)[r.fed:r.fed + take]
            start.append(start[-1] + take)
            length.append(self.pages.grow(r.seq, take))
        width = max(-(-n // self.model.page_size) for n in length)
        table = self.pages.table[[r.seq for r, _ in rows], :width]
        drawn = [r.fed + take >= len(r.prompt) for r, take in rows]  # the others are still inside their prompt
        settings = [((r.rng.random(dtype=np.float32) if d else 0.0), *r.settings) for (r, _), d in zip(rows, drawn)]
        # (prompts read all their pages, however they are cut into chunks)
        more = {} if getattr(self.model, "keep_pages", None) is None else {"lone": sum(r.fed >= len(r.prompt) for r, _ in rows)}
        picked = self.model.step(ids, table, start, length, settings, **more)
        made = []
        for (r, take), d, tok in zip(rows, drawn, picked):
            r.fed += take
            if not d:
                continue
            tok = int(tok)
            if tok >= 0 and tok != self.eos_id:
                r.tokens.append(tok)
                made.append((r.id, tok))
            if tok < 0 or tok == self.eos_id or len(r.tokens) == r.max_tokens:
                self.running.remove(r)
                self.finished[r.id] = r.tokens
                self.promised -= self._need(r)
                self.pages.release(r.seq)
                self.slots.append(r.seq)
        return made

    def run(self):
        """Steps until every request has ended; returns their tokens by id."""
        while not self.idle:
            self.step()
        return dict(self.finished)
