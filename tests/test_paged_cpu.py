"""Host side of the paged serving path without a GPU: the page table, the
generator's schedule against a model of plain Python, the rotation table, and
that the operators refuse to run on host tensors."""
import numpy as np
import pytest
import torch

from hypno_b200 import _lib, build, paged, sampling
from hypno_b200.paged_model import PagedGenerator


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


def test_page_table_grows_and_releases():
    t = paged.PageTable(5, 4, 3, 3)
    assert t.grow(0, 1) == 1 and t.grow(0, 3) == 4 and len(t.free) == 4   # one page holds four positions
    assert t.grow(0, 1) == 5 and len(t.free) == 3
    assert t.grow(2, 12) == 12 and len(t.free) == 0
    held = set(t.table[0][:2]) | set(t.table[2])
    assert held == set(range(5)) and t.table[0, 2] == -1 and np.all(t.table[1] == -1)
    assert not t.can_grow(1, 1) and not t.can_grow(2, 1) and t.can_grow(0, 3)
    with pytest.raises(ValueError):
        t.grow(1, 1)
    with pytest.raises(ValueError):
        t.grow(0, -1)
    t.release(2)
    assert len(t.free) == 3 and np.all(t.table[2] == -1) and t.lengths[2] == 0
    assert t.grow(1, 9) == 9 and len(set(t.free) | set(t.table[0][:2]) | set(t.table[1])) == 5
    with pytest.raises(ValueError):
        paged.PageTable(0, 4, 1, 1)


class Plain:
    """A model whose next token is a function of every token it has stored in
    its pages, so that a wrong page, length or order shows."""

    n_pages, page_size, max_pos = 12, 4, 40

    def __init__(self):
        self.pool = np.full((self.n_pages, self.page_size), -1, np.int64)
        self.rows = []

    def step(self, ids, table, q_start, kv_len, settings):
        out = []
        self.rows.append(len(ids))
        for b, n in enumerate(kv_len):
            new = ids[q_start[b]:q_start[b + 1]]
            for i, t in enumerate(new):
                p = n - len(new) + i
                self.pool[table[b][p // self.page_size], p % self.page_size] = t
            seen = [int(self.pool[table[b][p // self.page_size], p % self.page_size]) for p in range(n)]
            out.append(self.after(seen, settings[b][0]))
        return out

    @staticmethod
    def after(seen, u):
        return (sum((i + 1) * t for i, t in enumerate(seen)) + int(1000 * u)) % 97


@pytest.mark.parametrize("budget,max_seqs", [(1, 1), (3, 2), (7, 3), (1000, 8)])
def test_generator_equals_one_request_at_a_time(budget, max_seqs):
    g = np.random.default_rng(budget)
    m = Plain()
    gen = PagedGenerator(m, max_seqs=max_seqs, budget=budget)
    want = {}
    for i in range(9):
        prompt, n = [int(t) for t in g.integers(0, 97, size=int(g.integers(1, 20)))], int(g.integers(1, 9))
        rid = gen.submit(prompt, n, seed=i)
        rng, toks = np.random.Generator(np.random.PCG64(i)), []
        for _ in range(n):
            toks.append(Plain.after(prompt + toks, rng.random(dtype=np.float32)))
        want[rid] = toks
    assert gen.run() == want
    assert len(gen.pages.free) == m.n_pages and gen.promised == 0
    assert max(m.rows) <= max(budget, 0) + max_seqs


def test_generator_stops_at_the_end_token_and_refuses_what_cannot_fit():
    m = Plain()
    first = Plain.after([5], 0.0)
    gen = PagedGenerator(m, eos_id=first)
    gen.submit([5], 10)
    gen.running, r = [], gen.waiting[0]
    r.rng = type("zero", (), {"random": lambda self, dtype=None: 0.0})()
    assert gen.run() == {0: []}
    with pytest.raises(ValueError):
        gen.submit([], 3)
    with pytest.raises(ValueError):
        gen.submit([1] * 39, 2)
    with pytest.raises(ValueError):
        PagedGenerator(m, budget=0)


def test_rope_table_values():
    t = paged.rope_table(50, 16, 10000.0, "cpu").numpy().astype(np.float64)
    j, p = np.arange(8), np.arange(50)[:, None]
    a = p * 10000.0 ** (-2 * j / 16)
    # an angle of up to 50 in f32: half an ulp of the frequency and of the product, times the position
    assert np.abs(t[..., 0] - np.cos(a)).max() <= 50 * 2.0 ** -22 and np.abs(t[..., 1] - np.sin(a)).max() <= 50 * 2.0 ** -22
    with pytest.raises(_lib.HypnoCudaError):
        paged.rope_table(4, 7, 10000.0, "cpu")


def test_host_tensors_are_refused():
    z = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(TypeError):
        paged.PagedKV(z, z)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        paged.PagedBatch(i.view(1, 2), i, i[:1], 1, 1)
    with pytest.raises(TypeError):
        sampling.sample(torch.zeros((1, 8)), torch.zeros(1))


def test_a_device_is_current_within_the_block_and_the_former_after_it(monkeypatch):
    log, state = [], {"device": 3}
    monkeypatch.setattr(_lib, "current_device", lambda: state["device"])
    monkeypatch.setattr(_lib, "_set_device", lambda i: (log.append(i), state.update(device=i)))
    with _lib.on_device(1):
        assert state["device"] == 1
    assert state["device"] == 3 and log == [1, 3]
    with pytest.raises(RuntimeError):
        with _lib.on_device(0):
            raise RuntimeError
    assert state["device"] == 3 and log == [1, 3, 0, 3]
    with _lib.on_device(3):  # current already: no call
        pass
    assert log == [1, 3, 0, 3]


def test_product_workspaces_without_a_device(lib):
    import ctypes
    a, b = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.hc_q4_workspace_new(ctypes.byref(a)) == 0 and lib.hc_q4_workspace_new(ctypes.byref(b)) == 0
    assert a.value and b.value and a.value != b.value
    assert lib.hc_q4_workspace_check(a, None) == 0            # no product has run in it
    assert lib.hc_q4_workspace_new(None) == -1 and lib.hc_q4_workspace_check(None, None) == -1
    assert lib.hc_q4_matmul_ws_dev(None, None, 2, None, a, None) == -1
    assert lib.hc_q4_workspace_free(a) == 0 and lib.hc_q4_workspace_free(b) == 0 and lib.hc_q4_workspace_free(None) == 0


@pytest.mark.parametrize("bad", [[-1], [5, 97], [3, -2, 4], [2 ** 40]])
def test_ids_outside_the_vocabulary_are_refused(bad):
    m = Plain()
    m.vocab = 97
    gen = PagedGenerator(m)
    first = gen.submit([0, 96], 2)
    with pytest.raises(ValueError):
        gen.submit(bad, 2)
    assert len(gen.waiting) == 1 and gen.submit([1], 1) == first + 1    # nothing of the refused one is left
    assert sorted(gen.run()) == [first, first + 1]


def test_a_step_refuses_ids_before_any_device_work():
    from hypno_b200.paged_model import PagedModel
    m = PagedModel.__new__(PagedModel)      # without weights or a device
    m.vocab = 50
    for ids, error in (([3, 50], ValueError), ([-1], ValueError), ([1.5], TypeError)):
        with pytest.raises(error):
            m.step(ids, np.zeros((1, 1), np.int32), [0, len(ids)], [len(ids)], [(0.0, 0.0, 0, 1.0, 0.0)])


def test_what_a_handle_was_made_of_cannot_be_replaced():
    """The C structures hold the tensors' addresses, so another tensor must not be put in their place."""
    kv, batch = paged.PagedKV.__new__(paged.PagedKV), paged.PagedBatch.__new__(paged.PagedBatch)
    for obj, names in ((kv, ("k", "v")), (batch, ("block_table", "q_start", "kv_len", "max_q_len", "max_kv_len"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(obj, name, None)


@pytest.mark.parametrize("start,kv_len,settings", [([0, 2], [2], 1), ([1, 3], [2], 1), ([0, 2, 2, 3], [2, 1, 1], 3), ([0, 4, 3], [4, 1], 2), ([0], [], 0),
                                                   ([0, 1, 3], [1], 2), ([0, 1, 3], [1, 2], 1), ([0, 5], [5], 1)])
def test_a_step_refuses_rows_that_do_not_fit_together(start, kv_len, settings):
    """Before any device work, where a row past the end would fail an assertion."""
    from hypno_b200.paged_model import PagedModel
    m = PagedModel.__new__(PagedModel)
    m.vocab, m.device = 50, None
    with pytest.raises(ValueError):
        m.step([1, 2, 3], np.zeros((len(kv_len), 1), np.int32), start, kv_len, [(0.0, 0.0, 0, 1.0, 0.0)] * settings)
