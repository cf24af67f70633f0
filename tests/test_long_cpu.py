"""Host side of the 4-bit cache and of the attention over selected pages without
a GPU: what is refused, the structures of the C entry points, the plain forms."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from hypno_b200 import _lib, build, paged
from hypno_b200.paged_model import PagedGenerator, PagedModel

from . import _long as long
from .test_paged_cpu import Plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


def test_host_tensors_are_refused():
    c, s = torch.zeros((2, 2, 16, 32), dtype=torch.uint8), torch.zeros((2, 2, 16, 2), dtype=torch.float16)
    with pytest.raises(TypeError):
        paged.PagedKV4(c, s, c, s)
    b = torch.zeros((2, 2, 64), dtype=torch.int8)
    with pytest.raises(TypeError):
        paged.PageBounds(b, b, torch.zeros((2, 2)), 16)


def test_what_a_handle_was_made_of_cannot_be_replaced():
    for obj, names in ((paged.PagedKV4.__new__(paged.PagedKV4), ("pools",)), (paged.PageBounds.__new__(paged.PageBounds), ("lo", "hi", "scale"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(obj, name, None)


def test_structures_are_those_of_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hypno_cuda.h"\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(hc_paged_kv_q4), offsetof(hc_paged_kv_q4, k_scale), offsetof(hc_paged_kv_q4, vs_pos_stride), '
                   'sizeof(hc_page_lists), sizeof(hc_page_bounds), offsetof(hc_page_bounds, head_dim)); return 0; }\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    K, B = _lib.HcPagedKV4, _lib.HcPageBounds
    assert got == [ctypes.sizeof(K), K.k_scale.offset, K.vs_pos_stride.offset, _lib.HC_PAGE_LISTS.size, ctypes.sizeof(B), B.head_dim.offset]


def test_refusals_at_the_c_entries(lib):
    """Before any device work: the addresses are never read."""
    at = 1 << 20
    base = _lib.HcPagedKV(at, at, 2048, 1024, 32, 2048, 1024, 32, _lib.KV_Q4, 4, 16, 2, 64, 0)
    scales = (at, at, 64, 32, 2, 64, 32, 2)

    def kv(s=scales, **more):
        k = _lib.HcPagedKV4(base, *s)
        for name, x in more.items():
            setattr(k.base, name, x)
        return k

    batch = _lib.HC_PAGED_BATCH.pack(at, at, at, 8, 1, 8, 1, 1, 100, 0)
    rows = _lib.HC_ROWS.pack(at, 256, 64)
    need = ctypes.c_size_t()

    def attention(k, b=batch, heads=4, lists=None):
        if lists is None:
            return lib.hc_paged_attention_workspace(ctypes.addressof(k), b, heads, 0, 0, ctypes.byref(need))
        return lib.hc_paged_list_attention_workspace(ctypes.addressof(k), b, lists, heads, 0, 0, ctypes.byref(need))

    assert attention(kv()) == 0
    assert attention(kv(head_dim=48)) == -3 and attention(kv(head_dim=288)) == -3
    assert attention(kv(k_pos_stride=24)) == -1 and attention(kv(v=at + 8)) == -1 and attention(kv(kv_dtype=3)) == -3
    assert attention(kv(s=(at + 2, *scales[1:]))) == -1 and attention(kv(s=(None, *scales[1:]))) == -1
    assert attention(kv(s=(*scales[:4], 3, *scales[5:]))) == -1 and attention(kv(s=(*scales[:7], -2))) == -1
    lists = lambda p=at, r=8, h=4, w=4: _lib.HC_PAGE_LISTS.pack(p, r, h, w, 0)  # noqa: E731
    assert attention(kv(), lists=lists()) == 0
    for bad in (lists(p=0), lists(p=at + 1), lists(w=0), lists(w=-3), lists(r=-8), lists(h=-1)):
        assert attention(kv(), lists=bad) == -1
    assert lib.hc_paged_list_attention_workspace(ctypes.addressof(kv()), batch, None, 4, 0, 0, ctypes.byref(need)) == -1
    assert lib.hc_paged_list_attention_dev(ctypes.addressof(kv()), batch, None, rows, rows, None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_attention_dev(ctypes.addressof(kv()), batch, rows, _lib.HC_ROWS.pack(0, 0, 0), None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_values_dev(ctypes.addressof(kv()), None, at, None) == -1
    assert lib.hc_paged_values_dev(ctypes.addressof(kv()), at + 2, at, None) == -1
    assert lib.hc_paged_values_dev(ctypes.addressof(kv(kv_dtype=_lib.KV_FP16)), at, at, None) == -3

    def bounds(*a):
        return _lib.HcPageBounds(*(a or (at, at, at, 4, 16, 2, 64)))

    def select(b, q=rows, heads=4, budget=4, first=1, recent=2, out=at, ws=(at, 1 << 20)):
        return lib.hc_page_select_dev(ctypes.addressof(b), batch, q, heads, 0, budget, first, recent, out, ws[0], ws[1], None)

    def workspace(b=None, heads=4, pages=8):
        batch = _lib.HC_PAGED_BATCH.pack(at, at, at, pages, 1, pages, 1, 1, 100, 0)
        assert lib.hc_page_select_workspace(ctypes.addressof(b or bounds()), batch, heads, ctypes.byref(need)) == 0
        return need.value

    assert workspace() == 0 and workspace(pages=100000) == 2 * 100000 * 4 and workspace(bounds(at, at, at, 4, 16, 2, 68)) == 2 * 8 * 4
    assert lib.hc_page_select_workspace(ctypes.addressof(bounds()), batch, 3, ctypes.byref(need)) == -1
    for b, want in ((bounds(at, at, at, 4, 16, 2, 66), -3), (bounds(at, at, at, 4, 16, 2, 260), -3), (bounds(at + 8, at, at, 4, 16, 2, 64), -1),
                    (bounds(at, at, None, 4, 16, 2, 64), -1), (bounds(at, at, at, 0, 16, 2, 64), -1)):
        assert select(b) == want and lib.hc_page_bounds_values_dev(ctypes.addressof(b), at, at, None) == want
        assert lib.hc_page_bounds_update_dev(ctypes.addressof(b), ctypes.addressof(kv()), batch, None) == want
    for ws in ((None, 0), (at, 63), (at + 4, 64)):      # (heads of 68 elements take one)
        assert select(bounds(at, at, at, 4, 16, 2, 68), q=_lib.HC_ROWS.pack(at, 272, 68), ws=ws) == -1
    for bad in (dict(heads=3), dict(budget=2), dict(first=-1), dict(recent=4), dict(budget=0, first=0, recent=0), dict(out=None), dict(out=at + 2),
                dict(q=_lib.HC_ROWS.pack(0, 0, 0))):
        assert select(bounds(), **bad) == -1, bad
    assert lib.hc_page_bounds_update_dev(ctypes.addressof(bounds(at, at, at, 4, 32, 2, 64)), ctypes.addressof(kv()), batch, None) == -1
    assert lib.hc_page_bounds_values_dev(ctypes.addressof(bounds()), at, None, None) == -1


def test_the_workspace_fits_the_last_round_of_a_chunk_over_4_bits(lib):
    """Four sequences whose values fit three at a time: the last one alone is cut into more runs than the three together."""
    at, need = 1 << 20, ctypes.c_size_t()
    kv = _lib.HcPagedKV4(_lib.HcPagedKV(at, at, 1024, 1024, 64, 1024, 1024, 64, _lib.KV_Q4, 4, 16, 1, 128, 0), at, at, 64, 64, 4, 64, 64, 4)
    pages, each = 40000, 40000 * 16 * 128 * 2

    def bytes_of(seqs):
        batch = _lib.HC_PAGED_BATCH.pack(at, at, at, pages, seqs, pages, 800, 200, 640000, 0)
        assert lib.hc_paged_attention_workspace(ctypes.addressof(kv), batch, 1, 1, 0, ctypes.byref(need)) == 0
        return need.value

    runs = lambda seqs, together: bytes_of(seqs) - 2 * together * each - 4 * together * pages  # noqa: E731  (each part a multiple of 256)
    assert 2 * each * 3 <= 2 ** 30 < 2 * each * 4 and runs(1, 1) > runs(3, 3) > 0
    assert runs(4, 3) >= runs(1, 1)


def test_a_step_refuses_rows_that_are_not_single():
    m = PagedModel.__new__(PagedModel)
    m.vocab, m.device, m.keep_pages = 50, None, 4
    for start, lone in (([0, 1, 3], 2), ([0, 2, 3], 1), ([0, 1, 2, 3], -1)):
        n = len(start) - 1
        with pytest.raises(ValueError):
            m.step([1, 2, 3], np.zeros((n, 1), np.int32), start, [9] * n, [(0.0, 0.0, 0, 1.0, 0.0)] * n, lone=lone)


def test_the_generator_says_which_rows_are_generated_tokens():
    """... where the model reads a part of the pages for these: never for the last piece of a prompt."""
    class Model(Plain):
        keep_pages, said = 3, []

        def step(self, ids, table, q_start, kv_len, settings, lone):
            self.said.append((lone, list(np.diff(q_start))))
            assert lone <= len(kv_len) and all(n == 1 for n in np.diff(q_start)[:lone])
            return super().step(ids, table, q_start, kv_len, settings)

    def run(m):
        gen = PagedGenerator(m, max_seqs=3, budget=4)
        for i, n in enumerate((1, 5, 9, 3)):
            gen.submit(list(range(1, n + 1)), 4, seed=i)
        return gen.run()

    m = Model()
    assert run(m) == run(Plain())
    # four requests make 16 tokens: the first of each comes from its prompt's last row
    assert sum(lone for lone, _ in m.said) == 12 and any(lone < sum(n == 1 for n in rows) for lone, rows in m.said)


def test_the_plain_4_bit_form():
    g = np.random.default_rng(0)
    x = (g.standard_normal((200, 64)) * 10.0 ** g.uniform(-9, 3, (200, 1))).astype(np.float32)
    x[0], x[1, 5], x[2, 40], x[3] = 0, np.inf, np.nan, 7000
    codes, scales, v = long.quantize(x)
    assert np.array_equal(long.decode(codes, scales, 64), v, equal_nan=True)
    assert np.isnan(v[1, :32]).all() and np.isfinite(v[1, 32:]).all() and np.isnan(v[2, 32:]).all() and np.all(v[0] == 0) and np.all(v[3] == 6272)
    s = scales[4:, :2].astype(np.float64)
    top = np.abs(x[4:].astype(np.float64)).reshape(-1, 2, 32).max(-1)
    # not below a seventh, and by less than one step of seven bits (or of float16's smallest) above
    assert np.all(s >= top / 7 * (1 - 2.0 ** -23)) and np.all(s <= np.maximum(top / 7 * (1 + 2.0 ** -6), top / 7 + 2.0 ** -24) * (1 + 2.0 ** -23))
    m, _ = np.frexp(s)
    assert np.all(m * 128 == np.rint(m * 128))
    assert np.all(np.abs(v[4:].astype(np.float64) - x[4:]).reshape(-1, 2, 32) <= s[..., None] / 2 * (1 + 2.0 ** -22))
