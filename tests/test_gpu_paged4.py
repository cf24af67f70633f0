"""The paged cache in 4 bits: append and attention against their definitions on
the host, at the sizes and masks where they can go wrong, and what they refuse."""
import numpy as np
import pytest
import torch

from hypno_b200 import paged
from hypno_b200._lib import HypnoCudaError

from . import _long as long
from . import _paged as ref

pytestmark = pytest.mark.gpu

X = [np.float32, np.float16]
IDS = ["f32", "f16"]


def in_order(t, order):
    return t.transpose(1, 2).contiguous().transpose(1, 2) if order == "page" else t


def on_device(c, dev, order="head", fused=False):
    kv = paged.PagedKV4(*(in_order(torch.from_numpy(t).to(dev), order) for t in c.pools))
    batch = paged.PagedBatch(torch.from_numpy(c.table).to(dev), torch.from_numpy(c.q_start).to(dev),
                             torch.from_numpy(c.kv_len).to(dev), max(c.new, default=0), max(max(c.kv, default=0), 0))
    q, kn, vn = (torch.from_numpy(x).to(dev) for x in (c.q, c.kn, c.vn))
    if fused:  # heads side by side, as a fused projection writes them
        rows = torch.cat([q, kn, vn], 1)
        q, kn, vn = rows[:, :c.heads], rows[:, c.heads:c.heads + c.kv_heads], rows[:, c.heads + c.kv_heads:]
    return kv, batch, q, kn, vn


def compare(c, out, lse, want, want_lse, A, M):
    tol = ref.tolerance(c, A, M, c.q.dtype == np.float16)
    got = out.cpu().numpy().astype(np.float64)
    err = np.abs(got - want)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], float(np.nanmax(err)), float(tol.max()), int(bad.sum()), bad.size)
    got_lse = lse.cpu().numpy().astype(np.float64)
    seen = np.isfinite(want_lse)
    assert np.array_equal(seen, np.isfinite(got_lse)) and np.all(got_lse[~seen] == -np.inf)
    # the log of the sum: the scores' error, and f32 rounding of the sum and of the result
    room = A[..., 0] * 2.0 ** -20 + 2.0 ** -19 + np.abs(np.where(seen, want_lse, 0)) * 2.0 ** -22
    assert np.all(np.abs(got_lse[seen] - want_lse[seen]) <= room[seen])


def check_attention(c, dev, window=0, scale=None, order="head", fused=False, batch_edit=None):
    kv, batch, q, _, _ = on_device(c, dev, order, fused)
    if batch_edit:
        batch = batch_edit(batch)
    lse = torch.full((c.rows, c.heads), float("nan"), device=dev)
    out = paged.attention(kv, batch, q, window=window, scale=scale, lse=lse)
    assert out.shape == q.shape and out.dtype == q.dtype
    compare(c, out, lse, *ref.attention(c, window, scale))
    return out


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 1, 128), (4, 2, 32), (4, 4, 128), (32, 1, 64), (6, 2, 96), (3, 1, 160), (2, 2, 256), (8, 1, 224)])
@pytest.mark.parametrize("page", [16, 7])
def test_single_tokens(cuda_device, x, heads, kv_heads, dim, page):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 130, 513]
    check_attention(long.Case([1] * len(kv), kv, heads, kv_heads, dim, page, 1, x=x), cuda_device)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (4, 1, 128, 32), (3, 3, 128, 20), (2, 1, 32, 16), (4, 2, 96, 64), (4, 2, 192, 16)])
def test_chunks(cuda_device, x, heads, kv_heads, dim, page):
    """Whole prompts and chunks behind cached tokens, around the tiles' edges."""
    c = long.Case([128, 1, 129, 0, 31, 200, 257], [128, 77, 300, 50, 31, 263, 257], heads, kv_heads, dim, page, 2, x=x)
    check_attention(c, cuda_device)
    check_attention(c, cuda_device, window=70)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens", [[1] * 5, [3, 1, 2, 1, 4], [5] * 4, [9, 1, 33, 0, 2], [130]], ids=["single", "few", "equal", "ragged", "one"])
def test_over_many_runs(cuda_device, x, dim, tokens):
    lens = [2050, 777, 1300, 5, 1024][:len(tokens)]
    for window in (0, 600):
        check_attention(long.Case(tokens, lens, 8, 2, dim, 16, 12 + window, x=x), cuda_device, window=window)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("window", [1, 2, 16, 100, 129, 1000])
def test_windows(cuda_device, x, window):
    check_attention(long.Case([1, 150, 3, 40], [300, 290, 9, 40], 4, 2, 64, 16, 3, x=x), cuda_device, window=window)
    check_attention(long.Case([1, 4, 3], [300, 290, 9], 4, 2, 128, 16, 3, x=x), cuda_device, window=window)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(cuda_device, x, dim):
    """Empty sequences, more rows than positions, and rows over holes only."""
    for last in (70, 3):
        c = long.Case([0, 3, 5, 1, 2, last], [0, 0, 2, 33, 64, 140], 4, 2, dim, 16, 5, x=x)
        c.table[3, :] = -1               # no page at all
        c.table[4, 1] = c.k.shape[0]     # an entry past the pool
        c.table[5, 0:5] = -7
        out = check_attention(c, cuda_device)
        assert torch.all(out[0:3] == 0)
        check_attention(c, cuda_device, window=8)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("new,dim", [(1, 64), (150, 64), (3, 160)])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 70, 10 ** 9, -1, -2 ** 31])
def test_lengths_past_the_table(cuda_device, x, new, dim, length):
    c = long.Case([new], [48 + new], 4, 2, dim, 16, 17, x=x)
    c.table = np.ascontiguousarray(c.table[:, :3])
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    batch = paged.PagedBatch(batch.block_table, batch.q_start, torch.tensor([length], dtype=torch.int32, device=cuda_device), new, 48)
    lse = torch.empty((new, 4), device=cuda_device)
    before = [t.clone() for t in kv.pools]
    got = paged.attention(kv, batch, q, lse=lse)
    turned = paged.append(kv, batch, kn, vn, q=q, rope=paged.rope_table(48, dim, 1e4, cuda_device))
    assert bool(torch.isfinite(turned).all()) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv.pools, before))
    if length < 0:
        assert bool((got == 0).all()) and bool(torch.all(lse == -float("inf")))
    else:
        compare(c, got, lse, *ref.attention(c))
    assert bool((paged.attention(kv, batch, q, window=100) == 0).all())


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("stale", [np.nan, -65504.0])
def test_stale_slots_do_not_reach_a_row(cuda_device, x, dim, stale):
    """Unused slots of a page and spare pages hold NaN or the largest values."""
    check_attention(long.Case([1, 1, 40, 130], [5, 70, 91, 130], 4, 2, dim, 16, 6, x=x, stale=stale), cuda_device)
    check_attention(long.Case([1, 1, 2, 3], [5, 70, 91, 130], 4, 2, dim, 16, 6, x=x, stale=stale), cuda_device)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [3, 5, 150])
def test_later_tokens_do_not_reach_a_row(cuda_device, x, dim, new):
    """Blocks that are not finite at the chunk's later positions, and at positions that have left the window."""
    c = long.Case([new], [new + 60], 4, 2, dim, 16, 7, x=x)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    n, w = new + 60, 30
    clean = [paged.attention(kv, batch, q, window=y) for y in (0, w)]
    for p in (n - 2, 20):
        for t in (kv.pools[1], kv.pools[3]):
            t[int(c.table[0, p // 16]), :, p % 16, 0] = float("nan")
    full, windowed = (paged.attention(kv, batch, q, window=y) for y in (0, w))
    sees_20 = np.array([p < 20 + w for _, p in c.where()])
    late = np.array([p >= n - 2 for _, p in c.where()])
    ok = torch.from_numpy(~(late | sees_20)).to(cuda_device)
    assert bool((~torch.isfinite(full)).all())
    tol = 2.0 ** -9 if q.dtype == torch.float16 else 2.0 ** -17      # two evaluations of values below 6, other partial sums
    assert torch.all((windowed - clean[1]).abs()[ok] <= 6 * tol)
    assert bool((~torch.isfinite(windowed[~ok])).all())


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1), (16, 1), (24, 1)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (64, 32), (96, 16), (160, 16), (128, 20)])
@pytest.mark.parametrize("new", [1, 2, 3])
def test_what_has_left_the_window_does_not_reach_a_row(cuda_device, x, heads, kv_heads, dim, page, new):
    """Everything in front of the windows of a sequence's rows is not finite, up to the key before the first one's, for
    tiles of one token and of several, windows that begin at every place of a tile."""
    lens = [40, 47, 48, 49, 63, 300, 1111]
    c = long.Case([new] * len(lens), lens, heads, kv_heads, dim, page, 34, x=x)
    for window in (1, 15, 16, 30, 37):
        d = [t.copy() for t in c.pools]
        for b, n in enumerate(lens):
            for j in range(max(n - new - window + 1, 0)):
                for t in (d[1], d[3]):
                    t[c.page_of(b, j), :, j % page, :dim // 32] = np.nan
        held, c.pools = c.pools, d
        out = check_attention(c, cuda_device, window=window)
        assert bool(torch.isfinite(out).all())
        c.pools = held


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("order", ["head", "page"])
def test_strides(cuda_device, x, order):
    check_attention(long.Case([1, 9, 140], [33, 65, 200], 8, 2, 64, 16, 8, x=x), cuda_device, order=order, fused=True)
    check_attention(long.Case([1, 2, 1], [33, 65, 200], 8, 2, 128, 16, 8, x=x), cuda_device, order=order, fused=True)


def shifted(t):
    """The same values one element past an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    v = flat[1:].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("new", [1, 140])
def test_unaligned_rows(cuda_device, x, new):
    c = long.Case([new], [new + 100], 4, 2, 64, 16, 9, x=x)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    want = paged.attention(kv, batch, q).double()
    out = shifted(torch.zeros_like(q))
    paged.attention(kv, batch, shifted(q), out=out)
    assert torch.all((out.double() - want).abs() <= 6 * (2.0 ** -9 if q.dtype == torch.float16 else 2.0 ** -17))
    rope = paged.rope_table(256, 64, 1e4, cuda_device)
    turned = paged.append(kv, batch, kn, vn, q=q, rope=rope)
    held = [t.clone() for t in kv.pools]
    for t in kv.pools:
        t.zero_()
    again = paged.append(kv, batch, shifted(kn), shifted(vn), q=shifted(q), rope=rope, q_out=shifted(q))
    where = [(int(c.table[0, p // 16]), p % 16) for _, p in c.where()]
    assert torch.equal(again, turned) and all(torch.equal(a[g, :, s, :2], b[g, :, s, :2]) for a, b in zip(kv.pools, held) for g, s in where)


@pytest.mark.parametrize("x", X, ids=IDS)
def test_bounds_of_the_batch_do_not_change_results(cuda_device, x):
    """max_q_len and max_kv_len too small or far too large."""
    c = long.Case([1, 70, 5], [700, 170, 5], 8, 2, 64, 16, 10, x=x)
    for mq, mk in ((1, 1), (0, 0), (3, 100), (70, 700), (5000, 100000)):
        check_attention(c, cuda_device, batch_edit=lambda b: paged.PagedBatch(b.block_table, b.q_start, b.kv_len, mq, mk))


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("new", [2, 60])
def test_scales_of_the_scores(cuda_device, x, new):
    """Large scores, scales of zero and below, tiny ones, queries beyond the 16-bit range."""
    c = long.Case([1, new], [200, 130], 4, 2, 64, 16, 11, x=x, scale_q=30.0)
    for scale in (None, 0.01, 0.0, -0.02, 1e-30):
        check_attention(c, cuda_device, scale=scale)
    if x == np.float32:
        c.q *= np.float32(3e5)
        check_attention(c, cuda_device, scale=1e-6)


@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("new", [1, 3])
def test_scales_that_vanish(cuda_device, x, dim, new):
    """A scale of zero, or one that leaves nothing of a row's scores: every key weighs the same, of rows of zeros, of the
    smallest and of ordinary elements, over whole tiles and cut ones; rows that are not finite stay so."""
    c = long.Case([new] * 5, [32, 40, 75, 131, 500], 4, 2, dim, 16, 35, x=x)
    c.q[0], c.q[1, :2], c.q[-1, 1], c.q[2] = 0, 0, 0, np.finfo(x).tiny
    for scale in (0.0, 1e-45, 1e-38, 1e-30, -1e-30, 1e-8, None):
        check_attention(c, cuda_device, scale=scale)
        check_attention(c, cuda_device, scale=scale, window=21)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    q[0, 1, 5], q[-1, 2, 0] = float("nan"), float("inf")
    for scale in (0.0, 1e-30, None):
        got = paged.attention(kv, batch, q, scale=scale)
        nan = torch.isnan(got).all(-1)
        assert bool(nan[0, 1]) and bool(nan[-1, 2]) and int(nan.sum()) == 2 and bool(torch.isfinite(got[~nan]).all())


def test_wide_tables_take_several_rounds(cuda_device):
    """Prompts whose values do not fit the workspace together: 3 tables of 20,000 pages of 16."""
    c = long.Case([140, 170, 133], [200, 170, 333], 8, 8, 128, 16, 30, x=np.float16)
    wide = np.full((3, 20000), -1, np.int32)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    kv, batch, q, _, _ = on_device(c, cuda_device)
    import ctypes
    from hypno_b200._lib import load
    need = ctypes.c_size_t()
    assert load().hc_paged_attention_workspace(kv.ref, batch.pack(c.rows), 8, 1, 0, ctypes.byref(need)) == 0
    assert 20000 * 16 * 8 * 128 * 4 <= need.value <= 1.5 * 2 ** 30      # one sequence's values, no more
    check_attention(c, cuda_device)


def test_a_smaller_last_round(cuda_device):
    """Three sequences' values at a time, then the fourth's; the fourth's keys are cut into more runs."""
    c = long.Case([140, 170, 133, 100], [200, 170, 333, 1200], 2, 2, 128, 16, 32, x=np.float16)
    wide = np.full((4, 20000), -1, np.int32)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    check_attention(c, cuda_device, batch_edit=lambda b: paged.PagedBatch(b.block_table, b.q_start, b.kv_len, 170, 320000))


def test_rows_behind_the_last_sequence(cuda_device):
    """A padded batch: outputs, queries and pages of rows that belong to no sequence stay as they were."""
    for new in ([1, 2], [140, 30]):
        c = long.Case(new, [n + 60 for n in new], 4, 2, 128, 16, 33)
        kv, batch, q, kn, vn = on_device(c, cuda_device)
        q2, k2, v2 = (torch.cat([t, torch.full_like(t[:1], 9).repeat(5, 1, 1)]) for t in (q, kn, vn))
        out, turned = torch.full_like(q2, 3.0), torch.full_like(q2, 4.0)
        want = paged.attention(kv, batch, q)
        paged.attention(kv, batch, q2, out=out)
        assert torch.equal(out[:-5], want) and bool((out[-5:] == 3.0).all())
        rope = paged.rope_table(256, 128, 1e4, cuda_device)
        want = paged.append(kv, batch, kn, vn, q=q, rope=rope)
        held = kv.values()
        paged.append(kv, batch, k2, v2, q=q2, rope=rope, q_out=turned)
        assert torch.equal(turned[:-5], want) and bool((turned[-5:] == 4.0).all()) and all(torch.equal(a, b) for a, b in zip(kv.values(), held))


def test_large_pages(cuda_device):
    """Pages whose elements' eighths are more than a grid's second dimension takes, for a chunk and single tokens."""
    for new in (1, 60):
        check_attention(long.Case([new], [100], 8, 8, 128, 140000, 31, x=np.float16), cuda_device)


def test_long_cache_offsets(cuda_device):
    """Codes beyond 2^31 bytes of the pool."""
    dim, page, heads, dev = 128, 16, 8, cuda_device
    n_pages = (1 << 31) // (heads * page * dim // 2) + 700
    codes = torch.zeros((n_pages, heads, page, dim // 2), dtype=torch.uint8, device=dev)
    kv = paged.PagedKV4(codes, torch.zeros((n_pages, heads, page, 4), dtype=torch.float16, device=dev), codes.clone(),
                        torch.zeros((n_pages, heads, page, 4), dtype=torch.float16, device=dev))
    g = torch.Generator(device=dev).manual_seed(3)
    for new in (1, 130):
        n = 600 * page - 3
        kv.pools[0][-600:] = torch.randint(0, 256, (600, heads, page, dim // 2), generator=g, device=dev, dtype=torch.uint8)
        kv.pools[2][-600:] = torch.randint(0, 256, (600, heads, page, dim // 2), generator=g, device=dev, dtype=torch.uint8)
        for t in (kv.pools[1], kv.pools[3]):
            t[-600:] = (torch.randint(64, 128, (600, heads, page, 4), generator=g, device=dev) / 512).half()
        table = torch.arange(n_pages - 600, n_pages, dtype=torch.int32, device=dev)[None].contiguous()
        q = torch.randn((new, heads, dim), generator=g, device=dev).half()
        i32 = dict(dtype=torch.int32, device=dev)
        batch = paged.PagedBatch(table, torch.tensor([0, new], **i32), torch.tensor([n], **i32), new, n)
        out = paged.attention(kv, batch, q).double()

        def values(codes, scales):
            c = torch.stack((codes[-600:] & 15, codes[-600:] >> 4), -1).flatten(-2).double() - 8
            return (c.unflatten(-1, (4, 32)) * scales[-600:].double()[..., None]).flatten(-2).transpose(0, 1).reshape(heads, -1, dim)[:, :n]

        kk, vv = values(*kv.pools[:2]), values(*kv.pools[2:])
        s = torch.einsum("rhd,hnd->rhn", q.double(), kk) * dim ** -0.5
        i = torch.arange(n - new, n, device=dev)[:, None, None]
        s = s.masked_fill(torch.arange(n, device=dev) > i, -float("inf"))
        want = torch.einsum("rhn,hnd->rhd", s.softmax(-1), vv)
        assert torch.all((out - want).abs() <= 2.0 ** -10 * 2)      # values below 2


@pytest.mark.parametrize("x", X, ids=IDS)
def test_same_bits_on_other_streams_and_in_a_graph(cuda_device, x):
    """Append and attention in one graph, replayed with other contents of the same tensors."""
    for new in ([1, 1], [70, 200, 1], [3, 3, 3]):
        c, d = (long.Case(new, [n + 700 + i for n in new], 8, 2, 128, 16, 14 + i, x=x) for i in range(2))
        kv, batch, q, kn, vn = on_device(c, cuda_device)
        rope = paged.rope_table(1024, 128, 1e4, cuda_device)

        def step():
            return paged.attention(kv, batch, paged.append(kv, batch, kn, vn, q=q, rope=rope))

        first = step()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()) as _:
            assert torch.equal(step(), first)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for y in (d, c):
            for t, a in ((batch.block_table, y.table), (batch.kv_len, y.kv_len), (q, y.q), (kn, y.kn), (vn, y.vn), *zip(kv.pools, y.pools)):
                t.copy_(torch.from_numpy(a))
            g.replay()
            got = out.clone()
            assert torch.equal(got, step())
        assert torch.equal(got, first)


def test_another_device_than_the_current_one(cuda_device, monkeypatch):
    c = long.Case([1, 70], [900, 300], 8, 2, 128, 16, 13)
    kv, batch, q, kn, vn = on_device(c, cuda_device)

    def calls():
        return paged.append(kv, batch, kn, vn, q=q), paged.attention(kv, batch, q), *kv.values()

    want = calls()
    far = ref.Elsewhere(monkeypatch, paged)
    got = calls()
    assert far.device == 7
    assert {n for n, d in far.calls if d != 0} <= {"hc_paged_attention_workspace"}  # (host arithmetic)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("x", X, ids=IDS)
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dim,rot,page,order,fused", [(64, 64, 16, "head", False), (128, 64, 20, "page", True), (32, 32, 1, "head", True),
                                                      (96, 20, 7, "head", False), (128, 6, 3, "page", True), (128, 0, 16, "head", False),
                                                      (256, 256, 16, "head", True), (64, 24, 16, "head", False), (32, 2, 16, "head", False)])
def test_append(cuda_device, x, pairs, dim, rot, page, order, fused):
    c = long.Case([1, 0, 33, 2, 4], [1, 9, 40, 50, 2], 6, 2, dim, page, 20, x=x)
    c.table[3, 49 // page] = -1            # the last position of sequence 3 is a hole
    c.kn[3], c.vn[4, 1] = 0, 0
    c.kn[5] *= x(1e-6)
    c.vn[6] *= x(3e4)
    c.vn[7, 0, 3], c.kn[8, 1, dim - 1] = np.inf, np.nan
    kv, batch, q, kn, vn = on_device(c, cuda_device, order, fused)
    rope = paged.rope_table(64, rot, 10000.0, cuda_device) if rot else None
    before = [t.cpu().numpy() for t in kv.pools]
    out = paged.append(kv, batch, kn, vn, q=q, rope=rope, pairs=pairs)
    where = c.where()
    cs = np.zeros((c.rows, rot // 2, 2), np.float32)
    if rot:
        cs = rope.cpu().numpy()[np.maximum([p for _, p in where], 0)]
    with np.errstate(all="ignore"):
        # rotation in separately rounded steps, so equal to the last bit
        assert np.array_equal(out.cpu().numpy(), long.rotate32(c.q, cs, pairs).astype(x))
        kq, vq = long.quantize(long.rotate32(c.kn, cs, pairs)), long.quantize(c.vn)
    n = dim // 32
    for r, (b, p) in enumerate(where):
        pg = c.page_of(b, p)
        if pg >= 0:
            for i, (codes, scales, _) in enumerate((kq, vq)):
                before[2 * i][pg, :, p % page] = codes[r]
                before[2 * i + 1][pg, :, p % page, :n] = scales[r, :, :n]
    for t, want in zip(kv.pools, before):                              # everything else keeps its bits
        got = t.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want)) if got.dtype == np.float16 else True
        assert np.array_equal(np.nan_to_num(got), np.nan_to_num(want))
    for t, i in zip(kv.values(), (0, 2)):
        with np.errstate(invalid="ignore"):
            assert np.array_equal(t.cpu().numpy().astype(np.float64), long.decode(before[i], before[i + 1], dim), equal_nan=True)


@pytest.mark.parametrize("pairs,rot", [("adjacent", 64), ("halves", 64), ("halves", 40), ("halves", 16), ("halves", 6)])
def test_append_in_place_and_without_queries(cuda_device, pairs, rot):
    c = long.Case([3, 1], [30, 7], 4, 2, 64, 16, 21)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    rope = paged.rope_table(64, rot, 10000.0, cuda_device)
    want = paged.append(kv, batch, kn, vn, q=q, rope=rope, pairs=pairs)
    held = kv.values()
    pos = [(int(c.table[b, p // 16]), p % 16) for b, p in c.where()]
    for g, s in pos:
        kv.pools[0][g, :, s] = 0
    assert paged.append(kv, batch, kn, vn, rope=rope, pairs=pairs) is None
    assert paged.append(kv, batch, kn, vn, q=q, rope=rope, pairs=pairs, q_out=q) is q
    assert torch.equal(q, want)
    assert all(torch.equal(a[g, :, s], b[g, :, s]) for a, b in zip(kv.values(), held) for g, s in pos)


def test_a_value_is_off_by_half_a_step_at_most(cuda_device):
    """... of its block's scale, which is at most 1 + 2^-6 times a seventh of the largest magnitude."""
    c = long.Case([64], [64], 2, 2, 128, 16, 22)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    paged.append(kv, batch, kn, vn)
    got = np.stack([t.cpu().numpy()[c.table[0, np.arange(64) // 16], :, np.arange(64) % 16] for t in kv.values()]).astype(np.float64)
    want = np.stack([c.kn, c.vn]).astype(np.float64)
    top = np.abs(want).reshape(2, 64, 2, 4, 32).max(-1).repeat(32, -1).reshape(want.shape)
    assert np.all(np.abs(got - want) <= top / 14 * (1 + 2.0 ** -6) * (1 + 2.0 ** -22))


# ---------------------------------------------------------------- refusals

def test_refusals(cuda_device):
    dev = cuda_device
    c = long.Case([2, 1], [30, 7], 4, 2, 64, 16, 23)
    kv, batch, q, kn, vn = on_device(c, dev)
    kc, ks, vc, vs = kv.pools
    for bad, error in (((kc.int(), ks, vc, vs), TypeError), ((kc, ks.float(), vc, vs), TypeError), ((kc, ks[..., :1], vc, vs), ValueError),
                       ((kc[..., :24], ks, vc[..., :24], vs), ValueError), ((kc, ks, vc[1:], vs), ValueError), ((kc.cpu(), ks, vc, vs), TypeError),
                       ((kc[..., ::2], ks, vc[..., ::2], vs), ValueError)):
        with pytest.raises(error):
            paged.PagedKV4(*bad)
    odd = torch.zeros((kc.shape[0], 2, 16, 40), dtype=torch.uint8, device=dev)[..., 8:]      # strides of 40 bytes
    with pytest.raises(HypnoCudaError):
        paged.attention(paged.PagedKV4(odd, ks, vc, vs), batch, q)
    late = torch.zeros((kc.shape[0] * 2 * 16 * 2 + 1), dtype=torch.float16, device=dev)[1:].view(ks.shape)
    with pytest.raises(HypnoCudaError):
        paged.append(paged.PagedKV4(kc, late, vc, vs), batch, kn, vn)
    with pytest.raises(TypeError):
        paged.attention(kv, batch, q.double())
    with pytest.raises(ValueError):
        paged.attention(kv, batch, q[..., :32])
    with pytest.raises(HypnoCudaError):
        paged.append(kv, batch, kn, vn, rope=paged.rope_table(20, 64, 1e4, dev))      # 30 positions, a table of 20
    with pytest.raises(ValueError):
        paged.PagedKV4.alloc(2, 16, 2, 48, dev)


def test_empty_batches(cuda_device):
    kv = paged.PagedKV4.alloc(2, 16, 2, 64, device=cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    z = torch.zeros((0, 4, 64), device=cuda_device)
    empty = paged.PagedBatch(torch.zeros((0, 1), **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), 0, 0)
    idle = paged.PagedBatch(torch.zeros((2, 1), **i32), torch.zeros(3, **i32), torch.tensor([5, 0], **i32), 0, 5)
    for b in (empty, idle):
        assert paged.attention(kv, b, z).shape == (0, 4, 64)
        assert paged.append(kv, b, z[:, :2], z[:, :2], q=z).shape == (0, 4, 64)
    none = paged.PagedBatch(torch.zeros((1, 0), **i32), torch.tensor([0, 40], **i32), torch.tensor([50], **i32), 40, 50)   # a table without pages
    assert bool((paged.attention(kv, none, torch.ones((40, 4, 64), device=cuda_device)) == 0).all())
    assert all(bool((t == 0).all()) for t in kv.values())
