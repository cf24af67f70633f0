"""Paged append and attention (hc_paged_append_dev, hc_paged_attention_dev)
against their plain forms in 64 bits on the host: types, head layouts, page
sizes and lengths around every boundary, rows that see nothing, holes,
whatever lies in masked places, strides, streams, and what they refuse."""
import numpy as np
import pytest
import torch

from hypno_b200 import paged
from hypno_b200._lib import HypnoCudaError, call

from . import _paged as ref

pytestmark = pytest.mark.gpu

TYPES = [(np.float32, np.float16), (np.float16, np.float16), (np.float32, np.float32), (np.float16, np.float32)]
IDS = ["f32-f16", "f16-f16", "f32-f32", "f16-f32"]


def on_device(c, dev, order="head", fused=False):
    k, v = torch.from_numpy(c.k).to(dev), torch.from_numpy(c.v).to(dev)
    if order == "page":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    kv = paged.PagedKV(k, v)
    batch = paged.PagedBatch(torch.from_numpy(c.table).to(dev), torch.from_numpy(c.q_start).to(dev),
                             torch.from_numpy(c.kv_len).to(dev), max(c.new, default=0), max(max(c.kv, default=0), 0))
    q, kn, vn = (torch.from_numpy(x).to(dev) for x in (c.q, c.kn, c.vn))
    if fused:  # heads side by side, as a fused projection writes them
        rows = torch.cat([q, kn, vn], 1)
        q, kn, vn = rows[:, :c.heads], rows[:, c.heads:c.heads + c.kv_heads], rows[:, c.heads + c.kv_heads:]
    return kv, batch, q, kn, vn


def check_attention(c, dev, window=0, scale=None, order="head", fused=False, batch_edit=None):
    kv, batch, q, _, _ = on_device(c, dev, order, fused)
    if batch_edit:
        batch = batch_edit(batch)
    lse = torch.full((c.rows, c.heads), float("nan"), device=dev)
    out = paged.attention(kv, batch, q, window=window, scale=scale, lse=lse)
    want, want_lse, A, M = ref.attention(c, window, scale)
    tol = ref.tolerance(c, A, M, c.q.dtype == np.float16)
    got = out.cpu().numpy().astype(np.float64)
    assert got.shape == want.shape and out.dtype == q.dtype
    err = np.abs(got - want)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], float(np.nanmax(err)), float(tol.max()), int(bad.sum()), bad.size)
    got_lse = lse.cpu().numpy().astype(np.float64)
    seen = np.isfinite(want_lse)
    assert np.array_equal(seen, np.isfinite(got_lse)) and np.all(got_lse[~seen] == -np.inf)
    # the log of the sum: the scores' error, and f32 rounding of the sum and of the result
    room = A[..., 0] * 2.0 ** -20 + 2.0 ** -19 + np.abs(np.where(seen, want_lse, 0)) * 2.0 ** -22
    assert np.all(np.abs(got_lse[seen] - want_lse[seen]) <= room[seen])
    return out


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 1, 128), (4, 2, 16), (4, 4, 128), (32, 1, 64), (6, 2, 80)])
@pytest.mark.parametrize("page", [16, 7])
def test_single_tokens(cuda_device, types, heads, kv_heads, dim, page):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 130, 513]
    check_attention(ref.Case([1] * len(kv), kv, heads, kv_heads, dim, page, 1, *types), cuda_device)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (4, 1, 128, 32), (3, 3, 128, 20), (2, 1, 16, 16), (4, 2, 96, 64)])
def test_chunks(cuda_device, types, heads, kv_heads, dim, page):
    """Whole prompts and chunks behind cached tokens, around the tiles' edges."""
    c = ref.Case([128, 1, 129, 0, 31, 200, 257], [128, 77, 300, 50, 31, 263, 257], heads, kv_heads, dim, page, 2, *types)
    check_attention(c, cuda_device)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("window", [1, 2, 16, 100, 129, 1000])
def test_windows(cuda_device, types, window):
    check_attention(ref.Case([1, 150, 3, 40], [300, 290, 9, 40], 4, 2, 64, 16, 3, *types), cuda_device, window=window)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [1, 3, 8, 72, 160, 256])
def test_odd_head_sizes(cuda_device, types, dim):
    check_attention(ref.Case([1, 37], [40, 101], 4, 2, dim, 5, 4, *types), cuda_device)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("dim", [136, 192, 256])
@pytest.mark.parametrize("window", [0, 333])
def test_large_heads_over_many_runs(cuda_device, types, dim, window):
    check_attention(ref.Case([1, 3, 1, 20], [1500, 903, 0, 700], 6, 2, dim, 16, 11, *types), cuda_device, window=window)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 16), (128, 20)])
@pytest.mark.parametrize("tokens", [[5] * 4, [9, 1, 33, 0, 2], [130]], ids=["equal", "ragged", "one"])
def test_short_chunks_over_many_runs(cuda_device, types, dim, page, tokens):
    """Chunks whose row tiles are fewer than the SMs: the keys are cut into runs."""
    lens = [2050, 777, 1300, 5, 1024][:len(tokens)]
    check_attention(ref.Case(tokens, lens, 8, 2, dim, page, 12, *types), cuda_device)
    check_attention(ref.Case(tokens, lens, 8, 2, dim, page, 13, *types), cuda_device, window=600)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
def test_many_chunks_of_unlike_lengths(cuda_device, types):
    """More row tiles than SMs, of sequences whose lengths span every order of magnitude."""
    new = [1, 70, 0, 33, 5, 129, 64, 2, 90, 200] * 2
    kv = [n + (37 * i * i) % 900 * (i % 5 > 0) for i, n in enumerate(new)]
    kv[2], kv[12] = 0, 1200
    check_attention(ref.Case(new, kv, 16, 8, 64, 16, 14, *types), cuda_device)
    check_attention(ref.Case(new, kv, 16, 8, 64, 16, 15, *types), cuda_device, window=100)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_rows_that_see_nothing(cuda_device, types):
    """Empty sequences, more rows than positions, and rows over holes only."""
    c = ref.Case([0, 3, 5, 1, 2, 70], [0, 0, 2, 33, 64, 140], 4, 2, 64, 16, 5, *types)
    c.table[3, :] = -1               # no page at all
    c.table[4, 1] = c.k.shape[0]     # an entry past the pool
    c.table[5, 0:5] = -7
    out = check_attention(c, cuda_device)
    assert torch.all(out[0:3] == 0)
    check_attention(c, cuda_device, window=8)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("new,dim", [(1, 64), (150, 64), (1, 7), (40, 7), (3, 160)])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 70, 10 ** 9, -1, -2 ** 31])
def test_lengths_past_the_table(cuda_device, types, new, dim, length):
    """Positions past the table are holes however many the length names: such rows
    see all of the table's, stores go nowhere; a negative length sees nothing."""
    c = ref.Case([new], [48 + new], 4, 2, dim, 16, 17, *types)
    c.table = np.ascontiguousarray(c.table[:, :3])
    want, want_lse, A, M = ref.attention(c)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    batch = paged.PagedBatch(batch.block_table, batch.q_start, torch.tensor([length], dtype=torch.int32, device=cuda_device), new, 48)
    lse = torch.empty((new, 4), device=cuda_device)
    before = kv.k.clone(), kv.v.clone()
    got = paged.attention(kv, batch, q, lse=lse).cpu().numpy().astype(np.float64)
    turned = paged.append(kv, batch, kn, vn, q=q, rope=paged.rope_table(48, dim // 2 * 2, 1e4, cuda_device))
    assert bool(torch.isfinite(turned).all()) and torch.equal(kv.k, before[0]) and torch.equal(kv.v, before[1])
    if length < 0:
        assert np.all(got == 0) and bool(torch.all(lse == -float("inf")))
        return
    assert np.all(np.abs(got - want) <= ref.tolerance(c, A, M, types[0] == np.float16))
    room = A[..., 0] * 2.0 ** -20 + 2.0 ** -19 + np.abs(want_lse) * 2.0 ** -22
    assert np.all(np.abs(lse.cpu().numpy() - want_lse) <= room)
    # a window that reaches back from there leaves nothing, the widest one everything where there is something
    assert bool((paged.attention(kv, batch, q, window=100) == 0).all())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("new,dim", [(5, 64), (150, 64), (40, 7)])
def test_the_widest_window_with_more_rows_than_positions(cuda_device, types, new, dim):
    check_attention(ref.Case([new], [new - 4], 4, 2, dim, 16, 18, *types), cuda_device, window=2 ** 31 - 1)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("stale", [np.nan, np.inf, -65504.0])
def test_stale_slots_do_not_reach_a_row(cuda_device, types, stale):
    """Unused slots of a page and spare pages hold NaN, infinities or the lowest value."""
    c = ref.Case([1, 1, 40, 130], [5, 70, 91, 130], 4, 2, 64, 16, 6, *types, stale=stale)
    check_attention(c, cuda_device)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("new", [5, 150])
def test_later_tokens_do_not_reach_a_row(cuda_device, types, bad, new):
    """Keys and values that are not finite at the chunk's later positions, and at
    positions that have left the window: rows that do not see them are right, a
    row that sees such a value is not finite itself."""
    c = ref.Case([new], [new + 60], 4, 2, 64, 16, 7, *types)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    n, w = new + 60, 30
    clean = [paged.attention(kv, batch, q, window=x) for x in (0, w)]
    for p in (n - 2, 20):
        for t in (kv.k, kv.v):
            t[int(c.table[0, p // 16]), :, p % 16] = bad
    full, windowed = (paged.attention(kv, batch, q, window=x) for x in (0, w))
    sees_20 = np.array([p < 20 + w for _, p in c.where()])
    late = np.array([p >= n - 2 for _, p in c.where()])
    ok = torch.from_numpy(~(late | sees_20)).to(cuda_device)
    assert bool((~torch.isfinite(full)).all())                      # every row sees position 20
    tol = 2.0 ** -9 if q.dtype == torch.float16 else 2.0 ** -17      # two evaluations of values below 6, other partial sums
    assert torch.all((windowed - clean[1]).abs()[ok] <= 6 * tol)
    assert bool((~torch.isfinite(windowed[~ok])).all())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("new,heads,kv_heads,page,window,at", [(65, 4, 2, 16, 30, 50), (65, 4, 2, 20, 30, 50), (65, 4, 2, 16, 30, 94), (2, 128, 1, 16, 0, 61),
                                                              (3, 128, 1, 20, 0, 62), (3, 128, 1, 20, 0, 61),
                                                              (2, 128, 1, 16, 5, 56)])
def test_a_lone_token_does_not_see_its_neighbours_keys(cuda_device, types, bad, new, heads, kv_heads, page, window, at):
    """128 packed rows of which the last, or all, are one token's: a key or value
    that is not finite and that only the other rows see does not reach it."""
    c = ref.Case([new], [new + 60], heads, kv_heads, 64, page, 16, *types)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    clean = paged.attention(kv, batch, q, window=window)
    for t in (kv.k, kv.v):
        t[int(c.table[0, at // page]), :, at % page] = bad
    got = paged.attention(kv, batch, q, window=window)
    sees = torch.tensor([at <= p and (not window or at > p - window) for _, p in c.where()], device=cuda_device)
    assert 0 < int(sees.sum()) < new
    tol = 2.0 ** -9 if q.dtype == torch.float16 else 2.0 ** -17      # as above
    assert bool(((got - clean).abs()[~sees] <= 6 * tol).all())
    assert bool((~torch.isfinite(got[sees])).all())


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("order", ["head", "page"])
def test_strides(cuda_device, types, order):
    c = ref.Case([1, 9, 140], [33, 65, 200], 8, 2, 64, 16, 8, *types)
    check_attention(c, cuda_device, order=order, fused=True)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("new", [1, 140])
def test_unaligned_rows_and_pools(cuda_device, types, new):
    """Pools, queries and outputs that start one element past an aligned address."""
    c = ref.Case([new], [new + 100], 4, 2, 64, 16, 9, *types)
    kv, batch, q, _, _ = on_device(c, cuda_device)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v

    want = paged.attention(kv, batch, q).double()
    tol = 6 * (2.0 ** -9 if q.dtype == torch.float16 else 2.0 ** -17)
    kv2 = paged.PagedKV(shifted(kv.k), shifted(kv.v))
    assert torch.all((paged.attention(kv2, batch, q).double() - want).abs() <= tol)
    out = shifted(torch.zeros_like(q))
    paged.attention(kv, batch, shifted(q), out=out)
    assert torch.all((out.double() - want).abs() <= tol)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
def test_bounds_of_the_batch_do_not_change_results(cuda_device, types):
    """max_q_len and max_kv_len too small or far too large."""
    c = ref.Case([1, 70, 5], [700, 170, 5], 8, 2, 64, 16, 10, *types)
    for mq, mk in ((1, 1), (0, 0), (3, 100), (70, 700), (5000, 100000)):
        check_attention(c, cuda_device, batch_edit=lambda b: paged.PagedBatch(b.block_table, b.q_start, b.kv_len, mq, mk))


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
def test_wide_scores(cuda_device, types):
    """Large scores (one key takes all), a scale of its own, queries beyond the 16-bit range."""
    c = ref.Case([1, 60], [200, 130], 4, 2, 64, 16, 11, *types, scale_q=30.0)
    check_attention(c, cuda_device)
    check_attention(c, cuda_device, scale=0.01)
    if types[0] == np.float32:
        c.q *= np.float32(3e5)
        check_attention(c, cuda_device, scale=1e-6)
        c.q *= np.float32(1e-14)
        check_attention(c, cuda_device, scale=1e8)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("scale", [1e-8, 1e-30, 1e-45])
def test_tiny_scales_and_queries_of_zero(cuda_device, types, new, scale):
    """Scores of (nearly) 0 behind a mask: every visible key weighs the same."""
    c = ref.Case([new], [new + 20], 4, 2, 64, 16, 19, *types)
    c.q[::2] = 0
    check_attention(c, cuda_device, scale=scale)
    check_attention(c, cuda_device, scale=scale, window=9)


def test_long_cache_offsets(cuda_device):
    """Pages whose elements lie beyond 2^31 of the pool, and many splits."""
    dim, page, heads = 128, 16, 8
    n_pages = (1 << 31) // (heads * page * dim) + 700
    k = torch.zeros((n_pages, heads, page, dim), dtype=torch.float16, device=cuda_device)
    v = torch.zeros_like(k)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    for new in (1, 130):
        n = 600 * page - 3
        table = torch.arange(n_pages - 600, n_pages, dtype=torch.int32, device=cuda_device)[None].contiguous()
        k[-600:] = torch.randn((600, heads, page, dim), generator=g, device=cuda_device).half()
        v[-600:] = torch.randn((600, heads, page, dim), generator=g, device=cuda_device).half()
        q = torch.randn((new, heads, dim), generator=g, device=cuda_device).half()
        i32 = dict(dtype=torch.int32, device=cuda_device)
        batch = paged.PagedBatch(table, torch.tensor([0, new], **i32), torch.tensor([n], **i32), new, n)
        out = paged.attention(paged.PagedKV(k, v), batch, q).double()
        kk = k[-600:].transpose(0, 1).reshape(heads, -1, dim)[:, :n].double()
        vv = v[-600:].transpose(0, 1).reshape(heads, -1, dim)[:, :n].double()
        s = torch.einsum("rhd,hnd->rhn", q.double(), kk) * dim ** -0.5
        i = torch.arange(n - new, n, device=cuda_device)[:, None, None]
        s = s.masked_fill(torch.arange(n, device=cuda_device) > i, -float("inf"))
        want = torch.einsum("rhn,hnd->rhd", s.softmax(-1), vv)
        assert torch.all((out - want).abs() <= 2.0 ** -10 * 6)


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
def test_same_inputs_same_bits_and_other_streams(cuda_device, types):
    c = ref.Case([1, 1, 90], [4000, 300, 1500], 8, 2, 128, 16, 12, *types)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    a = paged.attention(kv, batch, q)
    torch.cuda.synchronize()
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            b = paged.attention(kv, batch, q)
        s.synchronize()
        assert torch.equal(a, b)


def test_graph_capture(cuda_device):
    c = ref.Case([1, 1], [900, 300], 8, 2, 128, 16, 13)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    want = paged.attention(kv, batch, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    out = torch.zeros_like(want)
    with torch.cuda.graph(g):
        paged.attention(kv, batch, q, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_another_device_than_the_current_one(cuda_device, monkeypatch):
    c = ref.Case([1, 70], [900, 300], 8, 2, 128, 16, 13)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    want = paged.append(kv, batch, kn, vn, q=q), paged.attention(kv, batch, q)
    far = ref.Elsewhere(monkeypatch, paged)
    got = paged.append(kv, batch, kn, vn, q=q), paged.attention(kv, batch, q)
    assert far.device == 7                                # as it was
    assert {n for n, d in far.calls if d == 0} >= {"hc_paged_append_dev", "hc_paged_attention_dev"}
    assert {n for n, d in far.calls if d != 0} <= {"hc_paged_attention_workspace"}  # (host arithmetic)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("types", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("new", [[1, 1], [70, 200, 1], [9, 9, 9]])
def test_a_captured_step(cuda_device, types, new):
    """Append and attention in one graph, replayed with other rows, lengths and pages in the same tensors."""
    c, d = (ref.Case(new, [n + 700 + i for n in new], 8, 2, 64, 16, 14 + i, *types) for i in range(2))
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    rope = paged.rope_table(1024, 64, 1e4, cuda_device)

    def step():
        return paged.attention(kv, batch, paged.append(kv, batch, kn, vn, q=q, rope=rope))

    first = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for x in (d, c):
        for t, a in ((kv.k, x.k), (kv.v, x.v), (batch.block_table, x.table), (batch.kv_len, x.kv_len), (q, x.q), (kn, x.kn), (vn, x.vn)):
            t.copy_(torch.from_numpy(a))
        g.replay()
        got = out.clone()
        assert torch.equal(got, step())
    assert torch.equal(got, first)


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dim,rot,page,order,fused", [(64, 64, 16, "head", False), (128, 64, 20, "page", True), (16, 16, 1, "head", True),
                                                      (80, 20, 7, "head", False), (9, 6, 3, "page", True), (128, 0, 16, "head", False)])
def test_append(cuda_device, types, pairs, dim, rot, page, order, fused):
    c = ref.Case([1, 0, 33, 2, 4], [1, 9, 40, 50, 2], 6, 2, dim, page, 20, *types)
    c.table[3, 49 // page] = -1            # the last position of sequence 3 is a hole
    kv, batch, q, kn, vn = on_device(c, cuda_device, order, fused)
    rope = paged.rope_table(64, rot, 10000.0, cuda_device) if rot else None
    before = [t.cpu().numpy() for t in (kv.k, kv.v)]
    out = paged.append(kv, batch, kn, vn, q=q, rope=rope, pairs=pairs)
    torch.cuda.synchronize()
    where = c.where()
    cs = np.zeros((c.rows, rot // 2, 2), np.float32)
    if rot:
        cs = rope.cpu().numpy()[np.maximum([p for _, p in where], 0)]
    qr, kr = ref.rotate(c.q, cs, pairs), ref.rotate(c.kn, cs, pairs)
    # two products and their difference in f32, then the rounding of the result
    f32 = 2.0 ** -22
    reach_q, reach_k = (np.max(np.abs(x.astype(np.float64))) * 2 for x in (c.q, c.kn))
    ux = 2.0 ** -11 if types[0] == np.float16 else 2.0 ** -24
    uc = 2.0 ** -11 if types[1] == np.float16 else 2.0 ** -24
    assert np.all(np.abs(out.cpu().numpy() - qr) <= reach_q * f32 + np.abs(qr) * ux + 2.0 ** -24)
    want_k, want_v = before[0].astype(np.float64), before[1].copy()
    room = np.zeros(want_k.shape)
    for r, (b, p) in enumerate(where):
        pg = c.page_of(b, p)
        if pg >= 0:
            want_k[pg, :, p % page] = kr[r]
            room[pg, :, p % page] = reach_k * f32 + np.abs(kr[r]) * uc + 2.0 ** -24
            want_v[pg, :, p % page] = c.vn[r].astype(types[1])
    assert np.all(np.abs(kv.k.cpu().numpy() - want_k) <= room)      # everything else keeps its bits
    assert np.array_equal(kv.v.cpu().numpy(), want_v)


def test_append_in_place_and_without_queries(cuda_device):
    c = ref.Case([3, 1], [30, 7], 4, 2, 64, 16, 21)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    rope = paged.rope_table(64, 64, 10000.0, cuda_device)
    want = paged.append(kv, batch, kn, vn, q=q, rope=rope)
    k = kv.k.clone()
    kv.k.zero_()
    assert paged.append(kv, batch, kn, vn, rope=rope) is None
    assert paged.append(kv, batch, kn, vn, q=q, rope=rope, q_out=q) is q
    assert torch.equal(q, want)
    pos = [(int(c.table[b, p // 16]), p % 16) for b, p in c.where()]
    assert all(torch.equal(kv.k[g, :, s], k[g, :, s]) for g, s in pos)


def test_rope_table_is_the_models(cuda_device):
    """The table rotates as hc_rope does (one head, several positions)."""
    from hypno_b200 import ops
    c = ref.Case([1], [38], 1, 1, 64, 16, 22, np.float32, np.float32)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    out = paged.append(kv, batch, kn, vn, q=q, rope=paged.rope_table(40, 64, 10000.0, cuda_device))
    a, b = c.q[0, 0].copy(), c.kn[0, 0].copy()
    ops.rope(a, b, 64, 37, 10000.0)
    assert np.allclose(out.cpu().numpy()[0, 0], a, rtol=0, atol=2.0 ** -21 * np.abs(c.q).max())
    assert np.allclose(kv.k[int(c.table[0, 2]), 0, 37 % 16].cpu().numpy(), b, rtol=0, atol=2.0 ** -21 * np.abs(c.kn).max())


# ---------------------------------------------------------------- refusals

def test_refusals(cuda_device):
    c = ref.Case([2, 1], [30, 7], 4, 2, 64, 16, 23)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    rope = paged.rope_table(64, 64, 10000.0, cuda_device)
    with pytest.raises(TypeError):
        paged.attention(kv, batch, q.double())
    with pytest.raises(ValueError):
        paged.attention(kv, batch, q[..., :32])
    with pytest.raises(ValueError):
        paged.attention(kv, batch, q.transpose(1, 2).contiguous().transpose(1, 2)[..., ::1][:, :, torch.arange(63, -1, -1)].flip(2)[..., ::2])
    with pytest.raises(HypnoCudaError):
        paged.attention(kv, batch, q[:, :3])                      # 3 query heads over 2 KV heads
    with pytest.raises(HypnoCudaError):
        paged.attention(kv, batch, q, window=-1)
    with pytest.raises(TypeError):
        paged.attention(kv, batch, q, lse=torch.zeros(3, device=cuda_device))
    with pytest.raises(HypnoCudaError):
        paged.append(kv, batch, kn, vn, rope=rope[:20].contiguous())  # 30 positions, a table of 20
    with pytest.raises(ValueError):
        paged.append(kv, batch, kn[:1], vn)
    with pytest.raises(ValueError):
        paged.append(kv, batch, kn, vn, pairs="both")
    with pytest.raises(TypeError):
        paged.append(kv, batch, kn, vn.half())
    with pytest.raises(HypnoCudaError):
        paged.append(kv, batch, kn, vn, rope=paged.rope_table(64, 66, 1e4, cuda_device))  # 66 of 64 elements
    with pytest.raises(TypeError):
        paged.PagedKV(kv.k.double(), kv.v.double())
    with pytest.raises(ValueError):
        paged.PagedKV(kv.k, kv.v[1:])
    with pytest.raises(TypeError):
        paged.PagedBatch(batch.block_table.long(), batch.q_start, batch.kv_len, 2, 30)
    with pytest.raises(ValueError):
        paged.PagedBatch(batch.block_table, batch.q_start[1:], batch.kv_len, 2, 30)
    big = paged.PagedKV.alloc(2, 16, 1, 264, device=cuda_device)
    with pytest.raises(HypnoCudaError) as e:
        paged.attention(big, batch, torch.zeros((3, 1, 264), dtype=torch.float16, device=cuda_device))
    assert e.value.code == -3


def test_refusals_at_the_c_entry(cuda_device):
    from hypno_b200._lib import HC_ROWS, load
    c = ref.Case([2, 1], [30, 7], 4, 2, 64, 16, 24)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    r, none = HC_ROWS.pack(q.data_ptr(), 256, 64), HC_ROWS.pack(0, 0, 0)
    lib = load()
    ref_b = batch.pack(3)
    assert lib.hc_paged_attention_dev(None, ref_b, r, r, None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_attention_dev(kv.ref, None, r, r, None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_attention_dev(kv.ref, ref_b, none, r, None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_attention_dev(kv.ref, ref_b, r, none, None, 4, 0, 0.1, 0, None, 0, None) == -1
    assert lib.hc_paged_attention_dev(kv.ref, ref_b, r, r, None, 4, 2, 0.1, 0, None, 0, None) == -3
    assert lib.hc_paged_append_dev(kv.ref, ref_b, none, r, None, None, 0, 0, None, 0, 0, 0, None) == -1
    assert lib.hc_paged_append_dev(kv.ref, ref_b, r, None, None, None, 0, 0, None, 0, 0, 0, None) == -1
    assert lib.hc_paged_append_dev(kv.ref, ref_b, r, r, r, None, 4, 0, None, 0, 0, 0, None) == -1
    assert lib.hc_paged_attention_workspace(kv.ref, ref_b, 4, 0, 0, None) == -1
    kv.struct.page_size = 0
    assert lib.hc_paged_attention_dev(kv.ref, ref_b, r, r, None, 4, 0, 0.1, 0, None, 0, None) == -1
    kv.struct.page_size, kv.struct.k_pos_stride = 16, -64
    assert lib.hc_paged_attention_dev(kv.ref, ref_b, r, r, None, 4, 0, 0.1, 0, None, 0, None) == -1


def test_empty_batches(cuda_device):
    kv = paged.PagedKV.alloc(2, 16, 2, 64, device=cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    empty = paged.PagedBatch(torch.zeros((0, 1), **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), 0, 0)
    z = torch.zeros((0, 4, 64), device=cuda_device)
    assert paged.attention(kv, empty, z).shape == (0, 4, 64)
    assert paged.append(kv, empty, z[:, :2], z[:, :2], q=z).shape == (0, 4, 64)
    idle = paged.PagedBatch(torch.zeros((2, 1), **i32), torch.zeros(3, **i32), torch.tensor([5, 0], **i32), 0, 5)
    assert paged.attention(kv, idle, z).shape == (0, 4, 64)
