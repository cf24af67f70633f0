"""Bounds of pages, the selection by them, and attention over lists of pages,
against their definitions on the host, and what they refuse."""
import numpy as np
import pytest
import torch

from hypno_b200 import paged
from hypno_b200._lib import HypnoCudaError

from . import _long as long
from . import _paged as ref
from .test_gpu_paged4 import compare, in_order, shifted
from .test_gpu_paged4 import on_device as on_device4

pytestmark = pytest.mark.gpu

CACHES = ["f32", "f16", "q4"]


def case(cache, *a, x=np.float32, **more):
    return long.Case(*a, x=x, **more) if cache == "q4" else ref.Case(*a, x=x, cache=np.float32 if cache == "f32" else np.float16, **more)


def on_device(c, dev, order="head", fused=False):
    if isinstance(c, long.Case):
        return on_device4(c, dev, order, fused)
    kv = paged.PagedKV(*(in_order(torch.from_numpy(t).to(dev), order) for t in (c.k, c.v)))
    batch = paged.PagedBatch(torch.from_numpy(c.table).to(dev), torch.from_numpy(c.q_start).to(dev),
                             torch.from_numpy(c.kv_len).to(dev), max(c.new, default=0), max(max(c.kv, default=0), 0))
    q, kn, vn = (torch.from_numpy(y).to(dev) for y in (c.q, c.kn, c.vn))
    if fused:
        rows = torch.cat([q, kn, vn], 1)
        q, kn, vn = rows[:, :c.heads], rows[:, c.heads:c.heads + c.kv_heads], rows[:, c.heads + c.kv_heads:]
    return kv, batch, q, kn, vn


def some_pages(c, width, seed):
    """Ascending lists of up to `width` of the pages that each row sees, every other one with its own last page."""
    g = np.random.default_rng(seed)
    out = np.full((c.rows, c.kv_heads, width), -1, np.int32)
    for r, (b, p) in enumerate(c.where()):
        n = max(p, -1) // c.page + 1
        for h in range(c.kv_heads):
            take = g.permutation(n)[:min(n, int(g.integers(0, width + 1)))]
            if (r + h) % 2 and n:
                take = np.append(take[:width - 1], n - 1)
            take = np.unique(take)
            out[r, h, :take.size] = take
    return out


def check_lists(c, dev, lists, window=0, scale=None, order="head", fused=False):
    kv, batch, q, _, _ = on_device(c, dev, order, fused)
    lse = torch.full((c.rows, c.heads), float("nan"), device=dev)
    out = paged.attention(kv, batch, q, window=window, scale=scale, lse=lse, pages=torch.from_numpy(lists).to(dev))
    compare(c, out, lse, *long.attention(c, lists, window, scale))
    return out


# ---------------------------------------------------------------- attention over lists

@pytest.mark.parametrize("x", [np.float32, np.float16], ids=["qf32", "qf16"])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 1, 128), (4, 2, 32), (24, 2, 64), (40, 1, 64), (3, 1, 160), (2, 1, 256)])
@pytest.mark.parametrize("page,width", [(16, 5), (7, 40), (64, 3)])
def test_single_tokens(cuda_device, x, cache, heads, kv_heads, dim, page, width):
    kv = [1, 2, 16, 17, 64, 65, 130, 513, 700]
    c = case(cache, [1] * len(kv), kv, heads, kv_heads, dim, page, 1, x=x)
    check_lists(c, cuda_device, some_pages(c, width, 2))


@pytest.mark.parametrize("x", [np.float32, np.float16], ids=["qf32", "qf16"])
@pytest.mark.parametrize("dim", [1, 7, 72])
@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_odd_heads(cuda_device, x, cache, dim):
    c = case(cache, [1, 3, 9], [70, 80, 333], 6, 2, dim, 5, 3, x=x)
    check_lists(c, cuda_device, some_pages(c, 9, 4))
    check_lists(c, cuda_device, some_pages(c, 9, 4), window=20)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new", [[1, 4, 0, 7], [33, 1, 150, 2]])
def test_several_rows_a_sequence_and_windows(cuda_device, cache, new):
    c = case(cache, new, [400, 900, 30, 350], 8, 2, 64, 16, 5, x=np.float16)
    lists = some_pages(c, 20, 6)
    for window in (0, 1, 100):
        check_lists(c, cuda_device, lists, window=window, order="page", fused=True)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("lens", [[3000, 1700, 64], [9000]])
def test_long_lists(cuda_device, cache, lens):
    """Runs of keys over many CTAs."""
    c = case(cache, [1] * len(lens), lens, 8, 2, 128, 16, 7)
    check_lists(c, cuda_device, some_pages(c, 150, 8))
    check_lists(c, cuda_device, np.tile(np.arange(600, dtype=np.int32), (c.rows, 2, 1)))      # all, and more than there are


@pytest.mark.parametrize("cache", CACHES)
def test_lists_of_every_kind(cuda_device, cache):
    """Empty, ending early, out of order, the same page twice, past the row, the table or the pool, holes, rows without positions."""
    c = case(cache, [1] * 10 + [3], [200] * 10 + [1], 4, 2, 64, 16, 9)
    c.table[3, 2], c.table[4, 0:4] = -1, c.k.shape[0]
    top = 2 ** 31 - 1
    rows = [[-1, 3, 4, 5, 6], [0, 5, -1, 7, 8], [5, 3, 6, 7, 8], [0, 2, 4, 12, -1], [0, 1, 2, 3, -1], [7, 7, 8, 9, 9], [-5, 0, 1, 2, 3],
            [11, 12, 13, 400, top], [0, top, 1, 2, 3], [0, 1, 2, 12, 12], [-2 ** 31, 0, 0, 0, 0], [0, 1, 2, 3, 4], [0, -1, -1, -1, -1], [0, 0, 0, 0, 0]]
    lists = np.array([rows[r % len(rows)] for r in range(c.rows)], np.int32)[:, None].repeat(2, 1)
    lists[:, 1] = np.array([rows[(r + 3) % len(rows)] for r in range(c.rows)])
    out = check_lists(c, cuda_device, lists)
    assert bool((out[0, :2] == 0).all())
    check_lists(c, cuda_device, np.ascontiguousarray(lists[..., :1]))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("stale", [np.nan, -65504.0])
def test_what_is_not_listed_does_not_reach_a_row(cuda_device, cache, dim, stale):
    """Slots behind the row, spare pages and pages that no list names hold NaN or the lowest values."""
    c = case(cache, [1, 2, 5], [75, 163, 330], 8, 2, dim, 16, 10, stale=stale)
    lists = some_pages(c, 6, 11)
    lists[np.isin(lists, [2])] = 1                       # nothing names page 2 (a list may end there)
    for b in range(3):
        g = c.table[b, 2]
        if isinstance(c, long.Case):
            c.pools[1][g], c.pools[3][g] = np.nan, np.nan
        c.k[g], c.v[g] = np.nan, np.nan
    out = check_lists(c, cuda_device, lists)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("cache", CACHES)
def test_lists_in_views_and_many_rows(cuda_device, cache):
    """Lists inside a wider tensor, heads in another order, unaligned queries, and rows enough for a CTA each."""
    c = case(cache, [1] * 300, [40 + 3 * i for i in range(300)], 4, 4, 64, 16, 12, x=np.float16)
    lists = some_pages(c, 7, 13)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    t = torch.from_numpy(lists).to(cuda_device)
    lse = torch.empty((300, 4), device=cuda_device)
    want = paged.attention(kv, batch, q, lse=lse, pages=t)
    compare(c, want, lse, *long.attention(c, lists))
    wide = torch.full((4, 300, 11), 3, dtype=torch.int32, device=cuda_device)
    wide[:, :, 2:9] = t.transpose(0, 1)
    assert torch.equal(paged.attention(kv, batch, q, pages=wide.transpose(0, 1)[:, :, 2:9]), want)
    out = shifted(torch.zeros_like(q))
    paged.attention(kv, batch, shifted(q), out=out, pages=t)
    assert torch.equal(out, want)


# ---------------------------------------------------------------- bounds

@pytest.mark.parametrize("cache,dim", [("f32", 64), ("f16", 128), ("q4", 128), ("f16", 4), ("f32", 12), ("f16", 72), ("q4", 32), ("q4", 256), ("f32", 256)])
@pytest.mark.parametrize("page", [16, 1, 7, 128])
@pytest.mark.parametrize("order", ["head", "page"])
def test_bounds(cuda_device, cache, dim, page, order):
    """Of the pages with new rows alone, over their filled slots alone."""
    c = case(cache, [1, 0, 33, 2, 1, 5, 3], [1, 9, 40, 50, 16, 2, 0], 2, 2, dim, page, 20, stale=np.nan)
    c.table[3, 48 // page] = -1
    kv, batch, _, _, _ = on_device(c, cuda_device, order)
    b = paged.PageBounds.alloc(kv)
    b.lo.fill_(5), b.hi.fill_(6), b.scale.fill_(7)
    want = [t.cpu().numpy() for t in (b.lo, b.hi, b.scale)]
    paged.update_bounds(b, kv, batch)
    for g, filled in long.touched(c):
        want[0][g], want[1][g], want[2][g] = long.bounds(c.k[g], filled)
    for t, w in zip((b.lo, b.hi, b.scale), want):
        assert np.array_equal(t.cpu().numpy(), w)
    lo, hi = b.values()
    assert np.array_equal(lo.cpu().numpy(), want[0].astype(np.float32) * want[2][..., None]) and np.array_equal(hi.cpu().numpy(), want[1] * want[2][..., None])


def test_bounds_hold_the_keys(cuda_device):
    """Every magnitude: subnormal, the type's largest, one of 127 / 64 steps, zeros, and keys that are not finite."""
    page, dim = 16, 8
    top = [0.0, 1e-45, 1e-38, 2.0 ** -121, 1.0, 127.0 / 64, np.nextafter(np.float32(127 / 64), np.float32(2)), 126.5, 127.0, 127.5, 3.4e38, np.inf, np.nan]
    k = np.random.default_rng(1).uniform(-1, 1, (len(top), 1, page, dim)).astype(np.float32)
    for i, t in enumerate(top):
        k[i] *= np.float32(t) if np.isfinite(t) else 1
        k[i, 0, 3, 5] = -t
    kv = paged.PagedKV(*(torch.from_numpy(k).to(cuda_device) for _ in range(2)))
    n = len(top)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    batch = paged.PagedBatch(torch.arange(n, **i32)[None].contiguous(), torch.tensor([0, n * page], **i32), torch.tensor([n * page], **i32), n * page, n * page)
    b = paged.PageBounds.alloc(kv)
    paged.update_bounds(b, kv, batch)
    lo, hi, s = (t.cpu().numpy() for t in (b.lo, b.hi, b.scale))
    for i in range(n):
        want = long.bounds(k[i], page)
        assert all(np.array_equal(a[i], w) for a, w in zip((lo, hi, s), want)), top[i]
        if np.isfinite(top[i]):
            u = s[i].astype(np.float64)[:, None]
            assert np.all(lo[i] * u <= k[i].min(1)) and np.all(hi[i] * u >= k[i].max(1)) and np.abs(k[i]).max() <= 127 * u.max()
            assert abs(int(lo[i].min())) <= 127


# ---------------------------------------------------------------- selection

def all_bounds(c):
    n = c.k.shape[0]
    out = [np.zeros((n, c.kv_heads, c.dim), np.int8), np.zeros((n, c.kv_heads, c.dim), np.int8), np.zeros((n, c.kv_heads), np.float32)]
    for g in range(n):
        out[0][g], out[1][g], out[2][g] = long.bounds(c.k[g], c.page)
    return out


def check_select(c, dev, b, budget, first=1, recent=2, fused=False):
    kv, batch, q, _, _ = on_device(c, dev, fused=fused)
    h = paged.PageBounds(*(torch.from_numpy(t).to(dev) for t in b), page_size=c.page)
    got = paged.select_pages(h, batch, q, budget, first, recent)
    assert got.dtype == torch.int32
    want = long.select(c, *b, budget, first, recent)
    assert np.array_equal(got.cpu().numpy(), want)
    return got


@pytest.mark.parametrize("x", [np.float32, np.float16], ids=["qf32", "qf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 1, 128), (4, 2, 32), (40, 1, 16), (6, 2, 72), (2, 1, 256), (4, 2, 12), (18, 2, 64)])
def test_select(cuda_device, x, heads, kv_heads, dim):
    c = case("f32", [1, 4, 1, 0, 9, 1], [700, 333, 16, 9, 80, 1], heads, kv_heads, dim, 16, 30, x=x)
    b = all_bounds(c)
    for budget, first, recent in ((8, 1, 2), (3, 1, 2), (1, 0, 0), (20, 0, 20), (43, 4, 4), (44, 1, 1), (200, 1, 2)):
        check_select(c, cuda_device, b, budget, first, recent, fused=budget % 2 == 0)


@pytest.mark.parametrize("page,length", [(1, 9000), (7, 2999), (16, 40000)])
def test_select_among_many(cuda_device, page, length):
    c = case("f16", [1, 2], [length, length // 2], 4, 2, 16, page, 31)
    b = all_bounds(c)
    for budget in (5, 257, 1000):
        check_select(c, cuda_device, b, budget)


def test_select_ties_and_odd_values(cuda_device):
    """Equal scores go by index; queries of zero, not finite or of any magnitude; pages of infinite bounds, holes."""
    c = case("f32", [1] * 8, [640] * 8, 2, 1, 16, 16, 32)
    b = all_bounds(c)
    same = [t.copy() for t in b]
    for t in same:
        t[:] = t[:1]
    check_select(c, cuda_device, same, 7)
    c.q[0], c.q[1, 0], c.q[2, 1, 3], c.q[3] = 0, np.nan, np.inf, np.inf
    c.q[4] *= np.float32(1e-38)
    c.q[5] *= np.float32(1e37)
    c.q[6] = -0.0
    b[2][c.table[0, 5]], b[2][c.table[4, 9]] = np.inf, np.inf
    c.table[2, 7], c.table[3, 0], c.table[4, 39], c.table[5, 10:38] = -1, -1, c.k.shape[0], -3
    for budget in (3, 9, 39):
        check_select(c, cuda_device, b, budget)
    for s in (1e-30, 2.0 ** -119, 1e30):
        d = [b[0], b[1], (np.abs(b[2]) > 0) * 2.0 ** np.round(np.log2(s))]
        d[2] = d[2].astype(np.float32)
        c.q[5] = np.clip(c.q[5], -1e30, 1e30)
        check_select(c, cuda_device, d, 9)


def test_select_with_a_wide_table_and_many_rows(cuda_device):
    """Tables whose keys do not fit one CTA's memory, and more rows than a grid's third dimension takes: the form in two kernels."""
    c = case("f32", [1, 3], [700, 333], 4, 2, 16, 16, 34)
    b = all_bounds(c)
    want = long.select(c, *b, 9)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    h = paged.PageBounds(*(torch.from_numpy(t).to(cuda_device) for t in b), page_size=16)
    wide = torch.full((2, 60000), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :c.table.shape[1]] = torch.from_numpy(c.table).to(cuda_device)
    other = paged.PagedBatch(wide, batch.q_start, batch.kv_len, 3, 700)
    assert np.array_equal(paged.select_pages(h, other, q, 9).cpu().numpy(), want)
    n = 70000
    i32 = dict(dtype=torch.int32, device=cuda_device)
    many = paged.PagedBatch(batch.block_table[:1].repeat(n, 1), torch.arange(n + 1, **i32), torch.full((n,), 700, **i32), 1, 700)
    got = paged.select_pages(h, many, q[:1].expand(n, -1, -1), 9)
    assert torch.equal(got, torch.from_numpy(want[:1]).to(cuda_device).expand(n, -1, -1))


@pytest.mark.parametrize("dim", [16, 12])      # in one kernel, in two
@pytest.mark.parametrize("x", [np.float32, np.float16], ids=["qf32", "qf16"])
@pytest.mark.parametrize("infinite", [1, 10, 37, 40])
@pytest.mark.parametrize("holes", [0, 1, 25])
def test_select_with_more_infinite_pages_than_places(cuda_device, dim, x, infinite, holes):
    """Beside finite pages, one or many, and holes; nothing behind the lists is written."""
    c = case("f32", [1, 2], [640, 635], 4, 2, dim, 16, 37, x=x)
    b = all_bounds(c)
    g = np.random.default_rng(infinite + holes)
    for s in range(2):
        at = g.permutation(40)
        b[2][c.table[s, at[:infinite]]] = np.inf
        c.table[s, at[max(40 - holes, 1):]] = -1
    kv, batch, q, _, _ = on_device(c, cuda_device)
    h = paged.PageBounds(*(torch.from_numpy(t).to(cuda_device) for t in b), page_size=16)
    for budget, first, recent in ((6, 1, 2), (3, 0, 0), (16, 1, 2), (39, 1, 1), (4, 2, 2)):
        room = torch.full((3 * 2 * budget + 256,), 77, dtype=torch.int32, device=cuda_device)
        out = room[:3 * 2 * budget].view(3, 2, budget)
        paged.select_pages(h, batch, q, budget, first, recent, out=out)
        assert np.array_equal(out.cpu().numpy(), long.select(c, *b, budget, first, recent))
        assert bool((room[3 * 2 * budget:] == 77).all())


def test_select_of_many_heads(cuda_device):
    """A group of 130 query heads."""
    c = case("f32", [2], [400], 130, 1, 256, 16, 35)
    check_select(c, cuda_device, all_bounds(c), 9)


def test_bounds_after_a_call_with_fewer_rows(cuda_device):
    """update_bounds goes by the row starts, whatever other calls with the batch have read."""
    c = case("f16", [1, 1, 33], [20, 40, 60], 4, 2, 64, 16, 36)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    b = paged.PageBounds.alloc(kv)
    paged.select_pages(b, batch, q[:2], 4)
    paged.update_bounds(b, kv, batch)
    want = [torch.zeros_like(t).cpu().numpy() for t in (b.lo, b.hi, b.scale)]
    for g, filled in long.touched(c):
        want[0][g], want[1][g], want[2][g] = long.bounds(c.k[g], filled)
    assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip((b.lo, b.hi, b.scale), want))


def test_rows_of_no_sequence_keep_their_lists(cuda_device):
    c = case("f32", [2, 1], [300, 200], 4, 2, 64, 16, 33)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    h = paged.PageBounds(*(torch.from_numpy(t).to(cuda_device) for t in all_bounds(c)), page_size=16)
    more = torch.cat([q, q])
    out = torch.full((6, 2, 5), 77, dtype=torch.int32, device=cuda_device)
    got = paged.select_pages(h, batch, more, 5, out=out)
    assert got is out and torch.equal(out[:3], paged.select_pages(h, batch, q, 5)) and bool((out[3:] == 77).all())
    res = torch.full_like(more, 3.0)
    paged.attention(kv, batch, more, out=res, pages=out)
    assert bool((res[3:] == 3.0).all()) and torch.equal(res[:3], paged.attention(kv, batch, q, pages=out[:3]))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new", [[1, 1, 2], [1, 70, 200]])
def test_a_part_of_a_steps_sequences(cuda_device, cache, new):
    """A batch whose rows begin behind others and end before others: the ones that belong to no sequence keep what they
    had, store nothing, and the rest is as without them."""
    c = case(cache, new, [n + 300 for n in new], 8, 2, 64, 16, 50)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    rope = paged.rope_table(512, 64, 1e4, cuda_device)
    b = paged.PageBounds(*(torch.from_numpy(t).to(cuda_device) for t in all_bounds(c)), page_size=16)
    pools = list(kv.pools) if cache == "q4" else [kv.k, kv.v]
    held = [t.clone() for t in pools]

    def step(batch, q, kn, vn, outs):
        for t, was in zip(pools, held):
            t.copy_(was)
        paged.append(kv, batch, kn, vn, q=q, rope=rope, q_out=outs[0])
        paged.update_bounds(b, kv, batch)
        paged.select_pages(b, batch, outs[0], 9, out=outs[1])
        paged.attention(kv, batch, outs[0], out=outs[2], lse=outs[3])
        paged.attention(kv, batch, outs[0], out=outs[4], pages=outs[1])
        return [t.clone() for t in (*pools, b.lo, b.hi, b.scale)]

    def empty(n):
        return [torch.full((n, 8, 64), 5.0, device=cuda_device), torch.full((n, 2, 9), 5, dtype=torch.int32, device=cuda_device),
                torch.full((n, 8, 64), 5.0, device=cuda_device), torch.full((n, 8), 5.0, device=cuda_device), torch.full((n, 8, 64), 5.0, device=cuda_device)]

    want = empty(c.rows)
    state = step(batch, q, kn, vn, want)
    wide = [torch.cat([torch.full_like(t[:1], 9).repeat(7, 1, 1), t, torch.full_like(t[:1], 9).repeat(4, 1, 1)]) for t in (q, kn, vn)]
    got = empty(c.rows + 11)
    part = paged.PagedBatch(batch.block_table, batch.q_start + 7, batch.kv_len, batch.max_q_len, batch.max_kv_len)
    again = step(part, *wide, got)
    for a, w in zip(got, want):
        assert torch.equal(a[7:-4], w) and bool((a[:7] == 5).all()) and bool((a[-4:] == 5).all())
    assert all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(again, state))


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("cache", CACHES)
def test_many_sequences(cuda_device, cache):
    """More than the 32 whose places are worked out together."""
    n = 75
    c = case(cache, [1 + (i % 7 == 3) for i in range(n)], [2 + (131 * i) % 900 for i in range(n)], 8, 2, 64, 16, 46)
    check_lists(c, cuda_device, some_pages(c, 11, 47))
    kv, batch, q, _, _ = on_device(c, cuda_device)
    lse = torch.empty((c.rows, 8), device=cuda_device)
    out = paged.attention(kv, batch, q, lse=lse)
    compare(c, out, lse, *ref.attention(c))
    b = all_bounds(c)
    check_select(c, cuda_device, b, 5)


@pytest.mark.parametrize("cache", CACHES)
def test_calls_on_two_streams_at_once(cuda_device, cache):
    c = case(cache, [1, 2], [3000, 1700], 8, 2, 128, 16, 48)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    pages = torch.from_numpy(some_pages(c, 90, 49)).to(cuda_device)
    want = paged.attention(kv, batch, q, pages=pages), paged.attention(kv, batch, q)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((paged.attention(kv, batch, q, pages=pages), paged.attention(kv, batch, q)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))



@pytest.mark.parametrize("cache", CACHES)
def test_a_captured_step(cuda_device, cache):
    """Append, bounds, selection and attention in one graph, replayed with other contents of the same tensors and on
    another stream; two such graphs, replayed in turn, do not disturb one another."""
    new = [1, 1, 3]
    cs = [case(cache, new, [n + 700 + i for n in new], 8, 2, 64, 16, 40 + i) for i in range(2)]
    sides = []
    for c in cs:
        kv, batch, q, kn, vn = on_device(c, cuda_device)
        b = paged.PageBounds(*(torch.from_numpy(t).to(cuda_device) for t in all_bounds(c)), page_size=16)
        rope = paged.rope_table(1024, 64, 1e4, cuda_device)

        def step(kv=kv, batch=batch, q=q, kn=kn, vn=vn, b=b, rope=rope):
            turned = paged.append(kv, batch, kn, vn, q=q, rope=rope)
            paged.update_bounds(b, kv, batch)
            pages = paged.select_pages(b, batch, turned, 9)
            return paged.attention(kv, batch, turned, pages=pages), pages

        first = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        sides.append((g, out, first, step, (kv, batch, q, kn, vn)))
    for g, out, first, step, _ in sides + sides[::-1]:
        for t in out:
            t.zero_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, first))
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        again = sides[0][3]()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, sides[0][2]))
    # other queries and lengths in the tensors of the first
    g, out, _, step, (kv, batch, q, kn, vn) = sides[0]
    q.copy_(torch.from_numpy(cs[1].q)), kn.copy_(torch.from_numpy(cs[1].kn)), batch.kv_len.sub_(5)
    g.replay()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("cache", CACHES)
def test_a_budget_for_all_pages_is_dense_attention(cuda_device, cache):
    c = case(cache, [1, 2], [500, 333], 8, 2, 64, 16, 42)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    b = paged.PageBounds.alloc(kv)
    pages = paged.select_pages(b, batch, q, 40)
    tol = 6 * 2.0 ** -17      # two evaluations of values below 6, other partial sums
    assert bool(((paged.attention(kv, batch, q, pages=pages) - paged.attention(kv, batch, q)).abs() <= tol).all())


def test_the_selected_pages_hold_the_heaviest_keys(cuda_device):
    """Keys that carry most of the weight: their pages are chosen, and the sparse result is near the dense one."""
    c = case("f16", [1], [4096], 4, 2, 64, 16, 43)
    heavy = [17, 100, 201]
    for h in range(2):
        for p in heavy:
            c.k[c.table[0, p], h, 3] = (c.q[0, 2 * h] * 1.5).astype(np.float16)
            c.k[c.table[0, p], h, 4] = (c.q[0, 2 * h + 1] * 1.5).astype(np.float16)
    got = check_select(c, cuda_device, all_bounds(c), 12)
    assert all(bool((got == p).any(-1).all()) for p in heavy)
    kv, batch, q, _, _ = on_device(c, cuda_device)
    dense, want = paged.attention(kv, batch, q), ref.attention(c)[0]
    # what is left out weighs less than 4096 e^(largest light score - heavy score); here both are known
    s = np.einsum("gd,nd->gn", c.q[0, :2].astype(np.float64), c.k[c.table[0, :256], 0].reshape(-1, 64).astype(np.float64)) / 8
    w = np.exp(s - s.max(1, keepdims=True))
    kept = np.isin(np.arange(4096) // 16, got.cpu().numpy()[0, 0])
    left_out = (w * ~kept).sum(1) / w.sum(1)
    sparse = paged.attention(kv, batch, q, pages=got)
    room = 2 * left_out.max() * np.abs(c.v.astype(np.float64)).max() + 1e-5
    assert np.all(np.abs(sparse[0, :2].cpu().numpy() - want[0, :2]) <= room) and np.all(np.abs(dense[0, :2].cpu().numpy() - want[0, :2]) <= 1e-5)


def test_another_device_than_the_current_one(cuda_device, monkeypatch):
    c = case("q4", [1, 2], [900, 300], 8, 2, 128, 16, 44)
    kv, batch, q, kn, vn = on_device(c, cuda_device)
    b = paged.PageBounds.alloc(kv)

    def calls():
        paged.update_bounds(b, kv, batch)
        pages = paged.select_pages(b, batch, q, 9)
        return pages, paged.attention(kv, batch, q, pages=pages), *b.values()

    want = calls()
    far = ref.Elsewhere(monkeypatch, paged)
    got = calls()
    assert far.device == 7
    assert {n for n, d in far.calls if d != 0} <= {"hc_paged_list_attention_workspace", "hc_page_select_workspace"}  # (host arithmetic)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- refusals

def test_refusals(cuda_device):
    dev = cuda_device
    c = case("f16", [2, 1], [30, 7], 4, 2, 64, 16, 45)
    kv, batch, q, _, _ = on_device(c, dev)
    b = paged.PageBounds.alloc(kv)
    pages = torch.zeros((3, 2, 4), dtype=torch.int32, device=dev)
    for bad, error in ((pages.long(), TypeError), (pages[0], TypeError), (pages.cpu(), TypeError), (pages[:2], ValueError), (pages[:, :1], ValueError),
                       (pages[..., :0], ValueError), (pages[..., ::2], ValueError)):
        with pytest.raises(error):
            paged.attention(kv, batch, q, pages=bad)
    with pytest.raises(HypnoCudaError):
        paged.attention(kv, batch, q[:, :3], pages=pages)
    with pytest.raises(HypnoCudaError):
        paged.attention(kv, batch, q, window=-1, pages=pages)
    for args, error in (((0,), ValueError), ((2,), HypnoCudaError), ((5, 3, 3), HypnoCudaError), ((5, -1, 2), HypnoCudaError), ((5, 1, -2), HypnoCudaError)):
        with pytest.raises(error):
            paged.select_pages(b, batch, q, *args)
    with pytest.raises(TypeError):
        paged.select_pages(b, batch, q.double(), 5)
    with pytest.raises(ValueError):
        paged.select_pages(b, batch, q[..., :32], 5)
    with pytest.raises(TypeError):
        paged.select_pages(b, batch, q, 5, out=pages)
    with pytest.raises(HypnoCudaError):
        paged.select_pages(b, batch, q[:, :3], 5)
    for bad, error in (((b.lo.int(), b.hi, b.scale, 16), TypeError), ((b.lo, b.hi[1:], b.scale, 16), ValueError), ((b.lo, b.hi, b.scale[:, :1], 16), ValueError),
                       ((b.lo.transpose(0, 1), b.hi.transpose(0, 1), b.scale, 16), ValueError), ((b.lo, b.hi.cpu(), b.scale, 16), TypeError)):
        with pytest.raises(error):
            paged.PageBounds(*bad)
    with pytest.raises(HypnoCudaError):
        paged.update_bounds(paged.PageBounds(b.lo, b.hi, b.scale, 32), kv, batch)      # bounds of other pages
    odd = paged.PagedKV.alloc(2, 16, 2, 66, device=dev)
    with pytest.raises(HypnoCudaError) as e:
        paged.update_bounds(paged.PageBounds.alloc(odd), odd, batch)
    assert e.value.code == -3


def test_empty_batches(cuda_device):
    kv = paged.PagedKV.alloc(2, 16, 2, 64, device=cuda_device)
    b = paged.PageBounds.alloc(kv)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    z = torch.zeros((0, 4, 64), device=cuda_device)
    empty = paged.PagedBatch(torch.zeros((0, 1), **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), 0, 0)
    idle = paged.PagedBatch(torch.zeros((2, 1), **i32), torch.zeros(3, **i32), torch.tensor([5, 0], **i32), 0, 5)
    for batch in (empty, idle):
        paged.update_bounds(b, kv, batch)
        pages = paged.select_pages(b, batch, z, 4)
        assert pages.shape == (0, 2, 4) and paged.attention(kv, batch, z, pages=pages).shape == (0, 4, 64)
    none = paged.PagedBatch(torch.zeros((1, 0), **i32), torch.tensor([0, 2], **i32), torch.tensor([50], **i32), 2, 50)   # a table without pages
    q = torch.ones((2, 4, 64), device=cuda_device)
    paged.update_bounds(b, kv, none)
    pages = paged.select_pages(b, none, q, 4)
    assert bool((pages == -1).all()) and bool((paged.attention(kv, none, q, pages=pages) == 0).all())
