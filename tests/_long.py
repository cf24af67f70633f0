"""Plain forms of the 4-bit cache, the pages' bounds, their selection and the
attention over lists of pages on the host, for their tests."""
import numpy as np

from . import _paged as ref


def slots(dim):
    return 2 if dim <= 64 else 4 if dim <= 128 else 8


def quantize(x):
    """Codes, scales and values of float32 [..., dim], by the definition in float32 (every step of it is rounded alike everywhere)."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        top = np.max(np.abs(g), axis=-1)
        t = (top / np.float32(7)).astype(np.float32)
        up = ((t.view(np.uint32) + np.uint32(0x1FFFF)) & np.uint32(0xFFFE0000)).view(np.float32)
        s = np.minimum(np.ceil(up.astype(np.float64) * 2.0 ** 24) * 2.0 ** -24, 896.0).astype(np.float32)
        s = np.where(np.isfinite(top), s, np.float32("nan"))
        c = np.rint(g / np.where(s > 0, s, 1)[..., None]).clip(-7, 7)
    c = np.where((s > 0)[..., None], c, 0)
    codes = (c + 8).astype(np.uint8).reshape(*x.shape)
    scales = np.zeros((*x.shape[:-1], slots(x.shape[-1])), np.float16)
    scales[..., :s.shape[-1]] = s
    assert np.array_equal(scales[..., :s.shape[-1]].astype(np.float32), s, equal_nan=True)     # a scale is a float16
    values = (c * s[..., None]).astype(np.float32).reshape(x.shape)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales, values


def decode(codes, scales, dim):
    c = np.empty((*codes.shape[:-1], dim))
    c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
    return (c - 8) * np.repeat(scales.astype(np.float64)[..., :dim // 32], 32, -1)


class Case(ref.Case):
    """ref.Case with a cache in 4 bits: k and v are what its pools stand for.  Slots past head_dim / 32 of the scales hold NaN."""

    def __init__(self, *a, x=np.float32, stale=None, **more):
        super().__init__(*a, x=x, cache=np.float32, stale=stale, **more)
        self.pools, held = [], []
        for t in (self.k, self.v):
            codes, scales, values = quantize(t)
            scales[..., t.shape[-1] // 32:] = np.nan
            self.pools += [codes, scales]
            with np.errstate(invalid="ignore"):
                held.append(values.astype(np.float16))
            assert np.array_equal(held[-1].astype(np.float32), values, equal_nan=True)       # values are exact as float16
        self.k, self.v = held


def rotate32(x, cs, pairs):
    """Rotation in float32, each product and sum rounded by itself."""
    y = x.astype(np.float32).copy()
    half = cs.shape[1]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    i = np.arange(half) * 2 if pairs == "adjacent" else np.arange(half)
    j = i + 1 if pairs == "adjacent" else i + half
    a, b = x[..., i].astype(np.float32), x[..., j].astype(np.float32)
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def listed(entries):
    """The pages that a list names: it ends before the first entry that is not above the one in front of it."""
    out, last = [], -1
    for e in entries:
        if e <= last:
            break
        out.append(int(e))
        last = e
    return out


def attention(c, lists, window=0, scale=None):
    """ref.attention over the listed pages of each row and KV head."""
    scale = c.dim ** -0.5 if scale is None else scale
    G = c.heads // c.kv_heads
    out = np.zeros((c.rows, c.heads, c.dim))
    lse = np.full((c.rows, c.heads), -np.inf)
    A, M = np.zeros((c.rows, c.heads, 1)), np.zeros((c.rows, c.heads, 1))
    for r, (b, p) in enumerate(c.where()):
        for kh in range(c.kv_heads):
            js = [j for e in listed(lists[r, kh]) if e < c.table.shape[1] for j in range(e * c.page, min((e + 1) * c.page, p + 1))
                  if c.page_of(b, j) >= 0 and (not window or j > p - window)]
            if not js:
                continue
            pg, sl = [c.page_of(b, j) for j in js], [j % c.page for j in js]
            k, v = c.k[pg, kh, sl].astype(np.float64), c.v[pg, kh, sl].astype(np.float64)
            for h in range(kh * G, kh * G + G):
                q = c.q[r, h].astype(np.float64)
                s = k @ q * scale
                e = np.exp(s - s.max())
                out[r, h] = e @ v / e.sum()
                lse[r, h] = s.max() + np.log(e.sum())
                A[r, h] = np.max(np.abs(k) @ np.abs(q)) * abs(scale)
                M[r, h] = np.max(np.abs(v))
    return out, lse, A, M


def unit(top):
    """The least power of two, from 2^-120 on, of which top is at most 127."""
    if not np.isfinite(top):
        return np.inf
    e = -120
    while float(top) > 127.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def bounds(k, filled):
    """lo, hi, scale of the keys [kv_heads, page, dim] of a page."""
    k = k[:, :filled].astype(np.float64)
    lo, hi, s = np.zeros((k.shape[0], k.shape[2]), np.int8), np.zeros((k.shape[0], k.shape[2]), np.int8), np.zeros(k.shape[0], np.float32)
    for h in range(k.shape[0]):
        s[h] = unit(np.max(np.abs(k[h])))
        if np.isfinite(s[h]):
            lo[h], hi[h] = np.floor(k[h].min(0) / float(s[h])), np.ceil(k[h].max(0) / float(s[h]))
    return lo, hi, s


def touched(c):
    """(page, filled slots) of the pages that hold a new row."""
    for b, (t, n) in enumerate(zip(c.new, c.kv)):
        for i in range(max(n - t, 0) // c.page, -(-n // c.page) if t and n > 0 else 0):
            g = c.page_of(b, i * c.page)
            if g >= 0:
                yield g, min(c.page, n - i * c.page)


def select(c, lo, hi, scale, budget, first=1, recent=2):
    out = np.full((c.rows, c.kv_heads, budget), -1, np.int32)
    G = c.heads // c.kv_heads
    for r, (b, p) in enumerate(c.where()):
        n = min(p // c.page + 1, c.table.shape[1]) if p >= 0 else 0
        for kh in range(c.kv_heads):
            if n <= budget:
                out[r, kh, :n] = np.arange(n)
                continue
            codes, t = [], []
            for h in range(kh * G, kh * G + G):
                q = c.q[r, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    u = unit(np.max(np.abs(q)))
                t.append(u if np.isfinite(u) else 0.0)
                codes.append(np.rint(q / u).astype(np.int64) if np.isfinite(u) else np.zeros(c.dim, np.int64))
            score = []
            for i in range(n):
                g = c.page_of(b, i * c.page)
                if g < 0:
                    score.append(-np.inf)
                elif not np.isfinite(scale[g, kh]):
                    score.append(np.inf)
                else:
                    l, u = lo[g, kh].astype(np.int64), hi[g, kh].astype(np.int64)
                    score.append(max(float(np.maximum(q * l, q * u).sum()) * x for q, x in zip(codes, t)) * float(scale[g, kh]))
            forced = [i < first or i >= n - recent for i in range(n)]
            order = sorted(range(n), key=lambda i: (not forced[i], -score[i], i))
            out[r, kh] = sorted(order[:budget])
    return out
