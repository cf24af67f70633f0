"""Plain 64-bit forms of the paged operators on the host, for their tests."""
import numpy as np


class Case:
    """A paged cache and one step's batch, as numpy arrays.  new / kv: rows and
    positions of each sequence; spare pages and slots past a sequence's end
    hold `stale` (None: noise)."""

    def __init__(self, new, kv, heads, kv_heads, dim, page, seed=0, x=np.float32, cache=np.float16, stale=None, scale_q=1.5):
        g = np.random.default_rng(seed)
        self.new, self.kv = list(new), list(kv)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        used = [-(-max(n, 0) // page) for n in self.kv]
        n_pages = sum(used) + 2
        shape = (n_pages, kv_heads, page, dim)
        if stale is None:
            self.k, self.v = (g.standard_normal(shape).astype(cache) for _ in range(2))
        else:
            self.k, self.v = (np.full(shape, stale, cache) for _ in range(2))
        self.table = np.full((len(self.kv), max(max(used, default=0), 1) + 1), -1, np.int32)
        free = g.permutation(n_pages)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = free[at:at + u]
            at += u
            for p in range(max(self.kv[b], 0)):
                pg, s = self.table[b, p // page], p % page
                self.k[pg, :, s] = g.standard_normal((kv_heads, dim)).astype(cache)
                self.v[pg, :, s] = g.standard_normal((kv_heads, dim)).astype(cache)
        self.rows = sum(self.new)
        self.q = (g.standard_normal((self.rows, heads, dim)) * scale_q).astype(x)
        self.kn = g.standard_normal((self.rows, kv_heads, dim)).astype(x)
        self.vn = g.standard_normal((self.rows, kv_heads, dim)).astype(x)
        self.q_start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.kv_len = np.array(self.kv, np.int32)

    def where(self):
        """(sequence, position) of every row."""
        return [(b, self.kv[b] - t + i) for b, t in enumerate(self.new) for i in range(t)]

    def page_of(self, b, p):
        """Page of a position, -1 for a hole."""
        if p < 0 or p // self.page >= self.table.shape[1]:
            return -1
        g = int(self.table[b, p // self.page])
        return g if 0 <= g < self.k.shape[0] else -1


def attention(c, window=0, scale=None):
    """(out, lse, reach) in 64 bits: reach[r, h] bounds the scores' magnitudes
    (sum |q| |k| scale) and the values', for the tolerance."""
    scale = c.dim ** -0.5 if scale is None else scale
    G = c.heads // c.kv_heads
    out = np.zeros((c.rows, c.heads, c.dim))
    lse = np.full((c.rows, c.heads), -np.inf)
    A, M = np.zeros((c.rows, c.heads, 1)), np.zeros((c.rows, c.heads, 1))
    for r, (b, p) in enumerate(c.where()):
        js = [j for j in range(max(0, p - window + 1) if window else 0, p + 1) if c.page_of(b, j) >= 0]
        if not js:
            continue
        pg, sl = [c.page_of(b, j) for j in js], [j % c.page for j in js]
        for h in range(c.heads):
            k, v = c.k[pg, h // G, sl].astype(np.float64), c.v[pg, h // G, sl].astype(np.float64)
            q = c.q[r, h].astype(np.float64)
            s = k @ q * scale
            m = s.max()
            e = np.exp(s - m)
            out[r, h] = e @ v / e.sum()
            lse[r, h] = m + np.log(e.sum())
            A[r, h] = np.max(np.abs(k) @ np.abs(q)) * abs(scale)
            M[r, h] = np.max(np.abs(v))
    return out, lse, A, M


def tolerance(c, A, M, half_out):
    """Bound of the kernels' error.  A score's relative error is at most 2^-20
    of sum |q| |k| (f32 products and sums of up to 256 terms, operands split to
    22 bits), so a weight's is at most 2 A 2^-20, and exp, the sums and the
    division add at most 2^-19; a 16-bit result adds the rounding of the
    weights and of the result, 2^-11 each.  All of it times max |v|."""
    return M * (2 * A * 2.0 ** -20 + 2.0 ** -19 + (2.0 ** -10 if half_out else 0.0))


def rotate(x, cs, pairs):
    """Rotation of [rows, heads, dim] by cs [rows, rot / 2, 2], in 64 bits."""
    y = x.astype(np.float64).copy()
    half = cs.shape[1]
    c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    i = np.arange(half) * 2 if pairs == "adjacent" else np.arange(half)
    j = i + 1 if pairs == "adjacent" else i + half
    a, b = x[..., i].astype(np.float64), x[..., j].astype(np.float64)
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def sample(l, u, T, k, p, least):
    """One row of sample() from its definition with exact integer masses:
    (token, share of the kept mass)."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float32)
    if not (l > -np.inf).any():
        return -1, 0.0
    order = np.argsort(-l, kind="stable")
    ranked = l[order]
    inv = np.float32(1.0) / np.float32(T) if T > 0 else np.float32(1.0)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(ranked == ranked[0], 1.0, np.exp(((ranked - ranked[0]) * inv).astype(np.float64)))
    mass = (w * 2.0 ** 40).astype(np.int64)
    n = 1 if not T > 0 or not p > 0 or not least <= 1 else (k if 0 < k < l.size else l.size)
    keep = np.arange(l.size) < n
    if p < 1:
        held = np.where(keep, mass, 0)
        before = np.cumsum(held) - held
        keep &= before.astype(np.float64) < np.float64(np.float32(p)) * np.float64(held.sum())
    keep &= w.astype(np.float32) >= np.float32(least)
    keep[0] = True
    held = np.zeros(l.size, np.int64)
    held[order[keep]] = mass[keep]
    total = int(held.sum())
    goal = min(int(np.floor(np.float64(np.float32(u)) * np.float64(total))), total - 1)
    t = int(np.argmax(np.cumsum(held) > goal))
    return t, held[t] / total, held, total


class Elsewhere:
    """Stands in for a process whose current CUDA device is another than the
    tensors': the package's view of the current device, and of every call into
    the library the device it was made on (the real one stays device 0)."""

    def __init__(self, monkeypatch, *modules):
        from hypno_b200 import _lib
        self.device, self.calls, lib = 7, [], _lib.load()
        monkeypatch.setattr(_lib, "current_device", lambda: self.device)
        monkeypatch.setattr(_lib, "_set_device", lambda i: setattr(self, "device", i))

        def of(name):
            def run(*args):
                self.calls.append((name, self.device))
                return getattr(lib, name)(*args)
            return run

        library = type("Library", (), {"__getattr__": lambda _, name: of(name)})()
        for m in (_lib, *modules):
            monkeypatch.setattr(m, "load", lambda: library)
