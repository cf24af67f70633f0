"""Measured cases of the long-context operators of the paged cache: a cache held
in 4 bits (append into it, attention over it), and sparse attention over the
pages that a cheap score selects for each query (the pages' bounds, the
selection, the attention).

A case is a dict of plain values.  prepare() makes its inputs on the GPU from a
seed, run() is one pass (the plain torch form, or the package's operators when
`own` is set), work() the bytes and operations a pass cannot do without, and
exact() the same outputs from the definitions in 64 bits.

The 4-bit cache: 32 elements of a head share a scale s, the least number of
seven significant bits (a float16, at most 896) that is not below a seventh of
the largest magnitude; an element is the code c = round(x / s) in [-7, 7], held
as c + 8, element 2 i in the low half of byte i and 2 i + 1 in the high half.

A page's bounds: per KV head the smallest and largest key of each element over
the page's filled slots, as whole multiples of s, rounded outwards, s the least
power of two (from 2^-120 on) of which the largest magnitude is at most 127.  A
query's score of a page is the largest, over the query heads of the group, of
t sum_d max(c_d lo_d, c_d hi_d) with c = round(q / t), t the same for the head's q,
times s: an upper bound of the scores inside, but for the query's rounding.
"""
import math

import torch

own = False

F = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2, "q4": 0.5625}


# ---------------------------------------------------------------- the cases

def _case(name, op, seqs, new, kv, heads, kv_heads, dim, page, x, cache, ragged, order="head", **more):
    return dict(name=name, op=op, seqs=seqs, new=new, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                x=x, cache=cache, ragged=ragged, order=order, **more)


def listed():
    return [
        # the decode step's append: one row for each of 32 short conversations
        _case("append_32", "append", 32, 1, 144, 32, 8, 128, 16, "f32", "q4", True, rot=128, pairs="adjacent"),
        # the append of four 2048-token prompts
        _case("append_prefill", "append", 4, 2048, 2048, 32, 8, 128, 16, "f32", "q4", False, rot=128, pairs="adjacent"),
        # one short conversation on the smallest model (9 query heads over 3 KV heads): latency
        _case("attend_one", "attention", 1, 1, 161, 9, 3, 64, 16, "f32", "q4", False),
        # the 32-sequence decode of the 8B shape, sequences of different lengths, f32 activations
        _case("attend_32", "attention", 32, 1, 2304, 32, 8, 128, 16, "f32", "q4", True),
        # eight long documents answered one token at a time on the 70B shape
        _case("attend_long", "attention", 8, 1, 32768, 64, 8, 128, 64, "f16", "q4", True),
        # a 512-token chunk of a long prompt whose beginning is cached already
        _case("attend_chunk", "attention", 1, 512, 16384, 64, 8, 128, 64, "f16", "q4", False),
        # the bounds of the pages that a decode step's rows went to
        _case("bounds_32", "bounds", 32, 1, 2304, 32, 8, 128, 16, "f32", "q4", True),
        # the bounds of four prompts' pages
        _case("bounds_prefill", "bounds", 4, 2048, 2048, 32, 8, 128, 16, "f32", "f16", False),
        # the pages one conversation's next token reads
        _case("select_one", "select", 1, 1, 16384, 32, 8, 128, 16, "f32", "q4", False, budget=128),
        # the pages that eight long documents' next tokens read
        _case("select_long", "select", 8, 1, 32768, 64, 8, 128, 16, "f16", "q4", True, budget=256),
        # eight long documents answered one token at a time, an eighth of their pages read
        _case("sparse_long", "sparse", 8, 1, 32768, 64, 8, 128, 64, "f16", "f16", True, budget=64),
        # 32 conversations, 128 pages each, from a cache in 4 bits
        _case("sparse_32", "sparse", 32, 1, 8192, 32, 8, 128, 16, "f32", "q4", True, budget=128),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(9, 3, 64), (32, 4, 64), (32, 8, 128), (64, 8, 128), (16, 16, 128), (8, 1, 128), (8, 2, 96), (6, 2, 32)]
PAGES = [16, 16, 32, 64, 128, 20]


def draw(rng):
    """One more case of the listed ranges: any head layout, page size, order and
    type, lengths from one token to the longest, ragged batches."""
    while True:
        op = rng.choice(["attention", "attention", "append", "bounds", "select", "sparse", "sparse"])
        heads, kv_heads, dim = rng.choice(HEADS)
        page, order, x = rng.choice(PAGES), rng.choice(["head", "head", "page"]), rng.choice(["f32", "f16"])
        seqs, ragged, more = _spread(rng, 1, 32), rng.random() < 0.6, {}
        cache = "q4" if op in ("attention", "append") else rng.choice(["q4", "f16"])
        if op in ("select", "sparse"):
            new = 1 if rng.random() < 0.7 else _spread(rng, 2, 8)
            kv = max(9 * page, _spread(rng, 64, 32768))
            more = dict(budget=min(_spread(rng, 4, 256), kv // page // 2))
        else:
            new = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
            kv = max(new, _spread(rng, 64, 32768 if op == "attention" else 4096))
        if op == "append":
            more = dict(rot=dim if rng.random() < 0.7 else dim // 2, pairs=rng.choice(["adjacent", "halves"]))
        c = _case("", op, seqs, new, kv, heads, kv_heads, dim, page, x, cache, ragged, order, **more)
        del c["name"]
        w = work(c)
        if w["bytes"] > 3e8 or w["flops"] > 2.7e11:
            continue
        if op == "attention" and seqs * heads * new * kv > 6e8:
            continue
        if seqs * kv * kv_heads * dim > (3e7 if op in ("append", "bounds") else 2.7e8):
            continue
        if op == "select" and seqs * new * kv_heads * -(-kv // page) * dim > 1.4e8:
            continue
        if op == "sparse" and seqs * new * kv_heads * more["budget"] * page * dim > 1.4e8:
            continue
        return c


def _lengths(case):
    """New and cached tokens of each sequence (the cached ones include the new):
    a fixed pattern of the case, so that the work does not depend on the seed."""
    B, T, L = case["seqs"], case["new"], case["kv"]
    new, kv = [], []
    for b in range(B):
        t, n = T, L
        if case["ragged"]:
            if T > 1:
                t = 1 if b % 3 else max(1, T - (b * 37) % (T // 2 + 1))
            n = max(t, L - (b * 2377) % (3 * L // 4 + 1))
        new.append(t)
        kv.append(n)
    return new, kv


def work(case):
    new, kv = _lengths(case)
    R, D, H, KH, sx, sc = sum(new), case["dim"], case["heads"], case["kv_heads"], SIZE[case["x"]], SIZE[case["cache"]]
    ps, B = case["page"], case["seqs"]
    pages = sum(-(-n // ps) for n in kv)
    meta = 4 * (pages + 2 * B + 1)
    if case["op"] == "append":
        # the rows, and the cache read back as float16 (its 4-bit values are what the pass returns)
        pool = 2 * (pages + 3) * ps * KH * D
        return {"bytes": R * D * (2 * H + 2 * KH) * sx + pool * (SIZE["q4"] + 2) + R * case["rot"] * 4 + 4 * (R + 2 * B),
                "flops": 3 * R * (H + KH) * case["rot"]}
    if case["op"] == "attention":
        seen = sum(t * (n - t) + t * (t + 1) // 2 for t, n in zip(new, kv))
        return {"bytes": 2 * R * H * D * sx + 2 * sum(kv) * KH * D * sc + meta, "flops": 4 * H * D * seen}
    if case["op"] == "bounds":
        # the touched pages' keys, and the bounds read back as float32
        keys = sum(n - (n - t) // ps * ps for t, n in zip(new, kv))
        return {"bytes": keys * KH * D * sc + (pages + 3) * KH * (2 * D * (1 + 4) + 4) + meta, "flops": 2 * keys * KH * D}
    spots = [-(-p // ps) for t, n in zip(new, kv) for p in range(n - t + 1, n + 1)]  # pages that each row sees
    if case["op"] == "select":
        return {"bytes": pages * KH * (2 * D + 4) + R * H * D * sx + R * KH * case["budget"] * 4 + meta,
                "flops": 2 * sum(spots) * H * D}
    # sparse: pages that several rows of a sequence select are counted once a row (which they share is the inputs' matter)
    keys = sum(min(s, case["budget"]) for s in spots) * ps
    return {"bytes": 2 * R * H * D * sx + 2 * min(keys, max(sum(kv), 1)) * KH * D * sc + R * KH * case["budget"] * 4 + meta,
            "flops": 4 * H * D * keys}


# ---------------------------------------------------------------- inputs

def _scale_slots(dim):
    return 2 if dim <= 64 else 4 if dim <= 128 else 8


def _to_q4(x):
    """Codes [..., dim / 2] and scales [..., slots] of float32 values [..., dim]."""
    g = x.unflatten(-1, (x.shape[-1] // 32, 32))
    top = g.abs().amax(-1)
    s = top / torch.full_like(top, 7.0)
    s = ((s.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)       # up to seven significant bits
    s = torch.ceil(s * 2.0 ** 24) * 2.0 ** -24                                  # a float16
    s = torch.where(torch.isfinite(top), s.clamp_max(896.0), math.nan)
    c = torch.round(g / torch.where(s > 0, s, 1.0)[..., None]).nan_to_num(0.0).clamp(-7, 7)
    c = (torch.where(torch.isfinite(top)[..., None], c, 0.0) + 8.0).flatten(-2).to(torch.uint8)
    scales = torch.zeros((*s.shape[:-1], _scale_slots(x.shape[-1])), dtype=torch.float16, device=x.device)
    scales[..., :s.shape[-1]] = s.to(torch.float16)
    return c[..., 0::2] | (c[..., 1::2] << 4), scales


def _from_q4(codes, scales):
    """The float32 values of codes and scales."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    s = scales[..., :c.shape[-1] // 32].float()
    return (c.unflatten(-1, (s.shape[-1], 32)) * s[..., None]).flatten(-2)


def _in_order(t, order):
    """The pool's memory in the case's order, as a [n_pages, kv_heads, page, ...] view."""
    return t.transpose(1, 2).contiguous().transpose(1, 2) if order == "page" else t


def _pool(case, g, kv, dev):
    """A pool with every page the sequences need and some spare ones, in a
    shuffled order, holding the keys and values of earlier tokens (and of earlier
    requests beyond them).  Keys of a page have something in common."""
    ps, KH, D = case["page"], case["kv_heads"], case["dim"]
    per = -(-case["kv"] // ps)
    used = [-(-n // ps) for n in kv]
    n_pages = sum(used) + 3
    k = torch.randn((n_pages, KH, ps, D), generator=g, device=dev)
    k += torch.randn((n_pages, KH, 1, D), generator=g, device=dev)
    v = torch.randn((n_pages, KH, ps, D), generator=g, device=dev)
    perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["seqs"], per), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    if case["cache"] == "q4":
        pool = [_in_order(t, case["order"]) for x in (k, v) for t in _to_q4(x)]
    else:
        pool = [_in_order(x.to(F[case["cache"]]), case["order"]) for x in (k, v)]
    return pool, table


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    new, kv = _lengths(case)
    pool, table = _pool(case, g, kv, dev)
    R, H, KH, D, dt, op = sum(new), case["heads"], case["kv_heads"], case["dim"], F[case["x"]], case["op"]
    # the rows of a fused q/k/v projection: heads side by side
    rows = torch.randn((R, H + 2 * KH, D), generator=g, device=dev)
    if op != "append":
        rows[:, :H] *= 2.0                                # scores of a trained model spread further than noise
    rows = rows.to(dt)
    start = [0]
    for t in new:
        start.append(start[-1] + t)
    s = dict(case=case, pool=pool, table=table, q=rows[:, :H], k=rows[:, H:H + KH], v=rows[:, H + KH:],
             q_start=torch.tensor(start, dtype=torch.int32, device=dev),
             kv_len=torch.tensor(kv, dtype=torch.int32, device=dev), max_new=max(new), max_kv=max(kv))
    if op == "append":
        j = torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64)
        a = torch.arange(case["kv"], device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * j / case["rot"])
        s["rope"] = torch.stack((a.cos(), a.sin()), -1).to(torch.float32).contiguous()  # [positions, rot / 2, 2]
    if op in ("bounds", "select"):
        n_pages = pool[0].shape[0]
        if op == "select":                                # every page's bounds, as earlier steps left them
            s["bounds"] = list(_bounds_of(_keys(s, torch.arange(n_pages, device=dev)), None))
            s["pool"] = []
        else:
            s["bounds"] = [torch.zeros((n_pages, KH, D), dtype=torch.int8, device=dev) for _ in range(2)]
            s["bounds"].append(torch.zeros((n_pages, KH), device=dev))
    if op == "sparse":
        # lists as a selection makes them: the first page, the last two, others between
        seq, tok = _rows_of(s)
        n = (_positions(s, seq, tok) // case["page"] + 1)[:, None, None]
        P = table.shape[1]
        i = torch.arange(P, device=dev)
        r = torch.rand((R, KH, P), generator=g, device=dev)
        r = torch.where((i == 0) | (i >= n - 2), 2.0, r).masked_fill_(i >= n, -1.0)
        r, i = torch.topk(r, min(case["budget"], P), dim=2)
        i = torch.where(r >= 0, i, P).sort(2).values
        s["pages"] = torch.full((R, KH, case["budget"]), -1, dtype=torch.int32, device=dev)
        s["pages"][:, :, :i.shape[2]] = torch.where(i < P, i, -1)
    if own:
        from hypno_b200 import paged
        # the handles a serving program keeps with its pool
        if s["pool"]:
            s["cache"] = paged.PagedKV4(*pool) if case["cache"] == "q4" else paged.PagedKV(*pool)
        if "bounds" in s:
            s["handle"] = paged.PageBounds(*s["bounds"], page_size=case["page"])
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return _own_pass(s, op)
    return {"append": _plain_append, "attention": _plain_attention, "bounds": _plain_bounds, "select": _plain_select,
            "sparse": _plain_sparse}[op](s)


def _own_pass(s, op):
    from hypno_b200 import paged
    batch = paged.PagedBatch(s["table"], s["q_start"], s["kv_len"], s["max_new"], s["max_kv"])
    if op == "attention":
        return paged.attention(s["cache"], batch, s["q"])
    if op == "sparse":
        return paged.attention(s["cache"], batch, s["q"], pages=s["pages"])
    if op == "select":
        return paged.select_pages(s["handle"], batch, s["q"], s["case"]["budget"])
    if op == "bounds":
        paged.update_bounds(s["handle"], s["cache"], batch)
        return s["handle"].values()
    q = paged.append(s["cache"], batch, s["k"], s["v"], q=s["q"], rope=s["rope"], pairs=s["case"]["pairs"])
    return q, *s["cache"].values()


def _rows_of(s):
    """Sequence and index within its new tokens of every packed row."""
    r = torch.arange(s["q"].shape[0], device=s["q"].device)
    seq = torch.searchsorted(s["q_start"][1:].long(), r, right=True)
    return seq, r - s["q_start"].long()[seq]


def _positions(s, seq, tok):
    t = (s["q_start"][1:] - s["q_start"][:-1]).long()
    return s["kv_len"].long()[seq] - t[seq] + tok


def _keys(s, pages):
    """The float32 keys of pages."""
    p = s["pool"]
    return _from_q4(p[0][pages], p[1][pages]) if s["case"]["cache"] == "q4" else p[0][pages].float()


def _values(s, pages):
    p = s["pool"]
    return _from_q4(p[2][pages], p[3][pages]) if s["case"]["cache"] == "q4" else p[1][pages].float()


def _plain_rotate(x, cs, pairs):
    rot = 2 * cs.shape[1]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    x = x.float()
    if pairs == "adjacent":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat((a * c - b * n, a * n + b * c), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_append(s):
    c = s["case"]
    seq, tok = _rows_of(s)
    pos = _positions(s, seq, tok)
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    cs = s["rope"][pos]
    kc, ks, vc, vs = s["pool"]
    kc[page, :, slot], ks[page, :, slot] = _to_q4(_plain_rotate(s["k"], cs, c["pairs"]))
    vc[page, :, slot], vs[page, :, slot] = _to_q4(s["v"].float())
    return (_plain_rotate(s["q"], cs, c["pairs"]).to(s["q"].dtype), _from_q4(kc, ks).to(torch.float16),
            _from_q4(vc, vs).to(torch.float16))


def _plain_attention(s):
    c = s["case"]
    H, KH, D, ps, T, L = c["heads"], c["kv_heads"], c["dim"], c["page"], s["max_new"], s["max_kv"]
    B, G, dev = c["seqs"], c["heads"] // c["kv_heads"], s["q"].device
    seq, tok = _rows_of(s)
    pages = s["table"].long().clamp_min(0)                               # [B, P]
    N = pages.shape[1] * ps
    K = _keys(s, pages).permute(0, 2, 4, 1, 3).reshape(B, KH, D, N)[..., :L]
    Q = torch.zeros((B, T, H, D), device=dev)
    Q[seq, tok] = s["q"].float()
    Q = Q.view(B, T, KH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KH, G * T, D)
    S = (Q @ K).view(B, KH, G, T, L)
    del K
    S *= 1.0 / math.sqrt(D)
    n, t = s["kv_len"].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    at = (n - t)[:, None] + torch.arange(T, device=dev)                    # [B, T]: each row's position
    seen = torch.arange(L, device=dev) <= at[..., None]
    S.masked_fill_(~seen[:, None, None], -math.inf)
    S -= S.amax(-1, keepdim=True).clamp_min(-3e38)
    S.exp_()
    total = S.sum(-1, keepdim=True)
    V = _values(s, pages).permute(0, 2, 1, 3, 4).reshape(B, KH, N, D)[:, :, :L]
    O = (S.view(B, KH, G * T, L) @ V).view(B, KH, G, T, D) / total.clamp_min(1e-37)
    return O.permute(0, 3, 1, 2, 4).reshape(B, T, H, D)[seq, tok].to(s["q"].dtype)


def _unit(top):
    """The least power of two, from 2^-120 on, of which `top` is at most 127; infinite where top is not finite."""
    bits = top.view(torch.int32)
    e = (bits >> 23) - 6 + ((bits & 0x7FFFFF) > 0x7E0000).int()
    return torch.where(torch.isfinite(top), (e.clamp_min(7) << 23).view(torch.float32), math.inf)


def _bounds_of(k, filled):
    """Bounds [..., kv_heads, dim] (two int8) and scales [..., kv_heads] of the
    keys [..., kv_heads, page, dim] of pages whose first `filled` slots count (None: all)."""
    lo = hi = k
    if filled is not None:
        out = torch.arange(k.shape[-2], device=k.device) >= filled[..., None]
        out = out[..., None, :, None]
        lo, hi = k.masked_fill(out, math.inf), k.masked_fill(out, -math.inf)
    lo, hi = lo.amin(-2), hi.amax(-2)
    s = _unit(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    by = s[..., None]
    lo8, hi8 = torch.floor(lo / by), torch.ceil(hi / by)
    fine = torch.isfinite(by)
    return torch.where(fine, lo8, 0.0).to(torch.int8), torch.where(fine, hi8, 0.0).to(torch.int8), s


def _plain_bounds(s):
    c = s["case"]
    ps, dev = c["page"], s["table"].device
    n, t = s["kv_len"].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    first, last = (n - t) // ps, (n - 1) // ps                             # pages that hold a new row
    i = torch.minimum(first[:, None] + torch.arange((s["max_new"] + ps - 2) // ps + 1, device=dev), last[:, None])
    page = s["table"].long().gather(1, i)
    lo, hi, scale = s["bounds"]
    lo[page], hi[page], scale[page] = _bounds_of(_keys(s, page), n[:, None] - i * ps)
    return lo.float() * scale[..., None], hi.float() * scale[..., None]


def _plain_select(s):
    """The first page, the last two, and of the others the ones with the largest
    scores (equal ones: the lower index first), `budget` in all, by index."""
    c = s["case"]
    KH, G, budget = c["kv_heads"], c["heads"] // c["kv_heads"], c["budget"]
    seq, tok = _rows_of(s)
    lo, hi, scale = s["bounds"]
    page = s["table"].long()[seq]                                          # [R, P]
    held, page = page >= 0, page.clamp_min(0)
    q = s["q"].float().unflatten(1, (KH, G))
    t = _unit(q.abs().amax(-1))
    c8 = torch.where(torch.isfinite(t)[..., None], torch.round(q / t[..., None]), 0.0)
    up, down = c8.clamp_min(0), c8.clamp_max(0)
    # (whole numbers below 2^24: exact in float32)
    I = up @ hi[page].permute(0, 2, 3, 1).float() + down @ lo[page].permute(0, 2, 3, 1).float()  # [R, KH, G, P]
    best = (I * torch.where(torch.isfinite(t), t, 0.0)[..., None]).clamp(-3e38, 3e38).amax(2)
    sc = scale[page].permute(0, 2, 1)                                      # [R, KH, P]
    score = torch.where(torch.isfinite(sc), best * sc, math.inf).masked_fill(~held[:, None], -math.inf)
    n = (_positions(s, seq, tok) // c["page"] + 1)[:, None, None]
    P = page.shape[1]
    i = torch.arange(P, device=page.device)
    order = torch.sort(score, dim=2, descending=True, stable=True).indices
    kind = torch.where((order == 0) | (order >= n - 2), 2, 1).masked_fill_(order >= n, 0)
    kind, at = torch.sort(kind, dim=2, descending=True, stable=True)
    order = order.gather(2, at)[:, :, :budget].masked_fill(kind[:, :, :budget] == 0, P).sort(2).values
    out = torch.full((order.shape[0], KH, budget), -1, dtype=torch.int32, device=page.device)
    out[:, :, :order.shape[2]] = torch.where(order < P, order, -1).int()
    return out


def _plain_sparse(s):
    c = s["case"]
    KH, D, ps, G = c["kv_heads"], c["dim"], c["page"], c["heads"] // c["kv_heads"]
    seq, tok = _rows_of(s)
    R, W = s["pages"].shape[0], c["budget"]
    i = s["pages"].long()                                                  # [R, KH, W]
    page = s["table"].long()[seq[:, None, None], i.clamp_min(0)].clamp_min(0)
    head = torch.arange(KH, device=i.device)[None, :, None]
    at = (i * ps)[..., None] + torch.arange(ps, device=i.device)
    seen = (at <= _positions(s, seq, tok)[:, None, None, None]) & (i >= 0)[..., None]
    here = (page, head)
    K = _keys(s, here).reshape(R, KH, W * ps, D)
    S = s["q"].float().unflatten(1, (KH, G)) @ K.transpose(2, 3) * (1.0 / math.sqrt(D))
    del K
    S.masked_fill_(~seen.view(R, KH, 1, W * ps), -math.inf)
    S -= S.amax(-1, keepdim=True).clamp_min(-3e38)
    S.exp_()
    O = S @ _values(s, here).reshape(R, KH, W * ps, D) / S.sum(-1, keepdim=True).clamp_min(1e-37)
    return O.reshape(R, KH * G, D).to(s["q"].dtype)


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "bounds": _exact_bounds, "select": _exact_select,
            "sparse": _exact_sparse}[case["op"]](case, s)


def _decoded(codes, scales, dim):
    out = torch.empty((*codes.shape[:-1], dim), dtype=torch.float64, device=codes.device)
    out[..., 0::2] = (codes % 16).double()
    out[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    return (out - 8) * torch.repeat_interleave(scales.double(), 32, dim=-1)[..., :dim]


def _k64(case, s, pages, h):
    p = s["pool"]
    return _decoded(p[0][pages, h], p[1][pages, h], case["dim"]) if case["cache"] == "q4" else p[0][pages, h].double()


def _v64(case, s, pages, h):
    p = s["pool"]
    return _decoded(p[2][pages, h], p[3][pages, h], case["dim"]) if case["cache"] == "q4" else p[1][pages, h].double()


def _exact_append(case, s):
    new, kv = _lengths(case)
    rot, ps, D = case["rot"], case["page"], case["dim"]

    def turned(x, cs):
        z = x.double().clone()
        first = torch.arange(rot // 2, device=x.device) * 2 if case["pairs"] == "adjacent" else torch.arange(rot // 2, device=x.device)
        second = first + (1 if case["pairs"] == "adjacent" else rot // 2)
        turn = torch.view_as_complex(cs.double().contiguous())[:, None]
        y = torch.complex(z[..., first], z[..., second]) * turn
        z[..., first], z[..., second] = y.real, y.imag
        return z

    def held(x):
        """What the cache keeps of x, [..., dim]."""
        y = x.clone()
        for i in range(0, D, 32):
            top = y[..., i:i + 32].abs().amax(-1, keepdim=True)
            m, e = torch.frexp(top / 7)
            scale = torch.ldexp(torch.ceil(m * 128) / 128, e)
            scale = torch.ceil(scale * 2.0 ** 24) / 2.0 ** 24
            scale = torch.minimum(scale, torch.full_like(scale, 896.0))
            part = torch.round(y[..., i:i + 32] / scale).clamp(-7, 7) * scale
            y[..., i:i + 32] = torch.where(top > 0, part, torch.zeros_like(part))
        return y

    at = torch.cat([torch.arange(L - t, L) for t, L in zip(new, kv)]).to(s["q"].device)
    owner = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(new)).to(s["q"].device)
    cs = s["rope"].index_select(0, at)
    page = s["table"][owner, torch.div(at, ps, rounding_mode="floor")].long()
    kp, vp = _decoded(s["pool"][0], s["pool"][1], D), _decoded(s["pool"][2], s["pool"][3], D)
    k, v = held(turned(s["k"], cs)), held(s["v"].double())
    for h in range(case["kv_heads"]):
        kp[page, h, at.remainder(ps)] = k[:, h]
        vp[page, h, at.remainder(ps)] = v[:, h]
    return turned(s["q"], cs), kp, vp


def _exact_attention(case, s):
    new, kv = _lengths(case)
    G = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    r = 0
    for b, (t, L) in enumerate(zip(new, kv)):
        pages = s["table"][b, :-(-L // case["page"])].long()
        for h in range(case["kv_heads"]):
            k, v = (f(case, s, pages, h).reshape(-1, case["dim"])[:L] for f in (_k64, _v64))
            i = torch.arange(L - t, L, device=k.device)[:, None]
            hidden = torch.arange(L, device=k.device)[None] > i
            for q in range(h * G, h * G + G):
                x = s["q"][r:r + t, q].double() @ k.T / math.sqrt(case["dim"])
                x[hidden] = -math.inf
                out[r:r + t, q] = torch.softmax(x, dim=1) @ v
        r += t
    return out


def _exact_bounds(case, s):
    new, kv = _lengths(case)
    ps = case["page"]
    lo, hi, scale = (x.double() for x in s["bounds"])
    lo, hi = lo * scale[..., None], hi * scale[..., None]
    for b, (t, L) in enumerate(zip(new, kv)):
        for i in range((L - t) // ps, (L - 1) // ps + 1):
            page = int(s["table"][b, i])
            for h in range(case["kv_heads"]):
                k = _k64(case, s, page, h)[:min(ps, L - i * ps)]
                unit = 2.0 ** max(math.ceil(math.log2(max(float(k.abs().max()), 1e-300) / 127)), -120)
                lo[page, h] = torch.floor(k.min(0).values / unit) * unit
                hi[page, h] = torch.ceil(k.max(0).values / unit) * unit
    return lo, hi


def _exact_select(case, s):
    return None  # a list of whole numbers: it is equal or it is not


def _exact_sparse(case, s):
    new, kv = _lengths(case)
    G, ps = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = [(b, L - t + i) for b, (t, L) in enumerate(zip(new, kv)) for i in range(t)]
    for r, (b, p) in enumerate(at):
        for h in range(case["kv_heads"]):
            i = s["pages"][r, h].long()
            i = i[i >= 0]
            pages = s["table"][b].long()[i]
            j = (i[:, None] * ps + torch.arange(ps, device=i.device)).flatten()
            fit = j <= p
            k, v = (f(case, s, pages, h).reshape(-1, case["dim"])[fit] for f in (_k64, _v64))
            q = s["q"][r, h * G:h * G + G].double()
            out[r, h * G:h * G + G] = torch.softmax(q @ k.T / math.sqrt(case["dim"]), dim=1) @ v
    return out
