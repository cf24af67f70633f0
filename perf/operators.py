"""Measured cases of the paged serving operators: appending rotated keys and
values to a paged cache, attention of new tokens over it, and drawing the next
token from given uniform numbers.

A case is a dict of plain values.  prepare() makes its inputs on the GPU from a
seed, run() is one pass (the plain torch form, or the package's operators when
`own` is set), work() the bytes and operations a pass cannot do without, and
exact() the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

F = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}


# ---------------------------------------------------------------- the cases

def _attn(name, seqs, new, kv, heads, kv_heads, dim, page, q, cache, ragged, window=0, order="head"):
    return dict(name=name, op="attention", seqs=seqs, new=new, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                x=q, cache=cache, ragged=ragged, window=window, order=order)


def _append(name, seqs, new, kv, heads, kv_heads, dim, page, x, cache, ragged, rot, pairs="adjacent", order="head"):
    return dict(name=name, op="append", seqs=seqs, new=new, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                x=x, cache=cache, ragged=ragged, rot=rot, pairs=pairs, order=order)


def _sample(name, rows, vocab, mode):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, mode=mode)


def listed():
    return [
        # one short conversation on the smallest model (9 query heads over 3 KV heads, FP32 cache): latency
        _attn("decode_one_f32", 1, 1, 161, 9, 3, 64, 16, "f32", "f32", False),
        # the 32-sequence decode of the 8B shape, sequences of different lengths, f32 activations over an FP16 cache
        _attn("decode_32", 32, 1, 2304, 32, 8, 128, 16, "f32", "f16", True),
        # eight long documents answered one token at a time on the 70B shape
        _attn("decode_long", 8, 1, 32768, 64, 8, 128, 64, "f16", "f16", True),
        # a 512-token chunk of a long prompt whose beginning is cached already
        _attn("chunk_long", 1, 512, 16384, 64, 8, 128, 64, "f16", "f16", False),
        # four prompts of 2048 tokens in one pass, with the framework's f32 activations
        _attn("prefill_4", 4, 2048, 2048, 32, 8, 128, 16, "f32", "f16", False),
        # a serving step: some sequences feed a chunk of their prompt, the others one token; odd lengths
        _attn("mixed", 24, 257, 4001, 32, 8, 128, 16, "f16", "f16", True),
        # the decode step's append: one row for each of 32 sequences
        _append("append_32", 32, 1, 2304, 32, 8, 128, 16, "f32", "f16", True, 128),
        # the append of four 2048-token prompts
        _append("append_prefill", 4, 2048, 2048, 32, 8, 128, 16, "f32", "f16", False, 128),
        # chunks of odd lengths, half-split pairs on part of the head, a page size that is no power of two
        _append("append_odd", 5, 333, 1777, 32, 4, 64, 20, "f16", "f16", True, 32, "halves", "page"),
        # one conversation's next token (the smallest model's vocabulary)
        _sample("sample_one", 1, 49152, "nucleus"),
        # the next token of 32 requests, each with its own settings
        _sample("sample_32", 32, 128256, "mixed"),
        # a large batch of requests
        _sample("sample_256", 256, 128256, "mixed"),
    ]


def _spread(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return v if v != 3072 else v + 1


HEADS = [(9, 3, 64), (32, 4, 64), (32, 8, 128), (64, 8, 128), (4, 2, 16), (16, 16, 128), (8, 1, 128)]
PAGES = [16, 16, 32, 64, 128, 20]


def draw(rng):
    """One more case of the listed ranges: any head layout, page size, order and
    type, lengths from one token to the longest, windows, ragged batches."""
    while True:
        op = rng.choice(["attention", "attention", "attention", "append", "sample"])
        if op == "sample":
            c = _sample("", _spread(rng, 1, 256), _spread(rng, 1000, 128256), rng.choice(["nucleus", "mixed", "plain", "topk"]))
        else:
            heads, kv_heads, dim = rng.choice(HEADS)
            page, order = rng.choice(PAGES), rng.choice(["head", "head", "page"])
            x, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
            seqs = _spread(rng, 1, 32)
            new = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
            if op == "attention":
                kv = max(new, _spread(rng, 64, 32768))
                window = _spread(rng, 64, 4096) if rng.random() < 0.2 else 0
                c = _attn("", seqs, new, kv, heads, kv_heads, dim, page, x, cache, rng.random() < 0.6, window, order)
            else:
                kv = max(new, _spread(rng, 64, 4096))
                rot = dim if rng.random() < 0.7 else dim // 2
                c = _append("", seqs, new, kv, heads, kv_heads, dim, page, x, cache, rng.random() < 0.6, rot,
                            rng.choice(["adjacent", "halves"]), order)
        del c["name"]
        w = work(c)
        if w["bytes"] > 7e8 or w["flops"] > 2.7e11:
            continue
        if op == "attention" and c["seqs"] * c["heads"] * c["new"] * c["kv"] > 2.2e9:
            continue
        if op != "sample" and c["seqs"] * c["kv"] * c["kv_heads"] * c["dim"] > 4e8:
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


def _visible(case):
    """Visible (query, key) pairs of the case, for one head."""
    n = 0
    for t, L in zip(*_lengths(case)):
        w = case["window"] or L
        first = L - t + 1                       # keys seen by the first new token without a window
        if first >= w:
            n += t * w
        else:
            grow = min(t, w - first)            # rows that still see fewer than w keys
            n += grow * first + grow * (grow - 1) // 2 + (t - grow) * w
    return n


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 28), "flops": case["rows"] * case["vocab"] * 4}
    new, kv = _lengths(case)
    R, D, H, KH, sx, sc = sum(new), case["dim"], case["heads"], case["kv_heads"], SIZE[case["x"]], SIZE[case["cache"]]
    meta = 4 * (sum(-(-n // case["page"]) for n in kv) + 2 * case["seqs"] + 1)
    if case["op"] == "append":
        rows = R * (H + KH) * case["rot"]
        return {"bytes": R * D * (2 * H * sx + 2 * KH * (sx + sc)) + R * case["rot"] * 4 + 4 * (R + 2 * case["seqs"] + 1),
                "flops": 3 * rows}
    keys = sum(min(n, (case["window"] or n) + t - 1) for t, n in zip(new, kv))
    return {"bytes": 2 * R * H * D * sx + 2 * keys * KH * D * sc + meta, "flops": 4 * H * D * _visible(case)}


# ---------------------------------------------------------------- inputs

def _pages(case, g, kv, dev):
    """A pool with every page the sequences need and some spare ones, in a
    shuffled order, holding the keys and values of earlier tokens (and of
    earlier requests beyond them)."""
    ps, KH, D, dt = case["page"], case["kv_heads"], case["dim"], F[case["cache"]]
    per = -(-case["kv"] // ps)
    used = [-(-n // ps) for n in kv]
    n_pages = sum(used) + 3
    shape = (n_pages, KH, ps, D) if case["order"] == "head" else (n_pages, ps, KH, D)
    pools = [torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt) for _ in range(2)]
    if case["order"] == "page":
        pools = [p.transpose(1, 2) for p in pools]       # [n_pages, kv_heads, page, dim] views
    perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["seqs"], per), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    return pools[0], pools[1], table


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        # logits of a language model: probabilities that fall like a power of a token's rank
        z = torch.rand((B, V), generator=g, device=dev)
        logits = -1.4 * torch.log1p(z * V) + 0.5 * torch.randn((B, V), generator=g, device=dev)
        kinds = {"nucleus": [(0.8, 0, 0.95, 0.0)], "plain": [(1.0, 0, 1.0, 0.0)], "topk": [(0.7, 50, 1.0, 0.0)],
                 "mixed": [(0.8, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05),
                           (0.6, 1000, 0.99, 0.01), (1.0, 0, 1.0, 0.0)]}[case["mode"]]
        col = [[kinds[b % len(kinds)][j] for b in range(B)] for j in range(4)]
        return dict(case=case, logits=logits, u=torch.rand(B, generator=g, device=dev),
                    temperature=torch.tensor(col[0], device=dev, dtype=torch.float32),
                    top_k=torch.tensor(col[1], device=dev, dtype=torch.int32),
                    top_p=torch.tensor(col[2], device=dev, dtype=torch.float32),
                    min_p=torch.tensor(col[3], device=dev, dtype=torch.float32))
    new, kv = _lengths(case)
    kp, vp, table = _pages(case, g, kv, dev)
    R, H, KH, D, dt = sum(new), case["heads"], case["kv_heads"], case["dim"], F[case["x"]]
    # the rows of a fused q/k/v projection: heads side by side
    rows = torch.randn((R, H + 2 * KH, D), generator=g, device=dev)
    if case["op"] == "attention":
        rows[:, :H] *= 2.0                                # scores of a trained model spread further than noise
    rows = rows.to(dt)
    start = [0]
    for t in new:
        start.append(start[-1] + t)
    s = dict(case=case, k_pages=kp, v_pages=vp, table=table, q=rows[:, :H], k=rows[:, H:H + KH], v=rows[:, H + KH:],
             q_start=torch.tensor(start, dtype=torch.int32, device=dev),
             kv_len=torch.tensor(kv, dtype=torch.int32, device=dev), max_new=max(new), max_kv=max(kv))
    if case["op"] == "append":
        j = torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64)
        a = torch.arange(case["kv"], device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * j / case["rot"])
        s["rope"] = torch.stack((a.cos(), a.sin()), -1).to(torch.float32).contiguous()  # [positions, rot / 2, 2]
    if own:
        from hypno_b200 import paged
        s["cache"] = paged.PagedKV(kp, vp)                # the handle a serving program keeps with its pool
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return _own_pass(s, op)
    return {"attention": _plain_attention, "append": _plain_append, "sample": _plain_sample}[op](s)


def _own_pass(s, op):
    if op == "sample":
        from hypno_b200 import sampling
        return sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    from hypno_b200 import paged
    batch = paged.PagedBatch(s["table"], s["q_start"], s["kv_len"], s["max_new"], s["max_kv"])
    if op == "attention":
        return paged.attention(s["cache"], batch, s["q"], window=s["case"]["window"])
    q = paged.append(s["cache"], batch, s["k"], s["v"], q=s["q"], rope=s["rope"], pairs=s["case"]["pairs"])
    return q, s["k_pages"], s["v_pages"]


def _rows_of(s):
    """Sequence and index within its new tokens of every packed row."""
    r = torch.arange(s["q"].shape[0], device=s["q"].device)
    seq = torch.searchsorted(s["q_start"][1:].long(), r, right=True)
    return seq, r - s["q_start"].long()[seq]


def _plain_attention(s):
    c = s["case"]
    H, KH, D, ps, T, L = c["heads"], c["kv_heads"], c["dim"], c["page"], s["max_new"], s["max_kv"]
    B, G, dev = c["seqs"], c["heads"] // c["kv_heads"], s["q"].device
    seq, tok = _rows_of(s)
    pos = torch.arange(L, device=dev)
    page = s["table"].long().clamp_min(0)[:, pos // ps]
    slot = (pos % ps)[None].expand(B, L)
    K = s["k_pages"][page, :, slot].float().permute(0, 2, 3, 1)          # [B, KH, D, L]
    Q = torch.zeros((B, T, H, D), device=dev)
    Q[seq, tok] = s["q"].float()
    Q = Q.view(B, T, KH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KH, G * T, D)
    S = (Q @ K).view(B, KH, G, T, L)
    del K
    S *= 1.0 / math.sqrt(D)
    n, t = s["kv_len"].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    at = (n - t)[:, None] + torch.arange(T, device=dev)                    # [B, T]: each row's position
    seen = pos <= at[..., None]
    if c["window"]:
        seen &= pos > at[..., None] - c["window"]
    S.masked_fill_(~seen[:, None, None], -math.inf)
    S -= S.amax(-1, keepdim=True).clamp_min(-3e38)
    S.exp_()
    total = S.sum(-1, keepdim=True)
    V = s["v_pages"][page, :, slot].float().permute(0, 2, 1, 3)          # [B, KH, L, D]
    O = (S.view(B, KH, G * T, L) @ V).view(B, KH, G, T, D) / total.clamp_min(1e-37)
    return O.permute(0, 3, 1, 2, 4).reshape(B, T, H, D)[seq, tok].to(s["q"].dtype)


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
    t = (s["q_start"][1:] - s["q_start"][:-1]).long()
    pos = s["kv_len"].long()[seq] - t[seq] + tok
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    cs = s["rope"][pos]
    s["k_pages"][page, :, slot] = _plain_rotate(s["k"], cs, c["pairs"]).to(s["k_pages"].dtype)
    s["v_pages"][page, :, slot] = s["v"].to(s["v_pages"].dtype)
    return _plain_rotate(s["q"], cs, c["pairs"]).to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _plain_sample(s):
    """Tokens in order of their logit (ties: the lower index first).  Kept: the
    first top_k; of these the shortest head that holds top_p of their mass; of
    these the ones with at least min_p times the largest probability.  The draw
    walks the kept tokens by index until their mass exceeds u times the total.
    Masses are whole multiples of 2^-40 of the largest, so their sums are exact
    in any order."""
    l, T = s["logits"], s["temperature"]
    l = torch.where(torch.isnan(l), -math.inf, l)
    greedy = T <= 0
    inv = torch.where(greedy, 1.0, 1.0 / T)
    ranked, index = torch.sort(l, dim=1, descending=True, stable=True)
    top = ranked[:, :1]
    w = torch.where(ranked == top, 1.0, torch.exp((ranked - top) * inv[:, None]))
    mass = (w * 2.0 ** 40).long()
    rank = torch.arange(l.shape[1], device=l.device)
    k = torch.where(greedy, 1, s["top_k"]).long()[:, None]
    keep = (k <= 0) | (rank < k)
    held = torch.where(keep, mass, 0)
    before = held.cumsum(1) - held
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (before.double() < p * held.sum(1, keepdim=True).double())
    keep &= w >= s["min_p"][:, None]
    keep |= rank == 0
    held = torch.zeros_like(mass).scatter_(1, index, torch.where(keep, mass, 0))
    total = held.sum(1, keepdim=True)
    goal = (s["u"].double()[:, None] * total.double()).floor().long().clamp_max(total - 1)
    token = (held.cumsum(1) > goal).int().argmax(1, keepdim=True)
    logprob = torch.log((held.gather(1, token).double() / total.double()).float())[:, 0]
    some = top[:, 0] > -math.inf
    return torch.where(some, token[:, 0], -1).int(), torch.where(some, logprob, -math.inf)


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "sample": _exact_sample}[case["op"]](case, s)


def _exact_attention(case, s):
    new, kv = _lengths(case)
    G = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    r = 0
    for b, (t, L) in enumerate(zip(new, kv)):
        pages = s["table"][b, :-(-L // case["page"])].long()
        for h in range(case["kv_heads"]):
            k = s["k_pages"][pages, h].double().reshape(-1, case["dim"])[:L]
            v = s["v_pages"][pages, h].double().reshape(-1, case["dim"])[:L]
            i = torch.arange(L - t, L, device=k.device)[:, None]
            j = torch.arange(L, device=k.device)[None]
            hidden = (j > i) | (j <= i - (case["window"] or L))
            for q in range(h * G, h * G + G):
                x = s["q"][r:r + t, q].double() @ k.T / math.sqrt(case["dim"])
                x[hidden] = -math.inf
                out[r:r + t, q] = torch.softmax(x, dim=1) @ v
        r += t
    return out


def _exact_append(case, s):
    new, kv = _lengths(case)
    rot, ps = case["rot"], case["page"]

    def turned(x, cs):
        z = x.double().clone()
        first = torch.arange(rot // 2, device=x.device) * 2 if case["pairs"] == "adjacent" else torch.arange(rot // 2, device=x.device)
        second = first + (1 if case["pairs"] == "adjacent" else rot // 2)
        turn = torch.view_as_complex(cs.double().contiguous())[:, None]
        y = torch.complex(z[..., first], z[..., second]) * turn
        z[..., first], z[..., second] = y.real, y.imag
        return z

    at = torch.cat([torch.arange(L - t, L) for t, L in zip(new, kv)]).to(s["q"].device)
    owner = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(new)).to(s["q"].device)
    cs = s["rope"].index_select(0, at)
    page = s["table"][owner, torch.div(at, ps, rounding_mode="floor")].long()
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    k, v = turned(s["k"], cs), s["v"].double()
    for h in range(case["kv_heads"]):
        kp[page, h, at.remainder(ps)] = k[:, h]
        vp[page, h, at.remainder(ps)] = v[:, h]
    return turned(s["q"], cs), kp, vp


def _exact_sample(case, s):
    token, logp = [], []
    for b in range(case["rows"]):
        l = s["logits"][b].double()
        T, k, p, least, u = (s[n][b].item() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        if T <= 0:
            k, T = 1, 1.0
        order = torch.argsort(-l, stable=True)
        if k > 0:
            order = order[:k]
        q = torch.softmax(l[order] / T, dim=0)
        if p < 1:
            order = order[:max(1, int((q.cumsum(0) - q < p).sum()))]
            q = q[:order.numel()]
        fit = q >= least * q[0]
        order, at = torch.sort(order[fit])
        q = q[fit][at]
        q = q / q.sum()
        i = min(int((q.cumsum(0) <= u).sum()), q.numel() - 1)
        token.append(order[i])
        logp.append(q[i].log())
    return torch.stack(token).int(), torch.stack(logp)
