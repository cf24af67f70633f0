"""sampling.sample (hc_sample_uniform_dev) against its definition with exact
integer masses on the host.  The device's weights are CUDA's expf (within 2
ulp), the host's 64-bit exp, so a draw may differ only where u lies within
that rounding of a boundary between two tokens: each such draw is shown to lie
within 2^-20 of the boundary, and there may be few."""
import numpy as np
import pytest
import torch

from hypno_b200 import sampling
from hypno_b200._lib import call, load

from . import _paged as ref

pytestmark = pytest.mark.gpu

SETTINGS = [  # temperature, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.0), (0.7, 0, 0.95, 0.0), (1.5, 0, 1.0, 0.1), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0),
    (1.0, 1000000, 0.5, 0.01), (0.5, 7, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 0.999999, 0.0), (2.0, 200, 0.3, 0.5),
    (1.0, 0, 1.0, 2.0), (-1.0, 5, 0.9, 0.0), (1e-3, 0, 0.99, 0.0), (50.0, 3000, 0.97, 0.0),
]


def draws(dev, logits, settings, u):
    """Every row of logits with every setting, against the host."""
    B, V = logits.shape
    T, k, p, m = (np.repeat([s[i] for s in settings], B) for i in range(4))
    l = np.tile(logits, (len(settings), 1))
    t = lambda x, d: torch.from_numpy(np.ascontiguousarray(x, d)).to(dev)  # noqa: E731
    token, logp = sampling.sample(t(l, np.float32), t(u, np.float32), t(T, np.float32), t(k, np.int32), t(p, np.float32), t(m, np.float32))
    token, logp = token.cpu().numpy(), logp.cpu().numpy()
    loose = 0
    for r in range(len(l)):
        want, share, *rest = ref.sample(l[r], u[r], float(T[r]), int(k[r]), float(p[r]), float(m[r]))
        if token[r] == want:
            # expf within 2 ulp, so a share within 4 ulp; log and its rounding
            assert want < 0 and logp[r] == -np.inf or abs(logp[r] - np.log(share)) <= 2.0 ** -20 * (1 + abs(np.log(share))), r
            continue
        held, total = rest
        a, b = sorted((int(token[r]), want))
        assert held[token[r]] > 0, (r, token[r], want)
        edge = held[:a + 1].sum() / total
        assert abs(edge - u[r]) <= 2.0 ** -20 and held[a + 1:b].sum() / total <= 2.0 ** -20, (r, token[r], want)
        loose += 1
    assert loose <= max(1, len(l) // 100), loose
    return token


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4097, 32000, 49152])
def test_against_the_definition(cuda_device, V):
    g = np.random.default_rng(V)
    l = (g.standard_normal((4, V)) * 3).astype(np.float32)
    l[1] = np.round(l[1])                                        # many ties
    l[2] = -1.4 * np.log1p(g.random(V) * V).astype(np.float32)   # a language model's
    l[3, g.random(V) < 0.5] = -np.inf
    l[3, 0] = 0.0
    draws(cuda_device, l, SETTINGS, g.random(4 * len(SETTINGS)).astype(np.float32))


def test_large_vocabulary(cuda_device):
    g = np.random.default_rng(5)
    l = (-1.4 * np.log1p(g.random((2, 128256)) * 128256) + 0.5 * g.standard_normal((2, 128256))).astype(np.float32)
    draws(cuda_device, l, SETTINGS[:8], g.random(16).astype(np.float32))


@pytest.mark.parametrize("V", [7, 5000, 70001])
def test_ties_go_to_the_lowest_index(cuda_device, V):
    """All logits equal: the kept set is a prefix of the indices, and the draw is u's share of it."""
    l = torch.full((1, V), 2.5, device=cuda_device)
    for k in (1, 3, V - 1, V):
        for u in (0.0, 0.5, 1.0 - 2.0 ** -24):
            t, p = sampling.sample(l, torch.tensor([u], device=cuda_device), top_k=k)
            assert int(t) == min(int(u * k), k - 1)
            assert abs(float(p) + np.log(k)) <= 2.0 ** -20 * (1 + np.log(k))
    t, _ = sampling.sample(l, torch.tensor([1.0 - 2.0 ** -24], device=cuda_device), top_p=0.25)
    assert int(t) == int(np.ceil(0.25 * V)) - 1


@pytest.mark.parametrize("V", [3000, 9000, 40001])
@pytest.mark.parametrize("spread", [1e-3, 0.5, 30.0])
def test_flat_and_steep_rows(cuda_device, V, spread):
    """Ends of the order in buckets with thousands of distinct logits, far below the
    maximum, and among ties of thousands."""
    g = np.random.default_rng(V)
    l = np.empty((4, V), np.float32)
    l[0] = spread * g.random(V)                                   # evenly spread
    l[1] = -spread * np.sqrt(g.random(V))                         # most of them at the far end
    l[2] = np.where(g.random(V) < 0.5, -spread, 0.0)              # two values
    l[3] = -spread * g.random(V) ** 8                             # most of them at the maximum
    s = [(1.0, 0, 0.3, 0.0), (1.0, 0, 0.97, 0.0), (1.0, V // 2, 1.0, 0.0), (0.7, V - 7, 0.5, 0.2), (3.0, 1500, 0.9, 0.0), (0.05, 700, 0.999, 0.0)]
    draws(cuda_device, l, s, g.random(4 * len(s)).astype(np.float32))


def test_special_rows(cuda_device):
    """NaN and -inf are never drawn, +inf and -0 / +0 are handled, a row without a logit gives -1."""
    nan, inf = np.nan, np.inf
    l = np.array([[nan, 1.0, nan, -inf], [nan, nan, nan, nan], [-inf] * 4, [inf, 1.0, inf, 0.0], [-0.0, 0.0, -1e30, -inf], [3e38, -3e38, 3e38, nan]],
                 np.float32)
    for s in SETTINGS:
        for u in (0.0, 0.49, 0.51, 0.99999):
            token = draws(cuda_device, l, [s], np.full(6, u, np.float32))
            assert token[0] == 1 and token[1] == token[2] == -1 and token[3] in (0, 2) and token[4] in (0, 1) and token[5] in (0, 2)


@pytest.mark.parametrize("V", [5, 3000, 40001])
@pytest.mark.parametrize("T", [1e-45, 1e-39, 2.9e-39, 2.0 ** -128, 2.0 ** -126, 1e-30])
def test_temperatures_whose_reciprocal_overflows(cuda_device, V, T):
    """Only the maxima have a mass, and they share it."""
    g = np.random.default_rng(V)
    l = (g.standard_normal((3, V)) * 3).astype(np.float32)
    l[1, g.permutation(V)[:V // 3 + 1]] = 20.0
    l[2] = -7.5
    s = [(T, k, p, m) for k in (0, 1, 3, V - 1) for p in (1.0, 0.6) for m in (0.0, 0.5, 1.0)]
    u = g.random(3 * len(s)).astype(np.float32)
    with np.errstate(over="ignore"):
        token = draws(cuda_device, l, s, u)
    top = np.tile(l == l.max(1, keepdims=True), (len(s), 1))
    assert all(0 <= t < V and top[r, t] for r, t in enumerate(token))


def test_frequencies(cuda_device):
    """Evenly spaced u visit every kept token in proportion to its share."""
    n = 4096
    g = np.random.default_rng(9)
    row = g.standard_normal(300).astype(np.float32)
    l = torch.from_numpy(np.tile(row, (n, 1))).to(cuda_device)
    u = (torch.arange(n, device=cuda_device) + 0.5) / n
    t, p = sampling.sample(l, u, temperature=0.9, top_k=50)
    t, p = t.cpu().numpy(), np.exp(p.cpu().numpy())
    kept = np.argsort(-row, kind="stable")[:50]
    w = np.exp(row[kept].astype(np.float64) / 0.9)
    for i, share in zip(kept, w / w.sum()):
        assert abs((t == i).mean() - share) <= 1.0 / n + 2.0 ** -20
    assert set(t) <= set(kept) and np.all(np.diff(t) >= 0)


def test_strided_rows_outputs_and_streams(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    l = torch.randn((8, 1111), generator=g, device=cuda_device)
    u = torch.rand(8, generator=g, device=cuda_device)
    want = sampling.sample(l[:, 5:1005].contiguous(), u, 0.9, 30, 0.9, 0.01)
    out, lp = torch.empty(8, dtype=torch.int32, device=cuda_device), torch.empty(8, device=cuda_device)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = sampling.sample(l[:, 5:1005], u, 0.9, 30, 0.9, 0.01, out=out, logprob=lp)
    s.synchronize()
    assert got[0] is out and got[1] is lp
    assert torch.equal(out, want[0]) and torch.equal(lp, want[1])


@pytest.mark.parametrize("B,V", [(1, 40001), (12, 5000)])
def test_graph_capture(cuda_device, B, V):
    g = torch.Generator(device=cuda_device).manual_seed(B)
    l, u = torch.randn((B, V), generator=g, device=cuda_device) * 3, torch.rand(B, generator=g, device=cuda_device)
    args = 0.8, 40, 0.9, 0.01
    sampling.sample(l, u, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(l, u, *args)
    for _ in range(3):
        l.copy_(torch.randn((B, V), generator=g, device=cuda_device) * 3)
        u.copy_(torch.rand(B, generator=g, device=cuda_device))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, sampling.sample(l, u, *args)))


def test_another_device_than_the_current_one(cuda_device, monkeypatch):
    g = torch.Generator(device=cuda_device).manual_seed(2)
    l, u = torch.randn((3, 500), generator=g, device=cuda_device), torch.rand(3, generator=g, device=cuda_device)
    want = sampling.sample(l, u, 0.9, 30)
    far = ref.Elsewhere(monkeypatch, sampling)
    got = sampling.sample(l, u, 0.9, 30)
    assert far.device == 7 and far.calls == [("hc_sample_uniform_dev", 0)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda_device):
    l, u = torch.zeros((2, 10), device=cuda_device), torch.zeros(2, device=cuda_device)
    with pytest.raises(TypeError):
        sampling.sample(l.half(), u)
    with pytest.raises(TypeError):
        sampling.sample(l, u[:1])
    with pytest.raises(TypeError):
        sampling.sample(l, u, top_k=torch.zeros(2, device=cuda_device))
    with pytest.raises(ValueError):
        sampling.sample(torch.zeros((10, 2), device=cuda_device).T, u)
    with pytest.raises(ValueError):
        sampling.sample(l[:, :0], u)
    with pytest.raises(ValueError):
        sampling.sample(l[:1].expand(2, 10), u)
    p = u.data_ptr()
    assert load().hc_sample_uniform_dev(l.data_ptr(), 9, 2, 10, p, p, p, p, p, p, p, None) == -1
    assert load().hc_sample_uniform_dev(None, 10, 2, 10, p, p, p, p, p, p, p, None) == -1
    assert load().hc_sample_uniform_dev(l.data_ptr(), 1 << 23, 2, 1 << 23, p, p, p, p, p, p, p, None) == -1
    assert sampling.sample(l[:0], u[:0])[0].shape == (0,)
