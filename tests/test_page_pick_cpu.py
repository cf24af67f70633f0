"""The choice of a row's pages from their keys (hc_page_select.cu, pick_pages),
restated in 32-bit arithmetic and checked by brute force on the host, no GPU: the
least key that is taken is found by histograms of 2,048 equal steps of the range
that still holds it.  Checked here: each histogram holds the key that is looked
for, the loop ends within three of them, and the pages taken are the ones of
largest keys, the lower index first among equals, never more than the budget."""
import numpy as np
import pytest

BINS = 2048
ZERO, HOLE, INF = 0x80000000, 1, 0xfffffffe
M32 = 0xffffffff


def pick(keys, n, budget, first, recent):
    scored = keys[first:n - recent].astype(np.int64)
    left = budget - first - recent
    lo, hi, above = int(scored.min()), int(scored.max()), M32
    shift = max((hi - lo).bit_length() - 11, 0)
    rounds = 0
    while left > 0:
        rounds += 1
        hist = np.bincount((scored[(scored >= lo) & (scored <= hi)] - lo) >> shift, minlength=BINS)
        assert hist.size == BINS and hist.sum() >= left, "a range without the key that is looked for"
        from_top = np.cumsum(hist[::-1])
        k = int(np.argmax(from_top >= left))
        b, held = BINS - 1 - k, int(hist[BINS - 1 - k])
        left -= int(from_top[k]) - held
        lo = lo + (b << shift) & M32
        hi = lo + min(hi - lo, (1 << shift) - 1) & M32
        if shift == 0 or held == left:
            above = lo - 1 if held == left else lo
            left = 0 if held == left else left
            break
        shift = max(shift - 11, 0)
    assert rounds <= 3
    kept = np.ones(n, bool)
    kept[first:n - recent] = scored > above
    equal = np.flatnonzero(np.append(np.zeros(first, bool), scored == above))[:left]
    kept[equal] = True
    return np.flatnonzero(kept)


def want(keys, n, budget, first, recent):
    forced = [i < first or i >= n - recent for i in range(n)]
    return sorted(sorted(range(n), key=lambda i: (not forced[i], -int(keys[i]), i))[:budget])


KINDS = {
    "finite": lambda g, n: g.integers(0x9EC00000, 0xA0000000, n),
    "close": lambda g, n: 0x9EC00000 + g.integers(0, 50, n),
    "any": lambda g, n: g.integers(2, INF, n),
    "equal": lambda g, n: np.full(n, ZERO),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("infinite", [0, 1, 10, 30, 39])
@pytest.mark.parametrize("holes", [0, 1, 20])
def test_pick(kind, infinite, holes):
    g = np.random.default_rng(infinite * 100 + holes)
    for n in (40, 64, 1000):
        for first, recent in ((0, 0), (1, 2)):
            for budget in (3, 6, 16, n - 1):
                keys = KINDS[kind](g, n).astype(np.int64)
                at = g.permutation(n)
                keys[at[:infinite]], keys[at[n - holes:]] = INF, HOLE
                assert pick(keys, n, budget, first, recent).tolist() == want(keys, n, budget, first, recent)
