"""How the copying warp and the four that compute hand pairs to one another in the
attention over 4 bits (hc_paged_q4_stream.cu, k_paged_q4), restated as a copying
process and four others over the CTA's barriers and a ring of stages, and run under
random schedules on the host, no GPU.  The bounded waits (for copies, for a free stage)
may run out at any time.  Checked here: every run ends; each process sees every
pair, whole, and its rows are finished: with a number if all its stages came, else
with NaN, also by a process whose own waits held; no barrier is left half full."""
import random

import pytest

S, ROWS, ALL = 3, 4, 5
TOLD, READ = 2, 4


class Cta:
    def __init__(self, pairs, fail, rng):
        self.pairs, self.fail, self.rng = pairs, fail, rng       # stages of each pair
        self.bars = {}
        self.full, self.empty = [0] * S, [0] * S                   # completed phases
        self.arrived = [0] * S
        self.abort = False
        self.work = [None, None]
        self.out = [[] for _ in range(ROWS)]

    def arrive(self, i):
        n = self.bars.setdefault(i, [0, 0])                        # arrivals, completed phases
        n[0] += 1
        if n[0] == ALL:
            n[0], n[1] = 0, n[1] + 1

    def sync(self, i):
        phase = self.bars.setdefault(i, [0, 0])[1]
        self.arrive(i)
        while self.bars[i][1] == phase:
            yield

    def wait(self, done):
        """A bounded wait: false once it has run out, or another one has."""
        while not done():
            if self.abort or self.rng.random() < self.fail:
                self.abort = True
                return False
            yield
        return True

    def copies(self):
        n, told, ok = 0, 0, True
        for pair in [*range(len(self.pairs)), None]:
            stages = -1 if pair is None else self.pairs[pair] if ok else 0
            if told >= 2:
                yield from self.sync(READ + (told & 1))
            self.work[told & 1] = None                             # (being written)
            yield
            self.work[told & 1] = (pair, stages, not ok)
            self.arrive(TOLD + (told & 1))
            told += 1
            for _ in range(stages if ok else 0):
                st = n % S
                if n >= S:
                    ok = yield from self.wait(lambda: self.empty[st] >= n // S)
                    if not ok:
                        break
                self.full[st] += 1
                n += 1
                yield
        if told >= 2:
            yield from self.sync(READ + (told & 1))

    def rows(self, warp):
        n, lost, pairs = 0, False, 0
        while True:
            yield from self.sync(TOLD + (pairs & 1))
            pair, stages, gone = self.work[pairs & 1]
            if stages < 0:
                return
            lost |= gone
            came = 0
            for _ in range(stages):
                st = n % S
                if not lost:
                    lost = not (yield from self.wait(lambda: self.full[st] > n // S))
                yield
                came += not lost
                self.arrived[st] += 1
                if self.arrived[st] == ROWS:
                    self.arrived[st], self.empty[st] = 0, self.empty[st] + 1
                n += 1
            assert self.work[pairs & 1] == (pair, stages, gone)
            self.out[warp].append((pair, "nan" if lost else came))
            self.arrive(READ + (pairs & 1))
            pairs += 1


@pytest.mark.parametrize("fail", [0.0, 1e-3, 0.02, 0.3])
@pytest.mark.parametrize("pairs", [[], [1], [0, 0, 0], [5], [1, 7, 0, 2, 9], [4] * 8])
def test_every_pair_is_answered(pairs, fail):
    for seed in range(60):
        rng = random.Random(seed)
        c = Cta(pairs, fail, rng)
        live = [c.copies(), *(c.rows(w) for w in range(ROWS))]
        for _ in range(200000):
            if not live:
                break
            p = rng.choice(live)
            try:
                next(p)
            except StopIteration:
                live.remove(p)
        assert not live, "a process that waits for good"
        assert all(n == 0 for n, _ in c.bars.values())
        for out in c.out:
            assert [p for p, _ in out] == list(range(len(pairs)))
            assert all(v == "nan" or v == pairs[p] for p, v in out)
            assert c.abort or all(v != "nan" for _, v in out)
