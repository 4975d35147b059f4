"""CPU tests of the barrier protocols of the attention kernels: each kernel's
warps as steps over modelled barriers, tensor pipe and copies, run in many
random orders.  No order may block, overrun a barrier (a waiter whose phase is
two behind would wait forever), or overwrite what is still to be read."""
from __future__ import annotations

import random
from collections import deque

import pytest


class Barrier:
    """Completes a phase after `count` arrivals."""

    def __init__(self, count=1):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def done(self, number):
        """Whether phase `number` has completed, as a wait by parity sees it."""
        assert self.phase - number <= 1, "overrun: a wait by parity would miss the phase"
        return self.phase > number


class Machine:
    """Warps as generators that yield what they wait for; the tensor pipe runs
    what was issued in order; copies land at any time."""

    def __init__(self, rng):
        self.rng, self.pipe, self.copies, self.warps = rng, deque(), [], []

    def issue(self, work):
        self.pipe.append(work)

    def copy(self, barrier, land=lambda: None):
        self.copies.append((barrier, land))

    def run(self, warps, limit=200000):
        waits = {w: None for w in warps}
        for _ in range(limit):
            if not waits and not self.pipe and not self.copies:
                return
            choices = [w for w, c in waits.items() if c is None or c()]
            if self.pipe:
                choices.append("pipe")
            if self.copies:
                choices.append("copy")
            assert choices, "blocked"
            chosen = self.rng.choice(choices)
            if chosen == "pipe":
                self.pipe.popleft()()
            elif chosen == "copy":
                barrier, land = self.copies.pop(self.rng.randrange(len(self.copies)))
                land()
                barrier.arrive()
            else:
                try:
                    waits[chosen] = next(chosen)
                except StopIteration:
                    del waits[chosen]
        raise AssertionError("not done")


class Cell:
    """A region of memory: what it holds, and how many readers still need it."""

    def __init__(self):
        self.value, self.readers = None, 0

    def write(self, value, readers):
        assert self.readers == 0, (self.value, value)
        self.value, self.readers = value, readers

    def read(self, value):
        assert self.value == value, (self.value, value)
        self.readers -= 1
        assert self.readers >= 0


def ring(machine, stages):
    full, empty, tiles = [Barrier() for _ in range(stages)], [Barrier() for _ in range(stages)], [Cell() for _ in range(stages)]

    def load(fill, readers):  # by the loading warp
        s = fill % stages
        if fill >= stages:
            yield lambda: empty[s].done(fill // stages - 1)
        machine.copy(full[s], lambda: tiles[s].write(fill, readers))

    def there(fill):
        return lambda: full[fill % stages].done(fill // stages)

    return load, there, empty, tiles


def forward(m, items, stages):
    """items: for each, the key tiles [from, to) of both query tiles."""
    load, there, empty, tiles = ring(m, stages)
    q_full, q_empty, s_full, o_done = ([Barrier() for _ in range(2)] for _ in range(4))
    p_full = [[Barrier(), Barrier()] for _ in range(2)]
    score, out = [Cell(), Cell()], [Cell(), Cell()]
    spans = []
    for item in items:
        active = [s for s in item if s[0] < s[1]]
        spans.append((min(s[0] for s in active), max(s[1] for s in active)) if active else (0, 0))

    def sees(item, i, j):
        return item[i][0] <= j < item[i][1]

    def loader():
        fills, loads = 0, [0, 0]
        for item, (first, last) in zip(items, spans):
            for i in range(2):
                if item[i][0] < item[i][1]:
                    if loads[i]:
                        yield lambda i=i: q_empty[i].done(loads[i] - 1)
                    loads[i] += 1
                    m.copy(q_full[i])
            for j in range(first, last):
                for _ in range(2):
                    yield from load(fills, sum(sees(item, i, j) for i in range(2)))
                    fills += 1

    def products():
        fill, used, done = 0, [0, 0], [0, 0]
        for item, (first, last) in zip(items, spans):
            if first == last:
                continue

            def ask(i, j, f):
                if j == item[i][0]:
                    number = used[i]
                    yield lambda: q_full[i].done(number)
                    used[i] += 1

                def work():
                    tiles[f % stages].read(f)
                    score[i].write(("s", j), 1)

                m.issue(work)
                m.issue(s_full[i].arrive)
                if j + 1 == item[i][1]:
                    m.issue(q_empty[i].arrive)

            yield there(fill)
            for i in range(2):
                if sees(item, i, first):
                    yield from ask(i, first, fill)
            m.issue(empty[fill % stages].arrive)
            for j in range(first, last):
                v, k = fill + 1, fill + 2
                yield there(v)
                more = j + 1 < last
                if more:
                    yield there(k)
                for i in range(2):
                    if sees(item, i, j):
                        for half in range(2):
                            yield lambda i=i, half=half, n=done[i]: p_full[i][half].done(n)

                        def work(i=i, j=j, v=v, start=item[i][0]):
                            score[i].read(("p", j))
                            tiles[v % stages].read(v)
                            if j == start:
                                out[i].write("o", 0)
                            out[i].value = ("o", j)

                        m.issue(work)
                        m.issue(o_done[i].arrive)
                        done[i] += 1
                    if more and sees(item, i, j + 1):
                        yield from ask(i, j + 1, k)
                m.issue(empty[v % stages].arrive)
                if more:
                    m.issue(empty[k % stages].arrive)
                fill += 2

    def softmax(i):
        done = 0
        for item in items:
            start, stop = item[i]
            for j in range(start, stop):
                yield lambda n=done: s_full[i].done(n)
                score[i].read(("s", j))
                if j > start and m.rng.random() < 0.3:  # the sums are scaled again
                    yield lambda n=done - 1: o_done[i].done(n)
                    assert out[i].value == ("o", j - 1)
                score[i].write(("p", j), 1)
                for half in range(2):
                    yield None
                    p_full[i][half].arrive()
                done += 1
            if start < stop:
                yield lambda n=done - 1: o_done[i].done(n)
                out[i].readers += 1
                yield None  # the results are read and written
                assert out[i].value == ("o", stop - 1)
                out[i].readers -= 1

    return [loader(), products(), softmax(0), softmax(1)]


def key_grads(m, items, stages):
    """items: for each, its number of tiles of queries."""
    load, there, empty, tiles = ring(m, stages)
    kv_full, kv_empty, s_full, dp_full, finished = (Barrier() for _ in range(5))
    p_done, ds_done = [Barrier(), Barrier()], [Barrier(), Barrier()]
    stat_full, stat_read, stat = [Barrier(), Barrier()], [Barrier(2), Barrier(2)], [Cell(), Cell()]
    score, dp, dv, dk, keys = [Cell(), Cell()], [Cell(), Cell()], Cell(), Cell(), Cell()

    def loader():
        fills = loads = g = 0
        for number, n in enumerate(items):
            if n == 0:
                continue
            if loads:
                yield lambda: kv_empty.done(loads - 1)
            loads += 1
            m.copy(kv_full, lambda number=number, n=n: keys.write(number, 2 * n))
            for _ in range(n):
                yield from load(fills, 2)
                if g >= 2:
                    yield lambda: stat_read[g % 2].done(g // 2 - 1)
                stat[g % 2].write(g, 4)
                stat_full[g % 2].arrive()
                yield from load(fills + 1, 2)
                fills, g = fills + 2, g + 1

    def scores(number, g, which):
        cell = score if which == 0 else dp

        def work():
            keys.read(number)
            tiles[(2 * g + which) % stages].read(2 * g + which)
            for h in range(2):
                cell[h].write(("in", g), 1)

        m.issue(work)
        m.issue((s_full if which == 0 else dp_full).arrive)

    def weighted(g, cells, barriers, to, tile, first):
        for h in range(2):
            yield lambda h=h: barriers[h].done(g)

            def work(h=h):
                cells[h].read(("out", g))
                if first and h == 0:
                    to.write(g, 0)
                to.value = g
                if h == 1:
                    tiles[tile % stages].read(tile)

            m.issue(work)

    def products():
        g = used = 0
        for number, n in enumerate(items):
            if n == 0:
                continue
            yield lambda: kv_full.done(used)
            used += 1
            yield there(2 * g)
            scores(number, g, 0)
            yield there(2 * g + 1)
            scores(number, g, 1)
            if n == 1:
                m.issue(kv_empty.arrive)
            for it in range(n):
                more = it + 1 < n
                if more:
                    yield there(2 * g + 2)
                yield from weighted(g, score, p_done, dv, 2 * g + 1, it == 0)
                if more:
                    scores(number, g + 1, 0)
                m.issue(empty[(2 * g + 1) % stages].arrive)
                if more:
                    yield there(2 * g + 3)
                yield from weighted(g, dp, ds_done, dk, 2 * g, it == 0)
                if more:
                    scores(number, g + 1, 1)
                    if it + 2 == n:
                        m.issue(kv_empty.arrive)
                else:
                    m.issue(finished.arrive)
                m.issue(empty[2 * g % stages].arrive)
                g += 1

    def half(h):
        g = used = 0
        for n in items:
            for _ in range(n):
                yield lambda: stat_full[g % 2].done(g // 2)
                stat[g % 2].read(g)
                yield lambda: s_full.done(g)
                score[h].read(("in", g))
                score[h].write(("out", g), 1)
                p_done[h].arrive()
                yield None
                stat[g % 2].read(g)
                stat_read[g % 2].arrive()
                yield lambda: dp_full.done(g)
                dp[h].read(("in", g))
                dp[h].write(("out", g), 1)
                ds_done[h].arrive()
                g += 1
            if n:
                yield lambda: finished.done(used)
                used += 1
                cell = dv if h == 0 else dk
                assert cell.value == g - 1
                cell.readers += 1
                yield None
                assert cell.value == g - 1
                cell.readers -= 1

    return [loader(), products(), half(0), half(1)]


def query_grads(m, items, stages, barriers=2):
    """items: for each, its number of tiles of keys; `barriers`: of ds, by turns."""
    load, there, empty, tiles = ring(m, stages)
    q_full, q_empty, dp_full, dp_read, finished = Barrier(), Barrier(), Barrier(), Barrier(2), Barrier()
    s_full = [Barrier(), Barrier()]
    ds_done = [[Barrier() for _ in range(barriers)] for _ in range(2)]
    score, dp, dq, rows = [[Cell(), Cell()], [Cell(), Cell()]], [Cell(), Cell()], Cell(), Cell()

    def loader():
        fills = loads = 0
        for number, n in enumerate(items):
            if n == 0:
                continue
            if loads:
                yield lambda: q_empty.done(loads - 1)
            loads += 1
            m.copy(q_full, lambda number=number, n=n: rows.write(number, 2 * n))
            for _ in range(n):
                yield from load(fills, 2)
                yield from load(fills + 1, 1)
                fills += 2

    def products():
        g = used = 0
        for number, n in enumerate(items):
            if n == 0:
                continue

            def ask(at):
                yield there(2 * at)

                def work():
                    rows.read(number)
                    tiles[2 * at % stages].read(2 * at)
                    for h in range(2):
                        score[at % 2][h].write(("in", at), 1)

                m.issue(work)
                m.issue(s_full[at % 2].arrive)

            def ask_dp(it, at):
                yield there(2 * at + 1)
                if at > 0:
                    yield lambda: dp_read.done(at - 1)

                def work():
                    rows.read(number)
                    tiles[(2 * at + 1) % stages].read(2 * at + 1)
                    for h in range(2):
                        dp[h].write(("in", at), 1)

                m.issue(work)
                m.issue(dp_full.arrive)
                m.issue(empty[(2 * at + 1) % stages].arrive)
                if it + 1 == n:
                    m.issue(q_empty.arrive)

            yield lambda: q_full.done(used)
            used += 1
            yield from ask(g)
            yield from ask_dp(0, g)
            for it in range(n):
                if it + 1 < n:
                    yield from ask(g + 1)
                    yield from ask_dp(it + 1, g + 1)
                for h in range(2):
                    yield lambda h=h: ds_done[h][g % barriers].done(g // barriers)

                    def work(h=h, at=g, first=it == 0):
                        score[at % 2][h].read(("out", at))
                        if first and h == 0:
                            dq.write(at, 0)
                        dq.value = at
                        if h == 1:
                            tiles[2 * at % stages].read(2 * at)

                    m.issue(work)
                m.issue(empty[2 * g % stages].arrive)
                if it + 1 == n:
                    m.issue(finished.arrive)
                g += 1

    def half(h):
        g = used = 0
        for n in items:
            for _ in range(n):
                yield lambda: s_full[g % 2].done(g // 2)
                score[g % 2][h].read(("in", g))
                yield lambda: dp_full.done(g)
                dp[h].read(("in", g))
                dp_read.arrive()
                yield None
                score[g % 2][h].write(("out", g), 1)
                ds_done[h][g % barriers].arrive()
                g += 1
            if n:
                yield lambda: finished.done(used)
                used += 1
                if h == 0:
                    assert dq.value == g - 1
                    dq.readers += 1
                    yield None
                    assert dq.value == g - 1
                    dq.readers -= 1

    return [loader(), products(), half(0), half(1)]


SEEDS = range(60)


@pytest.mark.parametrize("stages", [5, 8])
@pytest.mark.parametrize("seed", SEEDS)
def test_forward_protocol(stages, seed):
    rng = random.Random(seed)
    items = []
    for _ in range(rng.randint(1, 5)):
        start, width = rng.randint(0, 2), rng.randint(0, 5)
        shift = rng.choice([0, 1])
        items.append([(start, start + width), (start + shift, start + width + rng.choice([shift, 1])) if rng.random() < 0.8 else (0, 0)])
    m = Machine(rng)
    m.run(forward(m, items, stages))


@pytest.mark.parametrize("stages", [5, 8])
@pytest.mark.parametrize("seed", SEEDS)
def test_key_gradients_protocol(stages, seed):
    rng = random.Random(seed)
    m = Machine(rng)
    m.run(key_grads(m, [rng.choice([0, 1, 2, 3, 7]) for _ in range(rng.randint(1, 5))], stages))


@pytest.mark.parametrize("stages", [5, 8])
@pytest.mark.parametrize("seed", SEEDS)
def test_query_gradients_protocol(stages, seed):
    rng = random.Random(seed)
    m = Machine(rng)
    m.run(query_grads(m, [rng.choice([0, 1, 2, 3, 7]) for _ in range(rng.randint(1, 5))], stages))


def test_one_barrier_for_ds_would_be_overrun():
    """Why the queries' kernel has two: the model finds the order in which half
    of the warps is a phase ahead."""
    found = 0
    for seed in range(300):
        m = Machine(random.Random(seed))
        try:
            m.run(query_grads(m, [7, 7], 5, barriers=1))
        except AssertionError as error:
            found += "overrun" in str(error)
    assert found > 0
