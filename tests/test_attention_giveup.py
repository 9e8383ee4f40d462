"""CPU model of how the tensor-core attention kernel (csrc/attn_tc.cu) ends
when waits of it run out, under random schedules.

Only the control flow is modelled: which warp waits for what, which waits have
a limit, and the hardware barriers, which have none.  Any limited wait may run
out at any time, copies and products may never complete, and whatever happens
every role has to come to its end, with no hardware barrier arrived at twice by
a warp in one generation.  The barriers' numbers are the kernel's own, from
csrc/attn_giveup.cuh.  Planted mistakes are found.  With a clock, waits run out
by their limit alone, and rows done again (csrc/attn_rows.cuh) that take longer
than any limit make none of them run out.
"""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

PIECES = 2
CSRC = Path(__file__).resolve().parents[1] / "psp-ml_b200" / "csrc"


class Broken(AssertionError):
    pass


class Phase:
    """mbarrier: `count` arrivals complete a phase; a wait names a phase by its parity."""

    def __init__(self, count):
        self.count = self.left = count
        self.done = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1

    def passed(self, n):
        return self.done % 2 != n % 2


class Meeting:
    """A hardware barrier of `warps` warps; a generation ends with the last arrival."""

    def __init__(self, warps):
        self.warps, self.here, self.generation = warps, [], 0

    def arrive(self, who):
        if who in self.here:
            raise Broken(f"warp {who} arrived twice in one generation")
        self.here.append(who)
        if len(self.here) == self.warps:
            self.here, self.generation = [], self.generation + 1


@pytest.fixture(scope="module")
def barrier_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("giveup")
    (d / "x.cpp").write_text('#include "attn_giveup.cuh"\nextern "C" int id(int t, int h, unsigned n) '
                             "{ return pspml::prob_barrier(t, h, n); }\n")
    subprocess.run(["g++", "-std=c++17", "-D__host__=", "-D__device__=", "-I", str(CSRC), "-shared",
                    "-fPIC", "-o", str(d / "x.so"), str(d / "x.cpp")], check=True)
    return ctypes.CDLL(str(d / "x.so")).id


class Kernel:
    """items: (key tiles of A, of B, whether its pieces are joined)."""

    SLOTS = 5

    def __init__(self, items, rng, barrier_of, chance, lost, after="meet", common=True, limit=None,
                 again=0.0, again_time=0, pause=True):
        self.items, self.rng, self.barrier_of, self.chance, self.lost = (items, rng, barrier_of,
                                                                         chance, lost)
        self.after, self.common = after, common
        # Steps of the clock: a wait's limit, and rows done again at an item's end.
        self.limit, self.again, self.again_time, self.pause = limit, again, again_time, pause
        self.clock = self.busy = 0
        self.abort = False
        self.book = 0
        self.record = [None, None]
        self.q_full, self.q_empty = Phase(1), Phase(1)
        self.kv_full = [Phase(1) for _ in range(self.SLOTS)]
        self.kv_empty = [Phase(1) for _ in range(self.SLOTS)]
        self.s_full, self.o_done = [Phase(1), Phase(1)], [Phase(1), Phase(1)]
        self.item_full, self.item_empty = [Phase(1), Phase(1)], [Phase(9), Phase(9)]
        self.prob = {}
        self.group = Meeting(8)
        self.block = Meeting(10)
        self.flight = []          # copies: any order
        self.commits = []         # of the MMA warp: in order

    # What a role yields: (passed, limited).  The answer is whether it passed.
    def limited(self, bar, n):
        return (lambda: bar.passed(n)), True

    def meet(self, meeting, who):
        meeting.arrive(who)
        g = meeting.generation if who in meeting.here else meeting.generation - 1
        return (lambda: meeting.generation > g), False

    def prob_at(self, t, h, n):
        return self.prob.setdefault(self.barrier_of(t, h, n), Meeting(5))

    def take(self, it):
        """(item or None) for a warp; a generator to be delegated to."""
        if not (yield self.limited(self.item_full[it % 2], it // 2)):
            self.abort = True
            if not self.common:
                return None
            if self.book == it or self.book == -1:
                self.book = -1
                return None
        return self.record[it % 2]

    def publish(self, it, what):
        self.record[it % 2] = what
        if self.book != it and self.common:
            return False
        self.book = it + 1
        self.item_full[it % 2].arrive()
        return True

    def loader(self):
        entry = q_loads = 0
        ok = True
        for it in range(len(self.items) + 1):
            if it >= 2 and not (yield self.limited(self.item_empty[it % 2], it // 2 - 1)):
                self.abort, ok = True, False
            if self.common and (not ok or self.abort):
                self.book = -1
                break
            if not self.publish(it, self.items[it] if it < len(self.items) and ok else None):
                break
            if self.record[it % 2] is None:
                break
            n = max(self.items[it][:2])
            if n and q_loads and not (yield self.limited(self.q_empty, q_loads - 1)):
                self.abort, ok = True, False
            if n:
                q_loads += 1
                self.flight.append(self.q_full)
            for _ in range(2 * n):
                slot, turn = entry % self.SLOTS, entry // self.SLOTS
                if turn and not (yield self.limited(self.kv_empty[slot], turn - 1)):
                    self.abort, ok = True, False
                if not ok:
                    break
                self.flight.append(self.kv_full[slot])
                entry += 1
        yield self.meet(self.block, "loader")

    def mma(self):
        entry = q_items = it = 0
        done = [0, 0]

        def wait(bar, n):
            if not (yield self.limited(bar, n)):
                self.abort = True
        while True:
            item = yield from self.take(it)
            if item is None:
                break
            n = max(item[:2])
            if n:
                yield from wait(self.q_full, q_items)
                q_items += 1
                yield from wait(self.kv_full[entry % self.SLOTS], entry // self.SLOTS)
                for t in range(2):
                    if item[t]:
                        if done[t]:
                            yield from wait(self.o_done[t], done[t] - 1)
                        self.commits.append(self.s_full[t])
                self.commits.append(self.kv_empty[entry % self.SLOTS])
                if n == 1:
                    self.commits.append(self.q_empty)
                for i in range(n):
                    v, k = entry + 1, entry + 2
                    yield from wait(self.kv_full[v % self.SLOTS], v // self.SLOTS)
                    if i + 1 < n:
                        yield from wait(self.kv_full[k % self.SLOTS], k // self.SLOTS)
                    for t in range(2):
                        if i >= item[t]:
                            continue
                        for h in range(PIECES):
                            yield self.meet(self.prob_at(t, h, done[t] + i), "mma")
                        self.commits.append(self.o_done[t])
                        if t == 1 or i >= item[1]:
                            self.commits.append(self.kv_empty[v % self.SLOTS])
                        if i + 1 < item[t]:
                            yield from wait(self.o_done[t], done[t] + i)
                            self.commits.append(self.s_full[t])
                            if t == 1 or i + 1 >= item[1]:
                                self.commits.append(self.kv_empty[k % self.SLOTS])
                    if i + 2 == n:
                        self.commits.append(self.q_empty)
                    entry += 2
                for t in range(2):
                    done[t] += item[t]
            self.item_empty[it % 2].arrive()
            it += 1
        yield self.meet(self.block, "mma")

    def softmax(self, t, w):
        done = it = 0
        ok = True
        who = (t, w)
        while True:
            item = yield from self.take(it)
            if item is None:
                break
            for i in range(item[t]):
                n = done + i
                if (ok or self.after == "arrive") and not (yield self.limited(self.s_full[t], n)):
                    self.abort, ok = True, False
                for h in range(PIECES):
                    if ok or self.after == "arrive":
                        self.prob_at(t, h, n).arrive(who)
                        yield (lambda: True), False
                    else:
                        yield self.meet(self.prob_at(t, h, n), who)
            done += item[t]
            if item[t] and ok and not (yield self.limited(self.o_done[t], done - 1)):
                self.abort, ok = True, False
            if item[2]:
                yield self.meet(self.group, who)
                yield self.meet(self.group, who)
            if self.rng.random() < self.again:
                self.busy += 1
                until = self.clock + self.again_time
                yield (lambda: self.clock >= until), False
                self.busy -= 1
            self.item_empty[it % 2].arrive()
            it += 1
        yield self.meet(self.block, who)

    def complete(self):
        """One copy lands or one commit's barrier is arrived at; some never are."""
        where = [x for x in (self.flight, self.commits) if x]
        if not where:
            return False
        which = self.rng.choice(where)
        bar = which.pop(self.rng.randrange(len(which)) if which is self.flight else 0)
        if self.rng.random() >= self.lost:
            bar.arrive()
        return True

    def run(self):
        waits, slow, since = {}, {}, {}
        for r in [self.loader(), self.mma()] + [self.softmax(t, w) for t in range(2)
                                                for w in range(4)]:
            waits[r], since[r] = next(r), 0
            slow[r] = self.rng.choice([1, 1, 5, 25])

        def step(r, answer):
            try:
                waits[r], since[r] = r.send(answer), self.clock
            except StopIteration:
                del waits[r]
        while waits:
            self.clock += 1
            if self.busy and self.pause:
                since = dict.fromkeys(since, self.clock)
            roles = list(waits)
            r = self.rng.choices(roles, [slow[x] for x in roles])[0]
            passed, limited = waits[r]
            if passed():
                step(r, True)
            elif limited and (self.abort or self.rng.random() < self.chance):
                step(r, False)
            elif limited and self.limit is not None and self.clock - since[r] > self.limit:
                step(r, False)
            elif not self.complete() and not any(p() for p, _ in waits.values()):
                if self.busy:  # nothing else to do meanwhile
                    self.clock += self.again_time // 20
                    continue
                late = [x for x in waits if waits[x][1]]  # nothing will come: limits run out
                if not late:
                    raise Broken("roles wait without a limit for what does not come")
                step(self.rng.choice(late), False)


def _items(rng):
    out = []
    for _ in range(rng.randint(1, 7)):
        n1 = rng.choice([0, 1, 2, 3, 4, 6, 9])
        out.append((rng.choice([n1, n1, max(0, n1 - 1), rng.randint(0, 9)]), n1,
                    rng.random() < 0.3))
    return out


def _runs(barrier_of, seeds, **kw):
    """How many of the runs were broken, and in how many a wait ran out."""
    broken = gave_up = 0
    for seed in range(seeds):
        rng = random.Random(seed)
        k = Kernel(_items(rng), rng, barrier_of, rng.choice([0.0005, 0.003, 0.02]),
                   rng.choice([0.0, 0.0, 0.02, 0.2]), **kw)
        try:
            k.run()
        except Broken:
            broken += 1
        gave_up += k.abort
    return broken, gave_up


def test_every_role_ends_when_waits_run_out(barrier_of):
    broken, gave_up = _runs(barrier_of, 600)
    assert broken == 0 and gave_up > 250


def test_without_failures_nothing_gives_up(barrier_of):
    for seed in range(100):
        rng = random.Random(seed)
        k = Kernel(_items(rng), rng, barrier_of, 0.0, 0.0)
        k.run()
        assert not k.abort


@pytest.mark.parametrize("mistake", ["arrivals left after a failure", "one barrier for all tiles",
                                     "a book of its own for each warp"])
def test_planted_mistakes_are_found(barrier_of, mistake):
    ids, kw = barrier_of, {}
    if mistake.startswith("arrivals"):
        kw["after"] = "arrive"
    elif mistake.startswith("one"):
        def ids(t, h, n):
            return barrier_of(t, h, 0)
    else:
        kw["common"] = False
    assert _runs(ids, 200, **kw)[0] > 0


def test_barriers_are_the_hardwares_and_apart(barrier_of):
    ids = [barrier_of(t, h, n) for t in range(2) for h in range(PIECES) for n in range(2)]
    assert len(set(ids)) == 8 and min(ids) >= 2 and max(ids) < 16
    assert all(barrier_of(t, h, n) == barrier_of(t, h, n + 2)
               for t in range(2) for h in range(PIECES) for n in range(2))


@pytest.mark.parametrize("pause", [True, False])
def test_rows_done_again_outlast_the_limits(barrier_of, pause):
    gave_up = 0
    for seed in range(30):
        rng = random.Random(seed)
        k = Kernel(_items(rng), rng, barrier_of, 0.0, 0.0, limit=400000, again=0.1,
                   again_time=2000000, pause=pause)
        k.run()
        gave_up += k.abort
    assert gave_up == 0 if pause else gave_up > 0
