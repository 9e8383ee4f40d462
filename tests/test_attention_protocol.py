"""CPU model of the barrier protocol of the tensor-core attention kernel
(csrc/attn_tc.cu) under random schedules.

The roles are coroutines that run between their waits in any order; TMA loads
and MMAs complete at any later time, MMAs on different accumulators in any
order (the same accumulator's in issue order, which is all that the hardware
promises).  Every buffer knows what it holds and which unfinished operations
use it, so the model reports a deadlock, a wait that returns for the wrong
phase (its reader then finds the wrong contents), and every read or write
that overlaps an operation still in flight.  Planting a mistake (a dropped
wait, a wrong arrival count) makes it fail.
"""
import random

import pytest

PIECES = 2


class Broken(AssertionError):
    pass


class Barrier:
    """mbarrier: `count` arrivals complete a phase; a wait names the parity of the phase it
    waits for and passes when the current phase has the other one."""

    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return self.phase % 2 != parity % 2


class Meeting:
    """A named hardware barrier: `arrivals` calls of arrive() let one waiter pass."""

    def __init__(self, arrivals):
        self.need, self.got = arrivals, 0

    def arrive(self):
        self.got += 1
        if self.got > self.need:
            raise Broken("a named barrier was arrived at twice in one generation")

    def passed(self):
        return self.got == self.need


class Buffer:
    def __init__(self, name):
        self.name, self.holds = name, None
        self.readers, self.writers = 0, 0

    def read(self, want):
        if self.writers:
            raise Broken(f"{self.name} read while it is written")
        if self.holds != want:
            raise Broken(f"{self.name} holds {self.holds}, {want} was expected")

    def write(self, what):
        if self.writers or self.readers:
            raise Broken(f"{self.name} written while it is in use")
        self.holds = what


class Kernel:
    def __init__(self, items, slots, rng, drop=(), empty_count=9, rescale=0.3):
        self.items, self.n_slots, self.rng, self.drop = items, slots, rng, set(drop)
        self.rescale = rescale
        self.q = Buffer("Q")
        self.slots = [Buffer(f"slot {i}") for i in range(slots)]
        self.s = [Buffer(f"S of {t}") for t in range(2)]       # all of S
        self.p = [[Buffer(f"P {h} of {t}") for h in range(PIECES)] for t in range(2)]
        self.o = [Buffer(f"O of {t}") for t in range(2)]
        self.record = [None, None]
        self.q_full, self.q_empty = Barrier(1), Barrier(1)
        self.kv_full = [Barrier(1) for _ in range(slots)]
        self.kv_empty = [Barrier(1) for _ in range(slots)]
        self.s_full = [Barrier(1) for _ in range(2)]
        self.o_done = [Barrier(1) for _ in range(2)]
        self.item_full = [Barrier(1) for _ in range(2)]
        self.item_empty = [Barrier(empty_count) for _ in range(2)]
        # Four softmax warps a tile; the model's warps move one by one.
        self.prob = [[Meeting(4) for _ in range(PIECES)] for _ in range(2)]
        self.flight = []      # operations under way: [done?, finish, group, predecessors]
        self.outputs = {}

    # ---------------------------------------------------------- async work
    def launch(self, start, finish, after=()):
        op = {"started": False, "done": False, "start": start, "finish": finish,
              "after": list(after)}
        self.flight.append(op)
        return op

    def step_flight(self):
        ready = [op for op in self.flight if not op["done"] and
                 (op["started"] or all(a["done"] for a in op["after"]))]
        if not ready:
            return False
        op = self.rng.choice(ready)
        if not op["started"]:
            op["start"]()
            op["started"] = True
        else:
            op["finish"]()
            op["done"] = True
            self.flight.remove(op)
        return True

    def load(self, buf, what, bar):
        if buf.readers or buf.writers:
            raise Broken(f"{buf.name} loaded while it is in use")
        buf.writers += 1

        def finish():
            buf.writers -= 1
            buf.holds = what
            bar.arrive()
        self.launch(lambda: None, finish)

    # --------------------------------------------------------------- roles
    def producer(self):
        entry = q_loads = 0
        for it in range(len(self.items) + 1):
            if it >= 2:
                yield lambda: self.item_empty[it % 2].passed(it // 2 - 1)
            if it == len(self.items):
                self.record[it % 2] = None
                self.item_full[it % 2].arrive()
                return
            self.record[it % 2] = it
            self.item_full[it % 2].arrive()
            n = max(self.items[it])
            if n == 0:
                continue
            if q_loads and "q_empty" not in self.drop:
                yield lambda: self.q_empty.passed(q_loads - 1)
            self.load(self.q, it, self.q_full)
            q_loads += 1
            for i in range(n):
                for kind in "KV":
                    slot, turn = entry % self.n_slots, entry // self.n_slots
                    if "kv_empty" not in self.drop:
                        yield lambda: self.kv_empty[slot].passed(turn - 1) if turn else True
                    self.load(self.slots[slot], (kind, it, i), self.kv_full[slot])
                    entry += 1

    def mma(self):
        issued = []                       # every operation of this thread
        last = {}                         # accumulator -> its last operation
        done = [0, 0]
        entry, q_items = 0, 0

        def run(acc, reads, write, result):
            """An MMA: holds its operands from start to finish; same accumulator in order."""
            def start():
                for buf, want in reads:
                    buf.read(want)
                    buf.readers += 1
                if write.writers or write.readers:
                    raise Broken(f"{write.name} accumulated while it is in use")
                write.writers += 1

            def finish():
                for buf, _ in reads:
                    buf.readers -= 1
                write.writers -= 1
                write.holds = result(write.holds)
            op = self.launch(start, finish, [last[acc]] if acc in last else [])
            last[acc] = op
            issued.append(op)

        def commit(bar):
            waiting = [op for op in issued if not op["done"]]
            self.launch(lambda: None, bar.arrive, waiting)

        def qk(t, it, i, slot, free):
            def start_s(_):
                return ("S", it, i)
            # S lies over both pieces of P: writing it needs them read.
            for piece in self.p[t]:
                if piece.writers or piece.readers:
                    raise Broken(f"{piece.name} overwritten by the next scores while in use")
            run(("S", t), [(self.q, it), (self.slots[slot], ("K", it, i))], self.s[t], start_s)
            commit(self.s_full[t])
            if free:
                commit(self.kv_empty[slot])

        for it in range(len(self.items) + 1):
            yield lambda: self.item_full[it % 2].passed(it // 2)
            if self.record[it % 2] is None:
                break
            if self.record[it % 2] != it:
                raise Broken("the MMA warp took the wrong item")
            n0, n1 = self.items[it]
            n = max(n0, n1)
            if n > 0:
                yield lambda: self.q_full.passed(q_items)
                q_items += 1
                slot = entry % self.n_slots
                yield lambda: self.kv_full[slot].passed(entry // self.n_slots)
                for t in range(2):
                    if self.items[it][t] == 0:
                        continue
                    if done[t] and "o_done" not in self.drop:
                        yield lambda: self.o_done[t].passed(done[t] - 1)
                    qk(t, it, 0, slot, not (t == 0 and n1 > 0))
                if n == 1:
                    commit(self.q_empty)
                for i in range(n):
                    v, k = entry + 2 * i + 1, entry + 2 * i + 2
                    yield lambda: self.kv_full[v % self.n_slots].passed(v // self.n_slots)
                    if i + 1 < n:
                        yield lambda: self.kv_full[k % self.n_slots].passed(k // self.n_slots)
                    for t in range(2):
                        nt, other = self.items[it][t], n1 if t == 0 else 0
                        if i >= nt:
                            continue
                        for h in range(PIECES):
                            yield self.prob[t][h].passed
                            self.prob[t][h].got = 0

                            def add(old, it=it, i=i, h=h):
                                want = None if i == 0 and h == 0 else \
                                    ("O", it, i, h - 1) if h else ("O", it, i - 1, PIECES - 1)
                                if want is not None and old != want:
                                    raise Broken(f"O holds {old} instead of {want}")
                                return ("O", it, i, h)
                            run(("O", t), [(self.p[t][h], ("P", it, i)),
                                           (self.slots[v % self.n_slots], ("V", it, i))],
                                self.o[t], add)
                        commit(self.o_done[t])
                        if i >= other:
                            commit(self.kv_empty[v % self.n_slots])
                        if i + 1 >= nt:
                            continue
                        if "o_done" not in self.drop:
                            yield lambda: self.o_done[t].passed(done[t] + i)
                        qk(t, it, i + 1, k % self.n_slots, i + 1 >= other)
                    if i + 2 == n:
                        commit(self.q_empty)
                entry += 2 * n
                done[0] += n0
                done[1] += n1
            self.item_empty[it % 2].arrive()

    def softmax(self, t, warp):
        """One of a tile's four warps: its rows of S, P and O are its own, so the first warp
        stands for the contents and the others for their arrivals."""
        done = 0
        first = warp == 0
        for it in range(len(self.items) + 1):
            yield lambda: self.item_full[it % 2].passed(it // 2)
            if self.record[it % 2] is None:
                return
            if self.record[it % 2] != it:
                raise Broken("a softmax warp took the wrong item")
            nt = self.items[it][t]
            for i in range(nt):
                yield lambda: self.s_full[t].passed(done + i)
                if first:
                    self.s[t].read(("S", it, i))
                    if i > 0 and self.rng.random() < self.rescale:
                        self.o[t].read(("O", it, i - 1, PIECES - 1))
                        self.o[t].write(("O", it, i - 1, PIECES - 1))
                yield lambda: True
                for h in range(PIECES):
                    if first:
                        if self.s[t].writers:
                            raise Broken("P written while the next scores are")
                        self.p[t][h].write(("P", it, i))
                    self.prob[t][h].arrive()
                    yield lambda: True
            done += nt
            if nt > 0:
                yield lambda: self.o_done[t].passed(done - 1)
                if first:
                    self.o[t].read(("O", it, nt - 1, PIECES - 1))
                yield lambda: True
                if first:  # still there at the end of the epilogue
                    self.o[t].read(("O", it, nt - 1, PIECES - 1))
            if first:
                self.outputs[it, t] = nt
            self.item_empty[it % 2].arrive()

    def run(self):
        roles = [self.producer(), self.mma()] + [self.softmax(t, w) for t in range(2)
                                                 for w in range(4)]
        waits = {}
        for r in roles:
            waits[r] = next(r, None)
        roles = [r for r in roles if waits[r] is not None]
        # A few speeds, so that some role lags far behind in some runs.
        speed = {r: self.rng.choice([1, 1, 4, 16]) for r in roles}
        while roles:
            ready = [r for r in roles if waits[r]()]
            moved = False
            if ready and self.rng.random() < 0.6:
                r = self.rng.choices(ready, [speed[x] for x in ready])[0]
                waits[r] = next(r, None)
                if waits[r] is None:
                    roles.remove(r)
                moved = True
            else:
                moved = self.step_flight()
            if not moved and not ready and not self.step_flight():
                raise Broken("deadlock")
        while self.step_flight():
            pass
        want = {(it, t): n for it, pair in enumerate(self.items) for t, n in enumerate(pair)}
        if self.outputs != want:
            raise Broken("an output is missing")


def _items(rng):
    items = []
    for _ in range(rng.randint(1, 6)):
        n1 = rng.choice([0, 1, 2, 3, 5, 8])
        n0 = rng.choice([n1, n1, max(0, n1 - 1), rng.randint(0, 8)])
        items.append((n0, n1))
    return items


@pytest.mark.parametrize("slots", [5, 8, 4, 3])
def test_protocol_under_random_schedules(slots):
    for seed in range(150):
        rng = random.Random(1000 * slots + seed)
        Kernel(_items(rng), slots, rng).run()


@pytest.mark.parametrize("drop", ["o_done", "q_empty", "kv_empty"])
def test_a_dropped_wait_is_found(drop):
    found = 0
    for seed in range(60):
        rng = random.Random(seed)
        try:
            Kernel([(4, 5), (3, 3), (6, 6)], 5, rng, drop=[drop]).run()
        except Broken:
            found += 1
    assert found > 0


def test_a_wrong_arrival_count_is_found():
    with pytest.raises(Broken):
        for seed in range(20):
            Kernel([(2, 2)] * 6, 5, random.Random(seed), empty_count=10).run()
