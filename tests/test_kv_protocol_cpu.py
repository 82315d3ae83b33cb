"""The barriers of the prompt kernels (csrc/kv_prompt.cu), as a model on the
host: warps that meet on named barriers, wait for mbarriers with a limit, and
issue matrix products that complete in order at any later time.  Whatever the
order, every wait sees its phase and every product finds the operands that it
should; whichever waits give up, and even if no product ever completes, every
warp reaches the end, and a row whose products did not all find what they
should is marked."""
import random

import pytest

DEQUANT, SOFTMAX = "dequant", "softmax"


class Deadlock(Exception):
    pass


class Machine:
    """Warps are generators that yield one step at a time; `give_up(rng)` says whether a wait that could go on
    gives up; `stalled`: no product completes."""

    def __init__(self, rng, give_up, stalled):
        self.rng, self.give_up, self.stalled = rng, give_up, stalled
        self.named, self.mbar, self.queue, self.gave_up = {}, {}, [], False
        self.flag = False  # what the warps see of it

    late = False  # whether a warp that gave up says so at its end only

    def init(self, name, count):
        self.mbar[name] = [0, count, count]  # phases completed, arrivals missing, count

    def mbar_arrive(self, name):
        b = self.mbar[name]
        b[1] -= 1
        if b[1] == 0:
            b[0], b[1] = b[0] + 1, b[2]

    def passed(self, name, parity):
        return (self.mbar[name][0] & 1) != parity  # the phase of this parity is not the one in progress

    def run(self, warps):
        state = {w: ("go", None) for w in warps}
        while state:
            ready = []
            for w, (kind, arg) in state.items():
                if kind == "go":
                    ready.append((w, None))
                elif kind == "wait":
                    if self.passed(*arg):
                        ready.append((w, True))
                    elif self.give_up(self.rng):
                        ready.append((w, False))
            if self.queue and not self.stalled:
                ready.append((None, None))
            if not ready:
                # what is left are waits: with a limit they all give up, barriers have none
                ready = [(w, False) for w, (kind, _) in state.items() if kind == "wait"]
                if not ready:
                    raise Deadlock(dict(self.named))
            w, value = self.rng.choice(ready)
            if w is None:
                self.queue.pop(0)()
                continue
            if value is False:
                self.gave_up = True
                self.flag = self.flag or not self.late
            try:
                step = w.send(value)
            except StopIteration:
                self.flag = self.flag or self.gave_up
                del state[w]
                continue
            if step[0] in ("arrive", "sync"):
                _, name, count = step
                arrived, waiting = self.named.get(name, (0, []))
                arrived += 1
                waiting = waiting + ([w] if step[0] == "sync" else [])
                state[w] = ("blocked", name) if step[0] == "sync" else ("go", None)
                if arrived == count:
                    for x in waiting:
                        state[x] = ("go", None)
                    arrived, waiting = 0, []
                self.named[name] = (arrived, waiting)
            elif step[0] == "wait":
                state[w] = ("wait", step[1:])


class Kernel:
    apart = True  # as many barriers of a kind as arrivals may be outstanding, and one more
    meet = True   # a warp that gave up waits at its barriers

    def tell(self, ok, name, count):
        return ("arrive" if ok or not self.meet else "sync", name, count)

    def spoil(self, half, all_rows, rows=(False,) * 4):
        self.spoiled |= {(half, i) for i in range(4) if all_rows or rows[i]}

    def finish(self, ok, half, warp, complete):
        """A softmax warp is about to store its rows."""
        if ok and not self.m.flag and (not complete or (half, warp) in self.spoiled):
            self.unmarked.append((half, warp))

    def turn(self, name, j, turns, few):
        """The barrier of block j's arrival: `turns` in turn, `few` if they were no more than the waits need
        that do not give up."""
        return name, j % (turns if self.apart else few)


class Narrow(Kernel):
    """prompt_kernel: four slots (K, V, K, V), two halves.  Counts are in warps: 4 arrive, 1 takes part."""

    def __init__(self, m, blocks, two):
        self.m, self.blocks, self.two = m, blocks, two
        for i in range(4):
            m.init(("empty", i), 1)
            m.init(("mask", i), 4)
        for h in range(2):
            m.init(("s", h), 1)
        self.slots = [[None] * 4 for _ in range(4)]  # what each dequantizing warp last stored
        self.scores, self.weights = [None, None], [[None] * 4 for _ in range(2)]
        self.done, self.wrong = [], []
        self.spoiled, self.unmarked = set(), []  # (half, warp) whose rows a product took from elsewhere; and not marked

    def warps(self):
        out = [self.mma()] + [self.dequant(i) for i in range(4)]
        return out + [self.softmax(h, i) for h in range(2) for i in range(4)]

    def expect(self, have, want, what):
        if have != want:
            self.wrong.append((what, have, want))

    def mma(self):
        m, q = self.m, self.m.queue

        def qk(half, slot, j):
            def product():
                self.expect(self.slots[slot], [("K", j)] * 4, "K")
                self.spoil(half, self.slots[slot] != [("K", j)] * 4)
                self.scores[half] = j
            q.append(product)
            q.append(lambda: m.mbar_arrive(("s", half)))

        def pv(half, slot, j):
            def product():
                self.expect(self.slots[slot], [("V", j)] * 4, "V")
                self.expect(self.weights[half], [j] * 4, "P")
                self.spoil(half, self.slots[slot] != [("V", j)] * 4, [x != j for x in self.weights[half]])
                self.done.append((half, j))
            q.append(product)
        yield ("sync", "Q", 9)
        if self.blocks:
            yield ("sync", self.turn("K", 0, 4, 2), 5)
            qk(0, 0, 0)
            if self.two:
                qk(1, 0, 0)
            if self.blocks > 2:
                q.append(lambda: m.mbar_arrive(("empty", 0)))
            for j in range(self.blocks):
                v, k, more = (2 * j + 1) & 3, (2 * j + 2) & 3, j + 1 < self.blocks
                yield ("sync", self.turn("V", j, 4, 2), 5)
                if more:
                    yield ("sync", self.turn("K", j + 1, 4, 2), 5)
                for half in range(2 if self.two else 1):
                    yield ("sync", self.turn(("P", half), j, 2, 1), 5)
                    pv(half, v, j)
                    if more:
                        qk(half, k, j + 1)
                    else:
                        q.append(lambda half=half: m.mbar_arrive(("s", half)))
                if j + 2 < self.blocks:
                    q.append(lambda v=v: m.mbar_arrive(("empty", v)))
                if j + 3 < self.blocks:
                    q.append(lambda k=k: m.mbar_arrive(("empty", k)))
        yield ("sync", "end", 13)

    def dequant(self, warp):
        ok = True
        for j in range(self.blocks):
            for side, slot in (("K", (2 * j) & 3), ("V", ((2 * j) & 3) + 1)):
                if j >= 2 and ok:
                    ok = yield ("wait", ("empty", slot), ((j >> 1) - 1) & 1)
                if side == "K":
                    self.m.mbar_arrive(("mask", j % 4))
                self.slots[slot][warp] = (side, j)
                yield self.tell(ok, self.turn(side, j, 4, 2), 5)
        yield ("sync", "end", 13)

    def softmax(self, half, warp):
        ok = True
        yield ("arrive", "Q", 9)
        work = half == 0 or self.two
        for j in range(self.blocks if work else 0):
            if ok:
                ok = yield ("wait", ("mask", j % 4), (j // 4) & 1)
            if ok:
                ok = yield ("wait", ("s", half), j & 1)
            if ok and not self.m.gave_up:
                self.expect(self.scores[half], j, "S")
            self.weights[half][warp] = j
            yield self.tell(ok, self.turn(("P", half), j, 2, 1), 5)
        if work and self.blocks and ok:
            ok = yield ("wait", ("s", half), self.blocks & 1)
            if ok and not self.m.gave_up:
                self.expect((half, self.blocks - 1) in self.done, True, "O")
        if work and self.blocks:
            self.finish(ok, half, warp, (half, self.blocks - 1) in self.done)
        yield ("sync", "end", 13)


class Wide(Kernel):
    """prompt_wide_kernel: one K and one V tile with four warps each, two score buffers."""

    together = False  # whether the last P V has the others' barrier

    def __init__(self, m, blocks, two):
        self.m, self.blocks = m, blocks
        for i in range(2):
            m.init(("s", i), 1)
        m.init("o", 1)
        m.init("last", 1)
        for i in range(4):
            m.init(("mask", i), 4)
        self.tiles = {"K": [None] * 4, "V": [None] * 4}
        self.scores, self.weights = [None, None], [[None] * 4 for _ in range(2)]
        self.done, self.wrong = [], []
        self.spoiled, self.unmarked = set(), []

    expect = Narrow.expect

    def warps(self):
        return ([self.mma()] + [self.dequant(side, i) for side in "KV" for i in range(4)]
                + [self.softmax(i) for i in range(4)])

    def mma(self):
        m, q = self.m, self.m.queue

        def qk(j):
            def product():
                self.expect(self.tiles["K"], [j] * 4, "K")
                self.spoil(0, self.tiles["K"] != [j] * 4)
                self.scores[j & 1] = j
            q.append(product)
            q.append(lambda: m.mbar_arrive(("s", j & 1)))

        def pv(j):
            def product():
                self.expect(self.tiles["V"], [j] * 4, "V")
                self.expect(self.weights[j & 1], [j] * 4, "P")
                self.spoil(0, self.tiles["V"] != [j] * 4, [x != j for x in self.weights[j & 1]])
                self.done.append(j)
            q.append(product)
            q.append(lambda: m.mbar_arrive("o" if self.together or j + 1 < self.blocks else "last"))
        yield ("sync", "Q", 5)
        if self.blocks:
            yield ("sync", self.turn("K", 0, 2, 1), 5)
            qk(0)
        for j in range(self.blocks):
            if j + 1 < self.blocks:
                yield ("sync", self.turn("K", j + 1, 2, 1), 5)
                qk(j + 1)
            yield ("sync", self.turn("V", j, 2, 1), 5)
            yield ("sync", self.turn("P", j, 4, 2), 5)
            pv(j)
        yield ("sync", "end", 13)

    def dequant(self, side, warp):
        ok = True
        for j in range(self.blocks):
            if j and ok:
                if side == "V":
                    ok = yield ("wait", "o", (j - 1) & 1)
                else:
                    ok = yield ("wait", ("s", (j - 1) & 1), ((j - 1) >> 1) & 1)
            if side == "K":
                self.m.mbar_arrive(("mask", j % 4))
            self.tiles[side][warp] = j
            yield self.tell(ok, self.turn(side, j, 2, 1), 5)
        yield ("sync", "end", 13)

    def softmax(self, warp):
        ok = True
        yield ("arrive", "Q", 5)
        for j in range(self.blocks):
            if ok:
                ok = yield ("wait", ("mask", j % 4), (j // 4) & 1)
            if ok:
                ok = yield ("wait", ("s", j & 1), (j >> 1) & 1)
            if ok and not self.m.gave_up:
                self.expect(self.scores[j & 1], j, "S")
            if j and ok and self.m.rng.random() < 0.5:  # a rescale of O
                ok = yield ("wait", "o", (j - 1) & 1)
            self.weights[j & 1][warp] = j
            yield self.tell(ok, self.turn("P", j, 4, 2), 5)
        if self.together and self.blocks > 1 and ok:
            ok = yield ("wait", "o", (self.blocks - 2) & 1)
        if self.blocks and ok:
            ok = yield ("wait", "o", (self.blocks - 1) & 1) if self.together else ("wait", "last", 0)
            if ok and not self.m.gave_up:
                self.expect(self.done[-1:], [self.blocks - 1], "O")
        if self.blocks:
            self.finish(ok, 0, warp, self.done[-1:] == [self.blocks - 1])
        yield ("sync", "end", 13)


def play(kernel, seed, blocks, two, chance, stalled=False, machine=Machine):
    rng = random.Random(seed)
    m = machine(rng, lambda r: r.random() < chance, stalled)
    k = kernel(m, blocks, two)
    m.run(k.warps())
    return m, k


@pytest.mark.parametrize("kernel", [Narrow, Wide])
def test_operands_are_where_the_products_look(kernel):
    for seed in range(150):
        blocks = seed % 11
        m, k = play(kernel, seed, blocks, seed % 2, 0.0)
        assert not m.gave_up and not k.wrong, (seed, k.wrong[:3])
        assert len(k.done) == blocks * (2 if kernel is Narrow and seed % 2 else 1)
        assert all(arrived == 0 for arrived, _ in m.named.values())


class WideTogether(Wide):
    together = True


def test_one_barrier_for_all_products_would_miss_a_phase():
    """Why the last product has a barrier of its own: it may complete before a slow warp has looked for the one
    before it, whose phase is then over."""
    assert any(play(WideTogether, seed, seed % 11, 0, 0.0)[0].gave_up for seed in range(150))


@pytest.mark.parametrize("kernel", [Narrow, Wide])
@pytest.mark.parametrize("chance,stalled", [(0.002, False), (0.05, False), (0.5, False), (0.02, True), (1.0, True)])
def test_every_warp_ends_whichever_waits_give_up(kernel, chance, stalled):
    for seed in range(200):
        m, k = play(kernel, seed, seed % 13, seed % 2, chance, stalled)
        assert all(arrived == 0 for arrived, _ in m.named.values()), seed
        assert not k.unmarked, seed


def hangs(kernel):
    for seed in range(200):
        try:
            play(kernel, seed, 12, 1, 0.02)
        except Deadlock:
            return True
    return False


@pytest.mark.parametrize("base", [Narrow, Wide])
@pytest.mark.parametrize("apart,meet", [(False, False), (True, False), (False, True)])
def test_either_rule_alone_would_hang(base, apart, meet):
    """Why a warp that gave up waits at its barriers, and why they are used in turn: otherwise it can arrive
    twice before its partner, which then waits for arrivals that were counted already."""
    assert hangs(type("Planted", (base,), {"apart": apart, "meet": meet})) and not hangs(base)


class LateMachine(Machine):
    late = True


@pytest.mark.parametrize("kernel", [Narrow, Wide])
def test_said_at_the_end_only_rows_would_stay_unmarked(kernel):
    """Why a warp says that it gave up before it goes on: another may store rows made of what it wrote."""
    assert any(play(kernel, seed, 12, 1, 0.02, machine=LateMachine)[1].unmarked for seed in range(400))
