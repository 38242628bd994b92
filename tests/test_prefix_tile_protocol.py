"""The barriers of the tcgen05 tiles of shared-prefix attention (attention_prefix_tc.cu), restated as
a model and run under many schedules, on the CPU.

A barrier of the hardware tells a waiter one bit, the parity of a phase: a waiter that comes when the
next phase has ended too waits for good, and one that comes before the phase before has ended goes
on too early. So at each wait of the kernel the barrier may be neither a phase behind nor two ahead, at
any relative speed of the roles. The model has the kernel's roles (producer, issuer, two softmax
groups), copies that arrive in any order and products that end in the order of their issue; it checks
each wait, and that everything reads the block that it means."""

import random

import pytest


class Barrier:
    def __init__(self, name, count=1):
        self.name, self.count, self.pending, self.phase = name, count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count


class Late(AssertionError):
    """A wait met a barrier that had gone on by more than one phase: it would not return."""


class Model:
    """Roles are generators that yield (barrier, phase) to wait; products and copies end on their own."""

    def __init__(self, rng):
        self.rng, self.copies, self.products, self.mem = rng, [], [], {}

    # what the roles do
    def copy(self, slot, block, bar):
        self.copies.append((slot, block, bar))

    def product(self, reads, write, left=()):
        """reads: {place: content} checked when it runs; write: (place, content); left: the contents
        that the place may hold before."""
        self.products.append(("mma", reads, write, left))

    def commit(self, bar):
        self.products.append(("commit", bar))

    def put(self, place, content, over):
        assert self.mem.get(place) in over, (place, content, self.mem.get(place))
        self.mem[place] = content

    def run(self, roles):
        waits = {name: None for name in roles}
        speed = {name: self.rng.choice((0.02, 0.3, 1.0, 5.0)) for name in (*roles, "copies", "products")}
        live = dict(roles)
        while live or self.copies or self.products:
            ready = []
            for name in live:
                if waits[name] is None:
                    ready.append(name)
                else:
                    bar, phase = waits[name]
                    if bar.phase >= phase + 2:
                        raise Late(f"{name} waits for phase {phase} of {bar.name}, which is at {bar.phase}")
                    # the parity test passes when the phase in progress has the other parity
                    if bar.phase & 1 != phase & 1:
                        assert bar.phase == phase + 1, f"{name} went on before phase {phase} of {bar.name} ({bar.phase})"
                        ready.append(name)
            if self.copies:
                ready.append("copies")
            if self.products:
                ready.append("products")
            assert ready, f"nothing can go on: {[(n, w[0].name, w[1], w[0].phase) for n, w in waits.items() if w and n in live]}"
            name = self.rng.choices(ready, [speed[n] for n in ready])[0]
            if name == "copies":
                slot, block, bar = self.copies.pop(self.rng.randrange(len(self.copies)))
                self.mem[slot] = block
                bar.arrive()
            elif name == "products":
                op = self.products.pop(0)
                if op[0] == "commit":
                    op[1].arrive()
                    continue
                _, reads, (place, content), left = op
                for p, want in reads.items():
                    assert self.mem.get(p) == want, (p, want, self.mem.get(p))
                self.put(place, content, left)
            else:
                try:
                    waits[name] = next(live[name])
                except StopIteration:
                    del live[name]


def pair(m, nb, groups, slots_by_scores):
    """Tiles of 256 rows: each group has its own rows, its scores are overwritten by their weights.
    slots_by_scores: the producer waits for the last group's barriers, which pass at every block (what
    the kernel must not do), instead of one barrier per slot."""
    kfull, vfull, kfree, vfree = ([Barrier(f"{n}{i}") for i in range(2)] for n in ("kfull", "vfull", "kfree", "vfree"))
    sready, pvdone = ([Barrier(f"{n}{g}") for g in range(2)] for n in ("sready", "pvdone"))
    pready = [[Barrier(f"pready{g}{h}") for h in range(2)] for g in range(2)]
    last = groups - 1
    used = {}  # products that still have to read a slot's block

    def producer():
        def load(what, full, i):
            if i >= 2:
                assert used.get((what, i - 2), 0) == groups
            m.copy((what, i & 1), i, full[i & 1])

        def load_k(i):
            if i >= 2:
                yield (sready[last], i - 2) if slots_by_scores else (kfree[i & 1], (i >> 1) - 1)
            load("k", kfull, i)

        def load_v(i):
            if i >= 2:
                yield (pvdone[last], i - 2) if slots_by_scores else (vfree[i & 1], (i >> 1) - 1)
            load("v", vfull, i)

        yield from load_k(0)
        for i in range(nb):
            yield from load_v(i)
            if i + 1 < nb:
                yield from load_k(i + 1)

    def done(what, i):
        used[(what, i)] = used.get((what, i), 0) + 1

    def issuer():
        def scores(g, i):
            m.product({("k", i & 1): i}, (("s", g), ("scores", i)), [None] if i == 0 else [("used", i - 1)])
            m.commit(_Note(lambda: done("k", i)))
            m.commit(sready[g])
            if g == last and i + 2 < nb:
                m.commit(kfree[i & 1])

        def weigh(g, i):
            for h in range(2):
                yield (pready[g][h], i)
                want = ("weights", i) if h else m.mem.get(("s", g))
                assert want in (("half", i), ("weights", i))
                m.product({("v", i & 1): i}, (("o", g), i), [None, i, i - 1])
            m.product({("s", g): ("weights", i)}, (("s", g), ("used", i)), [("weights", i)])
            m.commit(_Note(lambda: done("v", i)))
            m.commit(pvdone[g])
            if g == last and i + 2 < nb:
                m.commit(vfree[i & 1])

        yield (kfull[0], 0)
        for g in range(groups):
            scores(g, 0)
        yield (vfull[0], 0)
        for i in range(nb):
            for g in range(groups):
                yield from weigh(g, i)
                if g == 0 and i + 1 < nb:
                    yield (kfull[(i + 1) & 1], (i + 1) >> 1)
                if i + 1 < nb:
                    yield (pvdone[g], i)
                    scores(g, i + 1)
                    if g == last:
                        yield (vfull[(i + 1) & 1], (i + 1) >> 1)

    def group(g):
        for i in range(nb):
            yield (sready[g], i)
            m.put(("s", g), ("half", i), [("scores", i)])
            pready[g][0].arrive()
            yield from pause()
            if i == nb - 1:  # the last block's V rows past the range are zeroed in shared memory
                yield (vfull[i & 1], i >> 1)
                assert m.mem[("v", i & 1)] == i
            m.put(("s", g), ("weights", i), [("half", i)])
            pready[g][1].arrive()
        yield (pvdone[g], nb - 1)
        assert m.mem[("s", g)] == ("used", nb - 1)

    return {"producer": producer(), "issuer": issuer(), **{f"group {g}": group(g) for g in range(groups)}}


def single(m, nb, parity_buffers=False):
    """Tiles of 128 rows: the groups take alternate blocks, whose scores and then weights lie in one of
    three buffers in turn. parity_buffers: barriers and buffers by the block's parity instead (what the
    kernel must not do: block i + 2's scores would overwrite weights in use)."""
    nbuf = 2 if parity_buffers else 3
    kfull, vfull = ([Barrier(f"{n}{i}") for i in range(2)] for n in ("kfull", "vfull"))
    sready, pvdone = ([Barrier(f"{n}{b}") for b in range(nbuf)] for n in ("sready", "pvdone"))
    pready = [[Barrier(f"pready{b}{h}") for h in range(2)] for b in range(nbuf)]
    refset = [Barrier(f"refset{g}") for g in range(2)]
    state = {"k": -1, "v": -1, "ref": -1}  # last block whose products have read K, V; that set the scale

    def at(bars, i):
        return bars[i % nbuf], i // nbuf

    def producer():
        def load_k(i):
            if i >= 2:
                yield at(sready, i - 2)
                assert state["k"] >= i - 2
            m.copy(("k", i & 1), i, kfull[i & 1])

        def load_v(i):
            if i >= 2:
                yield at(pvdone, i - 2)
                assert state["v"] >= i - 2
            m.copy(("v", i & 1), i, vfull[i & 1])

        yield from load_k(0)
        for i in range(nb):
            if i + 1 < nb:
                yield from load_k(i + 1)
            yield from load_v(i)

    def issuer():
        def scores(i):
            m.product({("k", i & 1): i}, (("s", i % nbuf), ("scores", i)), [None, ("used", i - nbuf)])
            m.commit(_Note(lambda: state.update(k=i)))
            m.commit(sready[i % nbuf])

        def weigh(i):
            bar, phase = at(pready, i)
            for h in range(2):
                yield (bar[h], phase)
                assert m.mem[("s", i % nbuf)] in ([("weights", i)] if h else [("half", i), ("weights", i)])
                m.product({("v", i & 1): i}, ("o", (i, h)), [(i - 1, 1) if i else None] if h == 0 else [(i, 0)])
            m.product({("s", i % nbuf): ("weights", i)}, (("s", i % nbuf), ("used", i)), [("weights", i)])
            m.commit(_Note(lambda: state.update(v=i)))
            m.commit(pvdone[i % nbuf])

        yield (kfull[0], 0)
        scores(0)
        if nb > 1:
            yield (kfull[1], 0)
            scores(1)
        yield (vfull[0], 0)
        for i in range(nb):
            if i + 2 < nb:
                yield (kfull[(i + 2) & 1], (i + 2) >> 1)
                if i > 0:
                    yield at(pvdone, i - 1)
                scores(i + 2)
            yield from weigh(i)
            if i + 1 < nb:
                yield (vfull[(i + 1) & 1], (i + 1) >> 1)

    def group(g):
        mine = range(g, nb, 2)
        for k, i in enumerate(mine):
            yield at(sready, i)
            assert m.mem[("s", i % nbuf)] == ("scores", i)
            if i > 0:
                yield (refset[1 - g], k if g else k - 1)
            assert state["ref"] == i - 1
            state["ref"] = i
            refset[g].arrive()
            if i > 0 and m.rng.random() < 0.5:  # the scale moves: every product before is in the accumulator
                yield at(pvdone, i - 1)
                assert m.mem["o"] == (i - 1, 1)
            m.put(("s", i % nbuf), ("half", i), [("scores", i)])
            bar, _ = at(pready, i)
            bar[0].arrive()
            yield from pause()
            if i == nb - 1:
                yield (vfull[i & 1], i >> 1)
                assert m.mem[("v", i & 1)] == i
            m.put(("s", i % nbuf), ("weights", i), [("half", i)])
            bar[1].arrive()
        if len(mine):
            yield at(pvdone, mine[-1])
            assert state["v"] >= mine[-1]

    return {"producer": producer(), "issuer": issuer(), "group 0": group(0), "group 1": group(1)}


class _Note:
    """Something noted when the products before it have ended."""

    def __init__(self, f):
        self.arrive = f


def pause():
    b = Barrier("pause")
    b.arrive()
    yield (b, 0)


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("nb", [1, 2, 3, 4, 5, 8, 13])
def test_tiles_of_256_rows(nb, groups):
    for seed in range(150):
        m = Model(random.Random(1000 * nb + seed))
        m.run(pair(m, nb, groups, False))


@pytest.mark.parametrize("nb", [1, 2, 3, 4, 5, 6, 7, 8, 13])
def test_tiles_of_128_rows(nb):
    for seed in range(300):
        m = Model(random.Random(5000 * nb + seed))
        m.run(single(m, nb))


def test_the_model_sees_too_few_buffers():
    """Two buffers for three blocks under way: overwritten weights, or a wait that is late or early."""
    wrong = 0
    for seed in range(300):
        m = Model(random.Random(seed))
        try:
            m.run(single(m, 8, True))
        except AssertionError:
            wrong += 1
    assert wrong > 0


def test_the_model_sees_a_barrier_that_passes_every_block():
    """The producer on the last group's own barriers: some schedule leaves it two phases behind."""
    late = 0
    for seed in range(300):
        m = Model(random.Random(seed))
        try:
            m.run(pair(m, 8, 2, True))
        except Late as e:
            assert "producer" in str(e)
            late += 1
    assert late > 0


@pytest.mark.parametrize("groups", [1, 2])
def test_nothing_runs_on_after_the_issuer_has_left(groups):
    """The issuer gives up at any of its waits, for whatever reason: its last commit comes after every
    product, those of a half block among them, and it leaves when that has passed."""
    for stop in range(40):
        m, drain = Model(random.Random(stop)), Barrier("drain")
        m.put = lambda *a: None  # what the products read no longer matters
        roles = pair(m, 6, groups, False)

        def issuer(role=roles["issuer"], stop=stop):
            for n, w in enumerate(role):
                if n == stop:
                    break
                w[0].phase = w[1] + 1  # as if it had come
                yield pause_at()
            m.commit(drain)
            yield (drain, 0)
            assert not m.products
            done.append(stop)

        done = []
        m.mem = _Anything()
        m.run({"issuer": issuer()})
        assert done == [stop]


def pause_at():
    b = Barrier("pause")
    b.arrive()
    return (b, 0)


class _Anything(dict):
    def get(self, place, default=None):
        return _Any()


class _Any:
    def __eq__(self, other):
        return True
