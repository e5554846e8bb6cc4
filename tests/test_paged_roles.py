"""CPU: the order in which the warps of the paged attention's kernel for many
rows (csrc/paged_attn_tc.cu) wait on one another, on a model of them.

The roles are generators that run, in a random order, whenever what they wait
for has come: loads, queries and edges, the issue of the products, the softmax
of the two tiles of rows; the tensor cores and the bulk copies finish what was
issued some time later, each issuing thread's products in order.  A barrier
shows only the parity of its phase, as the hardware's does, so a wait that is a
whole phase late or early is not told apart from the right one.  Checked: every
wait ends; and whatever is read -- a tile of the ring, queries, scores, weights,
the output, a job -- is the one meant and whole.

Planted mistakes show that the model finds them."""

import random

import pytest

JOBS = 3  # slots for pieces of work


class Barrier:
    """Arrivals of a phase; a wait names the phase's parity."""

    def __init__(self, count):
        self.count, self.arrived, self.phase = count, 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.arrived, self.phase = 0, self.phase + 1

    def passed(self, phase):
        return lambda: (self.phase & 1) != (phase & 1)


class NamedBarrier:
    """Two groups meet; a group that passes without waiting arrives only."""

    def __init__(self):
        self.arrived, self.met = 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == 2:
            self.arrived, self.met = 0, self.met + 1

    def sync(self):
        met = self.met
        self.arrive()
        return lambda: self.met > met


class Wrong(Exception):
    pass


def expect(condition, what):
    if not condition:
        raise Wrong(what)


class Kernel:
    """One CTA's roles over a list of pieces.  narrow: heads of 64 (a thread
    that issues for each tile, V and K of a slot of the ring share a barrier,
    weights in columns of their own, turns at the exponentials); otherwise heads
    of 128."""

    def __init__(self, narrow, pieces, rng, mistake=None):
        self.narrow, self.pieces, self.rng, self.mistake = narrow, pieces, rng, mistake
        self.issuers = 2 if narrow else 1
        self.ring = 6 if narrow else 5
        self.full = [Barrier(1) for _ in range(self.ring)]
        self.empty = [Barrier(self.issuers) for _ in range(self.ring)]
        pair = lambda: [Barrier(1), Barrier(1)]  # noqa: E731 (one a tile of rows)
        self.q_full, self.q_free, self.s_full, self.s_free = pair(), pair(), pair(), pair()
        self.p_full, self.pv_done = pair(), pair()
        self.edge_in, self.edge = Barrier(self.issuers), Barrier(1)
        readers = 2 + self.issuers + 1 + (0 if narrow else 1)
        self.job_full = [Barrier(1) for _ in range(JOBS)]
        self.job_empty = [Barrier(readers) for _ in range(JOBS)]
        self.turns, self.both = [NamedBarrier(), NamedBarrier()], NamedBarrier()
        self.jobs = [None] * JOBS
        # what memory holds: (step's V, step's K) in the ring, a piece's queries,
        # counts of scores, weights and products by tile
        self.slots = [(None, None)] * self.ring
        self.queries = [None, None]
        self.scores, self.taken, self.weights, self.products = [0, 0], [0, 0], [0, 0], [0, 0]
        self.zeroed = set()
        self.copies = []
        self.tensor = [[] for _ in range(self.issuers)]
        first = 0
        for i, piece in enumerate(pieces):
            piece["index"], piece["first"] = i, first  # steps counted over all pieces
            first += piece["steps"]

    # ---- roles
    def next_job(self, turn):
        yield self.job_full[turn % JOBS].passed(turn // JOBS)
        job = self.jobs[turn % JOBS]
        expect((job or {"index": len(self.pieces)})["index"] == turn, "a job of another turn")
        return job

    def load(self):
        turn = 0

        def claim(content):
            nonlocal turn
            slot = turn % self.ring
            if self.mistake != "ring not waited for":
                yield self.empty[slot].passed(turn // self.ring + 1)
            self.slots[slot] = (None, None)

            def landed():
                self.slots[slot] = content
                self.full[slot].arrive()

            self.copies.append(landed)
            turn += 1

        def step(v, k):
            if self.narrow:
                yield from claim((v, k))
            else:
                yield from claim((v, None))
                yield from claim((None, k))

        before = None
        for made, piece in enumerate(self.pieces + [None]):
            if piece is None and before is not None:
                yield from step(before, None)
            yield self.job_empty[made % JOBS].passed(made // JOBS + 1)
            self.jobs[made % JOBS] = piece
            self.job_full[made % JOBS].arrive()
            for j in range(piece["steps"] if piece else 0):
                yield from step(before, piece["first"] + j)
                before = piece["first"] + j

    def edges(self, tiles, zeroes):
        """Queries of the tiles, then rows of V that must not count."""
        made, edges, turn = [0, 0], 0, 0
        while True:
            job = yield from self.next_job(turn)
            if job is None:
                return
            for w in tiles:
                if job["from"][w] == job["to"][w]:
                    continue
                if made[w] > 0 and self.mistake != "queries not waited for":
                    yield self.q_free[w].passed(made[w] - 1)
                made[w] += 1
                self.queries[w] = None
                yield lambda: True
                self.queries[w] = job["index"]
                self.q_full[w].arrive()
            for j in sorted(job["edges"]) if zeroes else ():
                yield self.edge_in.passed(edges)
                edges += 1
                expect(any(v == job["first"] + j for v, _ in self.slots), "V to zero is not there")
                self.zeroed.add(job["first"] + j)
                self.edge.arrive()
            self.job_empty[turn % JOBS].arrive()
            turn += 1

    def issue(self, i):
        tiles = [i] if self.narrow else [0, 1]
        tensor = self.tensor[i]
        turn, job_turn, edges = 0, 0, 0
        queries, used, made = [0, 0], [0, 0], [0, 0]
        on, at_edge, v_step = [False, False], False, None

        def edge():
            nonlocal edges
            if at_edge:
                self.edge_in.arrive()
                edges += 1
                if self.mistake != "edge not waited for":
                    yield self.edge.passed(edges - 1)

        def product(w, slot):
            if not on[w]:
                return
            n, step, zero = used[w], v_step, at_edge
            used[w] += 1
            if self.mistake != "weights not waited for":
                yield self.p_full[w].passed(n)

            def run():
                expect(self.weights[w] == n + 1, "weights")
                expect(self.slots[slot][0] == step, "V")
                expect(not zero or step in self.zeroed, "V with rows that must not count")
                self.products[w] = n + 1
                self.pv_done[w].arrive()

            tensor.append(run)

        def score(w, j, job, slot):
            if not job["from"][w] <= j < job["to"][w]:
                return
            if j == job["from"][w]:
                queries[w] += 1
                yield self.q_full[w].passed(queries[w] - 1)
            if self.narrow and made[w] > 0 and self.mistake != "scores not waited for":
                yield self.s_free[w].passed(made[w] - 1)
            n, step = made[w], job["first"] + j
            made[w] += 1

            def run():
                expect(self.slots[slot][1] == step, "K")
                expect(self.queries[w] == job["index"], "queries")
                # what the scores replace: the ones before, at 128 with their weights
                expect(self.taken[w] == n if self.narrow else self.products[w] == n, "scores")
                self.scores[w] = n + 1
                self.s_full[w].arrive()
                if j + 1 == job["to"][w]:
                    self.q_free[w].arrive()

            tensor.append(run)

        while True:
            job = yield from self.next_job(job_turn)
            if job is None:
                break
            self.job_empty[job_turn % JOBS].arrive()
            job_turn += 1
            for j in range(job["steps"]):
                slot, k_slot = turn % self.ring, (turn + 1) % self.ring
                yield self.full[slot].passed(turn // self.ring)
                if self.narrow:
                    if j > 0:
                        yield from score(i, j, job, slot)
                    yield from edge()
                    yield from product(i, slot)
                    if j == 0:
                        yield from score(i, j, job, slot)
                    tensor.append(self.empty[slot].arrive)
                    turn += 1
                else:
                    yield self.full[k_slot].passed((turn + 1) // self.ring)
                    yield from edge()
                    yield from product(0, slot)
                    if j == 0:
                        yield from product(1, slot)
                    yield from score(0, j, job, k_slot)
                    if j > 0:
                        yield from product(1, slot)
                    tensor.append(self.empty[slot].arrive)
                    yield from score(1, j, job, k_slot)
                    tensor.append(self.empty[k_slot].arrive)
                    turn += 2
                for w in tiles:
                    on[w] = job["from"][w] <= j < job["to"][w]
                at_edge, v_step = j in job["edges"], job["first"] + j
        if turn > 0:
            yield self.full[turn % self.ring].passed(turn // self.ring)
            yield from edge()
            for w in tiles:
                yield from product(w, turn % self.ring)

    def softmax(self, w):
        turn, seen = 0, 0
        while True:
            job = yield from self.next_job(turn)
            if self.narrow:  # both tiles go on with a job or neither does
                yield self.both.sync()
            if job is None:
                return
            self.job_empty[turn % JOBS].arrive()
            turn += 1
            if w == 1 and not job["two"]:
                continue
            first, last, steps = job["from"][w], job["to"][w], job["steps"]
            turns = self.narrow and job["two"]
            if turns and w == 1:
                self.turns[0].arrive()
            for j in range(0 if turns else first, steps if turns else last):
                if not first <= j < last:
                    yield self.turns[w].sync()
                    if w == 0 or j + 1 < steps:
                        self.turns[w ^ 1].arrive()
                    continue
                yield self.s_full[w].passed(seen)
                expect(self.scores[w] == seen + 1, "scores read")
                if self.narrow:
                    self.taken[w] = seen + 1
                    self.s_free[w].arrive()
                if self.rng.random() < 0.3 and j > first:  # the output rows rescaled
                    yield self.pv_done[w].passed(seen - 1)
                    expect(self.products[w] == seen, "output rescaled")
                if turns:
                    yield self.turns[w].sync()
                yield lambda: True  # the exponentials
                if turns and (w == 0 or j + 1 < steps):
                    self.turns[w ^ 1].arrive()
                if self.narrow and j > first and self.mistake != "weights overwritten":
                    yield self.pv_done[w].passed(seen - 1)
                expect(self.products[w] == seen, "weights stored over those of a product")
                self.weights[w] = seen + 1
                self.p_full[w].arrive()
                seen += 1
            if first < last:
                yield self.pv_done[w].passed(seen - 1)
                expect(self.products[w] == seen, "output read")
                yield lambda: True  # the rows' way out
                expect(self.products[w] == seen, "output overwritten")

    # ---- all of them, in a random order at random speeds
    def run(self):
        if self.narrow:
            roles = [self.edges((0, 1), True)]
        else:
            roles = [self.edges((0,), True), self.edges((1,), False)]
        roles += [self.load(), self.softmax(0), self.softmax(1)]
        roles += [self.issue(i) for i in range(self.issuers)]
        waits = {role: next(role) for role in roles}
        speed = {x: self.rng.choice([1, 1, 5, 30])
                 for x in roles + ["copies"] + list(range(self.issuers))}
        while waits or self.copies or any(self.tensor):
            ready = [role for role, passed in waits.items() if passed()]
            ready += [i for i in range(self.issuers) if self.tensor[i]]
            ready += ["copies"] if self.copies else []
            expect(ready, "a wait that never ends")
            one = self.rng.choices(ready, [speed[x] for x in ready])[0]
            if one == "copies":
                self.copies.pop(self.rng.randrange(len(self.copies)))()
            elif isinstance(one, int):
                self.tensor[one].pop(0)()
            else:
                try:
                    waits[one] = next(one)
                except StopIteration:
                    del waits[one]


def some_pieces(rng):
    pieces = []
    for _ in range(rng.randint(1, 7)):
        steps, two = rng.randint(1, 9), rng.random() < 0.8

        def span():
            first = rng.choice([0, 0, rng.randint(0, steps)])
            last = rng.choice([steps, rng.randint(0, steps)])
            return (first, last) if first < last else (0, 0)

        spans = [span(), span() if two else (0, 0)]
        pieces.append({
            "steps": steps, "two": two, "from": [a for a, _ in spans], "to": [b for _, b in spans],
            "edges": {j for j in range(steps)
                      if rng.random() < 0.3 or j in (0, steps - 1) and rng.random() < 0.5}})
    return pieces


@pytest.mark.parametrize("narrow", [True, False])
def test_every_wait_ends_and_sees_what_it_waits_for(narrow):
    for seed in range(500):
        rng = random.Random(seed)
        Kernel(narrow, some_pieces(rng), rng).run()


@pytest.mark.parametrize("narrow,mistake", [
    (True, "scores not waited for"), (True, "weights overwritten"),
    *((narrow, mistake) for narrow in (True, False)
      for mistake in ("ring not waited for", "queries not waited for", "edge not waited for",
                      "weights not waited for"))])
def test_the_model_finds_mistakes(narrow, mistake):
    found = 0
    for seed in range(60):
        rng = random.Random(seed)
        try:
            Kernel(narrow, some_pieces(rng), rng, mistake).run()
        except Wrong:
            found += 1
    assert found
