"""Host model of the masked attention kernel's barriers (csrc/masked_attention.cu): the loading warp, the scheduling warp, a warp
of products and a group of softmax threads for each stream, with loads and products that finish at any later time, run in random
interleavings over random lists of items. No wait may be left, no barrier may complete a phase twice before its waiters have seen
it (a wait knows only the parity), and no buffer may be written while a reader is left."""
import random

import pytest

STAGES, RECORDS = 5, 4


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def done(self, n):
        """Whether use n (from 0) is over, as a wait on its parity sees it."""
        assert self.phase <= n + 1, "a phase went by unseen"
        return self.phase != n   # parity: phase n is current, or it is over


class World:
    def __init__(self, items, seed):
        self.items, self.rng = items, random.Random(seed)
        b = Barrier
        self.kv_full, self.kv_empty = [b(1) for _ in range(STAGES)], [b(2) for _ in range(STAGES)]
        self.rec_full, self.rec_empty = [b(1) for _ in range(RECORDS)], [b(5) for _ in range(RECORDS)]   # a group reads as one here
        self.q_full, self.q_empty = b(1), b(2)
        self.s_full, self.p_full, self.o_full = [b(1), b(1)], [b(1), b(1)], [b(1), b(1)]
        self.x_full, self.x_done = b(2), b(2)
        self.q, self.stage, self.s, self.o = None, [None] * STAGES, [None, None], [None, None]
        self.pending = []              # loads, finished in any order
        self.queue = [[], []]          # of a products warp, finished in order
        self.out = {}

    def read_records(self):
        n = 0
        while True:
            yield self.rec_full[n % RECORDS], n // RECORDS
            item = n if n < len(self.items) else None
            self.rec_empty[n % RECORDS].arrive()
            yield None
            if item is None:
                return
            n += 1
            yield ("item", item)

    def role(self, body):
        """Runs body(item), a generator of waits, for each record."""
        for step in self.read_records():
            if isinstance(step, tuple) and step[0] == "item":
                yield from body(step[1])
            else:
                yield step

    def produce(self):
        use = [0]

        def load(what):
            u = use[0]
            use[0] += 1
            if u >= STAGES:
                yield self.kv_empty[u % STAGES], u // STAGES - 1

            def land():
                self.stage[u % STAGES] = what
                self.kv_full[u % STAGES].arrive()

            self.stage[u % STAGES] = None
            self.pending.append(land)
            yield None

        def body(i):
            n, pair = self.items[i]
            if pair:
                for j in range(n):
                    yield from load((i, "K", j))
                    yield from load((i, "V", j))
            else:
                for j in range(n + 1):
                    if j < n:
                        yield from load((i, "K", j))
                    if j:
                        yield from load((i, "V", j - 1))

        yield from self.role(body)

    def schedule(self):
        uses = 0
        for n in range(len(self.items) + 1):
            if n >= RECORDS:
                yield self.rec_empty[n % RECORDS], n // RECORDS - 1
            self.rec_full[n % RECORDS].arrive()
            yield None
            if n == len(self.items) or self.items[n][0] == 0:
                continue
            if uses:
                yield self.q_empty, uses - 1
            uses += 1

            def land(n=n):
                self.q = n
                self.q_full.arrive()

            self.q = None
            self.pending.append(land)
            yield None

    def multiply(self, x):
        use, q_count, p_count = [0], [0], [0]

        def enqueue(*ops):
            self.queue[x].extend(ops)

        def next_stage():
            u = use[0]
            use[0] += 1
            return u % STAGES, (self.kv_full[u % STAGES], u // STAGES)

        def scores(i, j, last):
            st, wait = next_stage()
            yield wait

            def product():
                assert self.stage[st] == (i, "K", j) and self.q == i and (self.s[x] is None or self.s[x][0] == "spent"), (self.stage[st], self.q, self.s[x])
                self.s[x] = ("S", i, j)

            enqueue(product, self.s_full[x].arrive, self.kv_empty[st].arrive)
            if last:
                enqueue(self.q_empty.arrive)
            yield None

        def values(i, j, first):
            st, wait = next_stage()
            yield wait
            yield self.p_full[x], p_count[0]
            p_count[0] += 1

            def product():
                assert self.stage[st] == (i, "V", j) and self.s[x] == ("P", i, j), (self.stage[st], self.s[x])
                assert self.o[x] is None if first else self.o[x][:2] == (i, "sum"), self.o[x]
                self.o[x] = (i, "sum", ([] if first else self.o[x][2]) + [j])
                self.s[x] = ("spent",)

            enqueue(product, self.kv_empty[st].arrive)
            yield None

        def skip():
            st, wait = next_stage()
            yield wait
            self.kv_empty[st].arrive()
            yield None

        def body(i):
            n, pair = self.items[i]
            if n == 0:
                return
            yield self.q_full, q_count[0]
            q_count[0] += 1
            if pair:
                yield from scores(i, 0, n == 1)
                for j in range(n):
                    yield from values(i, j, j == 0)
                    if j + 1 < n:
                        yield from scores(i, j + 1, j + 2 == n)
            else:
                mine = (n + 1 - x) // 2
                yield from (scores(i, 0, mine == 1) if x == 0 else skip())
                if n > 1:
                    yield from (scores(i, 1, mine == 1) if x == 1 else skip())
                if mine == 0:
                    enqueue(self.q_empty.arrive)
                for j in range(n):
                    own = j % 2 == x
                    yield from (values(i, j, j < 2) if own else skip())
                    if j + 2 < n:
                        yield from (scores(i, j + 2, j + 4 >= n) if own else skip())
            if pair or n > x:
                enqueue(self.o_full[x].arrive)

        yield from self.role(body)

    def softmax(self, x):
        s_count, o_count, x_count = [0], [0], [0]

        def body(i):
            n, pair = self.items[i]
            for j in range(0 if pair else x, n, 1 if pair else 2):
                yield self.s_full[x], s_count[0]
                s_count[0] += 1
                assert self.s[x] == ("S", i, j)
                self.s[x] = ("P", i, j)
                yield None
                self.p_full[x].arrive()
            if n > (0 if pair else x):
                yield self.o_full[x], o_count[0]
                o_count[0] += 1
            if pair:
                if n:
                    assert self.o[x] == (i, "sum", list(range(n)))
                    self.o[x] = None
            else:
                self.x_full.arrive()
                yield self.x_full, x_count[0]
                for y in range(2):
                    if n > y:
                        assert self.o[y] == (i, "sum", list(range(y, n, 2))), (self.o, i, n)
                yield None
                self.x_done.arrive()
                yield self.x_done, x_count[0]
                x_count[0] += 1
                self.o[x] = None
            self.out[i, x] = True

        yield from self.role(body)

    def run(self):
        roles = [self.produce(), self.schedule(), self.multiply(0), self.multiply(1), self.softmax(0), self.softmax(1)]
        waits = [None] * len(roles)
        speeds = [self.rng.choice([1, 1, 5, 30]) for _ in range(len(roles) + 3)]
        while any(r is not None for r in roles):
            ready = [k for k, r in enumerate(roles) if r is not None and (waits[k] is None or waits[k][0].done(waits[k][1]))]
            choices = ready + [len(roles)] * bool(self.pending) + [len(roles) + 1 + x for x in range(2) if self.queue[x]]
            assert choices, ("nobody can go on", [w and w[1] for w in waits], self.items)
            k = self.rng.choices(choices, [speeds[c] for c in choices])[0]
            if k == len(roles):
                self.pending.pop(self.rng.randrange(len(self.pending)))()
            elif k > len(roles):
                self.queue[k - len(roles) - 1].pop(0)()
            else:
                try:
                    waits[k] = next(roles[k])
                except StopIteration:
                    roles[k] = None
        while self.pending or any(self.queue):
            (self.pending or self.queue[0] or self.queue[1]).pop(0)()
        assert len(self.out) == 2 * len(self.items)


@pytest.mark.parametrize("seed", range(40))
def test_random_interleavings(seed):
    rng = random.Random(seed)
    for k in range(12):
        items = [(rng.choice([0, 1, 1, 2, 3, 5, 8]), rng.random() < rng.choice([0.0, 0.5, 1.0])) for _ in range(rng.randrange(1, 14))]
        World([(n, pair) for n, pair in items], 1000 * seed + k).run()
