"""Host model of the masked attention kernel's barriers (csrc/masked_attention.cu): the loading warp, the scheduling warp, the warp of
products and a group of softmax threads for each stream, with loads and products that finish at any later time, run in random
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
        self.kv_full, self.kv_empty = [b(1) for _ in range(STAGES)], [b(1) for _ in range(STAGES)]
        self.rec_full, self.rec_empty = [b(1) for _ in range(RECORDS)], [b(4) for _ in range(RECORDS)]   # a group reads as one here
        self.q_full, self.q_empty = b(1), b(1)
        self.s_full, self.p_full, self.o_full = ([b(1), b(1)] for _ in range(3))
        self.x_full, self.x_done = b(2), b(2)
        self.told = [b(4), b(4)]       # an item of few rows: the warps of a stream tell each other their maxima
        self.weights = [None, None]    # of such a stream, where the other queries of a pair go
        self.q, self.stage, self.s, self.o = None, [None] * STAGES, [None, None], [None, None]
        self.pending = []              # loads, finished in any order
        self.queue = []                # products, finished in order
        self.out = {}

    def read_records(self):
        n = 0
        while True:
            if n:
                self.rec_empty[(n - 1) % RECORDS].arrive()
                yield None
            yield self.rec_full[n % RECORDS], n // RECORDS
            if n == len(self.items):
                return
            n += 1
            yield ("item", n - 1)

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
            n, pair, few = self.items[i]
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
                if self.items[n][1]:
                    assert self.weights == [None, None], "weights were overwritten"
                self.q_full.arrive()

            self.q = None
            self.pending.append(land)
            yield None

    def multiply(self):
        use, q_count, p_count = [0], [0], [0, 0]
        enqueue = lambda *ops: self.queue.extend(ops)   # noqa: E731

        def stage():
            return use[0] % STAGES, (self.kv_full[use[0] % STAGES], use[0] // STAGES)

        def scores(x, i, j, st):
            def product():
                assert self.stage[st] == (i, "K", j) and self.q == i and self.s[x] in (None, "spent"), (self.stage[st], self.q, self.s[x])
                self.s[x] = ("S", i, j)

            enqueue(product, self.s_full[x].arrive)

        def values(x, i, j, st, first):
            yield self.p_full[x], p_count[x]
            p_count[x] += 1

            def product():
                assert self.stage[st] == (i, "V", j) and self.s[x] == ("P", i, j), (self.stage[st], self.s[x])
                if self.items[i][2]:
                    assert self.weights[x] == (i, j)
                    self.weights[x] = None
                assert self.o[x] is None if first else self.o[x][0] == i, self.o[x]
                self.o[x] = (i, ([] if first else self.o[x][1]) + [j])
                self.s[x] = "spent"

            enqueue(product)

        def body(i):
            n, pair, few = self.items[i]
            if n == 0:
                return
            yield self.q_full, q_count[0]
            q_count[0] += 1
            for j in range(1 if pair else min(n, 2)):
                st, wait = stage()
                yield wait
                scores(j, i, j, st)
                if pair:
                    scores(1, i, j, st)
                enqueue(self.kv_empty[st].arrive)
                use[0] += 1
                yield None
            if not few and n <= (1 if pair else 2):
                enqueue(self.q_empty.arrive)
            for j in range(n):
                v, wait = stage()
                yield wait
                use[0] += 1
                more = j + (1 if pair else 2) < n
                for x in ((0, 1) if pair else (j % 2,)):
                    yield from values(x, i, j, v, j < (1 if pair else 2))
                    if not pair:
                        enqueue(self.kv_empty[v].arrive)
                    if not more:
                        if pair:
                            enqueue(self.o_full[x].arrive)
                        continue
                    k, wait = stage()
                    if x == 0 or not pair:
                        yield wait
                    scores(x, i, j + (1 if pair else 2), k)
                    yield None
                if pair:
                    enqueue(self.kv_empty[v].arrive)
                if more:
                    enqueue(self.kv_empty[k].arrive)
                    if not few and j + (2 if pair else 3) == n:
                        enqueue(self.q_empty.arrive)
                    use[0] += 1
                yield None
            if few:
                enqueue(self.q_empty.arrive)
            if not pair:
                enqueue(*[self.o_full[x].arrive for x in range(min(n, 2))])

        yield from self.role(body)

    def softmax(self, x):
        s_count, o_count, x_count, told = [0], [0], [0], [0]

        def body(i):
            n, pair, few = self.items[i]
            tiles = list(range(0 if pair else x, n, 1 if pair else 2))
            for j in tiles:
                yield self.s_full[x], s_count[0]
                s_count[0] += 1
                assert self.s[x] == ("S", i, j)
                if j != tiles[0]:   # where a maximum has grown the sums so far are rescaled
                    assert self.o[x] == (i, tiles[:tiles.index(j)])
                if few:   # this thread of control is one of the four warps, the others' are taken along
                    for _ in range(4):
                        self.told[x].arrive()
                        yield None
                    yield self.told[x], told[0]
                    told[0] += 1
                    assert self.weights[x] is None and self.q == i
                    self.weights[x] = (i, j)
                self.s[x] = ("P", i, j)
                yield None
                self.p_full[x].arrive()
            if tiles:
                yield self.o_full[x], o_count[0]
                o_count[0] += 1
            if pair:
                if n:
                    assert self.o[x] == (i, tiles)
            else:
                self.x_full.arrive()
                yield self.x_full, x_count[0]
                for y in range(2):
                    if n > y:
                        assert self.o[y] == (i, list(range(y, n, 2))), (self.o, i, n)
                yield None
                self.x_done.arrive()
                yield self.x_done, x_count[0]
                x_count[0] += 1
            self.o[x] = None
            self.out[i, x] = True

        yield from self.role(body)

    def run(self):
        roles = [self.produce(), self.schedule(), self.multiply(), self.softmax(0), self.softmax(1)]
        waits = [None] * len(roles)
        speeds = [self.rng.choice([1, 1, 5, 30]) for _ in range(len(roles) + 2)]
        while any(r is not None for r in roles):
            ready = [k for k, r in enumerate(roles) if r is not None and (waits[k] is None or waits[k][0].done(waits[k][1]))]
            choices = ready + [len(roles)] * bool(self.pending) + [len(roles) + 1] * bool(self.queue)
            assert choices, ("nobody can go on", [w and w[1] for w in waits], self.items)
            k = self.rng.choices(choices, [speeds[c] for c in choices])[0]
            if k == len(roles):
                self.pending.pop(self.rng.randrange(len(self.pending)))()
            elif k > len(roles):
                self.queue.pop(0)()
            else:
                try:
                    waits[k] = next(roles[k])
                except StopIteration:
                    roles[k] = None
        while self.pending or self.queue:
            (self.pending or self.queue).pop(0)()
        assert len(self.out) == 2 * len(self.items)


@pytest.mark.parametrize("seed", range(40))
def test_random_interleavings(seed):
    rng = random.Random(seed)
    for k in range(12):
        kinds = rng.choice([["pair"], ["few", "pair"], ["few", "alternate", "pair"], ["few", "alternate"], ["alternate", "pair"]])
        items = [(rng.choice([0, 1, 1, 2, 3, 5, 8]), rng.choice(kinds)) for _ in range(rng.randrange(1, 14))]
        World([(n, kind == "pair", kind == "few") for n, kind in items], 1000 * seed + k).run()
