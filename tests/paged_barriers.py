"""A model of the barriers of paged attention's tcgen05 form (`chunk_kernel`), run under random schedules.

Roles: two loaders (K with Q, V), for each query tile ("chain") a warp that issues scores and one that issues the products
with V, and four softmax warps; products run in order on one pipe, loads land in any order. A unit is (second chain idle,
key tiles, whether the sequence ends in its last tile). The model asserts that no wait mistakes a phase for another of the
same parity, no buffer is overwritten in use or read before it is there, and everything ends."""


class Bar:
    def __init__(self, count, name):
        self.count, self.name, self.phase, self.pending = count, name, 0, count

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, self.name
        if self.pending == 0:
            self.phase += 1
            self.pending = self.count

    def passed(self, k):
        """A wait for phase k, which sees its parity alone."""
        seen, true = (self.phase & 1) != (k & 1), self.phase > k
        assert seen == true, (self.name, 'phase', self.phase, 'waited for', k)
        return true


class Kernel:
    def __init__(self, units, stages, chains, rng):
        self.units, self.stages, self.chains, self.rng = units, stages, chains, rng
        bars = lambda n, count, name: [Bar(count, f'{name}{i}') for i in range(n)]  # noqa: E731
        pairs = lambda count, name: [bars(2, count, f'{name}{i}.') for i in range(chains)]  # noqa: E731
        self.q_full, self.q_empty = Bar(1, 'q_full'), Bar(chains, 'q_empty')
        self.k_full, self.k_empty = bars(stages, 1, 'k_full'), bars(stages, chains, 'k_empty')
        self.v_full, self.v_empty = bars(stages, 1, 'v_full'), bars(stages, chains, 'v_empty')
        self.v_end, self.drained = Bar(1, 'v_end'), Bar(2 * chains, 'drained')
        self.s_full, self.p_full, self.pv_done = pairs(1, 's_full'), pairs(4, 'p_full'), pairs(1, 'pv_done')
        self.pipe, self.loads = [], []                         # products in order, loads in flight
        self.k, self.v, self.q = [None] * stages, [None] * stages, None
        self.k_readers, self.v_readers, self.q_readers = [0] * stages, [0] * stages, 0
        self.s = [[None, None] for _ in range(chains)]        # ('S', tile) or ('P', tile, warps that wrote)
        self.o, self.o_read = [[] for _ in range(chains)], [0] * chains

    def idle(self, unit, chain):
        return chain == 1 and self.units[unit][0]

    def loader(self, is_v):
        full, empty = (self.v_full, self.v_empty) if is_v else (self.k_full, self.k_empty)
        ring, readers = (self.v, self.v_readers) if is_v else (self.k, self.k_readers)
        g = ends = 0
        for u, (_, tiles, ends_inside) in enumerate(self.units):
            if not is_v:
                if u:
                    yield lambda: self.q_empty.passed(u - 1)

                def land_q(u=u):
                    assert self.q_readers == 0
                    self.q = u
                    self.q_full.arrive()
                self.loads.append(land_q)
            for t in range(tiles):
                s = g % self.stages
                if g >= self.stages:
                    yield lambda: empty[s].passed(g // self.stages - 1)
                end = is_v and ends_inside and t == tiles - 1

                def land(s=s, g=g, end=end):
                    assert readers[s] == 0
                    ring[s] = ('raw', g) if end else g
                    (self.v_end if end else full[s]).arrive()
                self.loads.append(land)
                yield lambda: True
                if end:   # the rows past the sequence's end are cleared
                    yield lambda: self.v_end.passed(ends)
                    ends += 1
                    assert ring[s] == ('raw', g)
                    ring[s] = g
                    full[s].arrive()
                g += 1
        for x in range(max(0, g - self.stages), g):
            yield lambda: full[x % self.stages].passed(x // self.stages)
        if not is_v:
            yield lambda: self.q_full.passed(len(self.units) - 1)

    def scores(self, i):
        g = n = 0
        for u, (_, tiles, _) in enumerate(self.units):
            yield lambda: self.q_full.passed(u)
            for _ in range(tiles):
                s = g % self.stages
                yield lambda: self.k_full[s].passed(g // self.stages)
                if self.idle(u, i):
                    self.k_empty[s].arrive()
                    g += 1
                    continue
                if n >= 2:
                    yield lambda: self.pv_done[i][n & 1].passed((n - 2) >> 1)
                self.k_readers[s] += 1
                self.q_readers += 1

                def product(s=s, g=g, n=n, u=u):
                    assert self.k[s] == g and self.q == u
                    self.k_readers[s] -= 1
                    self.q_readers -= 1
                    self.s[i][n & 1] = ('S', n)
                    self.s_full[i][n & 1].arrive()
                    self.k_empty[s].arrive()
                self.pipe.append(product)
                g += 1
                n += 1
                yield lambda: True
            if self.idle(u, i):
                self.q_empty.arrive()
            else:
                self.pipe.append(self.q_empty.arrive)
        self.pipe.append(self.drained.arrive)

    def values(self, i):
        g = n = 0
        for u, (_, tiles, _) in enumerate(self.units):
            for t in range(tiles):
                s = g % self.stages
                yield lambda: self.v_full[s].passed(g // self.stages)
                if self.idle(u, i):
                    self.v_empty[s].arrive()
                    g += 1
                    continue
                yield lambda: self.p_full[i][n & 1].passed(n >> 1)
                self.v_readers[s] += 1

                def product(s=s, g=g, n=n, fresh=t == 0):
                    assert self.v[s] == g and self.s[i][n & 1] == ('P', n, 4)
                    self.v_readers[s] -= 1
                    assert not (fresh and self.o[i]), 'O is started afresh before it was read'
                    self.o[i].append(n)
                    self.pv_done[i][n & 1].arrive()
                    self.v_empty[s].arrive()
                self.pipe.append(product)
                g += 1
                n += 1
                yield lambda: True
        self.pipe.append(self.drained.arrive)

    def softmax(self, i, dead):
        first = 0
        for u, (_, tiles, _) in enumerate(self.units):
            if self.idle(u, i):
                continue
            for t in range(tiles):
                n = first + t
                yield lambda: self.s_full[i][n & 1].passed(n >> 1)
                assert self.s[i][n & 1] is not None and self.s[i][n & 1][1] == n
                if t and not dead and self.rng.random() < 0.3:   # the row's maximum grew: O is rescaled
                    yield lambda: self.pv_done[i][(n - 1) & 1].passed((n - 1) >> 1)
                    assert len(self.o[i]) == t
                now = self.s[i][n & 1]
                self.s[i][n & 1] = ('P', n, (now[2] if now[0] == 'P' else 0) + 1)
                self.p_full[i][n & 1].arrive()
                yield lambda: True
            last = first + tiles - 1
            yield lambda: self.pv_done[i][last & 1].passed(last >> 1)
            assert self.o[i] == list(range(first, first + tiles))
            yield lambda: True
            self.o_read[i] += 1
            if self.o_read[i] == 4:
                self.o_read[i] = 0
                self.o[i].clear()
            first += tiles

    def owner(self, roles):
        """The warp that frees tensor memory once every role is done."""
        yield lambda: sum(r is not None for r in roles) == 1
        yield lambda: self.drained.passed(0)
        assert not self.pipe and not self.loads

    def run(self):
        rng, roles = self.rng, []
        parts = [self.loader(False), self.loader(True)]
        for i in range(self.chains):
            parts += [self.scores(i), self.values(i)] + [self.softmax(i, rng.random() < 0.3) for _ in range(4)]
        roles += [(part, None) for part in parts]
        roles.append((self.owner(roles), None))
        # Every role, the pipe and the loads move at speeds of their own.
        lazy = [0.9 * rng.random() ** 3 for _ in roles]
        lazy_load, lazy_pipe, quiet = 0.9 * rng.random(), 0.9 * rng.random(), 0
        while any(roles) or self.pipe or self.loads:
            moved, order = False, list(range(len(roles)))
            rng.shuffle(order)
            for j in order:
                if roles[j] is None or rng.random() < lazy[j]:
                    continue
                part, ready = roles[j]
                if ready is not None and not ready():
                    continue
                try:
                    roles[j] = part, next(part)
                except StopIteration:
                    roles[j] = None
                moved = True
            if self.loads and rng.random() >= lazy_load:
                self.loads.pop(rng.randrange(len(self.loads)) if rng.random() < 0.5 else 0)()
                moved = True
            if self.pipe and rng.random() >= lazy_pipe:
                self.pipe.pop(0)()
                moved = True
            quiet = 0 if moved else quiet + 1
            assert quiet < 3000, ('deadlock', [j for j, role in enumerate(roles) if role])
