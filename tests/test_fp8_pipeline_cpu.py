"""The waits of the kernels of attention over caches in 8 bits, played through on the CPU.

A wait on an mbarrier knows the parity of a phase alone: it passes while the barrier's completed phases and the
awaited one differ in parity. Here the kernels' roles (one for TMA, one that issues products, those that widen V, those
of the softmax) are coroutines that wait, arrive, read and write as the kernels do; loads land and products run later, loads
in any order, products in theirs. Drawn schedules look for a wait that passes early or never, and for a slot, a
buffer or a page's scale that is read or written out of turn.
"""

import random

import pytest


class World:
    def __init__(self, seed):
        self.rng = random.Random(seed)
        self.done, self.pending, self.need = {}, {}, {}   # of a barrier: phases over, arrivals of this one, arrivals of a phase
        self.mem, self.loads, self.products, self.now = {}, [], [], 0

    def bar(self, name, need):
        self.done[name], self.pending[name], self.need[name] = 0, 0, need

    def arrive(self, name):
        self.pending[name] += 1
        assert self.pending[name] <= self.need[name]
        if self.pending[name] == self.need[name]:
            self.done[name] += 1
            self.pending[name] = 0

    def passes(self, name, count):
        if (self.done[name] & 1) == (count & 1):
            return False
        assert self.done[name] == count + 1, f"{name}: a wait for phase {count} passes after {self.done[name]}"
        return True

    def run(self, roles):
        """Roles yield (barrier, count) to wait, None to be set aside."""
        waits = {r: None for r in roles}
        while waits or self.loads or self.products:
            ready = [r for r, w in waits.items() if w is None or self.passes(*w)]
            moves = ready + (["load"] if self.loads else []) + (["product"] if self.products else [])
            assert moves, f"all wait: {[w for w in waits.values()]}"
            m = self.rng.choice(moves)
            if m == "load":
                self.loads.pop(self.rng.randrange(len(self.loads)))()
            elif m == "product":
                self.products.pop(0)()
            else:
                try:
                    waits[m] = next(m)
                except StopIteration:
                    del waits[m]


def many_rows(pieces, NS, seed, choose):
    """fp8_attn_kernel: pieces of so many tiles; choose(j) -> (the reference moves, the tile is masked)."""
    w = World(seed)
    scales = NS + 2
    for i in range(NS):
        for name, need in (("KF", 2), ("KE", 1), ("VF", 2), ("VE", 2)):
            w.bar((name, i), need)
    for i in range(2):
        for name, need in (("S", 2), ("P", 4), ("W", 2), ("O", 1)):
            w.bar((name, i), need)
    w.bar("Q", 1)
    m = w.mem
    m.update(out=0, first={}, read=[0, 0, 0, 0])
    first = [sum(pieces[:p]) for p in range(len(pieces) + 1)]

    def tma():
        n = 0
        for p, nt in enumerate(pieces):
            if n:
                yield ("KE", (n - 1) % NS), (n - 1) // NS
            assert m.get("qk", -1) == n - 1                 # products that read the queries of the piece before

            def land(p=p):
                m["Q"] = p
                w.arrive("Q")
            w.loads.append(land)
            for _ in range(nt):
                for kv in "KV":
                    slot = n % NS
                    if n >= NS:
                        yield (kv + "E", slot), n // NS - 1
                    w.loads.append(lambda kv=kv, slot=slot, n=n: (m.__setitem__((kv, slot), n), w.arrive((kv + "F", slot))))
                    yield None
                    if kv == "K":
                        left = m.get(("users", n % scales), 0)
                        assert left == 0, f"scales of tile {n - scales} are still read"
                        m["scale", n % scales] = n
                        m["users", n % scales] = 6              # softmax and widening warps
                    w.arrive((kv + "F", slot))
                    yield None
                n += 1

    def used(j):
        assert m["scale", j % scales] == j
        m["users", j % scales] -= 1

    def mma():
        j = 0

        def product(i, begins, due):
            yield ("W", i & 1), i >> 1
            yield ("P", i & 1), i >> 1

            def run():
                assert m["V16", i & 1] == [i, i] and m["P", i & 1] == [i] * 4
                if begins:
                    assert m["out"] >= due, "the output before has not been read"
                m["pv"] = i
            w.products.append(run)
            w.products.append(lambda: w.arrive(("O", i & 1)))

        for p, nt in enumerate(pieces):
            yield "Q", p
            for i in range(nt):
                yield ("KF", j % NS), j // NS
                if j >= 2:
                    yield ("O", j & 1), (j - 2) >> 1

                def run(j=j, p=p):
                    assert m["K", j % NS] == j and m["Q"] == p
                    assert j < 2 or m["pv"] >= j - 2            # weights there have been read
                    m["S", j & 1], m["qk"] = j, j
                    m["P", j & 1] = [None] * 4
                w.products.append(run)
                w.products.append(lambda j=j: w.arrive(("S", j & 1)))
                w.products.append(lambda j=j: w.arrive(("KE", j % NS)))
                w.arrive(("S", j & 1))
                yield None
                if i:
                    yield from product(j - 1, i == 1, 4 * p)
                j += 1
            yield from product(j - 1, nt == 1, 4 * p)

    def widen(r):
        for j in range(first[-1]):
            yield ("VF", j % NS), j // NS
            if j >= 2:
                yield ("O", j & 1), (j - 2) >> 1
            assert m["V", j % NS] == j and (j < 2 or m["pv"] >= j - 2)
            used(j)
            m.setdefault(("V16", j & 1), [None, None])[r] = j
            yield None
            w.arrive(("W", j & 1))
            w.arrive(("VE", j % NS))
            yield None

    def softmax(r):
        for p, nt in enumerate(pieces):
            for j in range(first[p], first[p + 1]):
                moves, masked = choose(j)
                yield ("S", j & 1), j >> 1
                assert m["S", j & 1] == j
                if moves and j > first[p]:
                    yield ("O", 1 - (j & 1)), (j - 1) >> 1
                    assert m["pv"] == j - 1
                if masked:
                    yield ("W", j & 1), j >> 1
                used(j)
                m["P", j & 1][r] = j
                yield None
                w.arrive(("P", j & 1))
                yield None
            last = first[p + 1] - 1
            yield ("O", last & 1), last >> 1
            assert m["pv"] == last
            m["out"] += 1
            yield None

    w.run([tma(), mma(), *(widen(r) for r in range(2)), *(softmax(r) for r in range(4))])
    assert m["out"] == 4 * len(pieces) and all(m["users", i] == 0 for i in range(min(scales, first[-1])))


def few_rows(tiles, NS, seed):
    """fp8_decode_kernel: K and V of a tile in two slots of one ring."""
    w = World(seed)
    scales = NS // 2 + 1
    for i in range(NS):
        w.bar(("full", i), 2)
        w.bar(("empty", i), 4)
    m = w.mem

    def tma():
        for n in range(2 * tiles):
            slot = n % NS
            if n >= NS:
                yield ("empty", slot), n // NS - 1
            w.loads.append(lambda slot=slot, n=n: (m.__setitem__(slot, n), w.arrive(("full", slot))))
            yield None
            if n % 2 == 0:
                assert m.get(("users", n // 2 % scales), 0) == 0
                m["scale", n // 2 % scales], m["users", n // 2 % scales] = n // 2, 4
            w.arrive(("full", slot))
            yield None

    def warp():
        for n in range(2 * tiles):
            yield ("full", n % NS), n // NS
            assert m[n % NS] == n
            if n % 2 == 0:
                assert m["scale", n // 2 % scales] == n // 2
                m["users", n // 2 % scales] -= 1
            yield None
            w.arrive(("empty", n % NS))
            yield None

    w.run([tma(), *(warp() for _ in range(4))])


@pytest.mark.parametrize("NS", [2, 3])
@pytest.mark.parametrize("pieces", [[1], [2], [1, 1, 1], [2, 1, 3], [7, 4], [1, 9, 2, 1, 1, 5], [13, 13]])
def test_many_rows(pieces, NS):
    for seed in range(40):
        r = random.Random(seed)
        share = r.choice([0.0, 0.3, 1.0]), r.choice([0.0, 0.3, 1.0])
        picks = [(r.random() < share[0], r.random() < share[1]) for _ in range(sum(pieces))]
        many_rows(pieces, NS, seed, lambda j: picks[j])


@pytest.mark.parametrize("NS", [4, 5, 8, 10])
@pytest.mark.parametrize("tiles", [1, 2, 5, 23])
def test_few_rows(tiles, NS):
    for seed in range(40):
        few_rows(tiles, NS, seed)


def test_a_missing_wait_is_seen():
    """The play itself: a wait that a phase too many has gone by is told from one that is over."""
    w = World(0)
    w.bar("b", 1)
    w.arrive("b")
    assert w.passes("b", 0) and not w.passes("b", 1)
    with pytest.raises(AssertionError, match="passes after"):
        w.passes("b", 2)
