"""What waits for what in the tree attention kernel, as a happens-before graph.

An mbarrier tells a waiter the parity of its phase and nothing else. A wait for completion c
of a barrier is sound if, when it starts, completion c - 1 is known to be over (else the
barrier, a phase further back, looks as if c were over too), and if completion c + 1 cannot be
over before the wait has looked (else it would never end). Both follow from program
order, completed waits, and copies and products that end after they are issued -- or they do not, and
some schedule breaks them. The roles of csrc/tree_attn.cu (K and V producers, a product warp and a
softmax group for each half) are written down here step by step for pieces of ``nt`` tiles, and
every wait, arrival and use of a slot is looked at in the graph. Products of the two product
warps are not taken to end in any order between them, commits of one warp arrive in order.
"""

import itertools
import random

import pytest

# what the kernel does beyond the plain chain of waits; without either there is a schedule that breaks it
SEES_K1 = "group 0's product warp sees K_1 land before its slot is free"
SEES_LOAD = "a producer sees the load before in a slot land before it waits for the slot"
RULES = frozenset([SEES_K1, SEES_LOAD])


def _k_load(i, lead):
    return i if i < lead else 2 * i - lead + 1


def _v_load(i, lead, nt):
    return min(lead, nt) + i + min(i, max(nt - lead, 0))


class Graph:
    def __init__(self):
        self.pred, self.name, self.last = [], [], {}
        self.done, self.arrivals = {}, {}    # (barrier, completion) -> node, arriving nodes
        self.waits, self.orders = [], []     # (before, after, barrier, completion, role); (a, b, what): a before b

    def node(self, name, *preds):
        self.pred.append([p for p in preds if p is not None])
        self.name.append(name)
        return len(self.pred) - 1

    def step(self, role, name, *preds):
        self.last[role] = self.node(name, self.last.get(role), *preds)
        return self.last[role]

    def completion(self, bar, c):
        if (bar, c) not in self.done:
            self.done[bar, c] = self.node(("done", bar, c))
        return self.done[bar, c]

    def wait(self, role, bar, c, taken=True):
        """taken: every schedule waits here; else only some do, and nothing may rest on it."""
        before = self.step(role, ("before", bar, c))
        after = self.node(("after", bar, c), before, self.completion(bar, c))
        if taken:
            self.last[role] = after
        self.waits.append((before, after, bar, c, role))

    def arrive(self, node, bar, c):
        self.pred[self.completion(bar, c)].append(node)
        self.arrivals.setdefault((bar, c), []).append(node)

    def close(self):
        """self.anc[n]: a bit for every node before n (n among them)."""
        n, state, self.anc = len(self.pred), [0] * len(self.pred), [0] * len(self.pred)
        for root in range(n):
            stack = [] if state[root] else [(root, iter(self.pred[root]))]
            state[root] = state[root] or 1
            while stack:
                x, it = stack[-1]
                for p in it:
                    assert state[p] != 1, f"a circle of waits at {self.name[p]}"
                    if state[p] == 0:
                        state[p] = 1
                        stack.append((p, iter(self.pred[p])))
                        break
                else:
                    state[x] = 2
                    self.anc[x] = 1 << x
                    for p in self.pred[x]:
                        self.anc[x] |= self.anc[p]
                    stack.pop()

    def before(self, a, b):
        return bool((self.anc[b] >> a) & 1)

    def over(self, bar, c, x):
        return self.before(self.done[bar, c], x) or all(self.before(n, x) for n in self.arrivals[bar, c])


def _pipeline(pieces, two, q_tma, slots, nodes, rules, rescales):
    """The graph of one CTA. pieces: tiles of each; two[i]: two groups of rows, else tiles in
    turn; slots of the ring; the last ``nodes`` tiles of a piece hold nodes; rescales: a tile's
    second half always moves the reference (else nothing may rest on that wait)."""
    g = Graph()
    issue, land, used, qk_ops, q_issue = {}, {}, {}, {}, []
    op_of, commit_of = {}, {}

    def full(k):
        return ("full", k % slots), k // slots

    def empty(k, c=0):
        return ("empty", k % slots), k // slots + c

    for role in "KV":
        base, before = 0, []
        for n, nt in enumerate(pieces):
            lead = 1 if two[n] else 2
            if q_tma and role == "K":
                for k in before:
                    g.wait(role, *empty(k))
                if n:
                    g.wait(role, "seen", n - 1)
                q_issue.append(g.step(role, ("Q", n)))
                g.arrive(g.node(("Q landed", n), q_issue[-1]), "Q", n)
            for i in range(nt):
                k = base + (_k_load(i, lead) if role == "K" else _v_load(i, lead, nt))
                if k >= slots:
                    if SEES_LOAD in rules:
                        g.wait(role, ("full", k % slots), k // slots - 1)
                    g.wait(role, *empty(k, -1))
                issue[k] = g.step(role, ("load", k))
                land[k] = g.node(("landed", k), issue[k])
                g.arrive(land[k], *full(k))
            before = [base + _k_load(i, lead) for i in range(max(nt - lead, 0), nt)]
            base += 2 * nt

    turns = [0, 0]
    for s in (0, 1):
        role, base, n_q, n_p, n_t, n_s, n_o, handed = f"product {s}", 0, 0, 0, 0, 0, 0, False

        def op(name, at):
            op_of[s] = g.node(name, at, op_of.get(s))

        def commit(bar, c):
            commit_of[s] = g.node(("commit", bar, c), g.last[role], op_of[s], commit_of.get(s))
            g.arrive(commit_of[s], bar, c)

        for n, nt in enumerate(pieces):
            lead = 1 if two[n] else 2
            first = 0 if two[n] else s

            def release(k, times):
                used.setdefault(k, []).append(op_of[s])
                for _ in range(times):
                    commit(*empty(k))

            def qk(i, times):
                nonlocal n_s
                k = base + _k_load(i, lead)
                at = g.step(role, ("QK", n, i))
                g.orders.append((land[k], at, ("K there", n, i)))
                op(("QK done", n, i), at)
                qk_ops.setdefault((n, s), []).append(op_of[s])
                commit(("S", s), n_s)
                n_s += 1
                release(k, times)

            each = 1 if two[n] else 2
            if q_tma:
                g.wait(role, "Q", n)
                g.arrive(g.step(role, "seen"), "seen", n)
            if first < nt:
                if not q_tma:
                    g.wait(role, ("Q", s), n_q)
                    n_q += 1
                g.wait(role, *full(base + _k_load(first, lead)))
                qk(first, 1 if SEES_K1 in rules and s == 1 and not two[n] else each)
            if SEES_K1 in rules and not two[n] and s == 0 and nt > 1:
                g.wait(role, *full(base + _k_load(1, lead)))
                g.arrive(g.step(role, "K_1 seen"), *empty(base + _k_load(1, lead)))
            for i in range(first, nt, lead):
                v, more = base + _v_load(i, lead, nt), i + lead < nt
                if s == 1 or i > first or handed:
                    g.wait(role, ("turn", s), n_t)
                    n_t += 1
                g.wait(role, *full(v))
                if more:
                    g.wait(role, *full(base + _k_load(i + lead, lead)))
                for half in (0, 1):
                    g.wait(role, ("P", half, s), n_p)
                    at = g.step(role, ("PV", n, i, half))
                    g.orders.append((land[v], at, ("V there", n, i)))
                    op(("PV done", n, i, half), at)
                    if half == 0:
                        commit(("half", s), n_p)
                n_p += 1
                release(v, each)
                if more:
                    qk(i + lead, each)
                else:
                    commit(("O", s), n_o)
                    n_o += 1
                if s == 1 or two[n] or i + 1 < nt:
                    g.arrive(g.step(role, "turn"), ("turn", 1 - s), turns[1 - s])
                    turns[1 - s] += 1
            base += 2 * nt
            handed = two[n] or nt % 2 == 0

    base, n_s, n_q, n_o = 0, [0, 0], [0, 0], [0, 0]
    for n, nt in enumerate(pieces):
        lead = 1 if two[n] else 2
        for s in (0, 1):
            role, mine = f"softmax {s}", two[n] or s < nt
            if mine and not q_tma:
                at = g.step(role, ("Q written", n))
                g.arrive(at, ("Q", s), n_q[s])
                n_q[s] += 1
                g.orders += [(o, at, ("Q free", n)) for o in qk_ops.get((n - 1, s), [])]
            for i in range(0 if two[n] else s, nt, lead):
                g.wait(role, ("S", s), n_s[s])
                if i >= nt - nodes:
                    v = base + _v_load(i, lead, nt)
                    g.wait(role, *full(v))
                    g.orders.append((land[v], g.step(role, "cleaned"), ("V there to clean", n, i)))
                g.arrive(g.step(role, "first half"), ("P", 0, s), n_s[s])
                g.wait(role, ("half", s), n_s[s], taken=rescales)
                g.arrive(g.step(role, "second half"), ("P", 1, s), n_s[s])
                n_s[s] += 1
            if mine:
                g.wait(role, ("O", s), n_o[s])
                n_o[s] += 1
        for _ in range(2):  # the groups meet before and after a piece's output
            g.last["softmax 0"] = g.last["softmax 1"] = g.node("meet", g.last.get("softmax 0"), g.last.get("softmax 1"))
        base += 2 * nt
    for n, at in enumerate(q_issue):
        g.orders += [(o, at, ("Q free", n)) for s in (0, 1) for o in qk_ops.get((n - 1, s), [])]
    for k, at in issue.items():
        g.orders += [(o, at, ("slot free", k)) for o in used.get(k - slots, [])]
    return g


def _unsound(pieces, two, q_tma, slots, nodes, rules):
    """(role, barrier) of every wait that some schedule breaks, and whatever else is out of order."""
    bad = set()
    for rescales in (False, True):
        g = _pipeline(pieces, two, q_tma, slots, nodes, rules, rescales)
        g.close()
        for before, after, bar, c, role in g.waits:
            kind = bar[0] if isinstance(bar, tuple) else bar
            if c > 0 and not g.over(bar, c - 1, before):
                bad.add((role, kind))
            if (bar, c + 1) in g.done and (kind != "half" or rescales) and \
                    not any(g.before(after, n) for n in g.arrivals[bar, c + 1]):
                bad.add((role, kind, "too late"))
        for (bar, c), nodes_ in g.arrivals.items():
            want = 2 if bar == "seen" or bar[0] == "empty" else 1
            if len(nodes_) != want or (c > 0 and not all(g.over(bar, c - 1, n) for n in nodes_)):
                bad.add(("arrivals", bar))
        bad |= {("order", what[0]) for a, b, what in g.orders if not g.before(a, b)}
    return bad


def _schedules(two, q_tma):
    """Pieces of a CTA: one, two and three in every short combination, longer lines at random."""
    rng = random.Random(1)
    lines = [[n] for n in range(1, 14)] + [list(p) for p in itertools.product(range(1, 8), repeat=2)]
    lines += [list(p) for p in itertools.product((1, 2, 3, 5), repeat=3)]
    lines += [[rng.randint(1, 8) for _ in range(rng.randint(4, 6))] for _ in range(25)]
    for pieces in lines:
        yield pieces, [two == "rows" or (two == "mixed" and rng.random() < 0.5) for _ in pieces]


@pytest.mark.parametrize("slots", [5, 10])     # heads of 128 and of 64
@pytest.mark.parametrize("two,q_tma", [("turns", True), ("rows", True), ("turns", False), ("rows", False), ("mixed", False)])
def test_every_wait_is_sound(two, q_tma, slots):
    for pieces, kinds in _schedules(two, q_tma):
        for nodes in (0, 1, 3):
            bad = _unsound(pieces, kinds, q_tma, slots, nodes, RULES)
            assert not bad, (pieces, kinds, nodes, bad)


def test_the_model_sees_a_missing_wait():
    assert ("softmax 0", "full") in _unsound([4], [False], True, 5, 2, RULES - {SEES_K1})
    assert ("V", "empty") in _unsound([2, 4], [False, False], True, 5, 0, RULES - {SEES_LOAD})
    assert ("K", "empty") in _unsound([2, 4], [False, True], False, 5, 0, RULES - {SEES_LOAD})
