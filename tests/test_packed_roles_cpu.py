"""The roles of attend_packed (csrc/dsk_prompt.cuh) in random interleavings: barriers with phases and waits by parity, products that run in order some time after they were issued.  Every use of a
unit of keys or values, of queries, scores, weights and results is checked against who wrote it last; a state in which nobody can go on is an error too.  This restates the kernel's protocol by
hand: whoever changes waits, commits or arrivals there changes them here."""
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def wait(self, parity):
        return lambda: (self.phase & 1) != parity & 1


AHEAD, EARLY = 4, 4                                          # tiles of keys under way, tiles ahead of the end at which more work is asked for
SHAPES = {64: (2, 1, 1, 6, 5), 128: (2, 2, 2, 6, 4), 192: (2, 3, 2, 5, 3), 256: (1, 4, 4, 6, 4)}      # row tiles, units of keys and of values a tile, places for them


def run(rng, dk, work, idle, moves, early=True):
    """work: items, each a list of (tiles of keys: (for each of its steps, the row tiles that see some of it; whether some row does not see all)) and whether the second row tile has rows.  idle:
    softmax warps without rows; early: the wait for the product ahead, where a reference moves."""
    tiles, per_k, per_v, KU, VU = SHAPES[dk]
    bars = lambda n, count: [Bar(count) for _ in range(n)]
    soft, per = 4 * tiles, tiles                             # steps of a tile: two with two row tiles, of half as many keys
    kfull, kempty, vfull, vempty, vok, vraw = bars(AHEAD, 1), bars(AHEAD, tiles), bars(VU, 1), bars(VU, tiles), bars(VU, 2), bars(VU, 1)
    qfull, qempty, odone, ifull = (bars(2, 1) for _ in range(4))
    sfull, pvdone, pfull = ([bars(2, n) for _ in range(2)] for n in (1, 1, 4))            # [row tile][place]
    iempty, flushed = bars(2, soft + 2 * tiles + 3), [bars(2, 1) for _ in range(2)]
    items, want = [None, None], Bar(1)
    keys, values, queries, looked = [None] * KU, [None] * VU, [None] * 2, [0] * VU
    scores, weights, through = [[None, None], [None, None]], [[{}, {}], [{}, {}]], [[], []]       # [row tile][place], steps whose product is through
    queue, flying = [], []                                   # products and commits in the order of their issue; copies in any order

    def take(state):
        slot = state["turn"] & 1
        yield ifull[slot].wait(state["turn"] >> 1)
        state["item"] = items[slot]
        yield None
        iempty[slot].arrive()
        state["turn"] += 1

    def deal():
        for r, n in enumerate(list(range(len(work))) + [None]):
            yield iempty[r & 1].wait((r >> 1) ^ 1)
            items[r & 1] = n
            ifull[r & 1].arrive()
            if n is not None:
                yield want.wait(r)
                yield None                                   # (the claim)

    def copies():
        me, took, vn, par = {"turn": 0}, [0, 0], 0, 0
        at = {"n": 0, "tile": 0, "freed": 0, "sent": 0}
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            walk, two = work[n]

            def tile(i):
                bar = kfull[at["tile"] % AHEAD]
                units = Bar(per_k)                           # (the barrier counts bytes: its phase ends with the last unit)
                for c in range(per_k):
                    while at["freed"] + AHEAD <= at["tile"] or at["freed"] * per_k + KU <= at["sent"]:
                        yield kempty[at["freed"] % AHEAD].wait(at["freed"] // AHEAD)
                        at["freed"] += 1
                    flying.append((keys, at["n"], (n, i, c), (units, bar)))
                    keys[at["n"]] = "under way"
                    at["sent"] += 1
                    at["n"] = (at["n"] + 1) % KU
                at["tile"] += 1

            def some(i, vn, par):
                for c in range(per_v):
                    yield vempty[vn].wait(par ^ 1)
                    looked[vn] = 0
                    flying.append((values, vn, (n, i, c), (vraw if walk[i][1] else vfull)[vn]))
                    values[vn] = "under way"
                    vn, par = (0, par ^ 1) if vn + 1 == VU else (vn + 1, par)
                return vn, par

            yield from tile(0)
            if len(walk) <= EARLY:
                want.arrive()
            for t in range(tiles):
                if t and not two:
                    continue
                yield qempty[t].wait((took[t] & 1) ^ 1)
                flying.append((queries, t, n, qfull[t]))
                queries[t] = "under way"
                took[t] += 1
            for i in range(1, len(walk)):
                if i == len(walk) - EARLY:
                    want.arrive()
                yield from tile(i)
                vn, par = yield from some(i - 1, vn, par)
            vn, par = yield from some(len(walk) - 1, vn, par)

    def look(_):
        me, n, par = {"turn": 0}, 0, [0] * VU
        while True:
            yield from take(me)
            if me["item"] is None:
                return
            for i, (_, masked) in enumerate(work[me["item"]][0]):
                for c in range(per_v):
                    if masked:
                        yield vraw[n].wait(par[n])
                        par[n] ^= 1
                        assert values[n] == (me["item"], i, c)
                        yield None
                        looked[n] += 1
                        vok[n].arrive()
                    n = (n + 1) % VU

    def product_of_scores(t, n, step, c, place, at):
        def product():
            assert keys[place] == (n, step // per, c) and queries[t] == n
            if c == 0:
                assert scores[t][at] is None or scores[t][at] in through[t]      # what lay there was handed over and read
                scores[t][at], weights[t][at] = None, {}
            if c == per_k - 1:
                scores[t][at] = (n, step)
        return product

    def product_of_results(t, n, step, units, at, masked):
        def product():
            assert all(values[place] == (n, step // per, c) and (not masked or looked[place] == 2) for c, place in units)
            assert scores[t][at] == (n, step) and all(idle[n][4 * t + w] or weights[t][at].get(w) == (n, step) for w in range(4))
            through[t].append((n, step))
        return product

    def scorer(t):
        me = {"turn": 0}
        kt = kn = steps = took = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                break
            walk, two = work[n]
            there = t == 0 or two
            if there:
                yield qfull[t].wait(took)
            for i, (who, _) in enumerate(walk):
                yield kfull[kt % AHEAD].wait(kt // AHEAD)
                for h in range(per):
                    if not there or t not in who[h]:
                        continue
                    at = steps & 1
                    if steps > 1:
                        yield pvdone[t][at].wait((steps >> 1) - 1)
                    queue.extend([product_of_scores(t, n, i * per + h, c, (kn + c) % KU, at) for c in range(per_k)] + [sfull[t][at]])
                    steps += 1
                if there:
                    queue.append(kempty[kt % AHEAD])
                else:
                    kempty[kt % AHEAD].arrive()
                kt, kn = kt + 1, (kn + per_k) % KU
            if there:
                queue.append(qempty[t])
                took += 1
        queue.append(flushed[0][t])
        yield flushed[0][t].wait(0)

    def adder(t):
        me = {"turn": 0}
        vn = steps = 0
        vpar = [[0] * VU, [0] * VU]
        units, each = max(1, per_v // per), max(1, per // per_v)                  # units of a step, steps of a unit
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                break
            walk, two = work[n]
            there = t == 0 or two
            for i, (who, masked) in enumerate(walk):
                for h in range(per):
                    places = [(vn + u) % VU for u in range(units)]
                    if h % each == 0:
                        for place in places:
                            yield (vok if masked else vfull)[place].wait(vpar[masked][place])
                            vpar[masked][place] ^= 1
                    if there and t in who[h]:
                        at, first = steps & 1, h * units if each == 1 else 0
                        yield pfull[t][at].wait(steps >> 1)
                        queue.extend([product_of_results(t, n, i * per + h, [(first + u, place) for u, place in enumerate(places)], at, masked), pvdone[t][at]])
                        steps += 1
                    if h % each == each - 1:
                        for place in places:
                            if there:
                                queue.append(vempty[place])
                            else:
                                vempty[place].arrive()
                        vn = (vn + units) % VU
            if there:
                queue.append(odone[t])
        queue.append(flushed[1][t])
        yield flushed[1][t].wait(0)

    def softmax(x):
        t, w = divmod(x, 4)
        me = {"turn": 0}
        passed = took = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            walk, two = work[n]
            if t and not two:
                continue
            last = None
            for step in range(len(walk) * per):
                if t not in walk[step // per][0][step % per]:
                    continue
                at = passed & 1
                yield sfull[t][at].wait(passed >> 1)
                if not idle[n][x]:
                    assert scores[t][at] == (n, step)
                    yield None
                    if last is not None and rng.random() < moves:     # results are scaled again
                        if early:
                            yield pvdone[t][at ^ 1].wait((passed - 1) >> 1)
                        assert through[t][-1:] == [last]
                        yield None
                        assert through[t][-1:] == [last]
                    assert scores[t][at] == (n, step)
                    weights[t][at][w] = (n, step)
                    yield None
                pfull[t][at].arrive()
                passed += 1
                last = (n, step)
            yield odone[t].wait(took)
            took += 1
            if not idle[n][x]:
                assert through[t][-1:] == [last]
                yield None

    roles = [deal(), copies(), *(scorer(t) for t in range(tiles)), *(adder(t) for t in range(tiles))] + [look(k) for k in range(2)] + [softmax(x) for x in range(soft)]
    speed = [rng.choice([1, 1, 1, 10, 0.05]) for _ in roles] + [rng.choice([1, 0.1, 10]) for _ in range(2)]
    at = [next(r, False) for r in roles]                      # what a role waits for: a test, None, or False at its end
    while queue or flying or any(a is not False for a in at):
        able = [k for k, a in enumerate(at) if a is None or (a is not False and a())] + ([len(roles)] if queue else []) + ([len(roles) + 1] if flying else [])
        assert able, "nobody can go on"
        k = rng.choices(able, [speed[j] for j in able])[0]
        if k == len(roles):
            job = queue.pop(0)
            job.arrive() if isinstance(job, Bar) else job()
        elif k > len(roles):
            where, place, what, bar = flying.pop(rng.randrange(len(flying)))
            where[place] = what
            if isinstance(bar, tuple):
                bar[0].arrive()
                if bar[0].phase:
                    bar[1].arrive()
            else:
                bar.arrive()
        else:
            at[k] = next(roles[k], False)


def draw(rng, dk):
    tiles = SHAPES[dk][0]
    work, idle = [], []
    for _ in range(rng.randint(1, 5)):
        two = tiles == 2 and rng.random() < 0.8
        walk = [([{0} if not two else rng.choice([{0, 1}, {0, 1}, {0, 1}, {0}, {1}, set()]) for _ in range(tiles)], rng.random() < 0.4) for _ in range(rng.randint(1, 7))]
        walk[0][0][0] = {0, 1} if two else {0}               # (a row tile that has rows sees something)
        work.append((walk, two))
        row = [rng.random() < 0.2 for _ in range(4 * tiles)]
        row[0] = False                                       # (a row tile that has rows has its first)
        if two:
            row[4] = False
        idle.append(row)
    return dict(dk=dk, work=work, idle=idle, moves=rng.choice([0, 0.3, 1]))


@pytest.mark.parametrize("dk", sorted(SHAPES))
def test_roles_meet_in_every_order(dk):
    rng = random.Random(dk)
    for _ in range(400):
        run(rng, **draw(rng, dk))


def test_the_wait_for_the_product_ahead_is_needed():
    """The check itself sees what it is for: without that wait, results are scaled while a product adds to them."""
    rng, found = random.Random(5), 0
    for _ in range(400):
        try:
            run(rng, **draw(rng, 256), early=False)
        except AssertionError:
            found += 1
    assert found > 20
