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


AHEAD = 4                                                    # tiles of keys under way
SHAPES = {64: (2, 1, 1, 6, 5), 128: (2, 2, 2, 6, 4), 192: (2, 3, 2, 5, 3), 256: (1, 4, 4, 6, 4)}      # row tiles, units of keys and of values a tile, places for them


def run(rng, dk, work, idle, moves, early=True):
    """work: items, each a list of (tiles of keys: (row tiles that see some of it, whether some row does not see all)) and whether the second row tile has rows.  idle: softmax warps without
    rows; early: the wait for the product ahead, where a reference moves with one row tile."""
    tiles, per_k, per_v, KU, VU = SHAPES[dk]
    bars = lambda n, count: [Bar(count) for _ in range(n)]
    soft = 4 * tiles
    kfull, kempty, vfull, vempty, vok, vraw = bars(AHEAD, 1), bars(AHEAD, tiles), bars(VU, 1), bars(VU, tiles), bars(VU, 3), bars(VU, 1)
    qfull, qempty, sfull, pvdone, odone, ifull, turns = *(bars(2, 1) for _ in range(6)), bars(2, 4)
    pfull, iempty, flushed = [bars(2, 4) for _ in range(2)], bars(2, soft + 7), bars(2, 1)
    items = [None, None]
    keys, values, queries, looked = [None] * KU, [None] * VU, [None] * 2, [0] * VU
    scores, weights, through = [None, None], [[{}, {}], [{}, {}]], [None, None]
    queue, flying = [], []                                   # products and commits in the order of their issue; copies in any order

    def take(state):
        slot = state["turn"] & 1
        yield ifull[slot].wait(state["turn"] >> 1)
        state["item"] = items[slot]
        yield None
        iempty[slot].arrive()
        state["turn"] += 1

    def deal():
        par = 0
        for r, n in enumerate(list(range(len(work))) + [None]):
            yield iempty[r & 1].wait(par ^ 1)
            items[r & 1] = n
            ifull[r & 1].arrive()
            if r & 1:
                par ^= 1

    def copy_keys():
        me, took = {"turn": 0}, [0, 0]
        at = {"n": 0, "tile": 0, "freed": 0, "sent": 0}
        while True:
            yield from take(me)
            if me["item"] is None:
                return
            walk, two = work[me["item"]]

            def tile(i):
                bar = kfull[at["tile"] % AHEAD]
                units = Bar(per_k)                           # (the barrier counts bytes: its phase ends with the last unit)
                for c in range(per_k):
                    while at["freed"] + AHEAD <= at["tile"] or at["freed"] * per_k + KU <= at["sent"]:
                        yield kempty[at["freed"] % AHEAD].wait(at["freed"] // AHEAD)
                        at["freed"] += 1
                    flying.append((keys, at["n"], (me["item"], i, c), (units, bar)))
                    keys[at["n"]] = "under way"
                    at["sent"] += 1
                    at["n"] = (at["n"] + 1) % KU
                at["tile"] += 1

            yield from tile(0)
            for t in range(tiles):
                if t and not two:
                    continue
                yield qempty[t].wait((took[t] & 1) ^ 1)
                flying.append((queries, t, me["item"], qfull[t]))
                queries[t] = "under way"
                took[t] += 1
            for i in range(1, len(walk)):
                yield from tile(i)

    def copy_values():
        me, n, par = {"turn": 0}, 0, 0
        while True:
            yield from take(me)
            if me["item"] is None:
                return
            for i, (_, masked) in enumerate(work[me["item"]][0]):
                for c in range(per_v):
                    yield vempty[n].wait(par ^ 1)
                    looked[n] = 0
                    flying.append((values, n, (me["item"], i, c), (vraw if masked else vfull)[n]))
                    values[n] = "under way"
                    n, par = (0, par ^ 1) if n + 1 == VU else (n + 1, par)

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

    def product_of_scores(t, n, i, c, place, buf):
        def product():
            assert keys[place] == (n, i, c) and queries[t] == n
            if c == 0:
                if scores[buf] is not None:                  # what lay there was handed over and read
                    assert through[buf if tiles == 1 else t] == scores[buf]
                scores[buf], weights[buf] = None, [{}, {}]
            if c == per_k - 1:
                scores[buf] = (n, i)
        return product

    def product_of_results(t, n, i, c, place, buf, masked, half, last):
        def product():
            assert values[place] == (n, i, c) and (not masked or looked[place] == 3) and scores[buf] == (n, i)
            for h in ([half] if half is not None else [0, 1]):
                assert all(idle[n][4 * t + w] or weights[buf][h].get(w) == (n, i) for w in range(4))
            if last:
                through[buf if tiles == 1 else t] = (n, i)
        return product

    def issue_scores(t, state, n, i, buf):
        places = [(state["kn"] + c) % KU for c in range(per_k)]
        queue.extend([product_of_scores(t, n, i, c, place, buf) for c, place in enumerate(places)] + [sfull[buf], kempty[state["kt"] % AHEAD]])

    def next_keys(state):
        state["kt"] += 1
        state["kn"] = (state["kn"] + per_k) % KU

    def keys_there(state):
        return kfull[state["kt"] % AHEAD].wait(state["kt"] // AHEAD)

    def values_there(state, masked):
        for c in range(per_v):
            place = (state["vn"] + c) % VU
            yield (vok if masked else vfull)[place].wait(state["vpar"][masked][place])
            state["vpar"][masked][place] ^= 1

    def issue_results(t, state, n, i, buf, parity, masked):
        steps = 8 // per_v
        for u in range(8):
            place = state["vn"]
            if u % 4 == 0:
                yield pfull[buf][u // 4].wait(parity)
            if u % steps == steps - 1 or u == 3:
                queue.append(product_of_results(t, n, i, u // steps, place, buf, masked, u // 4 if steps <= 4 else (0 if u == 3 else None), u == 7))
                if u == 7:
                    queue.append(pvdone[t if tiles == 2 else buf])
            if u % steps == steps - 1:
                if tiles == 2 and u == 7:
                    state["pend"] = place
                else:
                    queue.append(vempty[place])
                state["vn"] = (place + 1) % VU

    def give_back(state):
        if state["pend"] is not None:
            queue.append(vempty[state["pend"]])
            state["pend"] = None

    def issuer(x):
        me = {"turn": 0, "kt": 0, "kn": 0, "vn": 0, "vpar": [[0] * VU, [0] * VU], "pend": None}
        passed = took = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                break
            walk, two = work[n]
            if tiles == 2:
                there = x == 0 or two
                if there:
                    yield qfull[x].wait(took)
                yield keys_there(me)
                for i, (who, masked) in enumerate(walk):
                    mine = there and x in who
                    if mine:
                        if passed:
                            yield pvdone[x].wait(passed - 1)
                        issue_scores(x, me, n, i, x)
                    else:
                        kempty[me["kt"] % AHEAD].arrive()
                    give_back(me)
                    next_keys(me)
                    if i + 1 < len(walk):
                        yield keys_there(me)
                    elif there:
                        queue.append(qempty[x])
                    yield from values_there(me, masked)
                    if mine:
                        yield from issue_results(x, me, n, i, x, passed, masked)
                        passed += 1
                    else:
                        for _ in range(per_v):
                            vempty[me["vn"]].arrive()
                            me["vn"] = (me["vn"] + 1) % VU
                if there:
                    queue.append(odone[x])
                    took += 1
                give_back(me)
            elif x == 0:
                yield qfull[0].wait(took)
                for i in range(len(walk)):
                    yield keys_there(me)
                    if passed > 1:
                        yield pvdone[passed & 1].wait((passed >> 1) - 1)
                    issue_scores(0, me, n, i, passed & 1)
                    next_keys(me)
                    passed += 1
                queue.append(qempty[0])
                took += 1
            else:
                for i, (_, masked) in enumerate(walk):
                    yield from values_there(me, masked)
                    yield from issue_results(0, me, n, i, passed & 1, passed >> 1, masked)
                    passed += 1
                queue.append(odone[0])
        queue.append(flushed[x])
        yield flushed[x].wait(0)

    def softmax(x):
        t, w = divmod(x, 4)
        me = {"turn": 0}
        passed = took = gated = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            walk, two = work[n]
            if t and not two:
                continue
            last = None
            for i, (who, _) in enumerate(walk):
                if t not in who:
                    continue
                buf, par = (t, passed) if tiles == 2 else (passed & 1, passed >> 1)
                yield sfull[buf].wait(par)
                if not idle[n][x]:
                    assert scores[buf] == (n, i)
                    yield None
                    if last is not None and rng.random() < moves:     # results are scaled again
                        if tiles == 1 and early:
                            yield pvdone[buf ^ 1].wait((passed - 1) >> 1)
                        assert through[buf ^ 1 if tiles == 1 else t] == last
                        yield None
                gate = len(who) == 2
                if gate and not idle[n][x] and gated + t > 0:
                    yield turns[t].wait(gated - 1 + t)
                for half in (0, 1):
                    if not idle[n][x]:
                        assert scores[buf] == (n, i)
                        weights[buf][half][w] = (n, i)
                        yield None
                    if half and gate:
                        turns[t ^ 1].arrive()
                        gated += 1
                        yield None
                    pfull[buf][half].arrive()
                passed += 1
                last = (n, i)
            yield odone[t if tiles == 2 else 0].wait(took)
            took += 1
            if not idle[n][x]:
                assert through[t if tiles == 2 else (passed - 1) & 1] == last
                yield None

    roles = [deal(), copy_keys(), copy_values(), issuer(0), issuer(1)] + [look(k) for k in range(3)] + [softmax(x) for x in range(soft)]
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
        walk = []
        for _ in range(rng.randint(1, 6)):
            who = {0} if not two else rng.choice([{0, 1}, {0, 1}, {0}, {1}])
            walk.append((who, rng.random() < 0.4))
        walk[0] = ({0, 1} if two else {0}, walk[0][1])       # (a row tile that has rows sees some tile)
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
    """The check itself sees what it is for: without that wait, results of one row tile are scaled while a product adds to them."""
    rng, found = random.Random(5), 0
    for _ in range(400):
        try:
            run(rng, **draw(rng, 256), early=False)
        except AssertionError:
            found += 1
    assert found > 20
