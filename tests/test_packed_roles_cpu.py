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


EARLY = 8                                                    # tiles ahead of the end at which more work is asked for
SHAPES = {64: (2, 8, 8), 128: (2, 6, 4), 192: (2, 3, 3), 256: (1, 2, 3)}      # row tiles, places of keys and of values


def run(rng, dk, work, idle, moves, early=True, joint=False):
    """work: items, each a list of (tiles of keys: (row tiles that see some of it, whether some row does not see all)) and whether the second row tile has rows.  idle: softmax warps without rows;
    early: the wait for the product ahead, where a reference moves; joint: both row tiles have the same rows, each every second tile of keys."""
    tiles, KP, VP = SHAPES[dk]
    bars = lambda n, count: [Bar(count) for _ in range(n)]
    soft = 4 * tiles
    kfull, kempty, vfull, vempty, vok, vraw = bars(KP, 1), bars(KP, tiles), bars(VP, 1), bars(VP, tiles), bars(VP, 1), bars(VP, 1)
    qfull, qempty, odone, ifull = bars(2, 1), bars(2, 2 if joint else 1), bars(2, 1), bars(2, 1)
    joined, read, halves = Bar(4), Bar(4), [None] * 4        # what the second row tile has is ready, was read; by which item and step its warps' results are
    sfull, pvdone, pfull = ([bars(2, n) for _ in range(2)] for n in (1, 1, 4))            # [row tile][place]
    iempty, flushed = bars(2, soft + 2 * tiles + 3), [bars(2, 1) for _ in range(2)]
    items, want = [None, None], Bar(1)
    keys, values, queries, looked = [None] * KP, [None] * VP, [None] * 2, [0] * VP
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

    def copy_keys():
        me, took, at, par = {"turn": 0}, [0, 0], 0, 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            walk, two = work[n]
            for i in range(len(walk)):
                yield kempty[at].wait(par ^ 1)
                flying.append((keys, at, (n, i), kfull[at]))
                keys[at] = "under way"
                at, par = (0, par ^ 1) if at + 1 == KP else (at + 1, par)
                if i == max(0, len(walk) - EARLY):
                    want.arrive()
                for t in range(tiles if i == 0 else 0):
                    if t and (joint or not two):
                        continue
                    yield qempty[t].wait((took[t] & 1) ^ 1)
                    flying.append((queries, t, n, qfull[t]))
                    queries[t] = "under way"
                    took[t] += 1

    def copy_values():
        me, at, par = {"turn": 0}, 0, 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            for i, (_, masked) in enumerate(work[n][0]):
                yield vempty[at].wait(par ^ 1)
                looked[at] = 0
                flying.append((values, at, (n, i), (vraw if masked else vfull)[at]))
                values[at] = "under way"
                at, par = (0, par ^ 1) if at + 1 == VP else (at + 1, par)

    def look():
        me, at, par = {"turn": 0}, 0, [0] * VP
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            for i, (_, masked) in enumerate(work[n][0]):
                if masked:
                    yield vraw[at].wait(par[at])
                    par[at] ^= 1
                    assert values[at] == (n, i)
                    yield None
                    looked[at] += 1
                    vok[at].arrive()
                at = (at + 1) % VP

    def product_of_scores(t, n, i, unit, at):
        def product():
            assert keys[unit] == (n, i) and queries[0 if joint else t] == n
            assert scores[t][at] is None or scores[t][at] in through[t]          # what lay there was handed over and read
            scores[t][at], weights[t][at] = (n, i), {}
        return product

    def product_of_results(t, n, i, unit, at, masked):
        def product():
            assert values[unit] == (n, i) and (not masked or looked[unit] == 1)
            assert scores[t][at] == (n, i) and all(idle[n][4 * t + w] or weights[t][at].get(w) == (n, i) for w in range(4))
            through[t].append((n, i))
        return product

    def scorer(t):
        me = {"turn": 0}
        kn = par = passed = took = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                break
            walk, two = work[n]
            there = t == 0 or two
            if there:
                yield qfull[0 if joint else t].wait(took)
            for i, (who, _) in enumerate(walk):
                yield kfull[kn].wait(par)
                if there and t in who:
                    at = passed & 1
                    if passed > 1:
                        yield pvdone[t][at].wait((passed >> 1) - 1)
                    queue.extend([product_of_scores(t, n, i, kn, at), sfull[t][at]])
                    passed += 1
                if there:
                    queue.append(kempty[kn])
                else:
                    kempty[kn].arrive()
                kn, par = (0, par ^ 1) if kn + 1 == KP else (kn + 1, par)
            if there:
                queue.append(qempty[0 if joint else t])
                took += 1
        queue.append(flushed[0][t])
        yield flushed[0][t].wait(0)

    def adder(t):
        me = {"turn": 0}
        vn = passed = 0
        par = [[0] * VP, [0] * VP]
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                break
            walk, two = work[n]
            there = t == 0 or two
            for i, (who, masked) in enumerate(walk):
                yield (vok if masked else vfull)[vn].wait(par[masked][vn])
                par[masked][vn] ^= 1
                if there and t in who:
                    at = passed & 1
                    yield pfull[t][at].wait(passed >> 1)
                    queue.extend([product_of_results(t, n, i, vn, at, masked), pvdone[t][at]])
                    passed += 1
                if there:
                    queue.append(vempty[vn])
                else:
                    vempty[vn].arrive()
                vn = (vn + 1) % VP
            if there and any(t in who for who, _ in walk):
                queue.append(odone[t])
        queue.append(flushed[1][t])
        yield flushed[1][t].wait(0)

    def softmax(x):
        t, w = divmod(x, 4)
        me = {"turn": 0}
        passed = took = pairs = 0
        while True:
            yield from take(me)
            n = me["item"]
            if n is None:
                return
            walk, two = work[n]
            if t and not two:
                continue
            last = None
            for step, (who, _) in enumerate(walk):
                if t not in who:
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
            if any(t in who for who, _ in walk):
                yield odone[t].wait(took)
                took += 1
            if not idle[n][x] and last is not None:
                assert through[t][-1:] == [last]
                yield None
            if joint and t:
                halves[w] = (n, last)
                yield None
                joined.arrive()
                yield read.wait(pairs)
                pairs += 1
            elif joint:
                yield joined.wait(pairs)
                if not idle[n][x]:
                    assert halves[w] == (n, last and max(((n, i) for i, (who, _) in enumerate(walk) if 1 in who), default=None))
                    assert halves[w][1] is None or through[1][-1:] == [halves[w][1]]
                    yield None
                    assert (halves[w][1] is None or through[1][-1:] == [halves[w][1]]) and through[0][-1:] == [last]
                read.arrive()
                pairs += 1

    roles = [deal(), copy_keys(), copy_values(), *(scorer(t) for t in range(tiles)), *(adder(t) for t in range(tiles)), look()] + [softmax(x) for x in range(soft)]
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
            bar.arrive()
        else:
            at[k] = next(roles[k], False)


def draw(rng, dk):
    tiles = SHAPES[dk][0]
    work, idle = [], []
    for _ in range(rng.randint(1, 5)):
        two = tiles == 2 and rng.random() < 0.8
        walk = [({0} if not two else rng.choice([{0, 1}, {0, 1}, {0, 1}, {0}, {1}]), rng.random() < 0.4) for _ in range(rng.randint(1, 12))]
        walk[0] = ({0, 1} if two else {0}, walk[0][1])       # (a row tile that has rows sees something)
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


@pytest.mark.parametrize("dk", [64, 128, 192])
def test_roles_meet_where_row_tiles_share_their_rows(dk):
    rng = random.Random(dk + 1)
    for _ in range(400):
        x = draw(rng, dk)
        x["work"] = [([({i & 1}, masked) for i, (_, masked) in enumerate(walk)], True) for walk, _ in x["work"]]
        x["idle"] = [row[:4] * 2 for row in x["idle"]]
        run(rng, **x, joint=True)


def test_the_wait_for_the_product_ahead_is_needed():
    """The check itself sees what it is for: without that wait, results are scaled while a product adds to them."""
    rng, found = random.Random(5), 0
    for _ in range(400):
        try:
            run(rng, **draw(rng, 256), early=False)
        except AssertionError:
            found += 1
    assert found > 20


def test_what_rows_see_of_the_tiles():
    """walk_of and seen_by (csrc/dsk_prompt.cuh), restated, against the mask itself: every key that a token sees lies in a tile of the walk, once, and ranges say rightly which tiles some token sees and
    which ones all of them see whole."""
    T, rng = 64, random.Random(0)
    for _ in range(4000):
        window, keep = rng.choice([0, 0, 1, 2, rng.randint(1, 300), rng.randint(1, 900)]), rng.choice([0, 1, 64, 65, rng.randint(0, 400)])
        tok, n = rng.randint(0, 700), rng.choice([1, 2, 7, 32, 64, 128])
        length = tok + rng.randint(1, 2 * n)
        t1 = min(tok + 2 * n, length)
        low = max(0, tok + 1 - window) // T if window else 0
        first = -(-min(keep, t1) // T) if window else 0
        kept = min(first, low)
        tiles = [i if i < kept else low + i - kept for i in range(kept + -(-t1 // T) - low)]
        assert len(set(tiles)) == len(tiles)
        sees = lambda i, j: j <= i and (not window or i - j < window or j < keep)
        for a in (tok, tok + n):
            if a >= length:
                continue
            b, at = min(a + n, length) - 1, kept - low
            some, upto = max(0, a + 1 - window) // T + at if window else 0, b // T + 1 + at
            whole, end = max(-(-max(0, b + 1 - window) // T) + at, kept) if window else 0, (a + 1) // T + at
            seen = {j // T for i in (a, b, (a + b) // 2) for j in (0, keep - 1, i - window + 1, i) if 0 <= j and sees(i, j)}
            assert seen <= set(tiles)
            for i, tile in enumerate(tiles):
                keys = [tile * T, tile * T + T - 1]
                any_of = keys[0] <= b and (not window or a - keys[1] < window or keys[0] < keep)
                assert (i < upto and (i < first or i >= some)) == any_of
                if whole <= i < end:
                    assert all(sees(x, y) for x in (a, b) for y in keys)
                elif not window:
                    assert not all(sees(a, y) for y in keys)


def test_a_row_tile_by_itself_sees_something_of_every_tile():
    """Where both row tiles have the same rows, each every second tile of the walk (seen_by, csrc/dsk_prompt.cuh): a walk of two tiles or more has work for both."""
    T, rng = 64, random.Random(1)
    for _ in range(4000):
        window, keep = rng.choice([0, 0, 1, 2, rng.randint(1, 300), rng.randint(1, 900)]), rng.choice([0, 1, 64, 65, rng.randint(0, 400)])
        a, n = rng.randint(0, 700), rng.choice([1, 2, 7, 32, 64, 128])
        t1 = a + rng.randint(1, n)
        low = max(0, a + 1 - window) // T if window else 0
        first = -(-min(keep, t1) // T) if window else 0
        kept = min(first, low)
        some, upto = max(0, a + 1 - window) // T + kept - low if window else 0, (t1 - 1) // T + 1 + kept - low
        assert all(i < upto and (i < first or i >= some) for i in range(kept + -(-t1 // T) - low))


def deal(rng, given, users, waits=True):
    """The warp that deals out work, by itself: given are the CTAs whose work it gets, its own first and then one for each claim (True: there is a piece for it; False: none, so that it claims the
    next one), users the roles that take items, of which the first asks for more.  Several claims may come ahead of the first item, and between two.  waits: for an answer, ahead of reading it.
    Returns what each role took."""
    claimed, want, ifull, iempty = Bar(1), Bar(1), [Bar(1) for _ in range(2)], [Bar(users) for _ in range(2)]
    items, answer, flying, took = [None, None], [None], [], [[] for _ in range(users)]

    def dealer():
        at, asks, claims, got = 0, False, 0, 0
        r = 0
        while True:
            while at is not None and (asks or not given[at]):
                asks, got = False, got + 1
                flying.append(got if got < len(given) else None)          # (the answer lands some time later; None: no CTA is left, and no other may be asked for)
                if waits:
                    yield claimed.wait(claims)
                else:
                    yield None
                claims += 1
                at = answer[0]
                assert at == (got if got < len(given) else None)
                yield None
            yield iempty[r & 1].wait((r >> 1) ^ 1)
            items[r & 1] = at
            yield None
            ifull[r & 1].arrive()
            if at is None:
                return
            yield want.wait(r)
            asks = True
            r += 1

    def user(x):
        turn = 0
        while True:
            yield ifull[turn & 1].wait(turn >> 1)
            n = items[turn & 1]
            yield None
            assert items[turn & 1] == n
            iempty[turn & 1].arrive()
            turn += 1
            if n is None:
                return
            took[x].append(n)
            if x == 0:
                want.arrive()
            yield None

    roles = [dealer()] + [user(x) for x in range(users)]
    speed = [rng.choice([1, 10, 0.05]) for _ in range(users + 2)]
    at = [next(r, False) for r in roles]
    while flying or any(a is not False for a in at):
        able = [k for k, a in enumerate(at) if a is None or (a is not False and a())] + ([users + 1] if flying else [])
        assert able, "nobody can go on"
        k = rng.choices(able, [speed[j] for j in able])[0]
        if k == users + 1:
            answer[0] = flying.pop(0)
            claimed.arrive()
        else:
            at[k] = next(roles[k], False)
    return took


def test_claims_of_ctas_without_a_piece():
    rng = random.Random(7)
    for _ in range(1500):
        given = [rng.random() < rng.choice([0.2, 0.5, 1.0]) for _ in range(rng.randint(1, 12))]
        took = deal(rng, given, rng.choice([1, 2, 11]))
        assert all(x == [n for n, piece in enumerate(given) if piece] for x in took), (given, took)


def test_the_wait_for_an_answer_is_needed():
    rng, found = random.Random(8), 0
    for _ in range(200):
        try:
            deal(rng, [True, False, True], 3, waits=False)
        except AssertionError:
            found += 1
    assert found > 20
