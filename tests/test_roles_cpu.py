"""The roles of attend_rows (csrc/dsk_kv8_tc5.cuh) in random interleavings: barriers with phases and waits by parity, products that run in order some time after they were issued.  Every use
of a stage, of scores, weights, scales and results is checked against who wrote it last; a state in which nobody can go on is an error too.  This restates the kernel's protocol by hand: whoever
changes waits, commits or arrivals there changes them here."""
import random

import pytest

SLOTS = 4


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def wait(self, parity):
        return lambda: (self.phase & 1) != parity


def stages(tiles, dk):
    """Stages of keys and of values (k_stages, v_stages)."""
    return 3 if dk == 64 and tiles == 2 else 1 if dk == 256 else 2, 1 if dk == 256 or (dk == 192 and tiles == 2) else 3 if dk == 64 else 2


def run(rng, tiles, dk, n, idle, moves, ahead=True):
    """One CTA with n tiles of keys; idle: warps without rows; moves: how often a reference moves; ahead: the wait for the product before the last."""
    kst_n, vst_n = stages(tiles, dk)
    vw = 3 if tiles == 2 else 4
    bars = lambda k, count: [Bar(count) for _ in range(k)]
    kfull, kempty, vfull, vempty = bars(3, 4), bars(3, 1), bars(3, vw), bars(3, 1)
    sfull, pfull, pvdone, cfull = bars(2, 1), bars(2, 4), bars(2, 1), bars(SLOTS, 1)
    cdone, flushed, qfull = Bar(vw), Bar(1), Bar(4 * tiles)
    keys, values, scales = [[None] * 4 for _ in range(3)], [[None] * vw for _ in range(3)], [None] * SLOTS
    scores, weights, through, issued = [None, None], [{}, {}], [0, 0], [0, 0]
    queue = []                                               # products and commits, in the order of their issue
    where = lambda t, i: t if tiles == 2 else i & 1           # columns of a tile's scores and weights

    def score(t, i, stage):
        def product():
            assert all(x == i for x in keys[stage])
            if scores[where(t, i)] is not None:              # what lay there was read and handed over
                assert len(weights[where(t, i)]) == sum(not idle[4 * t + w] for w in range(4))
            scores[where(t, i)], weights[where(t, i)] = i, {}
        queue.extend([product, sfull[where(t, i)]])

    def values_in(t, i, stage):
        def product():
            assert all(x == i for x in values[stage]) and scores[where(t, i)] == i
            assert all(idle[4 * t + w] or weights[where(t, i)].get(w) == i for w in range(4))
            through[t] += 1
        issued[t] += 1
        queue.extend([product, pvdone[t]])

    def issuer():
        yield qfull.wait(0)
        yield kfull[0].wait(0)
        for t in range(tiles):
            score(t, 0, 0)
        queue.append(kempty[0])
        kst = vst = kturn = vturn = 0
        for i in range(n):
            more = i + 1 < n
            if more:
                kst += 1
                if kst == kst_n:
                    kst, kturn = 0, kturn ^ 1
            if tiles == 1:
                if more:
                    yield kfull[kst].wait(kturn)
                    if i > 0:
                        yield pvdone[0].wait((i - 1) & 1)
                    score(0, i + 1, kst)
                    queue.append(kempty[kst])
                yield vfull[vst].wait(vturn)
                yield pfull[i & 1].wait((i >> 1) & 1)
                values_in(0, i, vst)
                queue.append(vempty[vst])
            else:
                yield vfull[vst].wait(vturn)
                for t in range(2):
                    yield pfull[t].wait(i & 1)
                    values_in(t, i, vst)
                    if t == 1:
                        queue.append(vempty[vst])
                    if more:
                        if t == 0:
                            yield kfull[kst].wait(kturn)
                        yield pvdone[t].wait(i & 1)
                        score(t, i + 1, kst)
                        if t == 1:
                            queue.append(kempty[kst])
            vst += 1
            if vst == vst_n:
                vst, vturn = 0, vturn ^ 1
        queue.append(flushed)
        yield flushed.wait(0)
        assert not queue                                     # nothing is under way when TMEM is given back

    def bring(warp, ring, full, empty, count, which):
        stage, turn = 0, 1
        for i in range(n):
            yield empty[stage].wait(turn)
            if which == 0 and warp == 0:
                scales[i % SLOTS] = i
                cfull[i % SLOTS].arrive()
            yield None
            ring[stage][warp] = i
            full[stage].arrive()
            stage += 1
            if stage == count:
                stage, turn = 0, turn ^ 1
        if which == 1:
            cdone.arrive()

    def softmax(x):
        t, w = divmod(x, 4)
        qfull.arrive()
        for i in range(n):
            at = where(t, i)
            yield cfull[i % SLOTS].wait((i // SLOTS) & 1)
            yield sfull[t].wait(i & 1) if tiles == 2 else sfull[i & 1].wait((i >> 1) & 1)
            last = ahead and tiles == 1 and i > 0 and i + 1 == n
            if not idle[x]:
                assert scores[at] == i and scales[i % SLOTS] == i
                yield None
                assert scales[i % SLOTS] == i
                if i > 0 and rng.random() < moves:            # results are scaled again
                    if tiles == 1:
                        yield pvdone[0].wait((i - 1) & 1)
                    assert through[t] == issued[t] == i
                    yield None
                    assert through[t] == i
                weights[at][w] = i
                yield None
            if last:
                yield pvdone[0].wait((i - 1) & 1)
            pfull[at].arrive()
        yield cdone.wait(0)
        if rng.random() < 0.3:
            yield None
        yield pvdone[t].wait((n - 1) & 1)
        assert idle[x] or through[t] == n                    # the results are whole

    roles = [issuer()] + [bring(w, keys, kfull, kempty, kst_n, 0) for w in range(4)] + [bring(w, values, vfull, vempty, vst_n, 1) for w in range(vw)] + [softmax(x) for x in range(4 * tiles)]
    speed = [rng.choice([1, 1, 1, 10, 0.05]) for _ in roles] + [rng.choice([1, 0.1, 10])]
    at = [next(r, False) for r in roles]                      # what a role waits for: a test, None, or False at its end
    while queue or any(a is not False for a in at):
        able = [k for k, a in enumerate(at) if a is None or (a is not False and a())] + ([len(roles)] if queue else [])
        assert able, "nobody can go on"
        k = rng.choices(able, [speed[j] for j in able])[0]
        if k == len(roles):
            job = queue.pop(0)
            job.arrive() if isinstance(job, Bar) else job()
        else:
            at[k] = next(roles[k], False)


def draw(rng, tiles, dk):
    idle = [rng.random() < 0.2 for _ in range(4 * tiles)]
    idle[0] = False
    return dict(tiles=tiles, dk=dk, n=rng.randint(1, 11), idle=idle, moves=rng.choice([0, 0.3, 1]))


@pytest.mark.parametrize("tiles,dk", [(1, 64), (1, 128), (1, 192), (1, 256), (2, 64), (2, 128), (2, 192)])
def test_roles_meet_in_every_order(tiles, dk):
    rng = random.Random(dk + tiles)
    for _ in range(400):
        run(rng, **draw(rng, tiles, dk))


def test_results_are_read_early_without_the_wait_ahead_of_the_last_weights():
    """The check itself sees what it is for: without that wait, one row tile's results are read before its last product is through."""
    rng, early = random.Random(5), 0
    for _ in range(400):
        try:
            run(rng, **draw(rng, 1, 128), ahead=False)
        except AssertionError:
            early += 1
    assert early > 20
