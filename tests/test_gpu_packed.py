"""Packed rows: places in a cache, packed rows into the 8-bit cache, causal attention of packed prompts, against their float64 restatement (oracle/packed_oracle.py).

Tolerances of attention, from the arithmetic of the kernel: queries, keys and values are exact operands; a score's sum of d products in fp32 is off by at most (d + 4) 2^-23 sum |q k| scale, which changes
a weight by that factor, numerator and denominator alike; a weight is rounded once for the product with the values, by half a step of the type (bf16 2^-8, fp16 2^-11 of it, or 2^-25 where it is
below 2^-14: the largest weight is at least 2^6, so 2^-31 of that); the exponential is good to 2^-21; sums over L keys in fp32 to L 2^-23; the result is rounded to its type once."""
import numpy as np
import pytest
import torch

import dsk
import packed_oracle as po
import serve_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def starts_of(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32)


class Prompt:
    """Queries, keys and values of packed sequences; rows of no one hold NaN, the results' rows of no one a number that must stay."""

    def __init__(self, lens, H, G, dk, dv, dtype="bf16", spare=0, first=0, seed=0, spread=1.5, fused=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.G, self.dk, self.dv, self.dtype, self.first = list(lens), H, G, dk, dv, dtype, first
        self.starts, self.rows = starts_of(lens, first), first + sum(lens) + spare
        if fused:
            x = torch.randn(self.rows, H * dk + G * (dk + dv), generator=g).to(DT[dtype])
            x[:, :H * dk] *= spread
            q, k, v = x.split([H * dk, G * dk, G * dv], 1)
        else:
            q, k, v = torch.randn(self.rows, H * dk, generator=g) * spread, torch.randn(self.rows, G * dk, generator=g), torch.randn(self.rows, G * dv, generator=g)
            q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
        self.q, self.k, self.v = q.unflatten(1, (H, dk)), k.unflatten(1, (G, dk)), v.unflatten(1, (G, dv))
        nobody = torch.ones(self.rows, dtype=torch.bool)
        nobody[first:first + sum(lens)] = False
        for x in (self.q, self.k, self.v):
            x[nobody] = float("nan")

    def run(self, scale=None, window=0, keep=0, out=None, move=lambda x: x.to(DEV)):
        packed = dsk.Packed.of(torch.from_numpy(self.starts).to(DEV), self.rows)
        out = torch.full((self.rows, self.H, self.dv), 7.0, dtype=DT[self.dtype], device=DEV) if out is None else out
        got = packed.attend(move(self.q), move(self.k), move(self.v), scale=scale, window=window, keep_first=keep, out=out)
        packed.check()
        self.check(got, scale, window, keep)
        return got

    def check(self, got, scale=None, window=0, keep=0, left=7.0):
        s = self.dk ** -0.5 if scale is None else scale
        want, mass, size, top = po.attend(*(x.double().numpy() for x in (self.q, self.k, self.v)), self.starts, s, window, keep)
        L, half = max(self.lens + [1]), torch.finfo(DT[self.dtype]).eps / 2
        tol = mass * (half + 2 * (self.dk + 4) * 2.0 ** -23 * size + 2.0 ** -20 + L * 2.0 ** -23) + L * 2.0 ** -31 * top
        g = got.double().cpu().numpy()
        rows = slice(self.first, self.first + sum(self.lens))
        assert (g[:self.first] == left).all() and (g[self.first + sum(self.lens):] == left).all()
        w, g, tol = want[rows], g[rows], tol[rows]
        assert np.array_equal(np.isnan(w), ~np.isfinite(g)), np.argwhere(np.isnan(w) != ~np.isfinite(g))[:6]
        with np.errstate(invalid="ignore"):
            off, may = np.abs(g - w), tol + half * (np.abs(w) + tol) + 2.0 ** -25
            assert (np.isnan(w) | (off <= may)).all(), (float(np.nanmax(off / may)), np.argwhere(~(np.isnan(w) | (off <= may)))[:6])


# ---- attention ----------------------------------------------------------------------------------------------------------------------------------

DIMS = [(16, 16), (64, 64), (80, 80), (96, 64), (112, 128), (128, 128), (144, 32), (192, 128), (64, 256), (208, 240), (256, 256)]


@pytest.mark.parametrize("lens", [[1], [2], [16], [37], [64], [127], [128], [129], [255], [256], [257], [400]])
def test_one_prompt(lens):
    Prompt(lens, 4, 2, 128, 128).run()


@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_sizes(dk, dv, dtype):
    Prompt([1, 70, 300, 129], 6, 2, dk, dv, dtype=dtype, spare=3, seed=dk + dv).run()


@pytest.mark.parametrize("H,G", [(1, 1), (2, 2), (3, 1), (7, 1), (6, 2), (16, 4), (8, 1), (32, 1), (48, 1), (40, 2), (128, 1), (130, 1), (5, 5)])
@pytest.mark.parametrize("d", [64, 256])
def test_heads(H, G, d):
    Prompt([3, 150, 1, 64], H, G, d, d, seed=H).run()


@pytest.mark.parametrize("lens", [[0, 5, 0, 300, 0, 0, 7], [1] * 40, [128] * 3, [0, 0, 0], [2000], [1, 1000, 2, 999, 3], [17] * 300, [0] * 700 + [3, 200] + [0] * 100 + [1] * 200])
@pytest.mark.parametrize("spare,first", [(0, 0), (9, 0), (130, 5)])
def test_lengths(lens, spare, first):
    Prompt(lens, 4, 2, 64, 64, spare=spare, first=first, seed=len(lens), fused=True).run()


@pytest.mark.parametrize("window,keep", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 128), (129, 3), (300, 200), (500, 1000), (2000, 4), (2 ** 31 - 1, 5), (2 ** 30, 0), (7, 2 ** 31 - 1)])
@pytest.mark.parametrize("H,G,d", [(4, 4, 64), (8, 2, 128), (4, 1, 256)])
def test_windows(window, keep, H, G, d):
    Prompt([700, 1, 333], H, G, d, d, dtype="f16", spare=2, seed=window % 97).run(window=window, keep=keep)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 0.01, 1.0, 3.0])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales(scale, dtype):
    Prompt([200, 45], 4, 2, 64, 64, dtype=dtype, seed=3).run(scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_maxima_that_jump(dtype, d):
    """Keys whose scores rise by hundreds from tile to tile and within one, and fall again: references move in either half, first and later."""
    p = Prompt([900, 130], 2, 1, d, d, dtype=dtype, seed=8, spread=0.3)
    for at, size in ((0, 1.0), (70, 4.0), (130, 9.0), (200, 14.0), (300, 25.0), (440, 40.0), (441, 41.0), (700, 60.0)):
        p.k[at] = torch.sign(p.q[at + 1:at + 2, 0]) * size
    p.run()


def test_weights_follow_a_falling_maximum():
    """The first key has the largest score by far: all later references stay where it put them."""
    for dtype in ("bf16", "f16"):
        p = Prompt([600], 1, 1, 64, 64, dtype=dtype, seed=9, spread=0.5)
        p.q[:, 0, 0], p.k[:, 0, 0] = 8.0, 0.0
        p.k[0, 0, 0] = 9.0
        p.run()


@pytest.mark.parametrize("H,G,d", [(4, 2, 64), (4, 4, 128), (2, 1, 192), (2, 1, 256)])
@pytest.mark.parametrize("window,keep", [(0, 0), (50, 3)])
def test_what_is_not_finite_reaches_those_alone_that_see_it(H, G, d, window, keep):
    """NaN and infinities among values (of keys that some rows see, some do not), among keys and among queries."""
    p = Prompt([300, 140, 60], H, G, d, min(d, 128) if d == 192 else d, seed=5, spare=4)
    p.v[40, 0, 3], p.v[131, G - 1, 0], p.v[299, 0, 5], p.v[300, 0, 1], p.v[439, 0, 9], p.v[499, 0, 2] = (float(x) for x in ("nan", "inf", "-inf", "nan", "inf", "nan"))
    p.run(window=window, keep=keep)
    for x, row, value in ((p.q, 77, "nan"), (p.q, 310, "inf"), (p.k, 200, "nan"), (p.k, 450, "nan")):
        x[row, 0, 1] = float(value)
    with np.errstate(all="ignore"):
        p.run(window=window, keep=keep)


def test_scores_of_minus_infinity():
    p = Prompt([150, 20], 2, 1, 64, 64, dtype="bf16", seed=6)
    p.q[:, :, 0] = 1.0
    p.k[0:130, 0, 0] = -float("inf")                         # the first 130 rows see nothing but -inf: zeros
    got = p.run()
    assert (got[:130] == 0).all() and (got[130:150] != 0).any()


def test_masks_of_the_lowest_value():
    """A key whose entries are the type's lowest value: scores beyond 2^24, on either side."""
    for dtype in ("bf16", "f16"):
        low = torch.finfo(DT[dtype]).min
        p = Prompt([300], 1, 1, 64, 64, dtype=dtype, seed=7)
        p.q[:, 0, 0], p.k[:, 0, 0] = 1.0, 0.0
        p.k[5, 0, 0] = p.k[150, 0, 0] = p.k[299, 0, 0] = low
        p.run()
        q, k, v = p.q.clone(), p.k.clone(), p.v.clone()      # the highest: all weight on that key
        k[5, 0, 0] = k[150, 0, 0] = k[299, 0, 0] = 0
        k[20, 0, 0] = -low
        packed = dsk.Packed.of(ints([0, 300]), 300)
        got = packed.attend(q.to(DEV), k.to(DEV), v.to(DEV), scale=0.25).cpu()
        packed.check()
        # one weight w alone: the product has it rounded, the sum has not, so that v w (1 + d) / w is off by half a step, and rounding the result by another (2.01: of their product)
        off, half = (got[20:, 0].double() - v[20, 0].double()).abs(), torch.finfo(DT[dtype]).eps / 2
        assert (off <= 2.01 * half * v[20, 0].double().abs()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_at_the_ends_of_the_type(dtype):
    """Sums of weights times the largest values do not run over."""
    p = Prompt([500], 2, 1, 64, 64, dtype=dtype, seed=11, spread=0.01)
    p.v[:] = torch.finfo(DT[dtype]).max * 0.99
    packed = dsk.Packed.of(torch.from_numpy(p.starts).to(DEV), 500)
    got = packed.attend(p.q.to(DEV), p.k.to(DEV), p.v.to(DEV))
    packed.check()
    assert torch.isfinite(got).all() and ((got.double().cpu() / p.v[0, 0, 0].double() - 1).abs() <= 3 * torch.finfo(DT[dtype]).eps).all()


def test_orders_of_rows_and_heads():
    """Heads ahead of rows, gaps between rows, an output whose rows are not 16-byte aligned."""
    p = Prompt([90, 200], 4, 2, 64, 64, seed=12, spare=1)

    def heads_first(x):
        return x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)

    def gaps(x):
        y = torch.full((x.shape[0], x.shape[1] + 1, x.shape[2] + 24), float("nan"), dtype=x.dtype, device=DEV)
        y[:, 1:, 8:8 + x.shape[2]] = x.to(DEV)
        return y[:, 1:, 8:8 + x.shape[2]]

    p.run(move=heads_first)
    p.run(move=gaps)
    odd = torch.full((p.rows, 4 * 64 + 3), 7.0, dtype=torch.bfloat16, device=DEV)
    p.run(out=odd[:, 1:257].unflatten(1, (4, 64)))
    assert (odd[:, 0] == 7).all() and (odd[:, 257:] == 7).all()
    half = torch.full((p.rows, 4 * 64 + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    p.run(out=half[:, 8:].unflatten(1, (4, 64)))             # on 16 bytes, not on 32
    assert (half[:, :8] == 7).all()


def many(H):
    """Rows of no one behind the sequences, so many that CTAs have two row tiles each (with few rows both have the same rows, each every second tile of keys)."""
    return 42_000 // H


@pytest.mark.parametrize("dk,dv", [(16, 16), (64, 64), (112, 128), (128, 128), (192, 128)])
@pytest.mark.parametrize("lens", [[1], [64, 65], [300, 1, 0, 129], [700]])
def test_two_row_tiles(lens, dk, dv):
    Prompt(lens, 8, 4, dk, dv, dtype="f16" if dk == 64 else "bf16", spare=many(8), seed=dk + len(lens)).run()


@pytest.mark.parametrize("H,G", [(8, 8), (14, 2), (6, 2), (24, 2), (10, 1)])
@pytest.mark.parametrize("window,keep", [(0, 0), (100, 3), (1, 1), (64, 200)])
def test_two_row_tiles_heads_and_windows(H, G, window, keep):
    Prompt([400, 33], H, G, 64, 64, spare=many(H), seed=H).run(window=window, keep=keep)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_two_row_tiles_maxima_that_jump(dtype, d):
    p = Prompt([900, 130], 8, 4, d, d, dtype=dtype, seed=8, spread=0.3, spare=many(8))
    for at, size in ((0, 1.0), (70, 4.0), (130, 9.0), (200, 14.0), (300, 25.0), (440, 40.0), (441, 41.0), (700, 60.0)):
        p.k[at] = torch.sign(p.q[at + 1:at + 2, 0]) * size
    p.run()


@pytest.mark.parametrize("window,keep", [(0, 0), (50, 3)])
@pytest.mark.parametrize("spare", [0, many(8)])
def test_two_row_tiles_and_what_is_not_finite(spare, window, keep):
    p = Prompt([300, 140, 60], 8, 4, 64, 64, seed=5, spare=4 + spare)
    p.v[40, 0, 3], p.v[70, 2, 1], p.v[131, 3, 0], p.v[299, 0, 5], p.v[300, 0, 1], p.v[439, 0, 9] = (float(x) for x in ("nan", "-inf", "inf", "-inf", "nan", "inf"))
    p.k[450, 1, 0] = float("nan")
    p.run(window=window, keep=keep)


@pytest.mark.parametrize("seed", range(6))
def test_few_rows_whose_maximum_lies_in_either_half(seed):
    """Where both row tiles of a CTA have the same rows, either one's reference may be beyond the other's by more than a weight can say, or one may have no key of a row at all."""
    p = Prompt([130, 65, 64, 193], 2, 1, 64, 64, dtype="bf16" if seed % 2 else "f16", seed=seed, spread=0.5)
    g = torch.Generator().manual_seed(seed)
    for at in torch.randperm(450, generator=g)[:6].tolist():
        p.k[at] *= 2.0 ** (seed + 2)
    p.run()
    p.run(window=70, keep=2)


def test_rows_beyond_four_gigabytes():
    """Queries, keys, values and results as parts of rows that lie 16 KB apart: offsets beyond 2^32 bytes and 2^31 entries."""
    p = Prompt([90, 60], 2, 1, 64, 64, seed=16)
    rows = 290_000
    wide = torch.zeros(rows, 8192, dtype=torch.bfloat16, device=DEV)
    at = rows - 150
    for x, c in ((p.q, 0), (p.k, 4096), (p.v, 8128)):
        wide[at:, c:c + x.shape[1] * 64] = x.flatten(1).to(DEV)
    out = wide[:, 1024:1152].unflatten(1, (2, 64))
    dsk.Packed.of(ints([at, at + 90, rows]), rows).attend(wide[:, :128].unflatten(1, (2, 64)), wide[:, 4096:4160, None].transpose(1, 2), wide[:, 8128:, None].transpose(1, 2), out=out)
    p.check(out[at:].contiguous())
    assert (out[:at] == 0).all()


@pytest.mark.parametrize("H,G", [(1, 1), (16, 16), (16, 2)])
def test_more_heads_than_the_cache_holds(H, G):
    """Heads are worked on a few at a time where their keys and values are many: every piece of work is done once."""
    n = 300_000 if G == 1 else 150_000
    lens = [64] * 2 + [n - 300] + [1] * 40 + [70]
    g = torch.Generator(device=DEV).manual_seed(17)
    q, k, v = (torch.randn(n, h, 64, generator=g, device=DEV).to(torch.bfloat16) for h in (H, G, G))
    out = torch.full((n, H, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    packed = dsk.Packed.of(torch.from_numpy(starts_of(lens)).to(DEV), n)
    packed.attend(q, k, v, window=100, out=out)
    packed.check()
    end = sum(lens)
    assert torch.isfinite(out[:end]).all() and torch.isnan(out[end:]).all()
    for row, first in ((3, 0), (100, 64), (n // 2, 128), (128 + n - 301, 128), (128 + n - 300 + 39, 128 + n - 300 + 39), (end - 1, end - 70)):
        lo = max(first, row - 99)
        for h in (0, H - 1):
            kk, vv = k[lo:row + 1, h * G // H].double(), v[lo:row + 1, h * G // H].double()
            w = torch.softmax(kk @ q[row, h].double() * 64 ** -0.5, 0)
            # (as Prompt.check: weights, scores and the result are rounded)
            tol = (w @ vv.abs()) * 2.0 ** -7.5 + 2.0 ** -8 * (w @ vv).abs() + 2.0 ** -20
            assert ((out[row, h].double() - w @ vv).abs() <= tol).all()


def test_starts_that_fall_or_point_outside_stay_inside():
    """Whatever starts say, rows outside the tensors are not touched, and sequences that are sound come out right."""
    p = Prompt([100, 50], 2, 1, 64, 64, seed=13, spare=60)
    out = torch.zeros(p.rows, 2, 64, dtype=torch.bfloat16, device=DEV)
    packed = dsk.Packed.of(ints([0, 100, 150, 120, 1 << 30, -5, 90]), p.rows)
    packed.attend(p.q.to(DEV), p.k.to(DEV), p.v.to(DEV), out=out)
    packed.check()
    want = torch.zeros_like(out)
    dsk.Packed.of(ints([0, 100]), p.rows).attend(p.q.to(DEV), p.k.to(DEV), p.v.to(DEV), out=want)
    assert torch.equal(out[:90], want[:90])


def test_streams_and_graphs():
    """Calls on two streams at a time, and a captured call that is replayed with other values and other lengths."""
    a, b = Prompt([300, 20], 4, 2, 128, 128, seed=14), Prompt([64, 256], 4, 2, 128, 128, seed=15)
    dev = [[x.to(DEV) for x in (p.q, p.k, p.v)] for p in (a, b)]
    plans = [dsk.Packed.of(torch.from_numpy(p.starts).to(DEV), 320) for p in (a, b)]
    outs = [torch.full((320, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, x, plan, out in zip(streams, dev, plans, outs):
            with torch.cuda.stream(s):
                plan.attend(*x, out=out)
    torch.cuda.synchronize()
    a.check(outs[0])
    b.check(outs[1])
    q, k, v, starts, out = (x.clone() for x in (*dev[0], plans[0].starts, outs[0]))
    plan, g = dsk.Packed.of(starts, 320), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attend(q, k, v, out=out)
    for p, x in ((a, dev[0]), (b, dev[1])):
        for to, of in zip((q, k, v, starts), (*x, torch.from_numpy(p.starts).to(DEV))):
            to.copy_(of)
        out.fill_(7.0)
        g.replay()
        plan.check()
        p.check(out)


def test_attention_refuses():
    p = Prompt([10], 2, 1, 64, 64)
    q, k, v = (x.to(DEV) for x in (p.q, p.k, p.v))
    packed = dsk.Packed.of(ints([0, 10]), 10)
    for kw, text in ((dict(scale=-1.0), "not negative"), (dict(scale=float("nan")), "not negative"), (dict(window=-1), "negative"), (dict(keep_first=-2), "negative"),
                     (dict(out=torch.zeros(10, 2, 64, device=DEV)), "results of"), (dict(out=torch.zeros(9, 2, 64, dtype=torch.bfloat16, device=DEV)), "output"),
                     (dict(out=torch.zeros(10, 1, 64, dtype=torch.bfloat16, device=DEV).expand(10, 2, 64)), "overlap")):
        with pytest.raises(dsk.DskError, match=text):
            packed.attend(q, k, v, **kw)
    for x, text in (((q.float(), k.float(), v.float()), "F16 or BF16"), ((q, k.half(), v), "keys of"), ((q[:, :, :60], k[:, :, :60], v), "multiple of 16"), ((q[:9], k, v), "queries"), ((q, k[:, :, :48], v), "keys"),
                    ((q.cpu(), k, v), "CUDA"), ((q[:, :, None], k, v), "rows, heads"), ((q, k.expand(10, 3, 64), v.expand(10, 3, 64)), "multiple")):
        with pytest.raises(dsk.DskError, match=text):
            packed.attend(*x)
    odd = torch.zeros(10, 2 * 64 + 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(dsk.DskError, match="multiple of 8"):
        packed.attend(odd[:, :128].unflatten(1, (2, 64)), k, v)
    with pytest.raises(dsk.DskError, match="16-byte"):
        packed.attend(odd[:, 1:129].unflatten(1, (2, 64)), k, v)
    with pytest.raises(dsk.DskError, match="multiple of 8"):
        packed.attend(q, k.expand(10, 1, 64), v[:1].expand(10, 1, 64))
    with pytest.raises(dsk.DskError, match="come from"):
        dsk.Packed()


# ---- places -------------------------------------------------------------------------------------------------------------------------------------

class Pool:
    """A pool beside its restatement; half of the blocks belong to no sequence and are not free."""

    def __init__(self, n_blocks, block, batch, width, seed=0):
        self.rng = np.random.default_rng(seed)
        self.n_blocks, self.block = n_blocks, block
        self.free = self.rng.permutation(n_blocks)[:max(1, n_blocks // 2)].tolist()
        self.table = np.full((batch, width), -1, dtype=np.int32)
        self.pool = dsk.Blocks.of(ints(self.free), n_blocks, block)
        self.t = torch.from_numpy(self.table.copy()).to(DEV)

    def same(self):
        n = int(self.pool.n_free.item())
        assert n == len(self.free) and self.pool.free[:n].tolist() == self.free
        assert np.array_equal(self.t.cpu().numpy(), self.table)
        assert int(self.pool._top[1].item()) == 0

    def bits(self):
        b = int(self.pool.status.item())
        self.pool.status.zero_()
        return b

    def extend(self, lens, count, rows, out=None):
        starts, new, positions, slots, pieces, status = po.extend(self.free, self.table, lens, count, rows, self.n_blocks, self.block)
        plan = self.pool.extend(self.t, ints(lens), ints(count), rows, out=out)
        assert self.bits() == status
        assert plan.starts.tolist() == starts and plan.lens.tolist() == new and plan.positions.tolist() == positions and plan.slots.tolist() == slots
        got = plan._pieces.view(-1, 4).tolist()
        assert len(got) >= len(pieces) and got[:len(pieces)] == pieces and all(x[1] == 0 for x in got[len(pieces):])
        self.same()
        return plan, new, status

    def cut(self, lens, keep):
        status = po.cut(self.free, self.table, lens, keep, self.n_blocks, self.block)
        self.pool.cut(self.t, ints(lens), ints(keep))
        assert self.bits() == status
        self.same()
        return status


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("batch", [1, 2, 31, 33, 300, 1024])
def test_places_of_random_steps(block, batch):
    """Prompts, decoded tokens, drafts that go back, sequences that end and begin again, until blocks run out now and then."""
    p = Pool(6 * batch + 4, block, batch, 7, seed=batch + block)
    rng, lens, plans, short = p.rng, [0] * batch, {}, 0
    for step in range(12):
        most = [1, 5, block, 3 * block][step % 4]
        count = [int(c) for c in rng.integers(0, most + 1, size=batch)]
        count = [min(c, 7 * block - l) for c, l in zip(count, lens)]
        rows = sum(count) + int(rng.integers(0, 50)) if step % 5 else max(1, sum(count) - 3)
        plan, lens, status = p.extend(lens, count, rows, out=plans.get(rows))
        plans[rows] = plan
        short += status == po.SHORT
        keep = [l if rng.random() < 0.5 else int(rng.integers(0, l + 1)) if rng.random() < 0.8 else 0 for l in lens]
        assert p.cut(lens, keep) == 0
        lens = keep
    assert short


def test_cut_undoes_extend():
    p = Pool(400, 16, 20, 30, seed=3)
    _, lens, _ = p.extend([0] * 20, [int(x) for x in p.rng.integers(0, 100, size=20)], 3000)
    free, table = list(p.free), p.table.copy()
    _, more, _ = p.extend(lens, [17] * 20, 500)
    p.cut(more, lens)
    assert p.free == free and np.array_equal(p.table, table)


def test_many_tokens_at_once():
    """More packed rows than one CTA lays out, and a stack that many CTAs read while one sets its height."""
    p = Pool(40000, 16, 50, 6000, seed=4)
    lens, plan = [0] * 50, None
    for _ in range(3):
        plan, lens, _ = p.extend(lens, [int(x) for x in p.rng.integers(0, 4000, size=50)], 200_003, out=plan)
    p.cut(lens, [x // 2 for x in lens])


def test_what_does_not_fit():
    p = Pool(20, 16, 5, 4, seed=5)                           # 10 blocks are free
    assert p.extend([0] * 5, [40, 64, 65, 20, 1], 200)[2] == po.RANGE                    # a sequence beyond its table gets nothing, the others do
    p.cut([40, 64, 0, 20, 1], [0] * 5)
    assert p.extend([0] * 5, [64, 64, 64, 1, 0], 200)[2] == po.SHORT                    # the third does not fit, nor does what is behind it
    p.cut([64, 64, 0, 0, 0], [0] * 5)
    assert p.extend([0] * 5, [10, 20, 0, 5, 1], 30)[2] == po.SHORT                      # rows
    p.cut([10, 20, 0, 0, 0], [0] * 5)
    assert p.extend([0] * 5, [2 ** 31 - 1, -7, -2 ** 31, 3, 0], 30)[2] == po.RANGE
    p.cut([0, 0, 0, 3, 0], [0] * 5)
    assert p.extend([-1, 2 ** 31 - 1, 0, 0, 0], [5, 1, 64, 0, 1], 65)[2] == po.RANGE
    assert p.cut([0, 64, 64, -3, 65], [1, 65, -1, -3, 2]) == po.RANGE                   # kept more than there is, negative, beyond the table
    assert p.extend([0, 0, 64, 0, 1], [1, 1, 0, 1, 0], 0)[2] == po.SHORT
    p.pool.extend(p.t, ints([0] * 5), ints([64] * 5), 400)
    with pytest.raises(dsk.DskError, match="ran out"):
        p.pool.check()
    p.pool.check()


def test_numbers_that_are_no_blocks():
    p = Pool(20, 16, 3, 4, seed=6)
    p.table[0, :2], p.table[1, 0] = [500, 3], -1
    p.t.copy_(torch.from_numpy(p.table))
    assert p.extend([10, 5, 0], [10, 5, 20], 40)[2] == po.PAGE            # tokens of unknown blocks have no slot, the others do
    assert p.cut([20, 10, 20], [0, 0, 0]) == po.PAGE                     # what is no block does not go back
    p.free += [0] * 20
    p.free = p.free[:20]
    p.pool = dsk.Blocks.of(ints(p.free), 20, 16)
    p.table[0] = [1, 2, 3, 4]
    p.t.copy_(torch.from_numpy(p.table))
    assert p.cut([64, 0, 0], [0, 0, 0]) == po.TWICE                       # a full stack
    with pytest.raises(dsk.DskError, match="no block|outside the cache"):
        p.pool.cut(ints([-1]).view(1, 1), ints([5]), ints([0]))
        p.pool.check()


def test_places_without_sequences_or_rows():
    p = Pool(10, 16, 0, 3)
    plan = p.pool.extend(p.t, ints([]), ints([]), 5)
    assert plan.starts.tolist() == [0] and plan.slots.tolist() == [-1] * 5
    p.pool.cut(p.t, ints([]), ints([]))
    q = Pool(10, 16, 2, 3)
    assert q.pool.extend(q.t, ints([0, 0]), ints([0, 0]), 0).starts.tolist() == [0, 0, 0]
    p.pool.check()
    q.pool.check()


def test_a_fresh_pool_and_a_view_of_a_table():
    pool = dsk.Blocks(8, block=16, device=0)
    wide = torch.full((3, 9), -5, dtype=torch.int32, device=DEV)
    plan = pool.extend(wide[:, :2], ints([0, 0, 0]), ints([17, 1, 32]), 60)
    assert wide.tolist() == [[0, 1] + [-5] * 7, [2] + [-5] * 8, [3, 4] + [-5] * 7]
    assert plan.slots[:18].tolist() == list(range(17)) + [32] and int(pool.n_free.item()) == 3
    pool.cut(wide[:, :2], plan.lens, ints([0, 0, 0]))
    assert pool.free.tolist() == list(range(7, -1, -1)) and wide[:, :2].flatten().tolist() == [-1, -1, -1, -5, -1, -1]
    pool.check()


def test_captured_places():
    """A captured step: drafts go back, the next ones get places; replayed with other lengths."""
    p = Pool(300, 16, 8, 20, seed=7)
    _, lens, _ = p.extend([0] * 8, [50] * 8, 400)
    t_lens, t_keep, t_count = ints(lens), ints([40] * 8), ints([10] * 8)
    plan = p.pool.extend(p.t, ints(lens), ints([0] * 8), 100)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.pool.cut(p.t, t_lens, t_keep)
        p.pool.extend(p.t, t_keep, t_count, 100, out=plan)
    for step in range(6):
        keep = [int(x) for x in p.rng.integers(20, 50, size=8)]
        count = [int(x) for x in p.rng.integers(0, 12, size=8)]
        for t, x in ((t_lens, lens), (t_keep, keep), (t_count, count)):
            t.copy_(ints(x))
        g.replay()
        status = po.cut(p.free, p.table, lens, keep, 300, 16)          # (some keep more than there is: left alone, and noted)
        starts, lens, _, slots, _, more = po.extend(p.free, p.table, keep, count, 100, 300, 16)
        assert p.bits() == status | more
        assert plan.starts.tolist() == starts and plan.slots.tolist() == slots and plan.lens.tolist() == lens
        p.same()


def test_places_refuse():
    pool = dsk.Blocks(8, block=16, device=0)
    t, z = torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints([0, 0])
    plan = pool.extend(t, z, z, 5)
    for call, text in ((lambda: pool.extend(t, z, z, -1), "rows"), (lambda: pool.extend(t, z, z, 6, out=plan), "earlier call"), (lambda: pool.extend(t, plan.lens, z, 5, out=plan), "old ones"),
                       (lambda: pool.extend(t, z, plan.lens, 5, out=plan), "counts"), (lambda: pool.extend(t.long(), z, z, 5), "int32"), (lambda: pool.extend(t, z[:1], z, 5), "lens"),
                       (lambda: pool.extend(t.cpu(), z, z, 5), "CUDA"), (lambda: pool.cut(t, z, z.long()), "keep"), (lambda: pool.extend(t, z, z, (1 << 20) + 1), "2\\^20"),
                       (lambda: pool.extend(t[:, ::2], z, z, 5), "neighbours"), (lambda: pool.extend(t[:1].expand(2, 4), z, z, 5), "overlap"), (lambda: dsk.Blocks(8, block=48, device=0).cut(t, z, z), "16, 32, 64 or 128"),
                       (lambda: dsk.Blocks.of(ints(range(9)), 8), "at most 8"), (lambda: dsk.Blocks.of(torch.zeros(3, dtype=torch.int32), 8), "CUDA"), (lambda: dsk.Packed.of(z.cpu(), 5), "CUDA"),
                       (lambda: pool.extend(torch.zeros(1025, 2, dtype=torch.int32, device=DEV), ints([0] * 1025), ints([0] * 1025), 5), "1024")):
        with pytest.raises(dsk.DskError, match=text):
            call()
    pool.check()


# ---- packed rows into the cache, and a run of all of them ---------------------------------------------------------------------------------------

def cache_of(rng, blocks, H, block, dk, dv):
    k, v = (rng.integers(0, 127, size=(blocks, H, block, d)).astype(np.uint8) for d in (dk, dv))
    ks, vs = (2.0 ** rng.integers(-3, 20, size=(blocks, H)) for _ in range(2))
    t = lambda a: torch.from_numpy(a.copy()).to(DEV)
    return dsk.Cache8.of(t(k).view(F8), t(v).view(F8), t(ks.astype(np.float32)), t(vs.astype(np.float32))), k, ks, v, vs


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,dk,dv,block", [(1, 16, 16, 16), (2, 80, 64, 32), (3, 128, 128, 64), (2, 192, 128, 128), (1, 256, 256, 128), (5, 48, 240, 16)])
def test_append(dtype, H, dk, dv, block):
    """Prompts, decoded tokens and portions, one call behind the other: codes and scales are those of the definition, bit for bit, and all else stays."""
    p = Pool(40, block, 3, 6, seed=dk + block)
    cache, k, ks, v, vs = cache_of(p.rng, 40, H, block, dk, dv)
    lens = [0, 0, 0]
    for count, spare in (([1, 1, 1], 0), ([2, 0, 1], 5), ([block, 3, block - 1], 1), ([1, 1, 1], 0), ([block, 2 * block + 3, block // 2], 3), ([0, 0, 0], 2), ([5, 5, 5], 0)):
        plan, new, _ = p.extend(lens, count, sum(count) + spare)
        rows = sum(count) + spare
        size = torch.exp(2.5 * torch.randn(rows, H, 1))
        x, y = ((torch.randn(rows, H, d) * size).to(DT[dtype]) for d in (dk, dv))
        x[sum(count):], y[sum(count):] = float("nan"), float("inf")
        cache.append(x.to(DEV), y.to(DEV), plan)
        for b in range(3):
            at = slice(sum(count[:b]), sum(count[:b + 1]))
            so.write(k, ks, p.table[b:b + 1], [lens[b]], [count[b]], x[None, at].double().numpy())
            so.write(v, vs, p.table[b:b + 1], [lens[b]], [count[b]], y[None, at].double().numpy())
        lens = new
        assert np.array_equal(cache.k_scale.cpu().numpy(), ks) and np.array_equal(cache.v_scale.cpu().numpy(), vs)
        assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), k) and np.array_equal(cache.v.view(torch.uint8).cpu().numpy(), v)
    cache.check()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,dk,dv,block,odd", [(2, 128, 128, 64, 0), (1, 80, 256, 128, 0), (2, 192, 128, 128, 0), (1, 96, 80, 64, 3)])
def test_append_few_rows_to_many_sequences(dtype, H, dk, dv, block, odd):
    """Decoded tokens of many sequences with a prompt or two among them (odd: rows at odd pitches), infinities and NaN among the values: codes and scales are those of the definition, bit for bit."""
    B = 24
    p = Pool(200, block, B, 6, seed=dk + block)
    cache, k, ks, v, vs = cache_of(p.rng, 200, H, block, dk, dv)
    lens = [0] * B
    mixed = [1] * 18 + [0, 130, 3, block, 1, block + 1]
    for step, (count, spare) in enumerate(((mixed, 0), ([1] * B, 60), (mixed[::-1], 7), ([4] * B, 0), ([0] * 23 + [block - 1], 40))):
        plan, new, _ = p.extend(lens, count, sum(count) + spare)
        rows = sum(count) + spare
        size = torch.exp(2.5 * torch.randn(rows, H, 1))
        x, y = ((torch.randn(rows, H, d + odd) * size).to(DT[dtype]) for d in (dk, dv))
        x, y = x[..., odd:], y[..., :dv]
        x[sum(count):], y[sum(count):] = float("nan"), float("inf")
        if step in (0, 2):
            y[3, 0, 5], y[sum(count) - 1, H - 1, dv - 1], x[20, 0, 0] = float("inf"), float("-inf"), float("nan")
        cache.append(x.to(DEV) if not odd else torch.cat([x, x[..., :odd]], -1).to(DEV)[..., :dk], y.to(DEV) if not odd else torch.cat([y, y[..., :odd]], -1).to(DEV)[..., :dv], plan)
        for b in range(B):
            at = slice(sum(count[:b]), sum(count[:b + 1]))
            so.write(k, ks, p.table[b:b + 1], [lens[b]], [count[b]], x[None, at].double().numpy())
            so.write(v, vs, p.table[b:b + 1], [lens[b]], [count[b]], y[None, at].double().numpy())
        lens = new
        assert np.array_equal(cache.k_scale.cpu().numpy(), ks) and np.array_equal(cache.v_scale.cpu().numpy(), vs)
        for got, want in ((cache.k, k), (cache.v, v)):       # (a NaN's sign is nobody's)
            g = got.view(torch.uint8).cpu().numpy()
            assert ((g == want) | ((g & 0x7f == 0x7f) & (want & 0x7f == 0x7f))).all()
    cache.check()
    small = dsk.Cache8(3, H, dk, dv, block=block, device=0)  # fewer blocks than the plan has numbers: nothing outside is touched
    plan, _, _ = p.extend(lens, mixed, sum(mixed))
    x, y = (torch.ones(sum(mixed), H, d, dtype=DT[dtype], device=DEV) for d in (dk, dv))
    small.append(x, y, plan)
    with pytest.raises(dsk.DskError, match="outside the cache"):
        small.check()


def test_append_strided_and_refused():
    p = Pool(20, 16, 2, 4, seed=8)
    cache, k, ks, v, vs = cache_of(p.rng, 20, 2, 16, 64, 64)
    plan, _, _ = p.extend([0, 0], [33, 20], 60)
    whole = torch.randn(60, 2, 2 * 64 + 3, device=DEV).to(torch.bfloat16)        # odd pitches, an odd offset for the values
    x, y = whole[..., :64], whole[..., 65:129]
    cache.append(x, y, plan)
    for b, at in ((0, slice(0, 33)), (1, slice(33, 53))):
        so.write(k, ks, p.table[b:b + 1], [0], [at.stop - at.start], x[None, at].double().cpu().numpy())
        so.write(v, vs, p.table[b:b + 1], [0], [at.stop - at.start], y[None, at].double().cpu().numpy())
    assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), k) and np.array_equal(cache.v.view(torch.uint8).cpu().numpy(), v)
    other = dsk.Cache8(20, 2, 64, block=32, device=0)
    for call, text in ((lambda: other.append(x, y, plan), "blocks of 32"), (lambda: cache.append(x, y, dsk.Packed.of(ints([0, 60]), 60)), "places"), (lambda: cache.append(x, y.float(), plan), "values of"),
                       (lambda: cache.append(x[:59], y[:59], plan), "keys"), (lambda: cache.append(x[:, :1], y, plan), "keys"), (lambda: cache.append(x.cpu(), y, plan), "CUDA")):
        with pytest.raises(dsk.DskError, match=text):
            call()
    small = dsk.Cache8(3, 2, 64, block=16, device=0)         # fewer blocks than the plan has numbers: nothing outside is touched
    small.append(x, y, plan)
    with pytest.raises(dsk.DskError, match="outside the cache"):
        small.check()


def test_serving_with_packed_rows():
    """What a serving program does with them: prompts arrive and attend packed while their keys and values join the cache, drafted tokens follow in it, refused ones go back, a sequence ends, another
    one takes its blocks.  Attention over the cache sees what was appended."""
    H, G, d, block, B = 4, 2, 64, 32, 4
    rng = np.random.default_rng(20)
    pool, cache = dsk.Blocks(30, block=block, device=0), dsk.Cache8(30, G, d, block=block, device=0)
    table, lens = torch.full((B, 12), -1, dtype=torch.int32, device=DEV), [0] * B
    held = [np.zeros((0, 2, G, d)) for _ in range(B)]        # keys and values that every sequence has

    def rows_of(n):
        return [torch.randn(n, h, d).to(torch.bfloat16) for h in (H, G, G)]

    t_lens = ints(lens)
    for step, count in enumerate(([100, 0, 37, 260], [0, 65, 0, 0], [4, 4, 4, 4], [1, 1, 1, 1], [0, 130, 3, 0])):
        rows = sum(count)
        q, k, v = rows_of(rows)
        plan = pool.extend(table, t_lens, ints(count), rows)
        cache.append(k.to(DEV), v.to(DEV), plan)
        assert plan.starts.tolist() == starts_of(count).tolist()
        for b in range(B):
            at = slice(sum(count[:b]), sum(count[:b + 1]))
            held[b] = np.concatenate([held[b], np.stack([k[at].double().numpy(), v[at].double().numpy()], 1)])
        if step == 0:                                        # whole prompts: their own rows are all that they see
            out = plan.attend(q.to(DEV), k.to(DEV), v.to(DEV))
            want = po.attend(*(x.double().numpy() for x in (q, k, v)), plan.starts.tolist(), d ** -0.5)[0]
            assert np.abs(out.double().cpu().numpy() - want).max() <= 2.0 ** -6 * np.abs(want).max()
        t_lens = plan.lens
        lens = t_lens.tolist()
        last = torch.randn(B, 1, H, d).to(torch.bfloat16)    # the next query of every sequence, over the cache
        got = cache.attend(last.to(DEV), table, t_lens, count=ints([int(n > 0) for n in lens])).double().cpu().numpy()
        for b in range(B):
            if not lens[b]:
                assert (got[b] == 0).all()
                continue
            for h in range(H):
                w = np.exp((held[b][:, 0, h // 2] @ last[b, 0, h].double().numpy()) * d ** -0.5)
                want = w @ held[b][:, 1, h // 2] / w.sum()
                assert np.abs(got[b, 0, h] - want).max() <= 0.15          # (values of a few units in E4M3: half a step, 2^-4 of each)
        keep = {2: [lens[0] - 3, lens[1], lens[2] - 1, lens[3] - 4], 3: [0, lens[1], lens[2], 0]}.get(step, lens)
        pool.cut(table, t_lens, ints(keep))
        t_lens, lens = ints(keep), keep
        held = [x[:n] for x, n in zip(held, keep)]
    pool.check()
    cache.check()
    pool.cut(table, t_lens, ints([0] * B))
    assert sorted(pool.free[:30].tolist()) == list(range(30)) and int(pool.n_free.item()) == 30


def falling(batch, rows, seed):
    """Starts of which every eighth falls or lies outside, and the last one is not the highest."""
    rng = np.random.default_rng(seed)
    s = np.sort(rng.integers(0, rows + 1, size=batch + 1))
    odd = rng.permutation(batch + 1)[:batch // 8 + 1]
    s[odd] = rng.integers(-rows, 2 * rows, size=len(odd))
    s[-1] = rows // 3
    return s


@pytest.mark.parametrize("H,G,d,rows,starts", [
    (2, 1, 64, 210, [0, 100, 150, 120, 1 << 30, -5, 90]), (2, 1, 64, 210, [0, 100, 150, 120, 200, -5, 90]), (1, 1, 64, 300, [120, 40]), (16, 16, 64, 4096, [0, 4096, 0, 4096]),
    (4, 2, 128, 9000, [0, 9000] * 40), (16, 16, 192, 3000, [0, 2000, 100, 3000, -1, 3000]), (8, 4, 256, 2500, [7, 2500, 7, 2400, 2500, 0])]
    + [(4, 1, 64, 2000, falling(b, 2000, b)) for b in (7, 33, 256, 257, 300, 1024)] + [(16, 16, 128, 20000, falling(b, 20000, b)) for b in (5, 1000)])
def test_starts_that_fall_are_the_highest_ahead_of_them(H, G, d, rows, starts):
    """Results are those of the starts that include/dsk.h says they are taken as, and rows of no one stay what they were, in every call."""
    g = torch.Generator(device=DEV).manual_seed(rows + len(starts))
    q, k, v = (torch.randn(rows, n, d, device=DEV, dtype=torch.bfloat16, generator=g) for n in (H, G, G))
    taken = np.maximum.accumulate(np.clip(np.asarray(starts, dtype=np.int64), 0, rows))
    results = []
    for s in (taken, starts, starts):
        results.append(torch.full((rows, H, d), 7.0, dtype=torch.bfloat16, device=DEV))
        packed = dsk.Packed.of(ints(s), rows)
        packed.attend(q, k, v, out=results[-1])
        packed.check()
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])
    first, last = int(taken[0]), int(taken[-1])
    assert (results[1][:first] == 7.0).all() and (results[1][last:] == 7.0).all() and not (results[1][first:last] == 7.0).all(dim=(1, 2)).any()


def test_more_entries_come_back_than_31_bits_count():
    """Entries that repeat one block number, 2^31 and more of them in a call: the stack fills up and is reported, and nothing is written ahead of it or behind it."""
    batch, width, block, n = 1024, (1 << 21) + 2048, 16, 5
    around = torch.full((n + 200,), 77, dtype=torch.int32, device=DEV)
    free, status = around[100:100 + n], torch.zeros(1, dtype=torch.int32, device=DEV)
    free.copy_(ints([4, 2, -3, -3, -3]))
    top = ints([2, 0])
    table = torch.full((batch, width), 3, dtype=torch.int32, device=DEV)
    lens, keep = torch.full((batch,), width * block, dtype=torch.int32, device=DEV), torch.zeros(batch, dtype=torch.int32, device=DEV)
    args = dsk.BlocksArgs(free.data_ptr(), top.data_ptr(), status.data_ptr(), 0, n, block)
    assert dsk.lib().dsk_blocks_cut(args, table.data_ptr(), width, width, lens.data_ptr(), keep.data_ptr(), batch, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert free.tolist() == [4, 2, 3, 3, 3] and top.tolist() == [n, 0] and int(status) == po.TWICE
    assert (around[:100] == 77).all() and (around[100 + n:] == 77).all() and bool((table.view(-1)[:1 << 31] == -1).all()) and bool((table.view(-1)[1 << 31:] == -1).all())


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -149, 1e-40, 3e-39, 2e-38])
@pytest.mark.parametrize("H,d", [(2, 64), (16, 128)])
def test_scales_next_to_zero(scale, H, d):
    """Scores of up to 2^126 ahead of a scale that takes them to next to nothing: weights are all alike at 0.  (A scale off by 2^-150, as numbers that small are rounded, is off by 2^-24 in such a score.)"""
    p = Prompt([300, 45, 1], H, 1, d, d, seed=31)
    p.q *= 2.0 ** 59
    p.k *= 2.0 ** 59
    got = p.run(scale=scale)
    if scale == 0.0:
        mean = p.v[:300, 0].double().cumsum(0) / torch.arange(1, 301)[:, None]
        assert ((got[:300, 0].double().cpu() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -8 * p.v[:300, 0].double().abs().cumsum(0) / torch.arange(1, 301)[:, None] * 1.01).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,G,dk,dv,lens", [(4, 2, 64, 64, [300, 1, 70]), (16, 16, 128, 128, [500, 64, 65]), (3, 1, 192, 128, [200]), (2, 2, 256, 256, [150, 3]), (16, 16, 64, 64, [1] * 300)])
def test_a_row_that_sees_one_key_has_its_value(dtype, H, G, dk, dv, lens):
    """First rows of sequences, and every row of a window of 1, bit for bit: the one weight is the power of two that the reference lies ahead, up to what scores and the reference are rounded by.  Scores
    here are below 2^6, which makes that 2^-18 of the weight (two roundings of half a step, 2^-19 each), and 2^-17 of the result with the exponential and the sum: less than the quarter of a step, 2^-9 or
    2^-12, that takes a result to the next number."""
    p = Prompt(lens, H, G, dk, dv, dtype=dtype, seed=41)
    q, k, v = (x.to(DEV) for x in (p.q, p.k, p.v))
    want = v.repeat_interleave(H // G, 1)
    packed = dsk.Packed.of(torch.from_numpy(p.starts).to(DEV), p.rows)
    first = torch.from_numpy(p.starts[:-1]).long()
    assert torch.equal(packed.attend(q, k, v)[first], want[first])
    assert torch.equal(packed.attend(q, k, v, window=1), want)
    packed.check()


def test_sizes_that_no_structure_holds_are_refused():
    z, t = ints([0, 0]), torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    pool = dsk.Blocks(8, block=16, device=0)
    none = torch.zeros(4, 2, 0, dtype=torch.bfloat16, device=DEV)
    some = torch.zeros(4, 2, 16, dtype=torch.bfloat16, device=DEV)
    for call, text in ((lambda: dsk.Packed.of(z, 1 << 40), "2\\^20"), (lambda: dsk.Packed.of(z, -1), "2\\^20"), (lambda: pool.extend(t, z, z, 1 << 31), "2\\^20"), (lambda: pool.extend(t, z, z, 1 << 60), "2\\^20"),
                       (lambda: dsk.Blocks.of(z, (1 << 32) + 8), "2\\^31"), (lambda: dsk.Packed.of(z, 4).attend(none, none, some), "multiple of 16"), (lambda: dsk.Packed.of(z, 4).attend(some, some, none), "multiple of 16"),
                       (lambda: dsk.Packed.of(z, 4).attend(some[:, :0], some, some), "multiple"), (lambda: dsk.Packed.of(z, 4).attend(some, some[:, :0], some[:, :0]), "multiple")):
        with pytest.raises(dsk.DskError, match=text):
            call()
