"""The 8-bit key / value cache and attention over it against their float64 restatement (oracle/serve_oracle.py).

Tolerances of attention, from the arithmetic of the kernels: queries and codes are exact in fp16; a score's sum of d products in fp32 is off by at most (d + 4) 2^-23 sum |q k| scale, which
changes a weight by that factor, numerator and denominator alike; a weight is rounded to fp16, 2^-11 of it, or by 2^-25 of the reference where it is below 2^-14 of
that (the reference is at most the largest weight times its value scale); the exponential is good to 2^-21; sums over L keys in fp32 to L 2^-24; the result is rounded to its type once."""
import numpy as np
import pytest
import torch

import dsk
import serve_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Case:
    """A cache in which the blocks of all sequences lie scattered; what no token holds is NaN."""

    def __init__(self, lens, H, dk, dv, block, seed=0, spread=0.7, dead=127, share=False):
        self.rng = np.random.default_rng(seed)
        self.lens, self.H, self.dk, self.dv, self.block = list(lens), H, dk, dv, block
        self.B, per = len(lens), max(1, max(-(-max(n, 1) // block) for n in lens))
        self.blocks = self.B * per + 2
        self.table = self.rng.permutation(self.blocks)[:self.B * per].reshape(self.B, per).astype(np.int32)
        if share:
            self.table[1:] = self.table[0]
        self.k, self.v = (np.full((self.blocks, H, block, d), dead, dtype=np.uint8) for d in (dk, dv))
        self.ks, self.vs = np.ones((self.blocks, H)), np.ones((self.blocks, H))
        for codes, scales, d in ((self.k, self.ks, dk), (self.v, self.vs, dv)):
            x = self.rng.normal(size=(self.B, max(1, max(lens)), H, d)) * np.exp(spread * self.rng.normal(size=(self.B, max(1, max(lens)), H, 1)))
            so.write(codes, scales, self.table, [0] * self.B, lens, x)

    def device(self):
        t = lambda a: torch.from_numpy(a.copy()).to(DEV)
        self.cache = dsk.Cache8.of(t(self.k).view(F8), t(self.v).view(F8), t(self.ks.astype(np.float32)), t(self.vs.astype(np.float32)))
        self.t = t(self.table)
        return self.cache

    def bytes(self):
        return self.cache.k.view(torch.uint8).cpu().numpy(), self.cache.v.view(torch.uint8).cpu().numpy(), self.cache.k_scale.cpu().numpy(), self.cache.v_scale.cpu().numpy()


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def expect(c, q, count, heads, scale, window=0, keep=0, lens=None):
    """(what attention gives, how far it may be off before its last rounding)"""
    lens = c.lens if lens is None else lens
    want, mass, size, top = so.attend(c.k, c.ks, c.v, c.vs, c.table, lens, count, q, heads, scale, window, keep)
    L = max(max(lens), 1)
    tol = mass * (2.0 ** -11 + 2 * (c.dk + 4) * 2.0 ** -23 * size + 2.0 ** -20 + L * 2.0 ** -24) + L * 2.0 ** -25 * 448 * top
    return want, tol


def check(got, want, tol, count, dtype, left=None):
    got = got.double().cpu().numpy()
    half = torch.finfo(DT[dtype]).eps / 2
    for b, n in enumerate(count):
        w, g = want[b, :n], got[b, :n]
        assert np.array_equal(np.isnan(w), np.isnan(g)), (b, np.argwhere(np.isnan(w) != np.isnan(g))[:4])
        off, may = np.abs(g - w), tol[b, :n] + half * (np.abs(w) + tol[b, :n]) + 2.0 ** -25
        assert (np.isnan(w) | (off <= may)).all(), (b, float(np.nanmax(off / may)))
        if left is not None:
            assert (got[b, n:] == left).all()


# ---- write --------------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,dk,dv,block", [(1, 16, 16, 16), (2, 80, 64, 32), (3, 128, 128, 64), (2, 192, 128, 128), (1, 256, 256, 128), (5, 48, 240, 16)])
def test_write(dtype, H, dk, dv, block):
    """Calls of one token, of a few, across borders and of whole blocks, in turn, on ragged sequences: codes and scales are those of the definition, bit for bit."""
    c = Case([0, 0, 0], H, dk, dv, block, dead=0)
    per = 5
    c.blocks = 3 * per + 2
    c.table = c.rng.permutation(c.blocks)[:3 * per].reshape(3, per).astype(np.int32)
    c.k, c.v = (c.rng.integers(0, 127, size=(c.blocks, H, block, d)).astype(np.uint8) for d in (dk, dv))
    c.ks, c.vs = (2.0 ** c.rng.integers(-3, 20, size=(c.blocks, H)) for _ in range(2))
    cache = c.device()
    at = [0, 3, block - 1]
    for n, count in ((1, [1, 1, 1]), (2, [2, 1, 0]), (block, [block, 3, block - 1]), (1, [1, 0, 1]), (2 * block + 3, [block, 2 * block + 3, block // 2]), (5, [5, 5, 5])):
        size = np.exp(2.5 * c.rng.normal(size=(3, n, H, 1)))
        x, y = (torch.from_numpy(c.rng.normal(size=(3, n, H, d)) * size).to(DT[dtype]) for d in (dk, dv))
        cache.write(x.to(DEV), y.to(DEV), c.t, ints(at), ints(count))
        so.write(c.k, c.ks, c.table, at, count, x.double().numpy())
        so.write(c.v, c.vs, c.table, at, count, y.double().numpy())
        at = [a + m for a, m in zip(at, count)]
        k, v, ks, vs = c.bytes()
        assert np.array_equal(ks, c.ks) and np.array_equal(vs, c.vs)
        assert np.array_equal(k, c.k) and np.array_equal(v, c.v)
    cache.check()


def test_write_strided_and_unaligned():
    c = Case([0, 0], 2, 64, 64, 16, dead=0)
    c.table = np.array([[0, 1, 2], [3, 4, 5]], dtype=np.int32)
    c.blocks = 6
    c.k, c.v = (np.zeros((6, 2, 16, 64), dtype=np.uint8) for _ in range(2))
    c.ks, c.vs = np.ones((6, 2)), np.ones((6, 2))
    cache = c.device()
    whole = torch.randn(2, 2, 40, 2 * 64 + 3, device=DEV).to(torch.bfloat16)          # [batch, head, row, key | value | pad]: odd pitches, an odd offset for the values
    k, v = whole[..., :64].transpose(1, 2), whole[..., 65:129].transpose(1, 2)
    wide_table = torch.full((2, 7), -1, dtype=torch.int32, device=DEV)
    wide_table[:, :3] = c.t
    cache.write(k, v, wide_table[:, :3], ints([1, 0]), ints([40, 33]))
    so.write(c.k, c.ks, c.table, [1, 0], [40, 33], k.double().cpu().numpy())
    so.write(c.v, c.vs, c.table, [1, 0], [40, 33], v.double().cpu().numpy())
    gk, gv, ks, vs = c.bytes()
    assert np.array_equal(gk, c.k) and np.array_equal(gv, c.v) and np.array_equal(ks, c.ks) and np.array_equal(vs, c.vs)


def test_write_what_is_not_finite_and_the_ends_of_the_range():
    c = Case([0], 4, 16, 16, 16, dead=0)
    cache = c.device()
    x = torch.zeros(1, 6, 4, 16)
    x[0, 0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 2.0])   # head 0: 2 is the largest number
    x[0, 1, 0, 0] = -0.0
    x[0, :, 1] = float("nan")                                                        # head 1: nothing but NaN, then a number
    x[0, 2, 1, 3] = 1e-30
    x[0, 3, 2, 5] = 3e38                                                             # head 2: beyond the range of the scales
    x[0, 1, 3, :] = torch.linspace(-448, 448, 16) * 2.0 ** -30                         # head 3: below its neighbours' range
    x[0, 2, 3, 1] = 1.0
    for lo, hi in ((0, 2), (2, 6)):
        cache.write(x[:, lo:hi].to(DEV), x[:, lo:hi].to(DEV), c.t, ints([lo]))
        so.write(c.k, c.ks, c.table, [lo], [hi - lo], x[:, lo:hi].double().numpy())
    k, v, ks, vs = c.bytes()
    assert np.array_equal(ks, c.ks) and np.array_equal(vs, c.ks)
    assert np.array_equal(so.TABLE[k], so.TABLE[c.k], equal_nan=True) and np.array_equal(k, v)
    cache.check()


def test_write_and_read_outside_are_noted_and_skipped():
    c = Case([32, 32, 32], 2, 16, 16, 16)
    cache = c.device()
    before = c.bytes()
    bad = c.t.clone()
    bad[0, 1], bad[1, 1], bad[2, 1] = -1, c.blocks, 2 ** 31 - 1
    x = torch.randn(3, 16, 2, 16, device=DEV)
    cache.write(x, x, bad, ints([16, 16, 16]))
    with pytest.raises(dsk.DskError, match="block number"):
        cache.check()
    cache.check()
    cache.write(x, x, c.t, ints([-1, 32, 2 ** 31 - 1]))
    with pytest.raises(dsk.DskError, match="outside the table"):
        cache.check()
    for a, b in zip(before, c.bytes()):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")
    out = tuple(torch.full((3, 16, 2, 16), 7.0, device=DEV) for _ in range(2))
    cache.read(bad, ints([16, 16, 16]), 16, out=out)
    assert all((o == 7).all() for o in out)
    with pytest.raises(dsk.DskError, match="block number"):
        cache.check()


# ---- read ---------------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,dk,dv,block", [(1, 16, 16, 16), (3, 128, 96, 64), (2, 192, 128, 32), (1, 256, 256, 128)])
def test_read(dtype, H, dk, dv, block):
    c = Case([3 * block + 5, 1, block], H, dk, dv, block)
    cache = c.device()
    first, count, n = [block - 3, 0, block - 1], [2 * block + 8, 1, 1], 2 * block + 8
    out = tuple(torch.full((3, n, H, d), 7.0, device=DEV, dtype=DT[dtype]) for d in (dk, dv))
    cache.read(c.t, ints(first), n, ints(count), out=out)
    for o, codes, scales in zip(out, (c.k, c.v), (c.ks, c.vs)):
        for b in range(3):
            for h in range(H):
                x, _ = so.gather(codes, scales, c.table[b], first[b] + count[b], h)
                assert torch.equal(o[b, :count[b], h].cpu(), torch.from_numpy(x[first[b]:]).to(DT[dtype]))
            assert (o[b, count[b]:] == 7).all()
    k, v = cache.read(c.t, ints(first), n, ints(count), dtype=DT[dtype])
    assert torch.equal(k[0], out[0][0]) and (k[1, 1:] == 0).all() and torch.equal(v[0], out[1][0])
    odd = tuple(torch.zeros((3, n, H, d + 3), device=DEV, dtype=DT[dtype])[..., 1:d + 1] for d in (dk, dv))
    cache.read(c.t, ints(first), n, ints(count), out=odd)
    assert torch.equal(odd[0][0], out[0][0]) and torch.equal(odd[1][0], out[1][0])
    cache.check()


# ---- attention ----------------------------------------------------------------------------------------------------------------------------------

SHAPES = [
    # lens, count, rows, heads, kv_heads, dk, dv, block, dtype, window, keep
    ([1], [1], 1, 1, 1, 16, 16, 16, "bf16", 0, 0),
    ([17, 1, 0, 333], [1, 1, 1, 1], 1, 4, 2, 64, 64, 16, "f16", 0, 0),
    ([1000], [1], 1, 16, 4, 128, 128, 64, "bf16", 0, 0),
    ([700, 90, 2100], [1, 1, 1], 1, 16, 1, 128, 128, 128, "f16", 0, 0),
    ([700, 90, 2100], [5, 2, 0], 5, 8, 2, 128, 128, 64, "bf16", 0, 0),
    ([513, 64, 65], [3, 3, 3], 3, 24, 2, 192, 128, 32, "bf16", 0, 0),
    ([513, 64, 65], [1, 1, 1], 1, 2, 2, 192, 128, 64, "f16", 0, 0),
    ([300, 20], [2, 7], 7, 2, 1, 256, 256, 64, "bf16", 0, 0),
    ([300, 20], [2, 1], 2, 6, 2, 80, 48, 32, "f16", 0, 0),
    ([150, 31], [9, 4], 9, 6, 2, 96, 256, 16, "bf16", 0, 0),
    ([900, 40, 130], [1, 1, 1], 1, 8, 4, 64, 64, 64, "bf16", 100, 0),
    ([900, 40, 130], [5, 3, 2], 5, 8, 4, 128, 128, 32, "f16", 33, 4),
    ([900, 140, 13], [2, 2, 2], 2, 4, 4, 112, 128, 128, "f16", 16, 17),
    ([450, 450], [1, 4], 4, 4, 1, 64, 128, 16, "bf16", 1, 0),
    ([100, 3], [100, 3], 100, 4, 2, 64, 64, 16, "bf16", 0, 0),
    ([260, 70], [200, 70], 200, 3, 1, 128, 128, 64, "f16", 50, 3),
    ([257], [257], 257, 2, 2, 192, 128, 64, "bf16", 0, 0),
    ([300, 129, 70], [130, 129, 1], 130, 8, 1, 128, 128, 32, "bf16", 0, 0),
    ([400], [300], 300, 2, 1, 80, 96, 64, "f16", 0, 0),
    ([333], [140], 140, 40, 2, 64, 48, 128, "f16", 77, 20),
    ([700, 130], [40, 37], 40, 2, 1, 256, 256, 64, "bf16", 0, 0),
    ([1300], [200], 200, 4, 2, 256, 128, 128, "f16", 0, 0),
    ([600, 40, 257], [33, 0, 100], 100, 1, 1, 96, 256, 16, "bf16", 130, 7),
    ([2100], [7], 7, 4, 1, 64, 64, 64, "bf16", 0, 0),
    ([900, 5, 300], [12, 5, 7], 12, 16, 4, 128, 128, 32, "bf16", 0, 0),
    ([1500, 128], [128, 128], 128, 2, 2, 192, 128, 64, "f16", 200, 4),
    ([1500, 128], [31, 1], 31, 4, 1, 64, 64, 16, "f16", 0, 0),
    ([650], [16], 16, 2, 1, 256, 256, 32, "f16", 0, 0),
]


@pytest.mark.parametrize("lens,count,rows,heads,kv_heads,dk,dv,block,dtype,window,keep", SHAPES)
def test_attend(lens, count, rows, heads, kv_heads, dk, dv, block, dtype, window, keep):
    c = Case(lens, kv_heads, dk, dv, block, seed=len(lens) + dk)
    cache = c.device()
    q = (torch.randn(len(lens), rows, heads, dk, generator=torch.Generator().manual_seed(3)) * 1.5).to(DT[dtype])
    scale = dk ** -0.5
    out = torch.full((len(lens), rows, heads, dv), 7.0, device=DEV, dtype=DT[dtype])
    cache.attend(q.to(DEV), c.t, ints(lens), count=ints(count), window=window, keep_first=keep, out=out)
    want, tol = expect(c, q.double().numpy(), count, heads, scale, window, keep)
    check(out, want, tol, count, dtype, left=7.0)
    cache.check()
    if all(n == rows for n in count):
        again = cache.attend(q.to(DEV), c.t, ints(lens), window=window, keep_first=keep)
        assert torch.equal(again, out)                        # the same sums in the same order
    # the same behind a table with room for many more tokens (work is laid out for what the table could hold), whose other entries nobody may look at
    wide = torch.full((len(lens), 3000), -7, dtype=torch.int32, device=DEV)
    wide[:, :c.t.shape[1]] = c.t
    out = torch.full((len(lens), rows, heads, dv), 7.0, device=DEV, dtype=DT[dtype])
    cache.attend(q.to(DEV), wide, ints(lens), count=ints(count), window=window, keep_first=keep, out=out)
    check(out, want, tol, count, dtype, left=7.0)
    cache.check()


@pytest.mark.parametrize("heads,rows", [(4, 1), (8, 1), (12, 3), (8, 8), (16, 2), (8, 11)])
@pytest.mark.parametrize("window,keep", [(0, 0), (40, 5)])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_more_heads_than_processors(heads, rows, window, keep, d):
    """Many sequences of very unequal lengths: several heads to a CTA, pieces of one head in two, with and without a window."""
    B = 84
    lens = [(53 * b) % 170 + (1 if b % 7 else 0) for b in range(B)]
    count = [min(rows, 1 + b % rows if b % 3 else rows) for b in range(B)]
    c = Case(lens, 4, d, d, 32)
    cache = c.device()
    q = torch.randn(B, rows, heads, d, device=DEV, dtype=torch.bfloat16)
    out = torch.full((B, rows, heads, d), 7.0, device=DEV, dtype=torch.bfloat16)
    cache.attend(q, c.t, ints(lens), count=ints(count), window=window, keep_first=keep, out=out)
    want, tol = expect(c, q.double().cpu().numpy(), count, heads, d ** -0.5, window, keep)
    check(out, want, tol, count, "bf16", left=7.0)
    cache.check()


def test_attend_long_and_ragged():
    """Pieces of one head in many CTAs, and many heads in one: all joined in a fixed order."""
    lens = [9000, 1, 37, 4100, 64, 0, 2500]
    c = Case(lens, 2, 64, 64, 64, seed=9)
    cache = c.device()
    q = torch.randn(7, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    out = cache.attend(q, c.t, ints(lens))
    want, tol = expect(c, q.double().cpu().numpy(), [1] * 7, 4, 0.125)
    check(out, want, tol, [1] * 7, "bf16")
    assert (out[5] == 0).all()


def test_attend_strided_rows_and_an_unaligned_result():
    c = Case([100, 30], 2, 64, 64, 16)
    cache = c.device()
    qkv = torch.randn(2, 3, 8 * 64 + 5, device=DEV, dtype=torch.float16)
    q = qkv[..., 1:1 + 4 * 64].unflatten(-1, (4, 64))
    room = torch.zeros(2, 4, 3, 67, device=DEV, dtype=torch.float16)
    out = room[..., 1:65].transpose(1, 2)
    cache.attend(q, c.t, ints([100, 30]), out=out, scale=0.2)
    want, tol = expect(c, q.double().cpu().numpy(), [3, 3], 4, 0.2)
    check(out, want, tol, [3, 3], "f16")
    assert (room[..., 0] == 0).all() and (room[..., 65:] == 0).all()


@pytest.mark.parametrize("size", [64, 256])
@pytest.mark.parametrize("rows", [4, 40, 90])
def test_attend_nan_and_large_values_where_a_row_does_not_look(rows, size):
    """A NaN key or value reaches the rows that see its token, entry by entry, and no other row; +-448 everywhere else is no harm."""
    n = 200
    c = Case([n, n], 2, size, size, 64, dead=126)
    for b, t, h, d in ((0, n - 1, 0, 5), (0, n - 2, 1, 60), (1, n - rows // 2, 0, 0), (1, n - rows // 2, 0, 63)):
        c.v[c.table[b][t // 64], h, t % 64, d] = 127 if d % 2 else 255
    c.k[c.table[1][(n - 2) // 64], 1, (n - 2) % 64, 3] = 255
    cache = c.device()
    q = torch.randn(2, rows, 4, size, device=DEV, dtype=torch.bfloat16)
    out = cache.attend(q, c.t, ints([n, n]), scale=0.125)
    want, tol = expect(c, q.double().cpu().numpy(), [rows] * 2, 4, 0.125)
    assert np.isnan(want).any() and not np.isnan(want[:, 0]).any()
    check(out, want, np.nan_to_num(tol, nan=0.0), [rows] * 2, "bf16")


@pytest.mark.parametrize("rows", [1, 100])
def test_attend_windows_over_nan(rows):
    """Tokens that have left the window are not looked at, whatever they hold."""
    n = 500
    c = Case([n], 1, 128, 128, 32)
    for t in range(8, n - 60 - rows):
        c.v[c.table[0][t // 32], 0, t % 32] = 127
        c.k[c.table[0][t // 32], 0, t % 32, 7] = 127
    cache = c.device()
    q = torch.randn(1, rows, 2, 128, device=DEV, dtype=torch.float16)
    out = cache.attend(q, c.t, ints([n]), window=60, keep_first=8)
    want, tol = expect(c, q.double().cpu().numpy(), [rows], 2, 128 ** -0.5, 60, 8)
    assert not np.isnan(want).any()
    check(out, want, tol, [rows], "f16")


@pytest.mark.parametrize("rows", [1, 70])
def test_attend_scales_of_very_unequal_size(rows):
    """Value blocks of 2^-40 beside those of 2^20, queries of 1e-4 beside 1e4, scores of some hundreds."""
    c = Case([300], 1, 64, 64, 16, seed=4)
    for j in range(0, 19, 3):
        c.vs[c.table[0][j], 0] = 2.0 ** -40
    for j in range(1, 19, 3):
        c.vs[c.table[0][j], 0] = 2.0 ** 20
    cache = c.device()
    q = torch.randn(1, rows, 8, 64, device=DEV) * torch.tensor([1e-4, 1e-2, 1.0, 30.0] * 2, device=DEV)[:, None]
    q = q.to(torch.bfloat16)
    out = cache.attend(q, c.t, ints([300]))
    want, tol = expect(c, q.double().cpu().numpy(), [rows], 8, 0.125)
    check(out, want, tol, [rows], "bf16")


@pytest.mark.parametrize("rows", [2, 100])
def test_attend_queries_that_are_not_finite(rows):
    c = Case([120], 1, 64, 64, 16)
    cache = c.device()
    q = torch.randn(1, rows, 2, 64, device=DEV, dtype=torch.bfloat16)
    q[0, 0, 0, 3], q[0, 1, 1, 5] = float("nan"), float("nan")
    out = cache.attend(q, c.t, ints([120]))
    bad = torch.zeros(1, rows, 2, dtype=torch.bool)
    bad[0, 0, 0] = bad[0, 1, 1] = True
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad)


@pytest.mark.parametrize("rows", [1, 80])
def test_attend_blocks_outside_and_short_tables(rows):
    """A block outside the cache is not seen; more tokens than the table has are noted."""
    c = Case([200, 200], 1, 64, 64, 32)
    c.table[0, 2] = -5
    c.table[1, 6] = c.blocks
    cache = c.device()
    q = torch.randn(2, rows, 2, 64, device=DEV, dtype=torch.bfloat16)
    out = cache.attend(q, c.t, ints([200, 200]))
    want, tol = expect(c, q.double().cpu().numpy(), [rows] * 2, 2, 0.125)
    check(out, want, tol, [rows] * 2, "bf16")
    with pytest.raises(dsk.DskError, match="block number"):
        cache.check()
    c.table[0, 2], c.table[1, 6] = c.table[0, 1], c.table[1, 0]
    c.device()
    lens = [10 ** 6, -3]
    out = c.cache.attend(q, c.t, ints(lens))
    want, tol = expect(c, q.double().cpu().numpy(), [rows] * 2, 2, 0.125, lens=lens)
    check(out[:1], want[:1], tol[:1] * 2, [rows], "bf16")
    assert (out[1] == 0).all()
    with pytest.raises(dsk.DskError, match="outside the table"):
        c.cache.check()


@pytest.mark.parametrize("rows", [1, 80, 300])
def test_attend_lengths_and_windows_at_the_ends_of_their_type(rows):
    c = Case([160, 150, 150], 1, 64, 64, 32)
    q = torch.randn(3, rows, 2, 64, device=DEV, dtype=torch.bfloat16)
    for first, seen in (([-2 ** 31, -2 ** 31 + 5, 150], 2), ([2 ** 31 - 1, 150, 150], 0)):
        c.device()
        out = c.cache.attend(q, c.t, ints(first), window=2 ** 31 - 1, keep_first=2 ** 31 - 1)
        assert (out[:seen] == 0).all()
        want, tol = expect(c, q.double().cpu().numpy(), [rows] * 3, 2, 0.125, lens=[min(max(n, -1), 1000) for n in first])   # (behind the table's end a row sees all of it)
        check(out, want, tol, [rows] * 3, "bf16")
        assert torch.equal(out, c.cache.attend(q, c.t, ints(first))) and torch.equal(out, c.cache.attend(q, c.t, ints(first), window=2 ** 32 + 5))
        with pytest.raises(dsk.DskError, match="outside the table"):
            c.cache.check()


@pytest.mark.parametrize("rows", [1, 80])
@pytest.mark.parametrize("sign,size", [(1, 118), (-1, 118), (1, 28), (-1, 28), (1, 40)])
def test_attend_largest_queries(rows, sign, size):
    """Scores of +-2^30 to +-2^120, all of one sign: far apart, so that a row's result is the value of its largest one."""
    n = 90
    c = Case([n], 1, 64, 64, 32)
    c.k &= 0x7f
    cache = c.device()
    q = torch.full((1, rows, 2, 64), sign * 2.0 ** size, device=DEV, dtype=torch.bfloat16)
    out = cache.attend(q, c.t, ints([n]), scale=0.125).float().cpu().numpy()
    at = lambda codes, scales, t: so.decode_table()[codes[c.table[0][t // 32], 0, t % 32]] * scales[c.table[0][t // 32], 0]
    score = np.array([sign * at(c.k, c.ks, t).sum() for t in range(n)])
    for i in range(rows):
        seen = score[:n - rows + i + 1]
        best = np.sort(seen)[-2:]
        assert len(best) < 2 or best[1] - best[0] > 2.0 ** -20 * abs(score).max()
        want = torch.tensor(at(c.v, c.vs, int(seen.argmax()))).bfloat16().float().numpy()
        assert (out[0, i] == want).all(), i


def test_attend_sequences_that_share_blocks():
    c = Case([256, 256, 256], 2, 128, 128, 64, share=True)
    cache = c.device()
    q = torch.randn(3, 1, 4, 128, device=DEV, dtype=torch.bfloat16)
    lens = [256, 100, 7]
    out = cache.attend(q, c.t, ints(lens))
    want, tol = expect(c, q.double().cpu().numpy(), [1] * 3, 4, 128 ** -0.5, lens=lens)
    check(out, want, tol, [1] * 3, "bf16")


def test_attend_empty_calls():
    c = Case([20], 1, 64, 64, 16)
    cache = c.device()
    assert cache.attend(torch.zeros(1, 0, 2, 64, device=DEV, dtype=torch.bfloat16), c.t, ints([20])).shape == (1, 0, 2, 64)
    assert cache.attend(torch.zeros(0, 1, 2, 64, device=DEV, dtype=torch.bfloat16), c.t[:0], ints([])).shape == (0, 1, 2, 64)
    z = torch.zeros(1, 0, 1, 64, device=DEV)
    cache.write(z, z, c.t, ints([3]))
    out = cache.attend(torch.ones(1, 2, 2, 64, device=DEV, dtype=torch.bfloat16), c.t, ints([20]), count=ints([0]))
    assert (out == 0).all()
    cache.check()


@pytest.mark.parametrize("rows", [0, 1, 100])
def test_attend_no_sequences(rows):
    """A batch of none, of rows for either kernel: no workspace, nothing launched."""
    cache = Case([20], 1, 64, 64, 16).device()
    for heads in (1, 64):
        q = torch.zeros(0, rows, heads, 64, device=DEV, dtype=torch.bfloat16)
        for blocks in (0, 2, 3000):
            table = torch.zeros(0, blocks, dtype=torch.int32, device=DEV)
            for window in (0, 100):
                assert cache.attend(q, table, ints([]), window=window).shape == (0, rows, heads, 64)
                assert cache.attend(q, table, ints([]), count=ints([]), window=window).shape == (0, rows, heads, 64)
    cache.write(q[:, :, :1], q[:, :, :1], table, ints([]))
    assert cache.read(table, ints([]), rows)[0].shape == (0, rows, 1, 64)
    logits = torch.zeros(0, 4, 50, device=DEV)
    a, t = dsk.verify_drafts(logits, torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, 4, device=DEV))
    assert a.shape == (0,) and t.shape == (0, 4)
    cache.check()


def test_attend_many_sequences():
    B = 700
    lens = [(37 * b) % 90 for b in range(B)]
    c = Case(lens, 1, 16, 16, 16)
    cache = c.device()
    q = torch.randn(B, 1, 1, 16, device=DEV, dtype=torch.float16)
    out = cache.attend(q, c.t, ints(lens))
    want, tol = expect(c, q.double().cpu().numpy(), [1] * B, 1, 0.25)
    check(out, want, tol, [1] * B, "f16")


@pytest.mark.parametrize("rows", [1, 96])
def test_attend_captured_replayed_and_on_two_streams(rows):
    """A captured call serves other lengths; two captured calls and an eager one on streams of their own, on the same cache, do not meet."""
    c = Case([600, 600], 2, 128, 128, 64)
    cache = c.device()
    lens = ints([600, 600])
    q = torch.randn(2, rows, 8, 128, device=DEV, dtype=torch.bfloat16)
    outs = [torch.zeros(2, rows, 8, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    cache.attend(q, c.t, lens, out=outs[0])
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.attend(q, c.t, lens, out=o)
        graphs.append(g)
    for n in ([600, 600], [rows + 5, 431], [rows, 598]):
        lens.copy_(ints(n))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                third = cache.attend(q, c.t, lens)
        torch.cuda.synchronize()
        want, tol = expect(c, q.double().cpu().numpy(), [rows] * 2, 8, 128 ** -0.5, lens=n)
        check(outs[0], want, tol, [rows] * 2, "bf16")
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], third)


@pytest.mark.parametrize("far", [-1, -2 ** 31, -2 ** 32, -2 ** 40])
def test_attend_negative_windows_of_any_size_are_refused(far):
    c = Case([20], 1, 64, 64, 16)
    cache = c.device()
    q = torch.zeros(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16)
    for kw in (dict(window=far), dict(keep_first=far), dict(window=far, keep_first=far)):
        with pytest.raises(dsk.DskError, match="negative"):
            cache.attend(q, c.t, ints([20]), **kw)


def test_check_waits_for_every_stream():
    """What a call on another stream is still to meet is not missed, and is cleared once it was told."""
    c = Case([40], 1, 64, 64, 16)
    cache = c.device()
    bad = c.t.clone()
    bad[0, 0] = -1
    q = torch.randn(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16)
    lens, side = ints([40]), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)                       # (a fifth of a second)
        cache.attend(q, bad, lens)
    with pytest.raises(dsk.DskError, match="block number"):
        cache.check()
    torch.cuda.synchronize()
    cache.check()


def test_refusals():
    c = Case([20], 2, 64, 64, 16)
    cache = c.device()
    q = torch.zeros(1, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    bad = [
        (dict(q=q.float()), "F16 or BF16"), (dict(q=q[:, :, :3]), "multiple"), (dict(q=q[..., :32]), "queries"), (dict(q=q[..., ::2]), "queries"), (dict(q=q.cpu()), "CUDA"),
        (dict(table=c.t.long()), "table"), (dict(table=c.t.cpu()), "CUDA"), (dict(lens=ints([20, 20])), "lengths"), (dict(lens=ints([20]).long()), "lengths"), (dict(count=ints([1, 1])), "count"),
        (dict(window=-1), "negative"), (dict(keep_first=-1), "negative"), (dict(scale=float("nan")), "number"), (dict(out=q.half()), "results"), (dict(out=q[..., :32]), "output"),
        (dict(out=q[:, :, :1].expand(1, 1, 4, 64)), "overlap"), (dict(q=q.expand(1, 3, 4, 64), out=q.new_zeros(4096).as_strided((1, 3, 4, 64), (0, 64, 64, 1))), "overlap"), (dict(q=q[:, :, :0]), "multiple"),
    ]
    for kw, text in bad:
        a = dict(q=q, table=c.t, lens=ints([20]))
        a.update(kw)
        with pytest.raises(dsk.DskError, match=text):
            cache.attend(**a)
    x = torch.zeros(1, 1, 2, 64, device=DEV)
    for a, text in (((x.long(), x), "values of"), ((x.double(), x.double()), "float32"), ((x, x.half()), "values of"), ((x[:, :, :1], x), "keys"), ((x, x[..., :48]), "values"), ((x[0], x), "batch, rows")):
        with pytest.raises(dsk.DskError, match=text):
            cache.write(*a, c.t, ints([0]))
    with pytest.raises(dsk.DskError, match="one type"):
        cache.read(c.t, ints([0]), 1, out=(x, x.half()))
    with pytest.raises(dsk.DskError, match="contiguous"):
        dsk.Cache8.of(cache.k[:, :, ::2], cache.v, cache.k_scale, cache.v_scale)
    with pytest.raises(dsk.DskError, match="multiple of 16"):
        odd = dsk.Cache8(2, 1, 24)
        odd.write(torch.zeros(1, 1, 1, 24, device=DEV), torch.zeros(1, 1, 1, 24, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV), ints([0]))
    v = dsk.View(x.data_ptr(), 3, 128, 128, 64)
    s = dsk.Kv8Rows.from_buffer_copy(cache._rows(c.t, ints([0]), None, 1))
    assert dsk.lib().dsk_kv8_write(cache._c, s, v, v, None) != 0 and b"F32, F16 or BF16" in dsk.lib().dsk_last_error()
    a = b = dsk.View.from_buffer_copy(cache._view("q", q, q.shape))
    s.table_blocks = 1 << 20                                   # (a call that needs a workspace; refused ahead of its launch)
    assert dsk.lib().dsk_kv8_attn(cache._c, s, a, b, 4, 1.0, 0, 0, None, 0, None) != 0 and b"workspace" in dsk.lib().dsk_last_error()


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("rows", [3, 20, 90])
@pytest.mark.parametrize("order", [1, -1])
def test_attend_maxima_that_jump(rows, order, d):
    """Scores that grow (or fall) by some tens from one stretch of 16 keys to the next, up to some hundreds: references move inside tiles and between them, by much and by little."""
    n = 400
    c = Case([n], 1, d, d, 16, seed=11, spread=0.1)
    grow = np.concatenate([np.linspace(0, 9, 20), np.array([0, 60, -40, 90, 91])])[::order]
    q0 = c.rng.normal(size=d)
    x = np.zeros((1, n, 1, d))
    for t in range(n):
        x[0, t, 0] = q0 * grow[t // 16] / (q0 @ q0) * 8 + 0.01 * c.rng.normal(size=d)       # (score of q0 at 1/8: grow)
    so.write(c.k, c.ks, c.table, [0], [n], x)
    cache = c.device()
    q = torch.from_numpy(q0[None, None, None, :] * np.array([1.0, 0.5, -1.0, 4.0])[None, None, :, None] * np.ones((1, rows, 1, 1))).to(torch.bfloat16)
    out = cache.attend(q.to(DEV), c.t, ints([n]), scale=0.125)
    want, tol = expect(c, q.double().numpy(), [rows], 4, 0.125)
    check(out, want, tol, [rows], "bf16")


def scored(levels, d, heads, seed, values=None):
    """A sequence whose token t has the score levels[t] (in powers of two, at scale ln 2) with the one query of all rows: entry 0 of a key is its level, which E4M3 has exactly, entry 0 of the
    query 1; the other entries are noise of keys that queries do not look at."""
    n = len(levels)
    c = Case([n], 1, d, d, 64, seed=seed)
    for t, e in enumerate(levels):
        page, row = c.table[0][t // 64], t % 64
        c.k[page, 0, row, 0] = so.encode(np.array([float(e)]))[0]
        assert so.TABLE[c.k[page, 0, row, 0]] == e
        if values is not None:
            c.v[page, 0, row] = so.encode(np.full(d, float(values[t])))
    c.ks[:] = 1.0
    c.vs[:] = 1.0
    q = torch.zeros(1, heads, 1, d, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    return c, q.transpose(1, 2).contiguous()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [40, 200])
def test_attend_references_that_move_in_both_halves_of_a_tile(rows, d):
    """The newer 64 keys of a tile of 128 move a row's reference, then the older ones do: weights and results that were stored a moment ago are scaled again, in every tile but the first; and
    rows that see none of the newer keys."""
    levels = np.zeros(640)
    for i in range(5):
        levels[128 * i + 64:128 * (i + 1)] = 32 * i
        levels[128 * i:128 * i + 64] = 32 * i + 16
    levels[640 - 60:] = -20                                  # (the rows' own tokens)
    c, q = scored(levels, d, 1, seed=21)
    q = q.expand(1, rows, 1, d).contiguous()
    for n in (640, 400, 300, rows + 7):
        cache = c.device()
        out = cache.attend(q.to(DEV), c.t, ints([n]), scale=float(np.log(2.0)))
        want, tol = expect(c, q.double().numpy(), [rows], 1, float(np.float32(np.log(2.0))), lens=[n])
        check(out, want, tol, [rows], "bf16")


def many(c, q, rows, n, B=148):
    """What every one of B sequences in the same blocks gets, as many as there are processors: no row's keys are shared out."""
    cache = c.device()
    out = cache.attend(q.to(DEV).expand(B, rows, 1, c.dk), c.t.expand(B, -1).contiguous(), ints([n] * B), scale=float(np.log(2.0)))
    assert torch.equal(out, out[:1].expand_as(out))
    want, tol = expect(c, q.expand(1, rows, 1, c.dk).double().numpy(), [rows], 1, float(np.float32(np.log(2.0))), lens=[n])
    check(out[:1], want, tol, [rows], "bf16")
    return want


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [40, 200])
def test_attend_references_that_move_in_both_halves_of_every_tile(rows, d):
    """The same where a CTA has tile after tile: results are scaled twice in a tile as well."""
    levels = np.zeros(640)
    for i in range(5):
        levels[128 * i + 64:128 * (i + 1)] = 32 * i
        levels[128 * i:128 * i + 64] = 32 * i + 16
    levels[640 - 60:] = -20
    c, q = scored(levels, d, 1, seed=21)
    for n in (640, 400, 300, rows + 7):
        many(c, q, rows, n)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [40, 200])
def test_attend_weights_that_a_late_reference_makes_small(rows, d):
    """A reference that lags by 14, then moves by 25 and more once the newer half's weights are stored: those are 2^-11 of the largest each, 2^-5 of the row together."""
    levels = np.full(512, -20.0)
    levels[:128] = 1
    levels[192:256] = 15
    levels[150] = 26
    values = np.zeros(512)
    values[192:256] = 16
    c, q = scored(levels, d, 1, seed=22, values=values)
    assert many(c, q, rows, 512).min() > 0.4


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("rows", [1, 3, 20, 40])
def test_attend_scales_of_blocks_that_no_sequence_owns(rows, dk, dv):
    """Blocks of 16 tokens, lengths of every remainder by 32, where nobody ever wrote block 0 and scales that nobody wrote are NaN, by clusters and by the line."""
    lens = list(range(rows, rows + 33))
    c = Case(lens, 1, dk, dv, 16, seed=30)
    c.table = (c.rng.permutation(c.blocks - 1)[:c.table.size] + 1).reshape(c.table.shape).astype(np.int32)   # block 0 is nobody's
    for a, s, d in ((c.k, c.ks, dk), (c.v, c.vs, dv)):
        a[:] = 127
        s[:] = np.nan
        so.write(a, s, c.table, [0] * c.B, lens, c.rng.normal(size=(c.B, max(lens), 1, d)))
    cache = c.device()
    q = torch.randn(c.B, rows, 1, dk, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    want, tol = expect(c, q.double().numpy(), [rows] * c.B, 1, dk ** -0.5)
    wide = torch.full((c.B, 3000), -7, dtype=torch.int32, device=DEV)
    wide[:, :c.t.shape[1]] = c.t
    for t in (c.t, wide):
        out = cache.attend(q.to(DEV), t, ints(lens))
        check(out, want, tol, [rows] * c.B, "bf16")
    cache.check()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("rows", [1, 5, 20, 80])
def test_attend_more_tokens_than_an_odd_table_has(rows, block):
    """A row behind the table's end sees the table's tokens and nothing beside them."""
    c = Case([5 * block, 5 * block], 1, 64, 64, block, seed=31)
    cache = c.device()
    q = torch.randn(2, rows, 2, 64, device=DEV, dtype=torch.bfloat16)
    lens = [5 * block + rows + 40, 5 * block + rows + 16]
    out = cache.attend(q, c.t, ints(lens))
    want, tol = expect(c, q.double().cpu().numpy(), [rows] * 2, 2, 0.125, lens=lens)
    check(out, want, tol, [rows] * 2, "bf16")
    with pytest.raises(dsk.DskError, match="outside the table"):
        cache.check()


@pytest.mark.parametrize("rows", [1, 6, 40, 1024])
@pytest.mark.parametrize("sink", [0, 30000])
def test_attend_long_tails_beside_one_large_weight(rows, sink):
    """A key with nearly all of the weight and no value, and tens of thousands at 2^-25 of it, which are all of the result: each of their weights is off by 2^-11 of itself or 2^-31 of the
    large one."""
    n, kv, G, d = 32768, 8, 4, 64
    one, top = (int(so.encode(np.array([x]))[0]) for x in (1.0, 26.0))
    k = torch.zeros(n // 128, kv, 128, d, dtype=torch.uint8, device=DEV)
    v = torch.full((n // 128, kv, 128, d), one, dtype=torch.uint8, device=DEV)
    k[sink // 128, :, sink % 128, 0], v[sink // 128, :, sink % 128] = top, 0
    scale = torch.ones(n // 128, kv, device=DEV)
    cache = dsk.Cache8.of(k.view(F8), v.view(F8), scale, scale.clone())
    table = torch.arange(n // 128, dtype=torch.int32, device=DEV)[None]
    q = torch.zeros(1, rows, kv * G, d, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 0.96875
    out = cache.attend(q, table, ints([n]), scale=float(np.log(2.0)))[0].double().cpu().numpy()
    tail = np.arange(n - rows, n) * 2.0 ** (-26 * 0.96875)   # (row i sees n - rows + i keys beside the large one)
    want = (tail / (1 + tail))[:, None, None]
    assert (np.abs(out - want) <= want * (2.0 ** -11 + 2.0 ** -8 + 2.0 ** -18) + n * 2.0 ** -31).all(), np.abs(out / want - 1).max()


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "f16"), (192, "bf16"), (256, "f16")])
def test_attend_values_that_come_late(d, dtype):
    """One tile of rows to a CTA and more keys than L2 holds: a product that waits for its values is not through when the softmax of the next tile, the last one, is.  Every call gives the
    same bits, and those are right (float64 on the GPU; the tolerances of the whole file)."""
    B, H, rows, n, block, dv = 48, 4, 40, 5000, 32, min(d, 128)
    g = torch.Generator(device=DEV).manual_seed(d)
    per = -(-n // block)
    lens = [n - (61 * b) % 2300 for b in range(B)]
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(B, per).to(DEV)
    k, v = ((torch.randn(B * per, H, block, x, generator=g, device=DEV) * 100).clamp(-448, 448).to(F8) for x in (d, dv))
    scale = torch.full((B * per, H), 2.0 ** -7, device=DEV)
    cache = dsk.Cache8.of(k, v, scale, scale.clone())
    q = (torch.randn(B, rows, H, d, generator=g, device=DEV) * 4).to(DT[dtype])
    first = cache.attend(q, table, ints(lens))
    for _ in range(60):
        assert torch.equal(first, cache.attend(q, table, ints(lens)))
    half = torch.finfo(DT[dtype]).eps / 2
    for b in range(0, B, 5):
        L = lens[b]
        kk, vv = ((x[table[b].long()].double() * 2.0 ** -7).transpose(0, 1).flatten(1, 2)[:, :L] for x in (k, v))
        qq = q[b].double().transpose(0, 1)
        w = (qq @ kk.transpose(1, 2) * d ** -0.5).masked_fill(torch.arange(L, device=DEV) > torch.arange(L - rows, L, device=DEV)[:, None], -np.inf)
        p = torch.softmax(w, -1)
        size = (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * d ** -0.5
        tol = p @ vv.abs() * (2.0 ** -11 + 2 * (d + 4) * 2.0 ** -23 * size + 2.0 ** -20 + L * 2.0 ** -24) + L * 2.0 ** -25 * 448 * 2.0 ** -7 * p.amax(-1, keepdim=True)
        want = p @ vv
        off = (first[b].double().transpose(0, 1) - want).abs()
        assert (off <= tol + half * (want.abs() + tol) + 2.0 ** -25).all(), b


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("tiles", [1, 2, 3, 7])
def test_attend_no_wait_gives_up(tiles, d):
    """Thousands of CTAs of one row tile and a few tiles of keys, call after call: no wait runs out, every call gives the same bits."""
    B, H, n, dv = 64, 3, 128 * tiles - 5, min(d, 128) if d < 256 else d
    g = torch.Generator(device=DEV).manual_seed(d + tiles)
    per = -(-n // 64)
    table = torch.arange(B * per, dtype=torch.int32, device=DEV).reshape(B, per)
    k, v = ((torch.randn(B * per, H, 64, x, generator=g, device=DEV) * 100).clamp(-448, 448).to(F8) for x in (d, dv))
    scale = torch.full((B * per, H), 2.0 ** -7, device=DEV)
    cache = dsk.Cache8.of(k, v, scale, scale.clone())
    for rows, window, keep in ((40, 0, 0), (100, 7, 17)):
        q = torch.randn(B, rows, H, d, generator=g, device=DEV, dtype=torch.bfloat16)
        first = cache.attend(q, table, ints([n] * B), window=window, keep_first=keep)
        assert all(torch.equal(first, cache.attend(q, table, ints([n] * B), window=window, keep_first=keep)) for _ in range(100))
        for b, i in ((0, 0), (B - 1, rows - 1), (B // 2, rows // 2)):                # (a row each against float64)
            t, L = n - rows + i, n
            kk, vv = ((x[table[b].long()].double() * 2.0 ** -7).transpose(0, 1).flatten(1, 2)[:, :L] for x in (k, v))
            j = torch.arange(L, device=DEV)
            seen = (j <= t) & ((t - j < window) | (j < keep) if window else j <= t)
            p = torch.softmax((kk @ q[b, i].double()[:, :, None])[..., 0].mul(d ** -0.5).masked_fill(~seen, -np.inf), -1)
            want, mass = (p[:, None] @ vv)[:, 0], (p[:, None] @ vv.abs())[:, 0]
            size = (kk.abs() @ q[b, i].double().abs()[:, :, None]).amax(1) * d ** -0.5
            tol = mass * (2.0 ** -11 + 2 * (d + 4) * 2.0 ** -23 * size + 2.0 ** -20 + L * 2.0 ** -24) + L * 2.0 ** -25 * 448 * 2.0 ** -7 * p.amax(-1, keepdim=True)
            assert ((first[b, i].double() - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8 + 2.0 ** -25).all()
    cache.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_beyond_32_bits(rows):
    """A cache of more than 4 GB of keys: its last blocks are written, read and attended."""
    blocks, H, dk, dv, block = 40000, 8, 192, 16, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("12 GB of device memory are needed")
    k = torch.empty((blocks, H, block, dk), dtype=torch.uint8, device=DEV)
    v = torch.empty((blocks, H, block, dv), dtype=torch.uint8, device=DEV)
    assert k.numel() > 1 << 32
    cache = dsk.Cache8.of(k.view(F8), v.view(F8), torch.ones((blocks, H), device=DEV), torch.ones((blocks, H), device=DEV))
    table = torch.tensor([[blocks - 1, 3, blocks - 2]], dtype=torch.int32, device=DEV)
    n = 2 * block + 40
    g = torch.Generator().manual_seed(0)
    x, y = torch.randn(1, n, H, dk, generator=g), torch.randn(1, n, H, dv, generator=g)
    cache.write(x.to(DEV), y.to(DEV), table, ints([0]))
    c = Case([n], H, dk, dv, block)
    c.table = np.array([[0, 1, 2]], dtype=np.int32)
    so.write(c.k, c.ks, c.table, [0], [n], x.double().numpy())
    so.write(c.v, c.vs, c.table, [0], [n], y.double().numpy())
    for i, page in enumerate([blocks - 1, 3, blocks - 2]):
        m = min(block, n - i * block)
        assert np.array_equal(k[page, :, :m].cpu().numpy(), c.k[i, :, :m]) and np.array_equal(v[page, :, :m].cpu().numpy(), c.v[i, :, :m])
    rk, rv = cache.read(table, ints([0]), n, dtype=torch.float32)
    for h in range(H):
        assert torch.equal(rk[0, :, h].cpu().double(), torch.from_numpy(so.gather(c.k, c.ks, c.table[0], n, h)[0]))
    q = torch.randn(1, rows, H, dk, generator=g).to(torch.bfloat16)
    out = cache.attend(q.to(DEV), table, ints([n]))
    want, tol = expect(c, q.double().numpy(), [rows], H, dk ** -0.5)
    check(out, want, tol, [rows], "bf16")
    cache.check()


def test_write_captured_and_replayed():
    """One captured call appends token after token: its places come from the GPU."""
    c = Case([0, 0], 2, 64, 64, 16, dead=0)
    c.table = np.array([[0, 1, 2], [3, 4, 5]], dtype=np.int32)
    c.blocks = 6
    c.k, c.v = (np.zeros((6, 2, 16, 64), dtype=np.uint8) for _ in range(2))
    c.ks, c.vs = np.ones((6, 2)), np.ones((6, 2))
    cache = c.device()
    first, x, y = ints([0, 5]), torch.zeros(2, 1, 2, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.write(x, y, c.t, first)
        first += 1
    at = [0, 5]
    for step in range(40):
        a, b = (torch.from_numpy(c.rng.normal(size=(2, 1, 2, 64)) * np.exp(c.rng.normal())).to(torch.bfloat16) for _ in range(2))
        x.copy_(a)
        y.copy_(b)
        g.replay()
        so.write(c.k, c.ks, c.table, at, [1, 1], a.double().numpy())
        so.write(c.v, c.vs, c.table, at, [1, 1], b.double().numpy())
        at = [t + 1 for t in at]
    k, v, ks, vs = c.bytes()
    assert np.array_equal(k, c.k) and np.array_equal(v, c.v) and np.array_equal(ks, c.ks) and np.array_equal(vs, c.vs)


def test_steps_of_speculative_decoding():
    """Prompt, then steps of a token and its drafts: keys and values join the cache, all queries attend, a head makes logits, the drafts are verified, and the next step's tokens lie over the
    refused ones.  Every call's result is that of the definition on what the calls before left."""
    B, H, G, d, V, n = 3, 2, 2, 64, 300, 4
    g = torch.Generator().manual_seed(5)
    emb, wq, wk, wv, wo = (torch.randn(*s, generator=g, dtype=torch.float64) * f for s, f in (((V, d), 1.0), ((d, H * G * d), 0.15), ((d, H * d), 0.15), ((d, H * d), 0.15), ((H * G * d, V), 0.2)))
    c = Case([0] * B, H, d, d, 32, dead=0)
    c.table = np.arange(B * 4, dtype=np.int32).reshape(B, 4)
    c.blocks = B * 4
    c.k, c.v = (np.zeros((c.blocks, H, 32, d), dtype=np.uint8) for _ in range(2))
    c.ks, c.vs = np.ones((c.blocks, H)), np.ones((c.blocks, H))
    cache = c.device()
    lens = [40, 7, 33]
    rng = np.random.default_rng(6)
    tokens = torch.from_numpy(rng.integers(0, V, size=(B, 40)))
    count, drawn = list(lens), None
    first = [0] * B
    for step in range(5):
        x = emb[tokens]
        q, k, v = ((x @ w).to(torch.bfloat16).view(B, tokens.shape[1], -1, d) for w in (wq, wk, wv))
        cache.write(k.to(DEV), v.to(DEV), c.t, ints(first), ints(count))
        so.write(c.k, c.ks, c.table, first, count, k.double().numpy())
        so.write(c.v, c.vs, c.table, first, count, v.double().numpy())
        total = [a + m for a, m in zip(first, count)]
        out = cache.attend(q.to(DEV), c.t, ints(total), ints(count))
        want, tol = expect(c, q.double().numpy(), count, H * G, d ** -0.5, lens=total)
        check(out, want, tol, count, "bf16", left=0.0)
        kk, vv, ks, vs = c.bytes()
        assert np.array_equal(kk, c.k) and np.array_equal(vv, c.v) and np.array_equal(ks, c.ks) and np.array_equal(vs, c.vs)
        logits = (out.double().cpu().flatten(2) @ wo).float()
        if step:
            probs = torch.softmax(logits[:, :n] + 0.5 * torch.from_numpy(rng.normal(size=(B, n, V))).float(), -1)
            coins = torch.from_numpy(rng.random((B, n + 1)).astype(np.float32)).clamp(max=1 - 2.0 ** -24)
            drafts = tokens[:, 1:].to(torch.int32).contiguous()
            a, t = dsk.verify_drafts(logits.to(DEV), drafts.to(DEV), coins.to(DEV), probs=probs.to(DEV), count=ints([m - 1 for m in count]))
            wa, wt = so.verify(logits.double().numpy(), drafts.numpy(), coins.numpy(), probs.numpy(), [m - 1 for m in count], 1.0)
            assert np.array_equal(a.cpu().numpy(), wa) and np.array_equal(t.cpu().numpy(), wt)
            first = [f + 1 + int(m) for f, m in zip(first, wa)]           # (the refused drafts' places are written again)
            drawn = [int(wt[b, wa[b]]) for b in range(B)]
        else:
            first = list(lens)
            drawn = [int(logits[b, lens[b] - 1].argmax()) for b in range(B)]
        tokens = torch.from_numpy(rng.integers(0, V, size=(B, n + 1)))
        tokens[:, 0] = torch.tensor(drawn)
        count = [n + 1, n, 1 + step % n]
    cache.check()
