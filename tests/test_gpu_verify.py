"""Verification of drafted tokens against its float64 restatement (oracle/serve_oracle.py): whole numbers, equal."""
import numpy as np
import pytest
import torch

import dsk
import serve_oracle as so

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def make(B, n, V, seed=0, noise=0.7, temperature=1.0, dtype="f32"):
    rng = np.random.default_rng(seed)
    logits = torch.from_numpy(rng.normal(size=(B, n + 1, V)) * 2.5).to(DT[dtype])
    q = torch.softmax(logits[:, :n].double() / max(temperature, 0.25) + noise * torch.from_numpy(rng.normal(size=(B, n, V))), -1).float()
    drafts = torch.from_numpy(np.array([[rng.choice(V, p=(r / r.sum())) for r in s] for s in q.double().numpy()], dtype=np.int32).reshape(B, n))
    coins = torch.from_numpy(rng.random((B, n + 1)).astype(np.float32)).clamp(max=1 - 2.0 ** -24)
    return logits, q, drafts, coins


def run(logits, drafts, coins, q, count, temperature):
    a, t = dsk.verify_drafts(logits.to(DEV), drafts.to(DEV), coins.to(DEV), probs=q.to(DEV) if q is not None else None,
                             count=torch.tensor(count, dtype=torch.int32, device=DEV) if count is not None else None, temperature=temperature)
    return a.cpu().numpy(), t.cpu().numpy()


def same(logits, drafts, coins, q, count, temperature):
    got = run(logits, drafts, coins, q, count, temperature)
    n = drafts.shape[1]
    want = so.verify(logits.double().numpy(), drafts.numpy(), coins.numpy(), q.numpy() if q is not None else None, [n] * len(drafts) if count is None else count, temperature)
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), np.argwhere(got[1] != want[1])[:4]
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("temperature", [1.0, 0.75, 0.0, 2.5])
@pytest.mark.parametrize("B,n,V", [(1, 1, 2), (3, 4, 33), (5, 3, 1000), (2, 8, 1025), (4, 2, 32000), (2, 0, 4097)])
def test_verify(B, n, V, temperature, dtype):
    logits, q, drafts, coins = make(B, n, V, seed=V + n, temperature=temperature, dtype=dtype)
    count = [n - b % (n + 1) for b in range(B)]
    same(logits, drafts, coins, q, None, temperature)
    same(logits, drafts, coins, q, count, temperature)
    same(logits, drafts, coins, None, count, temperature)


def test_verify_large_vocabulary_and_many_sequences():
    logits, q, drafts, coins = make(6, 5, 129280, seed=1)
    a, _ = same(logits, drafts, coins, q, None, 1.0)
    assert len(set(a.tolist())) > 1
    logits, q, drafts, coins = make(300, 3, 257, seed=2)
    same(logits, drafts, coins, q, None, 1.0)


def test_verify_flat_rows_draw_the_right_neighbour():
    """100000 equal logits: a draw next to a border is decided by the 64-bit sums."""
    V = 100000
    logits = torch.zeros(8, 1, V) + 3.0
    coins = torch.linspace(0.05, 0.95, 8)[:, None].contiguous()
    same(logits, torch.zeros(8, 0, dtype=torch.int32), coins, None, None, 1.0)


def test_verify_coins_at_the_ends():
    logits, q, drafts, coins = make(4, 3, 500, seed=3)
    for c in (0.0, 1 - 2.0 ** -24):
        same(logits, drafts, torch.full_like(coins, c), q, None, 1.0)
        same(logits, drafts, torch.full_like(coins, c), None, None, 1.0)
    sure = torch.full((1, 2, 64), -float("inf"))
    sure[:, :, 17] = 2.0
    a, t = same(sure, torch.tensor([[17]], dtype=torch.int32), torch.full((1, 2), 1 - 2.0 ** -24), None, None, 1.0)
    assert a[0] == 1 and t[0].tolist() == [17, 17]


def test_verify_the_models_own_drafts_are_all_accepted():
    logits, _, drafts, coins = make(4, 6, 777, seed=4, noise=0.0)
    q = torch.softmax(logits[:, :6].double(), -1)
    a, _ = run(logits, drafts, coins.clamp(max=0.999), q.float(), None, 1.0)
    assert (a == 6).all()


def test_verify_next_to_the_border():
    """coin x q a 10^-7 part beside p, on either side: the row's sum is taken again."""
    logits, q, drafts, coins = make(16, 2, 3000, seed=5)
    p = torch.softmax(logits.double(), -1)
    for i in range(2):
        px, qx = (t[:, i].gather(1, drafts[:, i:i + 1].long())[:, 0].double() for t in (p, q))
        side = torch.tensor([1 + 2e-7 if b % 2 else 1 - 2e-7 for b in range(16)], dtype=torch.float64)
        coins[:, i] = (px / qx * side).clamp(0, 1 - 2.0 ** -24).float()
    same(logits, drafts, coins, q, None, 1.0)


def test_verify_masked_and_broken_rows():
    logits, q, drafts, coins = make(8, 3, 200, seed=6)
    logits[0, 0, :150] = -float("inf")                       # masked entries
    logits[1, 1] = -float("inf")                             # nothing left
    logits[2, 0, 5] = float("nan")
    logits[3, 2, 199] = float("inf")
    logits[4, 3, 0] = float("nan")
    logits[5, :, 1:] = -float("inf")                         # one entry
    drafts[6, 0], drafts[7, 1] = 200, -1                      # outside the vocabulary
    coins[:, :3] = 0.01
    for t in (1.0, 0.5, 0.0):
        same(logits, drafts, coins, q, None, t)
        same(logits, drafts, coins, None, None, t)


def draw(logits, coins, q=None):
    """The token drawn from one row for every coin: behind no draft, or with q in place of a draft outside the vocabulary."""
    B, n, V = len(coins), 0 if q is None else 1, logits.shape[-1]
    c = torch.zeros(B, n + 1, device=DEV)
    c[:, n] = torch.tensor(coins, device=DEV)
    a, t = dsk.verify_drafts(logits.to(DEV).expand(B, n + 1, V), torch.full((B, n), -1, dtype=torch.int32, device=DEV), c, probs=None if q is None else q.to(DEV).expand(B, 1, V))
    assert (a == 0).all() and (t[:, 1:] == -1).all()
    return t[:, 0].tolist()


def test_verify_probabilities_of_minus_zero():
    """-0 is 0: such tokens are drawn by what the model gives them; those whose probability is negative or a NaN are not."""
    q = torch.full((1, 1, 64), -0.0)
    q[..., 5] = 1.0
    coins = [0.0, 0.25, 0.5, 0.99]
    assert draw(torch.zeros(1, 1, 64), coins, q) == [0, 16, 32, 63]           # (63 tokens of equal weight, 5 not among them)
    logits, _, drafts, _ = make(4, 3, 500, seed=9)
    drafts[:, 0] = -1
    zeros = torch.zeros(4, 3, 500)
    zeros[:, :, ::2] = -0.0
    same(logits, drafts, torch.rand(4, 4, generator=torch.Generator().manual_seed(1)), zeros, None, 1.0)
    q[..., :5], q[..., 6:9] = -0.5, float("nan")
    assert draw(torch.zeros(1, 1, 64), [0.0], q) == [9]


def allowed(left, coin, token, bound):
    """Whether `token` is what a coin draws from `left` where running sums may be off by `bound` (p sums to 1)."""
    s = np.cumsum(left)
    border = np.longdouble(coin) * s[-1]
    return 0 <= token < len(left) and s[token] > border - bound and (s[token - 1] if token else 0) <= border + bound


@pytest.mark.parametrize("V", [1000, 129280, 1 << 17, (1 << 17) + 1, 1 << 20])
@pytest.mark.parametrize("depth", [30.0, 31.5, 33.0, 34.0, 36.0])
def test_verify_long_tails(V, depth):
    """One large logit ahead of or behind all the others: these have what the definition gives them, however small each is.  Terms are good to 2^-36 of each, a border lies between two sums
    of them (2^-35), what is cut off below a unit comes to 2^-40."""
    coins = [0.0, 2.0 ** -34, 2.0 ** -32, 2.0 ** -31, 2.0 ** -30, 2.0 ** -28, 2.0 ** -26, 2.0 ** -23, 0.5, 1 - 2.0 ** -24]
    for at in (0, V - 1):
        row = np.full(V, -depth, dtype=np.longdouble)
        row[at] = 0
        p = np.exp(row)
        p /= p.sum()
        for coin, token in zip(coins, draw(torch.from_numpy(row.astype(np.float32))[None, None], coins)):
            assert allowed(p, coin, token, 2.0 ** -34), (at, coin, token)


@pytest.mark.parametrize("V", [(1 << 17) + 5, 1 << 20])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_verify_vocabularies_beyond_2_17(V, temperature):
    logits, q, drafts, coins = make(2, 2, V, seed=42, temperature=temperature)
    same(logits, drafts, coins, q, None, temperature)
    same(logits, drafts, coins, None, [1, 2], temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_verify_as_many_drafts_as_there_may_be(dtype):
    logits, q, drafts, coins = make(3, 127, 300, seed=41, noise=0.02, dtype=dtype)
    coins[:2, :127] *= 0.9
    a, _ = same(logits, drafts, coins, q, [127, 127, 90], 1.0)
    assert a.max() > 100
    same(logits, drafts, coins, None, None, 0.0)
    same(logits, drafts, coins, None, [127, 64, 0], 1.0)


def test_verify_draws_from_differences():
    """p and q equal to the last bit of fp32 at one token, whose rest is then far below the bound, and 2^-20 apart at the others: a q x sum that is cut short leaves the first one too much.
    p_0 is good to 2^-36 of itself, q_0 x sum as well: 2^-36 each of less than a half."""
    rng = np.random.default_rng(40)
    rows = []
    while len(rows) < 24:
        ab = rng.uniform(-2, 0, size=(200000, 2)).astype(np.float32).astype(np.longdouble)
        whole = 1 + np.exp(ab).sum(1)
        p0 = 1 / whole
        rest = p0 - p0.astype(np.float32).astype(np.longdouble)
        bits = whole * 2 ** 31 / 2.0 ** np.floor(np.log2(whole))                 # (32 bits ahead of the point)
        rows += list(ab[(rest >= 0) & (rest < 2.0 ** -36) & (bits % 1 > 0.75) & (p0 > 0.35) & (p0 < 0.5)].astype(np.float32))
    coins = [float(np.float32(2.0 ** e)) for e in (-16, -14, -13.5, -13, -12.5, -12, -11, -8, -4, -1)]
    for a, b in rows[:24]:
        p = np.exp(np.array([0.0, a, b], dtype=np.longdouble))
        p /= p.sum()
        q = p.astype(np.float32)
        q[1:] *= np.float32(1 - 2.0 ** -20)
        left = np.maximum(p - q.astype(np.longdouble), 0)
        for coin, token in zip(coins, draw(torch.tensor([0.0, a, b])[None, None], coins, torch.from_numpy(q)[None, None])):
            assert allowed(left, coin, token, 2.0 ** -35), (a, b, coin, token, left)


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_verify_terms_one_by_one(temperature):
    """Two tokens whose p - q is 2^-20 of p, beside one that leaves nothing: a draw between them tells their exponentials apart to 2^-36.  An error of 2^-36 in p and as much in q x sum is
    2^-15 of p - q, which moves the border between two of about equal size by 2^-16 at most."""
    rng = np.random.default_rng(43)
    for _ in range(150):
        x = np.array([0, 0, 0], dtype=np.float32)
        x[0] = -rng.uniform(0, 14) * temperature
        x[1] = x[0] - rng.uniform(0, 1) * temperature
        e = np.exp(x.astype(np.longdouble) / np.longdouble(np.float32(temperature)))
        p = e / e.sum()
        q = (p * (1 - np.longdouble(2.0) ** -20)).astype(np.float32)
        q[2] = 1
        left = np.maximum(p - q.astype(np.longdouble), 0)
        border = float(left[0] / left.sum())
        coins = [float(np.float32(border - 2.0 ** -15)), float(np.float32(border + 2.0 ** -15))]
        a, t = dsk.verify_drafts(torch.from_numpy(x).to(DEV).expand(2, 2, 3), torch.full((2, 1), -1, dtype=torch.int32, device=DEV), torch.tensor([[0, c] for c in coins], device=DEV),
                                 probs=torch.from_numpy(q).to(DEV).expand(2, 1, 3), temperature=temperature)
        assert t[:, 0].tolist() == [0, 1], (x, border)


def test_verify_lowest_index_of_equal_logits():
    logits = torch.zeros(2, 2, 5000)
    logits[:, :, [4990, 1200, 77]] = 5.0
    drafts = torch.tensor([[77], [1200]], dtype=torch.int32)
    a, t = same(logits, drafts, torch.zeros(2, 2), None, None, 0.0)
    assert a.tolist() == [1, 0] and t.tolist() == [[77, 77], [77, -1]]


def test_verify_strides():
    logits, q, drafts, coins = make(3, 4, 1003, seed=7)
    room = torch.zeros(5, 3, 1010, device=DEV)
    room[..., 3:1006] = logits.transpose(0, 1)
    view = room[..., 3:1006].transpose(0, 1)
    qroom = torch.zeros(3, 4, 1009, device=DEV)
    qroom[..., :1003] = q.to(DEV)
    a, t = dsk.verify_drafts(view, drafts.to(DEV), coins.to(DEV), probs=qroom[..., :1003])
    want = so.verify(logits.double().numpy(), drafts.numpy(), coins.numpy(), q.numpy(), [4] * 3, 1.0)
    assert np.array_equal(a.cpu().numpy(), want[0]) and np.array_equal(t.cpu().numpy(), want[1])


def test_verify_captured_and_on_two_streams():
    logits, q, drafts, coins = make(4, 3, 9000, seed=8)
    dl, dq, dd, dc = (t.to(DEV) for t in (logits, q, drafts, coins))
    dsk.verify_drafts(dl, dd, dc, probs=dq)
    made = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = dsk.verify_drafts(dl, dd, dc, probs=dq)
        made.append((g, r))
    for seed in (9, 10):
        new = make(4, 3, 9000, seed=seed)
        for d, s in zip((dl, dq, dd, dc), new):
            d.copy_(s)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(4):
            for (g, _), s in zip(made, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = so.verify(new[0].double().numpy(), new[2].numpy(), new[3].numpy(), new[1].numpy(), [3] * 4, 1.0)
        for _, (a, t) in made:
            assert np.array_equal(a.cpu().numpy(), want[0]) and np.array_equal(t.cpu().numpy(), want[1])


def test_refusals():
    logits, q, drafts, coins = (t.to(DEV) for t in make(2, 3, 50))
    bad = [(dict(logits=logits.double()), "float32"), (dict(logits=logits[..., ::2]), "neighbouring"), (dict(logits=logits[0]), "drafts . 1"), (dict(drafts=drafts.long()), "drafts"),
           (dict(drafts=drafts[:, :2]), "drafts"), (dict(coins=coins[:, :3]), "coins"), (dict(coins=coins.double()), "coins"), (dict(probs=q[:, :2]), "probs"), (dict(probs=q.half()), "probs"),
           (dict(count=torch.tensor([1, 2], device=DEV)), "count"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(drafts=drafts.cpu()), "CUDA")]
    for kw, text in bad:
        a = dict(logits=logits, drafts=drafts, coins=coins, probs=q)
        a.update(kw)
        with pytest.raises(dsk.DskError, match=text):
            dsk.verify_drafts(**a)
