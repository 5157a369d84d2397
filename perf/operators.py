"""Timed cases of the operators that a serving program calls beside the models: a key / value cache held in 8 bits, attention over it, and the
verification of drafted tokens.

The cache is made of blocks of `block` tokens; a block holds, for each key / value head, `block` rows of E4M3 values and one scale, a power of two:
the value is code x scale.  Block `table[b, j]` has the tokens j * block .. of sequence b.

  write    tokens `start[b] .. start[b] + count[b] - 1` of every sequence join the cache.  Scale of a block and head: the smallest power of two s with
           |x| <= 448 s over the rows that it holds, never smaller than it was while rows from earlier calls are in the block; their codes are rounded
           again where it grew.  A block whose first row is written starts anew.
  read     the values of tokens `start[b] .. start[b] + count[b] - 1`
  attend   query i of sequence b is its token t = lens[b] - count[b] + i and sees the tokens j <= t with t - j < window or j < keep_first;
           query head h reads key / value head h / (heads / kv_heads)
  verify   speculative sampling from given uniform numbers: draft i is accepted while coin_i q_i(x_i) < p_i(x_i), p_i = softmax(logits_i / temperature);
           the first one that is not is replaced by a draw from max(p_i - q_i, 0), and behind accepted ones the next token is drawn from p: in both the
           lowest index whose running sum is over (last coin) x (whole sum).  Without q the drafts are taken as certain (q_i(x_i) = 1).
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LEAST, MOST = -40, 40           # exponents of a scale


def _dsk():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek.cpp_b200"))
    import dsk
    return dsk


def listed():
    return [
        # the token that one sequence has just decoded joins a block that is half full: latency
        dict(name="write_token", op="write", batch=1, new=1, most=1001, heads=4, dk=128, dv=128, block=64, dtype="bf16", full=1),
        # a batch that verifies drafts: a token and its seven drafts of each of 64 sequences, across borders of blocks
        dict(name="write_drafts", op="write", batch=64, new=8, most=8000, heads=4, dk=128, dv=128, block=16, dtype="f16", full=0),
        # prompts of four sequences, of unequal lengths, wide keys
        dict(name="write_prompts", op="write", batch=4, new=8191, most=9000, heads=16, dk=192, dv=128, block=64, dtype="bf16", full=0),
        # a short sequence is read back to be kept elsewhere
        dict(name="read_short", op="read", batch=1, new=161, most=300, heads=4, dk=64, dv=64, block=32, dtype="bf16", full=1),
        # long sequences are read back for a consumer that has no 8-bit form
        dict(name="read_long", op="read", batch=8, new=8000, most=9000, heads=4, dk=128, dv=128, block=64, dtype="bf16", full=0),
        # one decoded token behind a thousand: latency
        dict(name="attend_token", op="attend", batch=1, new=1, most=1000, heads=16, kv_heads=4, dk=128, dv=128, block=64, dtype="bf16", window=0, keep=0, full=1),
        # one decoded token for each of 64 sequences of very unequal lengths: bytes of the cache
        dict(name="attend_batch", op="attend", batch=64, new=1, most=16000, heads=16, kv_heads=4, dk=128, dv=128, block=64, dtype="bf16", window=0, keep=0, full=0),
        # a token and its drafts, sliding window with first tokens that stay visible
        dict(name="attend_drafts", op="attend", batch=16, new=5, most=8000, heads=16, kv_heads=4, dk=128, dv=128, block=32, dtype="f16", window=1024, keep=4, full=0),
        # the second portion of a prompt, a head for every key head, wide keys: arithmetic
        dict(name="attend_portion", op="attend", batch=1, new=2048, most=6000, heads=16, kv_heads=16, dk=192, dv=128, block=64, dtype="bf16", window=0, keep=0, full=1),
        # ragged portions of three sequences, small heads, windowed
        dict(name="attend_ragged", op="attend", batch=3, new=777, most=4000, heads=16, kv_heads=4, dk=64, dv=64, block=64, dtype="bf16", window=512, keep=4, full=0),
        # four drafts of one sequence: latency
        dict(name="verify_one", op="verify", batch=1, drafts=4, vocab=32000, temperature=1.0, certain=0, dtype="f32", full=1),
        # drafts of a batch over a large vocabulary
        dict(name="verify_batch", op="verify", batch=32, drafts=7, vocab=129280, temperature=0.75, certain=0, dtype="f32", full=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "verify"])
    if op == "verify":
        c = dict(op=op, batch=_log(rng, 1, 32), drafts=rng.randint(1, 8), vocab=_log(rng, 300, 129280), temperature=rng.choice([1.0, 0.75, 0.5, 0.0]),
                 certain=rng.randint(0, 1), dtype=rng.choice(["f32", "bf16"]), full=rng.randint(0, 1))
        while c["batch"] * (c["drafts"] + 1) * c["vocab"] > 32 * 8 * 129280:
            c["batch"] = max(1, c["batch"] // 2)
        return c
    dk, dv = rng.choice([(64, 64), (80, 80), (96, 64), (128, 128), (112, 128), (192, 128), (256, 256)])
    c = dict(op=op, batch=_log(rng, 1, 64), new=_log(rng, 1, 4000), most=0, heads=rng.choice([1, 2, 4, 8, 16]), dk=dk, dv=dv, block=rng.choice([16, 32, 64, 128]),
             dtype=rng.choice(["bf16", "f16"]), full=rng.randint(0, 1))
    if op != "attend":
        while c["batch"] * c["new"] * c["heads"] * (dk + dv) > 60_000_000:
            c["batch"], c["new"] = max(1, c["batch"] // 2), max(1, c["new"] * 2 // 3)
        c["most"] = c["new"] + _log(rng, 1, 4000)
        return c
    c["kv_heads"], c["heads"] = min(c["heads"], 8), min(c["heads"], 8) * rng.choice([1, 2, 3, 4, 8])
    c["window"], c["keep"] = rng.choice([(0, 0), (0, 0), (0, 0), (_log(rng, 16, 4000), rng.choice([0, 4, 17]))])
    if rng.random() < 0.5:                                                      # decoded tokens and drafts; otherwise portions
        c["new"] = rng.choice([1, 1, 1, 2, 4, 8])
    c["most"] = c["new"] + _log(rng, 1, 12000)
    while c["batch"] * c["most"] * c["kv_heads"] * (dk + dv) > 300_000_000 or c["batch"] * c["new"] * c["most"] * c["heads"] * (dk + dv) > 25_000_000_000:
        if c["batch"] > 1:
            c["batch"] //= 2
        else:
            c["most"] = max(c["new"], c["most"] * 2 // 3)
            c["new"] = min(c["new"], max(8, c["most"] // 2))
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------

def _numbers(case):
    """Tokens that every sequence has (the new ones among them) and how many are new: the first sequence is the longest one, the others are spread."""
    B, n, most = case["batch"], case["new"], case["most"]
    if case["full"] or B == 1:
        return [most] * B, [n] * B
    lens = [max(n, most - (most - n) * ((7 * b) % B) // B) for b in range(B)]
    count = [n if b % 4 == 0 or n == 1 else max(1, n - (n * ((5 * b) % B)) // (2 * B)) for b in range(B)]
    return lens, count


def _random(shape, g, dtype=torch.float32, spread=None):
    x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(generator=g)
    if spread is not None:
        x *= spread
    return x.to(dtype)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] == "verify":
        B, n, V = case["batch"], case["drafts"], case["vocab"]
        logits = _random((B, n + 1, V), g) * 2.5
        q = torch.softmax(logits[:, :n] / max(case["temperature"], 0.25) + 0.7 * _random((B, n, V), g), -1)      # a smaller model's opinion of the same tokens
        race = torch.empty((B, n, V), device=DEV).exponential_(generator=g)
        drafts = (q / race).argmax(-1).to(torch.int32)
        coins = torch.empty((B, n + 1), device=DEV).uniform_(generator=g)
        count = None if case["full"] else torch.tensor([n - (3 * b) % (n + 1) if b else n for b in range(B)], device=DEV, dtype=torch.int32)
        state = {"case": case, "logits": logits.to(TYPES[case["dtype"]]), "drafts": drafts, "coins": coins, "probs": None if case["certain"] else q, "count": count}
        if own:
            state["dsk"] = _dsk()
        return state
    B, n, most, block, dk, dv, dt = case["batch"], case["new"], case["most"], case["block"], case["dk"], case["dv"], TYPES[case["dtype"]]
    H = case["kv_heads"] if case["op"] == "attend" else case["heads"]
    per = -(-most // block)
    blocks = B * per + 3                                                        # blocks of all sequences lie scattered over the cache
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed)))[:B * per]
    table = order.to(torch.int32).reshape(B, per).to(DEV)
    lens, count = _numbers(case)
    state = {"case": case, "table": table, "count": None if case["full"] else torch.tensor(count, device=DEV, dtype=torch.int32)}
    for name, d in (("k", dk), ("v", dv)):
        e = torch.randint(-11, -6, (blocks, H), generator=g, device=DEV)        # entries of a few units: scales of 2^-7 and so on
        state[name + "_scale"] = _pow2(e)
        state[name] = (_random((blocks, H, block, d), g) * 100).clamp_(-448, 448).to(F8)
    if case["op"] == "attend":
        state["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        state["q"] = _random((B, n, case["heads"], dk), g, dt, spread=1.5)
        state["out"] = torch.zeros((B, n, case["heads"], dv), device=DEV, dtype=dt)
    else:
        state["start"] = torch.tensor([l - c for l, c in zip(lens, count)], device=DEV, dtype=torch.int32)
        size = torch.exp(0.7 * _random((B, n, H, 1), g))                        # tokens of unequal size
        if case["op"] == "write":
            state["new_k"], state["new_v"] = _random((B, n, H, dk), g, dt, spread=size), _random((B, n, H, dv), g, dt, spread=size)
        else:
            state["out"] = (torch.zeros((B, n, H, dk), device=DEV, dtype=dt), torch.zeros((B, n, H, dv), device=DEV, dtype=dt))
    if own:                                                                     # the handle that a program keeps next to its cache
        state["cache"] = _dsk().Cache8.of(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if c["op"] == "verify":
        if own:
            accepted, tokens = s["dsk"].verify_drafts(s["logits"], s["drafts"], s["coins"], probs=s["probs"], count=s["count"], temperature=c["temperature"])
            return {"accepted": accepted, "tokens": tokens}
        return _verify(s, c)
    if c["op"] == "write":
        if own:
            s["cache"].write(s["new_k"], s["new_v"], s["table"], s["start"], count=s["count"])
        else:
            _write(s, c, "k")
            _write(s, c, "v")
        return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "read":
        if own:
            s["cache"].read(s["table"], s["start"], c["new"], count=s["count"], out=s["out"])
        else:
            _read(s, c, "k", s["out"][0])
            _read(s, c, "v", s["out"][1])
        return {"k": s["out"][0], "v": s["out"][1]}
    scale = c["dk"] ** -0.5
    if own:
        s["cache"].attend(s["q"], s["table"], s["lens"], count=s["count"], scale=scale, window=c["window"], keep_first=c["keep"], out=s["out"])
    else:
        _attend(s, c, scale)
    return s["out"]


# ---- plain forms -------------------------------------------------------------------------------------------------------------------------------

def _tokens(s, c):
    """Place of the new tokens: whether there is one, block in the cache, row in it, all [batch, new]."""
    i = torch.arange(c["new"], device=DEV)
    at = s["start"][:, None].long() + i
    there = i < s["count"][:, None] if s["count"] is not None else torch.ones_like(at, dtype=torch.bool)
    j = (at // c["block"]).clamp(max=s["table"].shape[1] - 1)
    return there, s["table"].long().gather(1, j), at % c["block"]


def _write(s, c, name):
    codes, scale, x = s[name], s[name + "_scale"], s["new_" + name].float()
    there, phys, row = _tokens(s, c)
    blocks, H, block, d = codes.shape
    # scales that the new rows need
    most = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    at = torch.where(there, phys, blocks).reshape(-1, 1).expand(-1, H)
    need = torch.zeros((blocks + 1, H), device=DEV).scatter_reduce(0, at, most.reshape(-1, H), "amax")[:blocks]
    m, e = torch.frexp(need)
    e = torch.where(need > 0, e - 9 + (m > 0.875), LEAST).clamp(LEAST, MOST)
    touched = torch.zeros(blocks + 1, dtype=torch.bool, device=DEV)
    touched[torch.where(there, phys, blocks).reshape(-1)] = True
    kept = torch.zeros(blocks + 1, dtype=torch.long, device=DEV)               # rows of earlier calls in a block
    kept[torch.where(there[:, 0], phys[:, 0], blocks)] = row[:, 0]
    touched, kept = touched[:blocks, None], kept[:blocks, None]
    new = torch.where(touched, torch.where(kept > 0, torch.maximum(scale, _pow2(e)), _pow2(e)), scale)
    # the kept rows of every sequence's first block, in the new scale
    first = phys[:, 0]
    old = codes.view(torch.uint8)[first].view(F8).float()
    again = (old * (scale / new)[first][:, :, None, None]).to(F8).view(torch.uint8)
    still = (torch.arange(block, device=DEV)[None, :] < kept[first]) & there[:, :1]
    bytes_ = codes.view(torch.uint8)
    bytes_[first] = torch.where(still[:, None, :, None], again, bytes_[first])
    # the new rows
    fresh = (x / new[phys][..., None]).clamp(-448, 448).to(F8).view(torch.uint8)
    bytes_[phys[there], :, row[there]] = fresh[there]
    scale.copy_(new)


def _read(s, c, name, out):
    there, phys, row = _tokens(s, c)
    x = s[name].view(torch.uint8)[phys, :, row].view(F8).float() * s[name + "_scale"][phys][..., None]
    out.copy_(torch.where(there[..., None, None], x.to(out.dtype), out))


def _whole(s, name, length):
    """All cached values of every sequence in 32 bits: [batch, kv_heads, length, d]."""
    t = s["table"].long()
    x = s[name].view(torch.uint8)[t].view(F8).float() * s[name + "_scale"][t][..., None, None]      # [batch, blocks, heads, block, d]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :length]


def _attend(s, c, scale):
    B, n, H, dk = s["q"].shape
    G, L = s["k"].shape[1], c["most"]
    q = s["q"].float().view(B, n, G, H // G, dk).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, dk)
    w = (q @ _whole(s, "k", L).transpose(2, 3)).view(B, G, H // G, n, L) * scale
    i, j = torch.arange(n, device=DEV), torch.arange(L, device=DEV)
    lens = s["lens"].long()
    count = s["count"].long() if s["count"] is not None else torch.full_like(lens, n)
    t = (lens - count)[:, None] + i
    seen = j <= t[:, :, None]
    if c["window"]:
        seen &= (t[:, :, None] - j < c["window"]) | (j < c["keep"])
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w -= w.amax(-1, keepdim=True).clamp(min=-1e30)
    w.exp_()
    w /= w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (w.view(B, G, H // G * n, L) @ _whole(s, "v", L)).view(B, G, H // G, n, -1).permute(0, 3, 1, 2, 4).reshape(B, n, H, -1)
    s["out"].copy_(torch.where((i < count[:, None])[:, :, None, None], o.to(s["out"].dtype), s["out"]))


def _verify(s, c):
    logits, x, coins = s["logits"].double(), s["drafts"].long(), s["coins"].double()
    B, n1, V = logits.shape
    n = n1 - 1
    count = s["count"].long() if s["count"] is not None else torch.full((B,), n, device=DEV)
    if c["temperature"] == 0:
        p = torch.zeros_like(logits).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
    else:
        logits /= c["temperature"]
        logits -= logits.amax(-1, keepdim=True)
        p = logits.exp_()
        p /= p.sum(-1, keepdim=True)
    px = p[:, :n].gather(2, x[..., None])[..., 0]
    if c["temperature"] == 0:
        ok = px > 0
    else:
        ok = coins[:, :n] * (1.0 if s["probs"] is None else s["probs"].gather(2, x[..., None])[..., 0].double()) < px
    ok &= torch.arange(n, device=DEV) < count[:, None]
    accepted = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device=DEV)
    left, r = p[b, accepted], accepted.clamp(max=n - 1)
    if c["temperature"] > 0:
        drafted = accepted < count
        if s["probs"] is None:
            q = torch.zeros_like(left).scatter_(1, x[b, r][:, None], 1.0)
        else:
            q = s["probs"][b, r].double()
        left = (left - q * drafted[:, None]).clamp_(min=0)
    run_ = left.cumsum(1)
    token = (run_ <= coins[:, n:] * run_[:, -1:]).sum(1).clamp(max=V - 1)
    i = torch.arange(n1, device=DEV)
    tokens = torch.where(i < accepted[:, None], torch.nn.functional.pad(x, (0, 1)), torch.where(i == accepted[:, None], token[:, None], -1))
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------

def work(c):
    if c["op"] == "verify":
        rows = c["batch"] * (c["drafts"] + 1) * c["vocab"]
        size = 4 if c["dtype"] == "f32" else 2
        q = 0 if c["certain"] or c["temperature"] == 0 else c["batch"] * c["vocab"] * 4          # of the draft that is replaced
        return {"bytes": rows * size + q, "flops": 4 * rows}
    lens, count = _numbers(c)
    size, wide = (4 if c["dtype"] == "f32" else 2), c["dk"] + c["dv"]
    if c["op"] != "attend":
        values = sum(count) * c["heads"] * wide
        return {"bytes": values * (size + 1) + 8 * c["heads"] * sum(-(-m // c["block"]) for m in count), "flops": 2 * values}
    keys, pairs = 0, 0
    for length, m in zip(lens, count):
        if not c["window"]:
            keys += length
            pairs += sum(range(length - m + 1, length + 1))
            continue
        low = max(0, length - m + 1 - c["window"])
        keys += length - low + min(low, c["keep"])
        for t in range(length - m, length):
            low = max(0, t + 1 - c["window"])
            pairs += t + 1 - low + min(low, c["keep"])
    return {"bytes": keys * c["kv_heads"] * wide + sum(count) * c["heads"] * wide * size, "flops": 2 * pairs * c["heads"] * wide}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------------------

def _nearest8(x):
    """The E4M3 value next to x, ties to the even one: steps of 2^-9 below 2^-6, of an eighth of the power of two below |x| from there on, at most 448."""
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    power = torch.where(torch.exp2(power) > x.abs().clamp(min=2.0 ** -6), power - 1, power)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "verify":
        return _exact_verify(s, case)
    lens, count = _numbers(case)
    table = s["table"].tolist()
    block, n = case["block"], case["new"]
    if case["op"] == "write":
        result = {}
        for name in ("k", "v"):
            codes, scale = s[name].double(), s[name + "_scale"].double()
            for b, (length, m) in enumerate(zip(lens, count)):
                first = length - m
                for j in range(first // block, (length - 1) // block + 1):
                    lo, hi = max(first, j * block), min(length, (j + 1) * block)
                    rows = s["new_" + name][b, lo - first:hi - first].double().transpose(0, 1)           # [heads, rows, d]
                    need = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((1, 2)) / 448)))
                    at, kept = table[b][j], lo - j * block
                    if kept:
                        need = torch.maximum(need, scale[at])
                        codes[at, :, :kept] = _nearest8(codes[at, :, :kept] * (scale[at] / need)[:, None, None])
                    scale[at] = need
                    codes[at, :, kept:kept + hi - lo] = _nearest8(rows / need[:, None, None])
            result[name], result[name + "_scale"] = codes, scale
        return result
    if case["op"] == "read":
        result = {}
        for name, out in zip("kv", s["out"]):
            back = out.double()
            for b, (length, m) in enumerate(zip(lens, count)):
                x = s[name].view(torch.uint8)[s["table"][b].long()].view(F8).double()
                x = (x * s[name + "_scale"][s["table"][b].long()].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)
                back[b, :m] = x[:, length - m:length].transpose(0, 1)
            result[name] = back
        return result
    G, H = case["kv_heads"], case["heads"]
    back = s["out"].double()
    for b, (length, m) in enumerate(zip(lens, count)):
        at = s["table"][b].long()
        t = torch.arange(length - m, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None, :]
        hidden = j > t
        if case["window"]:
            hidden |= (j <= t - case["window"]) & (j >= case["keep"])
        for g in range(G):
            k, v = ((s[x].view(torch.uint8)[at, g].view(F8).double() * s[x + "_scale"][at, g].double()[:, None, None]).flatten(0, 1)[:length] for x in "kv")
            for h in range(g * (H // G), (g + 1) * (H // G)):
                w = s["q"][b, :m, h].double() @ k.T / math.sqrt(case["dk"])
                back[b, :m, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v
    return back


def _exact_verify(s, case):
    B, n, V = case["batch"], case["drafts"], case["vocab"]
    accepted = torch.zeros(B, dtype=torch.int32)
    tokens = torch.full((B, n + 1), -1, dtype=torch.int32)
    for b in range(B):
        m = n if s["count"] is None else int(s["count"][b])
        for i in range(m + 1):
            row = s["logits"][b, i].double()
            if case["temperature"] == 0:
                p = torch.zeros_like(row)
                p[torch.nonzero(row == row.max())[0, 0]] = 1.0
            else:
                p = torch.softmax(row / case["temperature"], 0)
            q = torch.zeros_like(row)
            if i < m:
                x, coin = int(s["drafts"][b, i]), float(s["coins"][b, i])
                if case["temperature"] > 0:
                    q = s["probs"][b, i].double() if s["probs"] is not None else q.index_fill(0, torch.tensor([x], device=DEV), 1.0)
                if (float(p[x]) > 0) if case["temperature"] == 0 else (coin * float(q[x]) < float(p[x])):
                    tokens[b, i] = x
                    accepted[b] += 1
                    continue
            left = (p - q).clamp(min=0)
            sums = torch.cumsum(left, 0)
            tokens[b, i] = int(torch.nonzero(sums > float(s["coins"][b, n]) * sums[-1])[0, 0])
            break
    return {"accepted": accepted, "tokens": tokens}
