"""Timed cases of the operators that take prompts of several sequences as packed rows, one sequence behind the other: tables of cache blocks and places of
tokens made on the GPU, packed rows joining the 8-bit cache, and attention of whole prompts.

  blocks   free blocks are a stack.  First sequences give back what lies behind their first keep[b] tokens, in the reverse of the order in which blocks are
           taken; then count[b] tokens join every sequence: a block number for every block that these are first in, sequence by sequence, off the end of the
           stack, and for every joining token, packed, its position and its slot, block number x block + row in it.  The pass of a case ends with the
           lengths that it began with, so that it can be made again.
  append   packed rows of keys and values join the 8-bit cache at the places that were laid out for them.  Scale of a block and head: the smallest power
           of two s with |x| <= 448 s over the rows that it holds, never smaller than it was while rows from earlier calls are in the block; their codes
           are rounded again where it grew.  A block whose first row is written starts anew.
  attend   causal attention of packed sequences: token i of a sequence sees its tokens j <= i with i - j < window or j < keep_first; query head h reads
           key / value head h / (heads / kv_heads)

Rows behind the last sequence belong to no one: they are neither read nor written.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEAST, MOST = -40, 40           # exponents of a scale


def _dsk():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek.cpp_b200"))
    import dsk
    return dsk


def listed():
    return [
        # between two steps of speculative decoding: refused drafts' blocks go back, the next token and drafts of 64 sequences get places.  Latency
        dict(name="blocks_step", op="blocks", batch=64, new=5, most=8000, block=64, spare=0, uneven=1),
        # 32 sequences have ended and prompts of their lengths take their place
        dict(name="blocks_prompts", op="blocks", batch=32, new=8000, most=8000, block=32, spare=1000, uneven=1),
        # a step that serves decoded tokens and portions of prompts at once
        dict(name="append_step", op="append", batch=48, new=700, most=6000, heads=4, dk=128, dv=128, block=64, dtype="bf16", spare=100, uneven=2),
        # prompts of eight sequences join, wide keys
        dict(name="append_prompts", op="append", batch=8, new=5001, most=5001, heads=16, dk=192, dv=128, block=64, dtype="bf16", spare=0, uneven=1),
        # one short prompt: latency
        dict(name="attend_one", op="attend", batch=1, new=37, heads=16, kv_heads=4, dk=128, dv=128, dtype="bf16", window=0, keep=0, spare=0, uneven=0, fused=1),
        # questions of a batch: many short prompts of unequal lengths
        dict(name="attend_short", op="attend", batch=64, new=200, heads=16, kv_heads=4, dk=128, dv=128, dtype="bf16", window=0, keep=0, spare=77, uneven=1, fused=1),
        # documents of unequal lengths, a key head for every query head, wide keys
        dict(name="attend_ragged", op="attend", batch=8, new=5001, heads=32, kv_heads=32, dk=192, dv=128, dtype="bf16", window=0, keep=0, spare=0, uneven=1, fused=0),
        # one long document
        dict(name="attend_long", op="attend", batch=1, new=16384, heads=16, kv_heads=4, dk=128, dv=128, dtype="bf16", window=0, keep=0, spare=0, uneven=0, fused=1),
        # sliding window with first tokens that stay visible, small heads
        dict(name="attend_window", op="attend", batch=4, new=8000, heads=16, kv_heads=4, dk=64, dv=64, dtype="f16", window=1024, keep=4, spare=500, uneven=1, fused=1),
        # the widest heads
        dict(name="attend_wide", op="attend", batch=3, new=2500, heads=16, kv_heads=8, dk=256, dv=256, dtype="bf16", window=0, keep=0, spare=0, uneven=1, fused=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["blocks", "append", "attend", "attend", "attend", "attend"])
    c = dict(op=op, batch=_log(rng, 1, 256), spare=rng.choice([0, 1, 17, 300]), uneven=rng.choice([0, 1, 1, 2]))
    if op == "blocks":
        c["block"], c["new"] = rng.choice([16, 32, 64, 128]), _log(rng, 1, 8000)
        while c["batch"] * c["new"] > 250_000:
            c["batch"], c["new"] = max(1, c["batch"] // 2), max(1, c["new"] * 2 // 3)
        c["most"] = c["new"] + rng.choice([0, _log(rng, 1, 8000)])
        return c
    dk, dv = rng.choice([(64, 64), (80, 80), (96, 64), (128, 128), (128, 128), (112, 128), (192, 128), (256, 256)])
    c.update(new=_log(rng, 1, 12000), dk=dk, dv=dv, dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "append":
        c["block"], c["heads"] = rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8, 16])
        while c["batch"] * c["new"] * c["heads"] * (dk + dv) > 180_000_000:
            c["batch"], c["new"] = max(1, c["batch"] // 2), max(1, c["new"] * 2 // 3)
        c["most"] = c["new"] + rng.choice([0, _log(rng, 1, 4000)])
        return c
    c["kv_heads"] = rng.choice([1, 2, 4, 8])
    c["heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    c["window"], c["keep"] = rng.choice([(0, 0), (0, 0), (0, 0), (_log(rng, 16, 4000), rng.choice([0, 4, 17]))])
    c["fused"] = rng.choice([0, 1])
    while c["batch"] * c["new"] * c["new"] * c["heads"] * (dk + dv) > 900_000_000_000 or c["batch"] * c["new"] * c["heads"] * (dk + dv) > 180_000_000:
        c["batch"], c["new"] = max(1, c["batch"] // 2), max(1, c["new"] * 2 // 3)
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------

def _numbers(case):
    """Tokens that every sequence has in the end, and how many of them are new.  uneven: 0 all alike, 1 spread, 2 one token each but for every 16th."""
    B, n = case["batch"], case["new"]
    most = case.get("most", n)
    if case["uneven"] == 0 or B == 1:
        return [most] * B, [n] * B
    if case["uneven"] == 2:
        count = [n if b % 16 == 0 else 1 for b in range(B)]
    else:
        count = [max(1, n - n * ((5 * b) % B) // B) for b in range(B)]
    if most == n:
        return list(count), count
    return [max(m, most - (most - m) * ((7 * b) % B) // B) for b, m in enumerate(count)], count


def _random(shape, g, dtype=torch.float32, spread=None):
    x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(generator=g)
    if spread is not None:
        x *= spread
    return x.to(dtype)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    lens, count = _numbers(case)
    B, rows = case["batch"], sum(count) + case["spare"]
    state = {"case": case, "rows": rows, "lens": _i32(lens), "count": _i32(count)}
    if case["op"] == "attend":
        H, G, dk, dv, dt = case["heads"], case["kv_heads"], case["dk"], case["dv"], TYPES[case["dtype"]]
        starts = [0]
        for n in count:
            starts.append(starts[-1] + n)
        state["starts"] = _i32(starts)
        if case["fused"]:                                                       # queries, keys and values of a token side by side, as one product leaves them
            x = _random((rows, H * dk + G * dk + G * dv), g, dt)
            x[:, :H * dk] *= 1.5
            q, k, v = x[:, :H * dk], x[:, H * dk:(H + G) * dk], x[:, (H + G) * dk:]
        else:
            q, k, v = _random((rows, H * dk), g, dt, spread=1.5), _random((rows, G * dk), g, dt), _random((rows, G * dv), g, dt)
        state["q"], state["k"], state["v"] = q.unflatten(1, (H, dk)), k.unflatten(1, (G, dk)), v.unflatten(1, (G, dv))
        state["out"] = torch.zeros((rows, H, dv), device=DEV, dtype=dt)
        if own:
            state["packed"] = _dsk().Packed.of(state["starts"], rows)
        return state
    block = case["block"]
    per = -(-max(lens) // block)
    blocks = B * per + 3
    held = [-(-(l - n) // block) for l, n in zip(lens, count)]                  # blocks of the tokens that sequences have had for long
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
    table = torch.full((B, per), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    free = order[at:]                                                           # taken from the end
    state["keep"] = state["lens"] - state["count"]
    if case["op"] == "blocks":                                                  # the sequences have their tokens, the new ones among them
        top = free.shape[0]
        for b, (l, h) in enumerate(zip(lens, held)):
            n = -(-l // block) - h
            table[b, h:h + n] = free[top - n:top].flip(0)
            top -= n
        state["table"] = table.to(DEV)
        if own:
            state["pool"] = _dsk().Blocks.of(free[:top].to(DEV), blocks, block)
        else:
            state["free"], state["n_free"] = torch.zeros(blocks, device=DEV, dtype=torch.int32), _i32([top])
            state["free"][:top] = free[:top].to(DEV)
        return state
    state["table"] = table.to(DEV)
    H, dk, dv, dt = case["heads"], case["dk"], case["dv"], TYPES[case["dtype"]]
    for name, d in (("k", dk), ("v", dv)):
        state[name + "_scale"] = _pow2(torch.randint(-11, -6, (blocks, H), generator=g, device=DEV))
        state[name] = (_random((blocks, H, block, d), g) * 100).clamp_(-448, 448).to(F8)
    size = torch.exp(0.7 * _random((rows, H, 1), g))                            # tokens of unequal size
    state["new_k"], state["new_v"] = _random((rows, H, dk), g, dt, spread=size), _random((rows, H, dv), g, dt, spread=size)
    if own:                                                                     # the cache's handle, and the places that the step was given
        dsk = _dsk()
        state["cache"] = dsk.Cache8.of(state["k"], state["v"], state["k_scale"], state["v_scale"])
        state["pool"] = dsk.Blocks.of(free.to(DEV), blocks, block)
        state["packed"] = state["pool"].extend(state["table"], state["keep"], state["count"], rows)
    else:
        full = torch.zeros(blocks, device=DEV, dtype=torch.int32)
        full[:free.shape[0]] = free.to(DEV)
        _, _, state["positions"], state["slots"] = _extend(state["table"], state["keep"], state["count"], rows, block, full, _i32([free.shape[0]]))
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if c["op"] == "blocks":
        if own:
            pool = s["pool"]
            pool.cut(s["table"], s["lens"], s["keep"])
            plan = pool.extend(s["table"], s["keep"], s["count"], s["rows"])
            return {"table": s["table"], "free": pool.free, "n_free": pool.n_free, "starts": plan.starts, "lens": plan.lens, "positions": plan.positions, "slots": plan.slots}
        _cut(s["table"], s["lens"], s["keep"], c["block"], s["free"], s["n_free"])
        starts, lens, positions, slots = _extend(s["table"], s["keep"], s["count"], s["rows"], c["block"], s["free"], s["n_free"])
        return {"table": s["table"], "free": s["free"], "n_free": s["n_free"], "starts": starts, "lens": lens, "positions": positions, "slots": slots}
    if c["op"] == "append":
        if own:
            s["cache"].append(s["new_k"], s["new_v"], s["packed"])
        else:
            _append(s, c, "k")
            _append(s, c, "v")
        return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if own:
        s["packed"].attend(s["q"], s["k"], s["v"], window=c["window"], keep_first=c["keep"], out=s["out"])
    else:
        _attend(s, c)
    return s["out"]


# ---- plain forms -------------------------------------------------------------------------------------------------------------------------------

def _cut(table, lens, keep, block, free, n_free):
    j = torch.arange(table.shape[1], device=DEV)
    back = (j >= (keep[:, None] + block - 1) // block) & (j < (lens[:, None] + block - 1) // block)
    flat = back.flatten().flip(0)
    to = n_free + flat.cumsum(0) - 1
    stack = torch.cat([free, free[:1]])                                         # one more place, for what does not go back
    stack[torch.where(flat, to, free.shape[0])] = table.flatten().flip(0)
    free.copy_(stack[:-1])
    n_free += flat.sum().to(torch.int32)
    table.masked_fill_(back, -1)


def _extend(table, lens, count, rows, block, free, n_free):
    B = table.shape[0]
    had, has = (lens + block - 1) // block, (lens + count + block - 1) // block
    need = has - had
    fits = (need.cumsum(0) <= n_free) & (count.cumsum(0) <= rows)
    count, need = torch.where(fits, count, 0), torch.where(fits, need, 0)
    taken = need.cumsum(0)
    j = torch.arange(table.shape[1], device=DEV)
    new = (j >= had[:, None]) & (j < (had + need)[:, None])
    at = n_free - 1 - ((taken - need)[:, None] + j - had[:, None])
    table.copy_(torch.where(new, free[at.clamp(0, free.shape[0] - 1)], table))
    n_free -= taken[-1].to(torch.int32)
    starts = torch.nn.functional.pad(count.cumsum(0), (1, 0)).to(torch.int32)
    i = torch.arange(rows, device=DEV)
    b = torch.searchsorted(starts[1:], i, right=True).clamp(max=B - 1)
    t = lens[b] + i - starts[b]
    there = i < starts[-1]
    slot = table[b, (t // block).clamp(0, table.shape[1] - 1)] * block + t % block
    return starts, lens + count, torch.where(there, t, -1).to(torch.int32), torch.where(there, slot, -1).to(torch.int32)


def _append(s, c, name):
    codes, scale, x, block = s[name], s[name + "_scale"], s["new_" + name].float(), c["block"]
    blocks, H, _, d = codes.shape
    there = s["slots"] >= 0
    slot = s["slots"].long().clamp(min=0)
    page, row = torch.where(there, slot // block, blocks), slot % block         # (a place behind the cache for rows of no one)
    most = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    need = torch.zeros((blocks + 1, H), device=DEV).scatter_reduce(0, page[:, None].expand(-1, H), most, "amax")[:blocks]
    m, e = torch.frexp(need)
    e = torch.where(need > 0, e - 9 + (m > 0.875), LEAST).clamp(LEAST, MOST)
    kept = torch.full((blocks + 1,), block, device=DEV, dtype=torch.long).scatter_reduce(0, page, row, "amin")[:blocks, None]   # rows of earlier calls
    new = torch.where(kept < block, torch.where(kept > 0, torch.maximum(scale, _pow2(e)), _pow2(e)), scale)
    # the kept rows of every sequence's first block, in the new scale
    first = torch.div(s["keep"].long(), block, rounding_mode="floor").clamp(max=s["table"].shape[1] - 1)
    first = s["table"].long().gather(1, first[:, None])[:, 0].clamp(min=0)
    old = codes.view(torch.uint8)[first].view(F8).float()
    again = (old * (scale / new)[first][:, :, None, None]).to(F8).view(torch.uint8)
    bytes_ = codes.view(torch.uint8)
    still = torch.arange(block, device=DEV)[None, :] < kept[first]
    bytes_[first] = torch.where(still[:, None, :, None], again, bytes_[first])
    # the new rows
    fresh = (x / torch.cat([new, new[:1]])[page][..., None]).clamp(-448, 448).to(F8).view(torch.uint8)
    bytes_[page[there], :, row[there]] = fresh[there]
    scale.copy_(new)


def _attend(s, c):
    H, G, dk, dv, scale = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["dk"] ** -0.5
    at = 0
    for n in _numbers(c)[1]:
        k, v = s["k"][at:at + n].float().transpose(0, 1), s["v"][at:at + n].float().transpose(0, 1)     # [kv_heads, n, d]
        step = max(1, min(n, 400_000_000 // (n * H)))                          # queries at a time
        for i0 in range(0, n, step):
            i1 = min(n, i0 + step)
            q = s["q"][at + i0:at + i1].float().unflatten(1, (G, H // G)).permute(1, 2, 0, 3).flatten(1, 2)
            w = (q @ k[:, :i1].transpose(1, 2)).view(G, H // G, i1 - i0, i1) * scale
            i, j = torch.arange(i0, i1, device=DEV)[:, None], torch.arange(i1, device=DEV)
            seen = j <= i
            if c["window"]:
                seen &= (i - j < c["window"]) | (j < c["keep"])
            w.masked_fill_(~seen, -math.inf)
            w -= w.amax(-1, keepdim=True)
            w.exp_()
            w /= w.sum(-1, keepdim=True)
            o = w.view(G, -1, i1) @ v[:, :i1]
            s["out"][at + i0:at + i1] = o.view(G, H // G, i1 - i0, dv).permute(2, 0, 1, 3).reshape(i1 - i0, H, dv).to(s["out"].dtype)
        at += n


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------

def work(c):
    lens, count = _numbers(c)
    tokens = sum(count)
    if c["op"] == "blocks":                                                     # block numbers there and back, in stack and table; positions and slots; starts, lengths, counts
        rows = tokens + c["spare"]
        moved = sum(-(-l // c["block"]) - -(-(l - n) // c["block"]) for l, n in zip(lens, count))
        return {"bytes": 8 * rows + 16 * moved + 4 * 6 * c["batch"], "flops": 2 * rows}
    if c["op"] == "append":
        values = tokens * c["heads"] * (c["dk"] + c["dv"])
        return {"bytes": 3 * values + 8 * c["heads"] * sum(-(-n // c["block"]) for n in count), "flops": 2 * values}
    pairs = 0
    for n in count:
        w = min(c["window"], n) if c["window"] else n
        pairs += w * (w + 1) // 2 + (n - w) * w
        if c["window"]:                                                         # first tokens that the window has left behind
            pairs += sum(max(0, n - w - j) for j in range(min(c["keep"], n)))
    wide = c["dk"] + c["dv"]
    return {"bytes": 2 * tokens * (c["heads"] + c["kv_heads"]) * wide, "flops": 2 * pairs * c["heads"] * wide}


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
    lens, count = _numbers(case)
    if case["op"] == "blocks":                                                  # on the host, block by block and token by token
        block, table = case["block"], s["table"].tolist()
        stack, top = s["free"].tolist(), int(s["n_free"])
        for b in reversed(range(len(lens))):
            for j in reversed(range(-(-(lens[b] - count[b]) // block), -(-lens[b] // block))):
                stack[top] = table[b][j]
                top += 1
        starts, positions, slots = [0], [], []
        for b, (l, n) in enumerate(zip(lens, count)):
            for t in range(l - n, l):
                if t % block == 0:
                    top -= 1
                    table[b][t // block] = stack[top]
                positions.append(t)
                slots.append(table[b][t // block] * block + t % block)
            starts.append(len(slots))
        rest = [-1] * case["spare"]
        values = {"table": table, "free": stack, "n_free": [top], "starts": starts, "lens": lens, "positions": positions + rest, "slots": slots + rest}
        return {name: torch.tensor(x, dtype=torch.int32) for name, x in values.items()}
    if case["op"] == "append":
        block, table, result = case["block"], s["table"].tolist(), {}
        for name in ("k", "v"):
            codes, scale, at = s[name].double(), s[name + "_scale"].double(), 0
            for b, (l, n) in enumerate(zip(lens, count)):
                first = l - n
                for j in range(first // block, (l - 1) // block + 1):
                    lo, hi = max(first, j * block), min(l, (j + 1) * block)
                    x = s["new_" + name][at + lo - first:at + hi - first].double().transpose(0, 1)         # [heads, rows, d]
                    m, e = torch.frexp(x.abs().amax((1, 2)) / 448)                       # m x 2^e, m from a half up to 1
                    need = torch.ldexp(torch.ones_like(m), e - (m == 0.5).to(e.dtype))
                    page, kept = table[b][j], lo - j * block
                    if kept:
                        need = torch.maximum(need, scale[page])
                        codes[page, :, :kept] = _nearest8(codes[page, :, :kept] * (scale[page] / need)[:, None, None])
                    scale[page] = need
                    codes[page, :, kept:kept + hi - lo] = _nearest8(x / need[:, None, None])
                at += n
            result[name], result[name + "_scale"] = codes, scale
        return result
    out, at = s["out"].double(), 0
    group = case["heads"] // case["kv_heads"]
    for n in count:
        for h in range(case["heads"]):
            k, v = s["k"][at:at + n, h // group].double(), s["v"][at:at + n, h // group].double()
            for i0 in range(0, n, 8192):
                i1 = min(n, i0 + 8192)
                i, j = torch.arange(i0, i1, device=DEV)[:, None], torch.arange(n, device=DEV)[None, :]
                hidden = j > i
                if case["window"]:
                    hidden |= (j <= i - case["window"]) & (j >= case["keep"])
                x = s["q"][at + i0:at + i1, h].double() @ k.T / math.sqrt(case["dk"])
                out[at + i0:at + i1, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
        at += n
    return out
