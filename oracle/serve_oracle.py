"""serve_oracle.py — float64 restatement of the operators on device memory (include/dsk.h): the 8-bit key / value cache, attention over it, and the verification of
drafted tokens.  Plain loops over sequences, blocks, heads and rows."""
import numpy as np

EXP = 40


def decode_table():
    """The 256 E4M3 values (exponent bias 7, three fraction bits, 0x7f and 0xff are NaN, no infinities)."""
    out = np.empty(256)
    for b in range(256):
        s, e, f = -1.0 if b & 128 else 1.0, (b >> 3) & 15, b & 7
        out[b] = np.nan if (b & 127) == 127 else s * (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
    return out


TABLE = decode_table()


def encode(x):
    """Codes of the E4M3 values next to x, ties to the even code, at most +-448; NaN is 0x7f with the sign dropped."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    mags = TABLE[:127]
    hi = np.clip(np.searchsorted(mags, a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up = (mags[hi] - a < a - mags[lo]) | ((mags[hi] - a == a - mags[lo]) & (hi % 2 == 0))
    code = np.where(up, hi, lo).astype(np.uint8)
    code = np.where(np.signbit(x), code | 128, code)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def scale_for(amax):
    """The smallest power of two s with amax <= 448 s, exponent within +-EXP."""
    if amax == 0:
        return 2.0 ** -EXP
    m, e = np.frexp(amax)
    return 2.0 ** min(EXP, max(-EXP, int(e) - 9 + (1 if m > 0.875 else 0)))


def write(codes, scales, table, first, count, x):
    """codes [blocks, heads, block, d] uint8 and scales [blocks, heads] change in place; x [batch, rows, heads, d] float64."""
    block = codes.shape[2]
    for b in range(len(table)):
        n, i = int(count[b]), 0
        while i < n:
            t = int(first[b]) + i
            j, kept = t // block, t % block
            m = min(n - i, block - kept)
            page = int(table[b][j]) if 0 <= j < len(table[b]) else -1
            if 0 <= page < len(codes):
                for h in range(codes.shape[1]):
                    rows = x[b, i:i + m, h]
                    fin = np.abs(rows[np.isfinite(rows)])
                    s = scale_for(fin.max() if fin.size else 0.0)
                    if kept:
                        old = scales[page, h]
                        s = max(s, old)
                        if s != old:
                            codes[page, h, :kept] = requantise(codes[page, h, :kept], old / s)
                    scales[page, h] = s
                    codes[page, h, kept:kept + m] = encode(rows / s)
            i += m


def requantise(codes, ratio):
    return encode(TABLE[codes] * ratio)


def gather(codes, scales, table_row, length, head):
    """Values [length, d] of a sequence's head; tokens of blocks outside the cache are None rows (mask)."""
    block, d = codes.shape[2:]
    out, there = np.zeros((length, d)), np.ones(length, dtype=bool)
    for t in range(length):
        page = int(table_row[t // block])
        if 0 <= page < len(codes):
            out[t] = TABLE[codes[page, head, t % block]] * scales[page, head]
        else:
            there[t] = False
    return out, there


def attend(k, ks, v, vs, table, lens, count, q, heads, scale, window=0, keep=0, rows_out=None):
    """(result, sum p |v|, sum |q k| scale (largest over seen keys), largest p x value scale) of every row [batch, rows, heads, ...]; rows from count on are NaN."""
    batch, rows = q.shape[:2]
    block, G = k.shape[2], heads // k.shape[1]
    dv = v.shape[3]
    out, mass = np.full((batch, rows, heads, dv), np.nan), np.zeros((batch, rows, heads, dv))
    size, top = np.zeros((batch, rows, heads, 1)), np.zeros((batch, rows, heads, 1))
    for b in range(batch):
        L, n = int(lens[b]), int(count[b])
        L_here = max(0, min(L, len(table[b]) * block))
        for g in range(k.shape[1]):
            kk, there = gather(k, ks, table[b], L_here, g)
            vv, _ = gather(v, vs, table[b], L_here, g)
            sv = np.array([vs[int(table[b][t // block]), g] if there[t] else 0.0 for t in range(L_here)])
            for i in range(n):
                t = L - n + i
                j = np.arange(L_here)
                seen = there & (j <= t)
                if window:
                    seen &= (t - j < window) | (j < keep)
                for h in range(g * G, (g + 1) * G):
                    if not seen.any():
                        out[b, i, h] = 0.0
                        continue
                    x = q[b, i, h].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        w = kk[seen] @ x * scale
                        p = np.exp(w - w.max())
                        p /= p.sum()
                        out[b, i, h] = p @ vv[seen]
                        mass[b, i, h] = p @ np.abs(vv[seen])
                        size[b, i, h] = (np.abs(kk[seen]) @ np.abs(x)).max() * abs(scale)
                        top[b, i, h] = (p * sv[seen]).max()
    return out, mass, size, top


def verify(logits, drafts, coins, probs, count, temperature):
    batch, n1, V = logits.shape
    n = n1 - 1
    accepted, tokens = np.zeros(batch, dtype=np.int32), np.full((batch, n1), -1, dtype=np.int32)
    for b in range(batch):
        for i in range(int(count[b]) + 1):
            row = logits[b, i].astype(np.float64)
            drafted = i < count[b]
            x = int(drafts[b, i]) if drafted else -1
            bad = np.isnan(row).any() or not (row > -np.inf).any() or (temperature > 0 and (row == np.inf).any())
            if bad:
                break
            if temperature == 0:
                best = int(np.argmax(row))
                if drafted and x == best:
                    tokens[b, i] = x
                    accepted[b] += 1
                    continue
                tokens[b, i] = best
                break
            p = np.exp((row - row.max()) / temperature)
            p /= p.sum()
            q = np.zeros(V)
            if drafted:
                if probs is not None:
                    q = probs[b, i].astype(np.float64)
                elif 0 <= x < V:
                    q[x] = 1.0
                if 0 <= x < V and float(coins[b, i]) * q[x] < p[x]:
                    tokens[b, i] = x
                    accepted[b] += 1
                    continue
            left = np.maximum(p - q, 0)
            sums = np.cumsum(left)
            over = np.nonzero(sums > float(coins[b, n]) * sums[-1])[0]
            some = np.nonzero(left > 0)[0]
            tokens[b, i] = over[0] if len(over) else some[-1] if len(some) else -1
            break
    return accepted, tokens
