"""packed_oracle.py — float64 restatement of the operators on packed rows (include/dsk.h): places of tokens in the blocks of a cache, and causal attention of packed prompts.  Plain loops over
sequences, blocks, tokens and heads; packed rows into the 8-bit cache are serve_oracle.write, one sequence behind the other."""
import numpy as np

SHORT, PAGE, RANGE, TWICE = 8, 1, 2, 16


def extend(free, table, lens, count, rows, n_blocks, block):
    """free (a list, taken from its end) and table change in place.  Returns starts, lens, positions, slots, pieces (first row, rows, block, place), status."""
    starts, new, positions, slots, pieces, status, full = [0], [], [], [], [], 0, False
    left_blocks, left_rows = len(free), rows
    for b, (l, c) in enumerate(zip(lens, count)):
        c = max(c, 0)
        if l < 0 or l + c > len(table[b]) * block:
            status |= RANGE
            c = 0
            n = 0
        else:
            n = -(-(l + c) // block) - -(-l // block)
            left_blocks -= n                                 # (what does not fit is taken all the same: nothing behind it fits either)
            left_rows -= c
        if left_blocks < 0 or left_rows < 0:
            status |= SHORT if c else 0
            c = 0
        for i in range(c):
            t = l + i
            if t % block == 0:
                table[b][t // block] = free.pop()
            page = int(table[b][t // block])
            known = 0 <= page < n_blocks
            if not known:
                status |= PAGE
            if t % block == 0 or i == 0:
                pieces.append([len(slots), 0, page, t % block])
            if known:
                pieces[-1][1] += 1
            positions.append(t)
            slots.append(page * block + t % block if known else -1)
        starts.append(len(slots))
        new.append(l + c)
    return starts, new, positions + [-1] * (rows - len(slots)), slots + [-1] * (rows - len(slots)), pieces, status


def cut(free, table, lens, keep, n_blocks, block):
    """free and table change in place; returns the status."""
    status = 0
    for b in reversed(range(len(lens))):
        if not (0 <= keep[b] <= lens[b] <= len(table[b]) * block):
            status |= RANGE
            continue
        for j in reversed(range(-(-keep[b] // block), -(-lens[b] // block))):
            page = int(table[b][j])
            table[b][j] = -1
            if not 0 <= page < n_blocks:
                status |= PAGE
            elif len(free) < n_blocks:
                free.append(page)
            else:
                status |= TWICE
    return status


def attend(q, k, v, starts, scale, window=0, keep=0):
    """q [rows, heads, dim_k], k, v [rows, kv_heads, dim] float64.  Returns (results, mass: sum of weights x |values|, size: the largest sum of |q k| x scale, top: the largest |value| seen), the
    last three for tolerances; rows of no one are NaN.  Infinite and NaN values make results NaN."""
    rows, H, _ = q.shape
    G, dv = k.shape[1], v.shape[2]
    out, mass = (np.full((rows, H, dv), np.nan) for _ in range(2))
    size, top = (np.zeros((rows, H, 1)) for _ in range(2))
    odd = ~np.isfinite(v)
    vf = np.where(odd, 0.0, v)
    for b in range(len(starts) - 1):
        s, e = int(starts[b]), int(starts[b + 1])
        n = e - s
        if n <= 0:
            continue
        i, j = np.arange(n)[:, None], np.arange(n)[None, :]
        seen = j <= i
        if window > 0:
            seen &= (i - j < window) | (j < keep)
        for h in range(H):
            g = h // (H // G)
            with np.errstate(all="ignore"):
                x = np.where(seen, q[s:e, h] @ k[s:e, g].T * scale, -np.inf)
                top_x = x.max(1, keepdims=True)
                w = np.exp(x - np.where(top_x == -np.inf, 0.0, top_x))
                total = w.sum(1, keepdims=True)
                w = np.where(total == 0, 0.0, w / np.where(total == 0, 1.0, total))
                out[s:e, h] = w @ vf[s:e, g]
                out[s:e, h] = np.where((seen @ odd[s:e, g].astype(np.int64)) > 0, np.nan, out[s:e, h])
                mass[s:e, h] = w @ np.abs(vf[s:e, g])
                size[s:e, h, 0] = np.where(seen, np.abs(np.nan_to_num(q[s:e, h])) @ np.abs(np.nan_to_num(k[s:e, g])).T * abs(scale), 0.0).max(1)
                top[s:e, h, 0] = np.where(seen, np.abs(vf[s:e, g]).max(1)[None, :], 0.0).max(1)
    return out, mass, size, top
