"""The operators around a forest's leaves in 64 bits, in numpy: what tests compare with."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def groups(leaf, leaves):
    """leaf [rows, trees] -> order [trees, rows], begin and count [trees, leaves]."""
    rows, trees = leaf.shape
    order = np.empty((trees, rows), np.int32)
    begin = np.empty((trees, leaves), np.int32)
    count = np.empty((trees, leaves), np.int32)
    for t in range(trees):
        at = 0
        for l in range(leaves):
            mine = np.flatnonzero(leaf[:, t] == l)
            order[t, at:at + len(mine)] = mine
            begin[t, l], count[t, l] = at, len(mine)
            at += len(mine)
        order[t, at:] = np.flatnonzero((leaf[:, t] < 0) | (leaf[:, t] >= leaves))
    return order, begin, count


def product(x, w, b, leaf, leaves):
    """(y, the sum of the magnitudes that were added) for leaf [rows, trees]."""
    y = np.zeros((len(x), w.shape[1]))
    size = np.zeros_like(y)
    for t in range(leaf.shape[1]):
        for l in range(leaves):
            n = np.flatnonzero(leaf[:, t] == l)
            g = t * leaves + l
            y[n] += x[n] @ w[g].T
            size[n] += np.abs(x[n]) @ np.abs(w[g]).T
            if b is not None:
                y[n] += b[g]
                size[n] += np.abs(b[g])
    return y, size


def product_dx(dy, w, leaf, leaves):
    dx = np.zeros((len(dy), w.shape[2]))
    size = np.zeros_like(dx)
    for t in range(leaf.shape[1]):
        for l in range(leaves):
            n = np.flatnonzero(leaf[:, t] == l)
            dx[n] += dy[n] @ w[t * leaves + l]
            size[n] += np.abs(dy[n]) @ np.abs(w[t * leaves + l])
    return dx, size


def product_dw(dy, x, leaf, leaves):
    """(dw, its size, db, its size)"""
    G = leaf.shape[1] * leaves
    dw = np.zeros((G, dy.shape[1], x.shape[1]))
    db = np.zeros((G, dy.shape[1]))
    dw_size, db_size = np.zeros_like(dw), np.zeros_like(db)
    for g in range(G):
        n = np.flatnonzero(leaf[:, g // leaves] == g % leaves)
        dw[g], db[g] = dy[n].T @ x[n], dy[n].sum(0)
        dw_size[g], db_size[g] = np.abs(dy[n]).T @ np.abs(x[n]), np.abs(dy[n]).sum(0)
    return dw, dw_size, db, db_size


def philox(block, offset, seed):
    """Philox4x32-10: uint32 [len(block), 4] for the counters (block, offset), key seed."""
    block = np.asarray(block, np.uint64)
    c = [block & M32, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF),
         np.full_like(block, offset >> 32)]
    for r in range(10):
        k0 = np.uint64((seed + 0x9E3779B9 * r) & 0xFFFFFFFF)
        k1 = np.uint64(((seed >> 32) + 0xBB67AE85 * r) & 0xFFFFFFFF)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & M32, (a >> np.uint64(32)) ^ c[3] ^ k1, a & M32]
    return np.stack(c, 1).astype(np.uint32)


def kept(units, p, seed, offset=0):
    """Which of the units are kept, and the share that is."""
    t = int(np.floor(p * 65536 + 0.5))
    words = philox(np.arange((units + 7) // 8), offset, seed)
    fields = np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)
    return fields[:units] >= t, 1 - t / 65536


def scores(x, kind, bias=None, mask=None, mask_rows=None, ids=None, offsets=None,
           penalties=None):
    """(answers, size of the terms of s) for x [rows, classes]; mask uint32 [masks, words],
    penalties [rows, 3]."""
    rows, V = x.shape
    out = np.empty((rows, V))
    size = np.zeros((rows, V))
    for n in range(rows):
        s = x[n].astype(np.float64)
        big = np.abs(s)
        if ids is not None:
            lo = min(max(int(offsets[n]), 0), len(ids))
            hi = min(max(int(offsets[n + 1]), lo), len(ids))
            mine = ids[lo:hi].astype(np.int64)
            c = np.bincount(mine[(mine >= 0) & (mine < V)], minlength=V)
            r, f, p = penalties[n]
            with np.errstate(invalid="ignore"):
                s = np.where(c > 0, np.where(s > 0, s / r, s * r) - f * c - p, s)
                big = np.where(c > 0, big * max(r, 1 / r) + abs(f) * c + abs(p), big)
        if bias is not None:
            s = s + bias
            big = big + np.abs(bias)
        m = -1
        if mask is not None:
            m = mask_rows[n] if mask_rows is not None else (0 if len(mask) == 1 else n)
        if 0 <= m < (0 if mask is None else len(mask)):
            j = np.arange(V)
            s = np.where((mask[m][j // 32] >> (j % 32).astype(np.uint32)) & 1, s, -np.inf)
        if kind == "transformed":
            top = s.max()
            if top == -np.inf:
                s = np.zeros(V)
            else:
                with np.errstate(invalid="ignore"):
                    e = np.where(s == -np.inf, 0.0, np.exp(s - top))
                s = e / e.sum()
        out[n], size[n] = s, big
    return out, size


def whole_numbers(rng, rows, cols):
    """Whole numbers of -3 .. 5 without 0 and of positive mean.  Products of two are at most
    25, so float32 sums of up to 2^24 / 25 = 671088 of them are exact in any order, and a
    gradient of the maps that leaves out or repeats a row differs in every element of its
    leaf."""
    v = rng.integers(-3, 5, (rows, cols))
    return np.where(v >= 0, v + 1, v).astype(np.float64)
