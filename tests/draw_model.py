"""A draw from one row by one wave in numpy, in the order in which the device adds: the weights of a
lane pairwise, then a scan over 64 lanes (inside rows of 16 lanes, then the last lane of a row to the
next ones).  The scan's sums are of the same lanes in different associations, so they need not grow
from lane to lane where a lane adds nothing."""
import numpy as np

LANES = 64


def pairwise(w):
    """Sums over the last axis of 4 or 8."""
    while w.shape[-1] > 1:
        w = w[..., 0::2] + w[..., 1::2]
    return w[..., 0]


def scan(v):
    """Inclusive sums over the last axis of 64 lanes."""
    v = v.copy()
    for step in (1, 2, 4, 8):
        rows = v.reshape(v.shape[:-1] + (4, 16))
        moved = np.zeros_like(rows)
        moved[..., step:] = rows[..., :-step]
        v = (rows + moved).reshape(v.shape)
    v[..., 16:32] += v[..., 15:16]
    v[..., 48:64] += v[..., 47:48]
    v[..., 32:64] += v[..., 31:32]
    return v


def weights(x):
    """exp(x - max) of rows (rows, 64 * vec) as (rows, 64, vec)."""
    with np.errstate(invalid="ignore"):
        w = np.exp(x - x.max(1, keepdims=True))
    return w.reshape(len(x), LANES, -1)


def draw(w, u):
    """The index that numbers u (rows,) fall on, from weights w (rows, 64, vec): the first lane with a
    weight whose sum passes the target (else the last with a weight), and in it the first entry with a
    weight whose running sum does (else the last)."""
    mine = pairwise(w)
    upto = scan(mine)
    target = u * upto[:, -1]
    out = np.zeros(len(w), np.int64)
    for r in range(len(w)):
        some = mine[r] > 0
        hits = np.nonzero(some & (upto[r] > target[r]))[0]
        lane = hits[0] if len(hits) else np.nonzero(some)[0][-1]
        run = upto[r, lane - 1] if lane else 0.0
        at = -1
        for e in range(w.shape[2]):
            run += w[r, lane, e]
            if w[r, lane, e] > 0:
                at = e
                if run > target[r]:
                    break
        out[r] = lane * w.shape[2] + at
    return out


def order_key(x):
    """Unsigned integers that order like float32 values, both zeros alike."""
    b = int(np.array([np.float32(x) + np.float32(0.0)], np.float32).view(np.uint32)[0])
    return b ^ (0xFFFFFFFF if b >> 31 else 0x80000000)


def key_value(key):
    b = key ^ (0x80000000 if key >> 31 else 0xFFFFFFFF)
    return float(np.array([b], np.uint32).view(np.float32)[0])


def search(values, v, answer, near=4):
    """The values that the search for top_p's cut looks at, starting from v: values is the row's,
    answer(v) 1, -1 or 0 for a cut above, below or at v."""
    values = sorted(set(values))
    lowest, largest = values[0], values[-1]
    below, beyond = order_key(lowest) - 1, order_key(largest) + 1
    key, went, last, seen, step = order_key(v), 0, False, [], 0
    while True:
        seen.append(v)
        go = answer(v)
        if last or go == 0 or go == -went:
            return seen
        if go > 0:
            below = key
        else:
            beyond = key
        went = go if step < near else 0
        last = step >= near and beyond - below <= 1
        if step >= near and not last:
            key = below + (beyond - below) // 2
            v = key_value(key)
        else:
            if last:
                v = key_value(below)
            v = min(y for y in values if y > v) if last or go > 0 else max(y for y in values if y < v)
            key = order_key(v)
        step += 1
