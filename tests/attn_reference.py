"""The attention operators in 64 bits with numpy: per-head norms and rotations,
the 8-bit cache's values, block tables, attention; and the error bounds that the
device's results are held to."""
import numpy as np

BLOCK, NONE = 32, 0xFFFFFFFF
U32 = 2.0 ** -24  # half a step of fp32, relative


def rope(x, w, pos, n_rot, base, style, eps=1e-6, norm=True, one_plus=False, factors=None):
    """(values, bounds) of x [T, H, D] (float32) normalised and rotated.

    The bound counts half steps of fp32: the squares' sum in groups (log2 of the lanes and the elements of a lane, D / 32
    at most, the mean's, root's and quotient's roundings; halved by the root), three products, the sine and
    cosine (2 steps each), two products and a sum: under 16 + D / 32 of them on |a| + |b|."""
    x = np.asarray(x, np.float64)
    T, H, D = x.shape
    g = np.ones(D)
    if norm and w is not None:
        g = np.asarray(w, np.float64) + (1.0 if one_plus else 0.0)
    y = x * (1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)) if norm else x.copy()
    y = y * g
    half = n_rot // 2
    f = np.ones(half) if factors is None else np.asarray(factors, np.float64)
    angle = np.asarray(pos, np.float64)[:, None, None] * (base ** (-2.0 * np.arange(half) / max(n_rot, 1)) / f)
    c, s = np.cos(angle), np.sin(angle)
    ia = np.arange(half) if style == "neox" else 2 * np.arange(half)
    ib = ia + half if style == "neox" else ia + 1
    a, b = y[..., ia], y[..., ib]
    out, size = y.copy(), np.abs(y)
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    # (an angle counted in 64 bits: the rate has half a step of it, the product another)
    wrong = np.zeros_like(size)
    wrong[..., ia] = wrong[..., ib] = np.abs(angle) * 2.0 ** -51
    return out, size * ((16 + D / 32) * U32 + wrong) + 1e-37


def codes(x):
    """(codes, scale) of a block's tokens x [n, D] of one head, as the header defines them."""
    x = np.asarray(x, np.float32)
    if not np.isfinite(x).all():
        return np.zeros(x.shape), np.float32(np.nan)
    s = np.float32(np.float64(np.abs(x).max(initial=0.0)) / 127)
    if s == 0:
        return np.zeros(x.shape), s
    return np.clip(np.rint(x.astype(np.float64) / np.float64(s)), -127, 127), s


def values(x):
    """float32 values that the cache holds for a sequence's tokens x [n, kv, D] from position 0 on."""
    x = np.asarray(x, np.float32)
    out = np.empty_like(x)
    for b in range(0, len(x), BLOCK):
        for h in range(x.shape[1]):
            c, s = codes(x[b:b + BLOCK, h])
            out[b:b + BLOCK, h] = c.astype(np.float32) * s
    return out


def attention(q, k, v, pos, scale, window=0):
    """(out, bound) of queries q [n, H, D] at positions pos over values k, v [L, kv, D] (float64, NaN allowed).

    The bound, with s a logit and w its weight: q is off by 2^-22 of itself, the product's sum of 2 D
    terms by (D + 8) half steps of sum |q k|, the logit's scaling and the exponential by 8 half steps of max(1, |s|);
    an error e of the logits moves the output by 2 e sum w |v|.  The weights are off by 2^-22, sums of 32 run in
    the instruction and then over a wavefront's blocks (at most a quarter of them) and the parts."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, H, D = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for i in range(n):
        lo = max(0, pos[i] - window + 1) if window else 0
        kk, vv = k[lo:pos[i] + 1], v[lo:pos[i] + 1]
        steps = 32 + len(kk) / BLOCK / 4 + 24
        for h in range(H):
            s = kk[:, h // G] @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv[:, h // G]
            size = np.abs(kk[:, h // G]) @ np.abs(q[i, h]) * abs(scale)
            e = (size * (4 + D + 8) + np.maximum(1, np.abs(s)) * 8) * U32
            spread = w @ np.abs(vv[:, h // G])
            bound[i, h] = (2 * e.max() + (steps + 8) * U32 + 2.0 ** -22) * spread
    return out, bound + 1e-36


def plan(past, new, table, free, used, room):
    """(table, len, start, used, positions, slots, served) of lt_kv_plan."""
    past, new, table = (np.array(a, np.int64) for a in (past, new, table))
    n, width = table.shape
    served, most, at = np.ones(n, bool), used, used
    for i in range(n):
        b0, b1 = -(-past[i] // BLOCK), -(-(past[i] + new[i]) // BLOCK)
        served[i] = b1 <= width and at + b1 - b0 <= len(free)
        for j in range(b0, min(b1, width)):
            table[i, j] = free[at + j - b0] if served[i] else NONE
        at += b1 - b0
        if served[i]:
            most = max(most, at)
    start = np.concatenate([[0], np.cumsum(new)])
    pos, slots = np.zeros(room, np.int64), np.full(room, NONE)
    for i in range(n):
        for j in range(new[i]):
            t = start[i] + j
            if t < room:
                pos[t] = past[i] + j
                b = table[i, pos[t] // BLOCK] if pos[t] // BLOCK < width else NONE
                slots[t] = b * BLOCK + pos[t] % BLOCK if b != NONE else NONE
    u = lambda a: np.asarray(a).astype(np.uint32)  # noqa: E731
    return u(table), u(past + new), u(start), most, u(pos), u(slots), served
