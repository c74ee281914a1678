"""MXFP4 in 64 bits with numpy: the format's definition, its quantisation, and
the error bounds that the device's products are held to."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def decode(blocks, cols):
    """float64 [..., cols] of MXFP4 block bytes [..., cols / 32 * 17]."""
    b = np.asarray(blocks, np.uint8).reshape(-1, cols // 32, 17)
    q = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    v = np.where(q & 8, -1.0, 1.0) * MAGNITUDES[q & 7]
    e = b[..., :1].astype(np.int64)
    v = np.where(e == 255, np.nan, np.ldexp(v, (e - 127).astype(np.int32)))
    return v.reshape(np.asarray(blocks).shape[:-1] + (cols,))


def quantize(x):
    """uint8 blocks of float32 rows [..., cols]."""
    x = np.asarray(x, np.float32)
    v = x.astype(np.float64).reshape(-1, 32)
    a = np.abs(v)
    top = a.max(-1, keepdims=True)
    bad = ~np.isfinite(v).all(-1, keepdims=True)
    safe = np.where(bad | (top == 0), 1.0, top)
    e = np.clip(np.frexp(safe)[1] - 1 - 2, -127, 127)
    e = np.where(top == 0, -127, e)
    m = np.where(bad, 0.0, a) / np.ldexp(1.0, e)
    code = np.zeros(v.shape, np.uint8)
    for i in range(7):
        middle = (MAGNITUDES[i] + MAGNITUDES[i + 1]) / 2
        code += (m >= middle) if i % 2 else (m > middle)
    code = np.where(bad, 0, code | np.where(np.signbit(v), 8, 0)).astype(np.uint8)
    out = np.empty((v.shape[0], 17), np.uint8)
    out[:, 0] = np.where(bad[:, 0], 255, e[:, 0] + 127)
    out[:, 1:] = code[:, :16] | code[:, 16:] << 4
    return out.reshape(x.shape[:-1] + (x.shape[-1] // 32 * 17,))


def product(w, x):
    """(x w^T, bound) for w [rows, cols], x [..., cols] in float64.

    The bound.  Every activation is exact to 2^-24 of its block's largest.  A
    matrix instruction adds 128 exact products to its sum with an error of at
    most 2^-20 of the largest of them (128 terms cut at 2^-27), and there is
    one for each 128 columns and limb; the results' additions (groups of 128,
    limbs, waves, lanes: fewer than cols / 128 * 5 + 64) round by 2^-24 of
    what has been summed.  Both are against sum |w| max|x of the block|, times
    2 for the limbs' magnitudes, which add up to at most 1.07 of a block's
    largest value."""
    w, x = np.asarray(w, np.float64), np.asarray(x, np.float64)
    n = x.shape[-1]  # (a last block in part: zeros behind it)
    top = np.pad(np.abs(x), [(0, 0)] * (x.ndim - 1) + [(0, -n % 32)])
    top = top.reshape(x.shape[:-1] + (-1, 32)).max(-1).repeat(32, -1)[..., :n]
    scale = top @ np.abs(w).T
    return x @ w.T, 2 * scale * (2.0 ** -20 + (w.shape[1] / 128 * 5 + 64) * 2.0 ** -24)


def act(kind, g):
    if kind == 0:
        return g / (1 + np.exp(-g))
    return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))


def gated(gate, up, x, kind):
    """(act(gate x) * (up x), bound).  Both activations change by at most 1.13
    times their argument's change; exp, tanh, the division and the products
    round to about 4 ulp each, relative to g (the gelu's 1 + tanh may cancel)."""
    g, dg = product(gate, x)
    u, du = product(up, x)
    h = act(kind, g) * u
    return h, 1.13 * dg * (np.abs(u) + du) + np.abs(g) * du + 2.0 ** -20 * np.abs(g * u)


def down(w, h, dh):
    """(h w^T, bound) for h known to within dh."""
    y, dy = product(w, h)
    return y, dy * (1 + 2.0 ** -10) + dh @ np.abs(np.asarray(w, np.float64)).T * (1 + 2.0 ** -10)
