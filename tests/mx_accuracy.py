"""What the MXFP4 products keep of fp32 activations, in L2: a bound that a lost part of them
breaks, and numpy models of the two conversions to show that it does."""
import numpy as np


def block_tops(x):
    """The largest |x| of each block of 32, in every element's place."""
    top = np.abs(np.asarray(x, np.float64))
    return top.reshape(top.shape[:-1] + (-1, 32)).max(-1).repeat(32, -1)


def l2_limit(w, x):
    """For w [rows, cols], x [T, cols] with cols <= 2112: what ||y - x w^T|| over a vector's rows
    may be, [T].

    With s_r^2 = sum_i w_ri^2 M_i^2, M the largest of the activation's block.  An activation kept
    to 2^-24 M leaves an error of at most 2^-24 s in the mean over the weights' signs.  The sums
    are one rounding a matrix instruction: at most n = 5 * 2112 / 64 + 64 = 229 of them, each of
    0.41 * 2^-24 of a partial sum in the mean (uniform in half a step, the mantissa's mean 1.4);
    partial sums grow like sqrt(k / n) y, so together 0.41 sqrt(n / 2) 2^-24 |y|, and |y| is s / 2
    in the mean, as the largest of 32 normal numbers is 2.1 times their size.  In all
    sqrt(1 + 2.2^2) 2^-24 s = 2^-22.7 s; 2^-22 leaves half again for a vector's own luck."""
    s2 = block_tops(x) ** 2 @ (np.asarray(w, np.float64) ** 2).T
    return 2.0 ** -22 * np.sqrt(s2.sum(-1))


def within_l2(y, w, x):
    """Each vector's error over its limit, at most 1."""
    y, w, x = (np.asarray(a, np.float64) for a in (y, w, x))
    return np.linalg.norm(y - x @ w.T, axis=-1) / l2_limit(w, x)


def bf16_parts(x, n):
    """The sum of the first n bf16 numbers cut off from the top of x."""
    rest, total = np.asarray(x, np.float32).copy(), np.zeros(np.shape(x))
    for _ in range(n):
        part = (rest.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        total += part
        rest = rest - part
    return total


def fp6_limbs(x, n):
    """The sum of the first n E2M3 limbs of x's blocks of 32."""
    x64 = np.asarray(x, np.float32).astype(np.float64)
    top = block_tops(x64)
    unit = np.exp2(np.floor(np.log2(top)) - 2)
    unit = np.where(top / unit > 7.75, 2 * unit, unit)
    rest, total = x64 / unit, np.zeros(x64.shape)
    for j in (0, 4, 9, 14, 19)[:n]:
        r = rest * 2.0 ** j
        step = np.where(np.abs(r) < 2, 0.125, np.where(np.abs(r) < 4, 0.25, 0.5))
        q = np.clip(np.round(r / step) * step, -7.5, 7.5) * 2.0 ** -j
        total += q
        rest = rest - q
    return total * unit


def low_bits(g, rows, cols, synth_matrix, T):
    """(blocks, x) whose products live in the activations' last bits alone: x = 1 + j 2^-23, and
    the weight of element 16 + i of a block is minus that of element i."""
    m = synth_matrix(rows, cols)
    codes = m.reshape(rows, cols // 32, 17)[..., 1:]
    low = codes & 15
    codes[...] = low | (low ^ 8) << 4
    return m, (1 + g.integers(0, 64, (T, cols)) * 2.0 ** -23).astype(np.float32)


def low_bits_limit(w, x):
    """Sums of exact terms w (x - 1), 5 limbs of at most twice them: cols / 64 * 5 + 64 roundings
    at most.  The leading parts, w times 1, cancel inside each instruction, but a matrix instruction
    aligns the sum so far with the largest of its products and keeps 24 bits of that: those of the
    leading parts, one for each 64 columns, cut up to 2^-23 max |w| each from the sum, as fp32
    additions of these terms would in any order.  (An fp32 sum of the products as they are would
    be held to 2^-24 of sum |w|.)"""
    n = w.shape[1] / 64 * 5 + 64
    aligned = -(-w.shape[1] // 64) * 2.0 ** -23 * np.abs(w).max(1)
    return n * 2.0 ** -24 * 2 * (np.asarray(x, np.float64) - 1) @ np.abs(w).T + aligned
