"""Attention cut into parts along the keys, and what a batch that contradicts itself leaves behind: against the
64-bit reference (attn_reference.py)."""
import numpy as np
import pytest

import attn_reference as ref
import llmtoy_amd as lt
from llmtoy_amd.hip import DeviceArray, Graph, check, hip
from llmtoy_amd.lib import DeviceError
from test_gpu_attention import Seqs, _attend, _expect, close, dev, filled, gen, heads, read, same

pytestmark = pytest.mark.gpu

# D, KV, group, tokens before, new tokens: parts in groups of groups, rows that fill a tile and that do not, few and many rows
PARTS = [
    (64, 1, 16, [40000], [1]), (96, 1, 16, [30000], [1]), (128, 1, 16, [30000], [1]), (192, 1, 16, [30000], [1]),
    (256, 1, 16, [30000], [1]), (512, 1, 16, [20000], [1]), (64, 1, 1, [30000], [1]), (192, 1, 11, [20000], [1]),
    (256, 1, 3, [20000], [2]), (512, 1, 5, [20000], [3]), (128, 2, 8, [9000, 100, 5000], [2, 1, 4]),
    (128, 1, 8, [9000], [9]), (512, 1, 8, [5000], [9]), (256, 1, 8, [9000, 30], [5, 20]), (64, 2, 1, [9000], [40]),
    (192, 1, 8, [7000, 9000], [5, 1]),
]


@pytest.mark.parametrize("D,KV,G,past,new", PARTS)
def test_gpu_attention_in_many_parts(ctx, D, KV, G, past, new):
    print(f"parts {D} {KV}x{G} {past} {new}", flush=True)
    g, s, k, v, c, q, total, scale = _attend(ctx, D, KV, G, past, new, 0, seed=3)
    want, bound = _expect(k, v, q, total, new, scale, 0)
    b, qd = s.batch(total, new), dev(q)
    first = None
    for _ in range(4):  # whichever part comes last: the same sums
        out = dev(np.full(q.shape, 5, np.float32))
        ctx.attention(out, qd, c, b, scale)
        ctx.sync()
        got = out.numpy()
        first = got if first is None else first
        assert np.array_equal(got, first)
    close(first, want, bound)
    assert np.linalg.norm(first - want) / np.linalg.norm(want) < 2e-6
    c.free()


# more than 512 rows a sequence, and just as many: whole tiles and pieces of them, windows, odd groups
ROWS = [
    (64, 1, 3, [0], [171], 0), (64, 1, 4, [500], [128], 0), (96, 1, 5, [77], [131], 0), (96, 2, 2, [0, 3], [300, 256], 40),
    (128, 1, 7, [1000], [90], 300), (128, 2, 3, [0], [1500], 0), (192, 1, 4, [90], [150], 0), (192, 1, 9, [0], [60], 17),
    (256, 1, 11, [333], [60], 0), (256, 2, 2, [0, 64], [270, 1], 0), (512, 1, 16, [100], [40], 0), (512, 1, 3, [40], [180], 64),
    (64, 8, 1, [3000], [520], 0), (128, 1, 128, [31], [5], 0), (64, 2, 8, [0] * 12, [70] * 12, 0), (512, 2, 8, [6000], [65], 0),
]


@pytest.mark.parametrize("D,KV,G,past,new,window", ROWS)
def test_gpu_attention_of_many_rows(ctx, D, KV, G, past, new, window):
    print(f"rows {D} {KV}x{G} {past[:3]} {new[:3]} {window}", flush=True)
    g, s, k, v, c, q, total, scale = _attend(ctx, D, KV, G, past, new, window, seed=4)
    want, bound = _expect(k, v, q, total, new, scale, window)
    b, qd = s.batch(total, new, len(q) + 2), dev(np.concatenate([q, q[:2]]))
    first = None
    for _ in range(2):
        out = dev(np.full((len(q) + 2,) + q.shape[1:], 5, np.float32))
        ctx.attention(out, qd, c, b, scale, window)
        ctx.sync()
        got = out.numpy()
        first = got if first is None else first
        assert np.array_equal(got, first)
    close(first[:len(q)], want, bound)
    assert (first[len(q):] == 5).all()
    c.free()


@pytest.mark.parametrize("G,new", [(8, 80), (4, 129)])
def test_gpu_many_rows_see_no_further_than_their_mask(ctx, G, new):
    print(f"many rows: NaN and infinities in and out of sight, nothing in sight but zeros {G} {new}", flush=True)
    D, KV, window = 64, 1, 40
    g, s, k, v, c, q, total, scale = _attend(ctx, D, KV, G, [200], [new], window)
    c.free()
    k[0][5, 0, 3], v[0][40, 0, 2] = np.inf, np.nan  # blocks 0 and 1: out of every window
    v[0][170:240] = 0  # blocks of nothing
    k[0][224:256] = 0
    q[3] = 0
    clean = [x.copy() for x in (k[0], v[0])]
    for x in clean:
        x[:64] = 0
    want, bound = _expect([clean[0]], [clean[1]], q, total, [new], scale, window)
    c = filled(ctx, s, k, v, KV, D)
    out = DeviceArray(q.shape)
    ctx.attention(out, dev(q), c, s.batch(total, [new]), scale, window)
    ctx.sync()
    close(out.numpy(), want, bound)
    want, bound = _expect([clean[0]], [clean[1]], q, total, [new], 0.0, window)  # all keys alike
    ctx.attention(out, dev(q), c, s.batch(total, [new]), 0.0, window)
    ctx.sync()
    close(out.numpy(), want, bound)
    c.free()
    k[0][225, 0, 1] = np.nan  # a block that some see
    c = filled(ctx, s, k, v, KV, D)
    ctx.attention(out, dev(q), c, s.batch(total, [new]), scale, window)
    ctx.sync()
    pos = np.arange(200, 200 + new)
    sees = (pos >= 224) & (pos - window + 1 <= 255)
    got = out.numpy()
    assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()
    c.free()


@pytest.mark.parametrize("G,max_new,news", [(3, 1, [1, 30, 1]), (3, 12, [12, 30, 12]), (30, 20, [20, 30, 20])])
def test_gpu_tokens_beyond_max_new_are_left_alone(ctx, G, max_new, news):
    print(f"tokens beyond max_new {G} {max_new}", flush=True)
    g, s, k, v, c, q, total, scale = _attend(ctx, 64, 1, G, [100] * 3, news, 0)
    want, bound = _expect(k, v, q, total, news, scale, 0)
    out = dev(np.full(q.shape, 5, np.float32))
    ctx.attention(out, dev(q), c, s.batch(total, news, max_new=max_new), scale)
    with pytest.raises(DeviceError, match="sequence 1: the batch contradicts itself"):
        ctx.sync()
    got, at = out.numpy(), news[0]
    assert np.isnan(got[at:at + max_new]).all() and (got[at + max_new:at + news[1]] == 5).all()
    good = np.r_[0:at, at + news[1]:len(q)]
    close(got[good], want[good], bound[good])
    c.free()


@pytest.mark.parametrize("each,past", [(6, 3000), (40, 1000), (160, 1000)])
def test_gpu_overlapping_sequences_do_not_spoil_later_calls(ctx, each, past):
    print(f"overlapping sequences {each} {past}", flush=True)
    G, n = 4, 9
    g, s, k, v, c, q, total, scale = _attend(ctx, 64, 1, G, [past], [each], 0)
    table = np.repeat(s.table, n, 0)
    start = np.array([0, each] * ((n + 1) // 2))
    out = DeviceArray(q.shape)
    bad = lt.KvBatch(dev(start, np.uint32), dev(np.full(n, total[0]), np.uint32), dev(table), each)
    ctx.attention(out, dev(q), c, bad, scale)
    with pytest.raises(DeviceError, match="the batch contradicts itself"):
        ctx.sync()
    want, bound = _expect(k, v, q, total, [each], scale, 0)
    for _ in range(2):
        out = DeviceArray(q.shape)
        ctx.attention(out, dev(q), c, s.batch(total, [each]), scale)
        ctx.sync()
        close(out.numpy(), want, bound)
    c.free()


def test_gpu_two_graphs_share_the_scratch(ctx):
    """Captured calls of different shapes, replayed in turn with eager ones between them on the context's stream."""
    print("two graphs in turn", flush=True)
    runs = []
    for D, KV, G, past, new in ((128, 1, 8, [9000], [1]), (512, 1, 8, [3000, 40], [9, 1]), (64, 2, 4, [7000], [2])):
        g, s, k, v, c, q, total, scale = _attend(ctx, D, KV, G, past, new, 0, seed=5)
        b, qd = s.batch(total, new, max_new=max(new)), dev(q)
        out = DeviceArray(q.shape)
        ctx.attention(out, qd, c, b, scale)
        ctx.sync()
        runs.append((out, qd, c, b, scale, out.numpy()))
        close(runs[-1][5], *_expect(k, v, q, total, new, scale, 0))
    graphs = []
    for out, qd, c, b, scale, _ in runs[:2]:
        def once(out=out, qd=qd, c=c, b=b, scale=scale):
            for _ in range(3):
                ctx.attention(out, qd, c, b, scale)
        graphs.append(Graph(ctx.stream, once))
    for turn in range(4):
        for i, gr in enumerate(graphs):
            zero = np.zeros(runs[i][5].shape, np.float32)
            check(hip().hipMemcpy(runs[i][0].ptr, zero.ctypes.data, zero.nbytes, 1), "hipMemcpy")
            gr.launch()
            out, qd, c, b, scale, want = runs[2]
            ctx.attention(out, qd, c, b, scale)
            ctx.sync()
            assert np.array_equal(runs[i][0].numpy(), runs[i][5]), (turn, i)
            assert np.array_equal(out.numpy(), want), turn
    for gr in graphs:
        gr.destroy()
    for r in runs:
        r[2].free()


@pytest.mark.parametrize("D", [64, 96, 512])
@pytest.mark.parametrize("begin,steps", [(5, [60, 1, 31]), (32, [96, 5]), (31, [65, 40, 1]), (1, [31, 64, 33]), (40, [24, 24, 80])])
def test_gpu_appends_that_end_two_blocks_on(ctx, D, begin, steps):
    """The fp32 tokens of the last two blocks, where a block that goes on and a later one share a place."""
    print(f"append {D} {begin} {steps}", flush=True)
    g, kv = gen(D, begin), 2
    n = begin + sum(steps)
    s = Seqs(g, [n])
    k, v = heads(g, n, kv, D), heads(g, n, kv, D)
    v[n // 2, 0, 3] = 300.0
    c = ctx.kv_cache(s.pool, kv, D, 1)
    at = 0
    for m in [begin] + steps:
        c.append(dev(k[at:at + m]), dev(v[at:at + m]), s.batch([at + m], [m]))
        at += m
        a, b = read(c, s.slots(0, 0, at))
        assert same(a, ref.values(k[:at])) and same(b, ref.values(v[:at])), at
    ctx.sync()
    c.free()


def test_gpu_codes_next_to_a_border(ctx):
    """Values a few steps of fp32 beside the middle of two codes, at scales of every size."""
    print("codes next to a border", flush=True)
    D, g = 64, gen(11)
    blocks = []
    for e in range(-149, 121, 9):
        top = np.float32(np.ldexp(1 + g.random(), e))
        s = np.float32(np.float64(top) / 127)
        mid = ((g.integers(-127, 127, (32, D)) + 0.5) * np.float64(s)).astype(np.float32)
        x = mid
        for _ in range(3):
            x = np.where(g.random(x.shape) < 0.4, np.nextafter(x, np.float32(np.inf) * g.choice([-1, 1], x.shape).astype(np.float32)), x)
        x = np.clip(x, -top, top).astype(np.float32)
        x[0, 0] = top
        blocks.append(x)
    k = np.concatenate(blocks)[:, None]
    s = Seqs(g, [len(k)])
    c = filled(ctx, s, [k], [k[::-1].copy()], 1, D)
    a, b = read(c, s.slots(0, 0, len(k)))
    assert np.array_equal(a, ref.values(k)) and np.array_equal(b, ref.values(k[::-1]))
    c.free()
