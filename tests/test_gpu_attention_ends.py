"""What attention's operators do at their ends: many sequences and few tokens, blocks of nothing, tiles that cross a
block of NaN, full rows of a table, sequences in another row, reports; against the 64-bit reference
(attn_reference.py)."""
import numpy as np
import pytest

import attn_reference as ref
import llmtoy_amd as lt
from llmtoy_amd import ggml
from llmtoy_amd.hip import DeviceArray, Graph
from llmtoy_amd.lib import DeviceError, rmsnorm
from test_gpu_attention import Seqs, _attend, _expect, close, dev, filled, gen, heads, read, same, u32

pytestmark = pytest.mark.gpu


# sequences of a batch, those with tokens in it, tokens before, max_new (0: not known)
FEW_OF_MANY = [(2000, [1] * 16, 90, 128), (1025, [1], 40, 4096), (2000, [3, 1], 33, 0), (4096, [1] * 5, 20, 1 << 24),
               (1500, [100, 1, 1], 50, 100), (1500, [100, 1, 70], 50, 0)]


@pytest.mark.parametrize("n,new,past,max_new", FEW_OF_MANY)
def test_gpu_few_tokens_of_many_sequences(ctx, n, new, past, max_new):
    """More sequences than the many-row kernel cuts in pieces for, and fewer rows than a tile of it."""
    print(f"few of many {n} {new} {past} {max_new}", flush=True)
    D, KV, G = 128, 1, 8
    g = gen(n, len(new), 21)
    rows = np.sort(g.permutation(n)[:len(new)])
    total, adds = np.zeros(n, int), np.zeros(n, int)
    total[rows], adds[rows] = past + np.array(new), new
    s = Seqs(g, total)
    k, v = ([heads(g, m, KV, D) for m in total] for _ in range(2))
    c = filled(ctx, s, k, v, KV, D)
    q = g.standard_normal((sum(new), KV * G, D)).astype(np.float32)
    want, bound = _expect(k, v, q, total, adds, D ** -0.5, 0)
    out = dev(np.full(q.shape, 5, np.float32))
    ctx.attention(out, dev(q), c, s.batch(total, adds, max_new=max_new), D ** -0.5)
    ctx.sync()
    close(out.numpy(), want, bound)
    c.free()


@pytest.mark.parametrize("D,new", [(64, 1), (64, 90), (512, 2), (128, 80)])
@pytest.mark.parametrize("size,lift", [(1e-6, 0.0), (1e-8, 0.0), (1e-10, 0.0), (1.0, 15.0), (1.0, 40.0), (1e-6, 15.0)])
def test_gpu_attention_beside_a_block_of_nothing(ctx, D, new, size, lift):
    """A block whose values are all zero beside others of `size`; its logits higher than theirs by about `lift`."""
    print(f"block of nothing {D} {new} {size} {lift}", flush=True)
    KV, G, past, scale = 1, 8, 600, D ** -0.5  # (past: two blocks and more a wavefront)
    g = gen(D, new, int(lift), 22)
    n = past + new
    s = Seqs(g, [n])
    k, v, q = heads(g, n, KV, D), size * heads(g, n, KV, D), 0.3 * g.standard_normal((new, KV * G, D)).astype(np.float32)
    way = np.ones(D, np.float32)  # (every query has sqrt(D) of it)
    q += way
    k[32:64] += lift / (D * scale) * way
    v[32:64] = 0
    v = v.astype(np.float32)
    c = filled(ctx, s, [k], [v], KV, D)
    want, bound = _expect([k], [v], q, [n], [new], scale, 0)
    out = DeviceArray(q.shape)
    ctx.attention(out, dev(q), c, s.batch([n], [new]), scale)
    ctx.sync()
    close(out.numpy(), want, bound)
    # nothing but such blocks in sight
    w = np.zeros_like(v)
    w[:32] = v[:32]
    c.append(dev(k), dev(w), s.batch([n], [n]))
    want, bound = _expect([k], [w], q, [n], [new], scale, 0)
    ctx.attention(out, dev(q), c, s.batch([n], [new]), scale)
    ctx.sync()
    close(out.numpy(), want, bound)
    ctx.attention(out, dev(q), c, s.batch([n], [new]), scale, 64)
    ctx.sync()
    assert (out.numpy() == 0).all()
    c.free()


@pytest.mark.parametrize("D,G,past,new,window", [
    (64, 4, 222, 4, 40), (64, 4, 229, 4, 40), (64, 4, 478, 4, 0), (128, 8, 479, 2, 0), (512, 4, 478, 4, 0), (64, 4, 521, 4, 300),
    (64, 4, 198, 130, 40), (128, 8, 221, 70, 40), (512, 8, 222, 66, 40), (128, 8, 221, 70, 0)])
@pytest.mark.parametrize("what", ["keys", "values", "lost"])
def test_gpu_rows_of_a_tile_before_a_block_of_nan(ctx, D, G, past, new, window, what):
    """Rows that do not see a block which others of their tile see: it changes nothing for them."""
    print(f"block of NaN {D} {G} {past} {new} {window} {what}", flush=True)
    KV, n, scale = 1, past + new, D ** -0.5
    g, s, k, v, c, q, total, _ = _attend(ctx, D, KV, G, [past], [new], window, seed=23)
    pos = np.arange(past, n)
    c.free()
    for block in {b for b in (past // 32, past // 32 + 1, (past - window + 2) // 32 if window else 0) if b * 32 < n}:
        sees = (pos >= block * 32) & (pos - (window or n) + 1 < block * 32 + 32)
        k1, v1, table = k[0].copy(), v[0].copy(), s.table
        if what == "keys":
            k1[block * 32, 0, 3] = np.nan
        elif what == "values":
            v1[block * 32, 0, 3] = np.inf
        c = filled(ctx, s, [k1], [v1], KV, D)
        if what == "lost":
            s.table = table.copy()
            s.table[0, block] = ref.NONE
        want, bound = _expect(k, v, q, total, [new], scale, window)
        out = DeviceArray(q.shape)
        ctx.attention(out, dev(q), c, s.batch(total, [new]), scale, window)
        if what == "lost" and sees.any():
            with pytest.raises(DeviceError, match="sequence 0: the table has no block"):
                ctx.sync()
        ctx.sync()
        s.table = table
        got = out.numpy()
        assert np.isnan(got[sees]).all()
        close(got[~sees], want[~sees], bound[~sees])
        c.free()


def plan(past, new, table, free, used):
    """(table, used) of lt_kv_plan where every length fits 32 bits: a sequence whose row is full takes no blocks; from
    one that the list is too short for on, none does."""
    table, at, short = np.array(table, np.int64), used, False
    for i in range(len(past)):
        b0, b1 = -(-int(past[i]) // 32), -(-int(past[i] + new[i]) // 32)
        full = b1 > table.shape[1]
        if not full and b1 > b0:
            short |= at + b1 - b0 > len(free)
        take = not full and not short
        for j in range(b0, min(b1, table.shape[1])):
            table[i, j] = free[at + j - b0] if take else ref.NONE
        at += b1 - b0 if take else 0
    return u32(table), at


@pytest.mark.parametrize("n,width,most", [(3, 4, 40), (9, 4, 70), (200, 6, 100), (1500, 5, 60)])
@pytest.mark.parametrize("short", [False, True])
def test_gpu_plan_with_full_rows_among_others(ctx, n, width, most, short):
    print(f"plan with full rows {n} {width} {most} {short}", flush=True)
    g = gen(n, width, short, 24)
    past = g.integers(0, width * 32 + 1, n)
    new = g.integers(0, most, n)
    past[0], new[0] = width * 32, 33
    new[1] = 1 << 30  # far beyond any row
    past[2], new[2] = 31, 2
    held, after = -(-past // 32), -(-(past + new) // 32)
    order = g.permutation(int(held.sum() + after[after <= width].sum()) + 9)
    table = np.full((n, width), ref.NONE, np.int64)
    for i in range(n):
        table[i, :held[i]] = order[held[:i].sum():held[:i + 1].sum()]
    need = int((after - held)[after <= width].sum())
    free = order[held.sum():held.sum() + (need * 2 // 3 if short else need + 3) + 2]
    tokens = new.copy()
    tokens[1] = 0
    want, used = plan(past, tokens, table, free, 2)
    if not short:
        assert used == 2 + need
    room = int(new[0]) + 70  # (the second sequence has all of the others' room)
    b = lt.KvBatch(DeviceArray((n + 1,), np.uint32), DeviceArray((n,), np.uint32), dev(table, np.uint32), room)
    us, pos, sl = DeviceArray((1,), np.uint32), DeviceArray((room,), np.uint32), DeviceArray((room,), np.uint32)
    ctx.kv_plan(b, dev(past, np.uint32), dev(new, np.uint32), dev(free, np.uint32), dev([2], np.uint32), us, pos, sl)
    with pytest.raises(DeviceError, match="plan"):
        ctx.sync()
    got = b.table.numpy()
    # (the second sequence's: those before its full row are none)
    for j in range(held[1], width):
        want[1, j] = ref.NONE
    assert np.array_equal(got, want) and us.numpy()[0] == used
    fresh = (got != u32(table)) & (got != ref.NONE)
    assert fresh.sum() == used - 2  # what counts as taken is in a table
    assert (sl.numpy()[:new[0]] == ref.NONE).all()


@pytest.mark.parametrize("n,most", [(5, 3), (300, 40)])
def test_gpu_plan_again_and_again_loses_no_block(ctx, n, most):
    """A replayed plan beside a sequence whose row is full: every block that counts as taken is in a table."""
    print(f"plan replayed beside a full row {n} {most}", flush=True)
    g = gen(n, 25)
    width, steps = 6, 12
    past = u32(g.integers(0, 20, n))
    past[1] = width * 32 - 1
    new = u32(g.integers(1, most + 1, n))
    new[1] = 20  # (full from the first step on)
    free = u32(g.permutation(n * width * 2))
    room = int(new.sum())
    table = np.full((n, width), ref.NONE, np.uint32)
    for i in range(n):
        h = -(-int(past[i]) // 32)
        table[i, :h] = 100000 + 10 * i + np.arange(h)
    ln, used = dev(past), dev(u32([0]))
    b = lt.KvBatch(DeviceArray((n + 1,), np.uint32), ln, dev(table), room)
    pos, slots, nd, fd = DeviceArray((room,), np.uint32), DeviceArray((room,), np.uint32), dev(new), dev(free)
    graph = Graph(ctx.stream, lambda: ctx.kv_plan(b, ln, nd, fd, used, used, pos, slots))
    at = past.astype(int)
    for _ in range(steps):
        graph.launch()
        with pytest.raises(DeviceError, match="no room in the table's row"):
            ctx.sync()
        at = at + new
        fresh = b.table.numpy()
        fresh = fresh[(fresh != ref.NONE) & (fresh < 100000)]
        assert used.numpy()[0] == len(fresh) == len(set(fresh.tolist()))
        assert np.array_equal(ln.numpy(), at)
    graph.destroy()


def test_gpu_a_sequence_in_another_row(ctx):
    """The open block's tokens are the row's: a sequence that goes on in another row is told, and never gets the tokens
    of the row's last sequence; at a block's border it may move."""
    print("append: a sequence in another row", flush=True)
    g, kv, D = gen(26), 2, 64
    for case in ("same index", "same block", "both"):
        total = [40, 36, 64]
        s = Seqs(g, total)
        k = [heads(g, n, kv, D) for n in total]
        spare = next(p for p in range(s.pool) if p not in s.table)
        c = ctx.kv_cache(s.pool, kv, D, 3)
        if case == "same block":  # the first sequence ends, and its last block becomes the second one's
            first = s.table[0].copy()
            c.append(dev(k[0]), dev(k[0]), s.batch([40, 0, 0], [40, 0, 0]))
            s.table[1, 1] = first[1]
            c.append(dev(np.concatenate(k[1:])), dev(np.concatenate(k[1:])), s.batch([40, 36, 64], [0, 36, 64]))
        else:
            c.append(dev(np.concatenate(k)), dev(np.concatenate(k)), s.batch(total, total))
        if case == "both":  # the other way round too: two sequences change places
            s.table[[0, 1]] = s.table[[1, 0]]
            one = heads(g, 2, kv, D)
            c.append(dev(one), dev(one), s.batch([37, 41, 64], [1, 1, 0]))
            rows = [(0, 37), (1, 41)]
        else:
            s.table[0] = s.table[1]
            one = heads(g, 1, kv, D)
            c.append(dev(one), dev(one), s.batch([37, 0, 64], [1, 0, 0]))
            rows = [(0, 37)]
        with pytest.raises(DeviceError, match="append: the block's earlier tokens are not held"):
            ctx.sync()
        for i, n in rows:
            a, b = read(c, s.slots(i, 32, n))
            assert np.isnan(a).all() and np.isnan(b).all()
            assert np.isfinite(read(c, s.slots(i, 0, 32))[0]).all()
        # a whole block: no tokens from before are needed
        s.table[1] = s.table[2]
        s.table[1, 2] = spare
        more = heads(g, 3, kv, D)
        c.append(dev(more), dev(more), s.batch([0, 67, 64], [0, 3, 0]))
        c.append(dev(more[:1]), dev(more[:1]), s.batch([0, 68, 64], [0, 1, 0]))
        ctx.sync()
        assert same(read(c, s.slots(1, 0, 68))[0], ref.values(np.concatenate([k[2], more, more[:1]])))
        c.free()


@pytest.mark.parametrize("new", [1, 70])
def test_gpu_rows_and_blocks_used_again(ctx, new):
    """Rows and blocks of sequences that ended, for others: nothing is left of the former."""
    print(f"append: rows and blocks used again {new}", flush=True)
    g, kv, D, n = gen(27, new), 2, 96, 3
    s = Seqs(g, [160] * n, extra=0)
    c = ctx.kv_cache(s.pool, kv, D, n)
    order = s.table.copy()
    for turn in range(4):
        s.table = order[np.roll(np.arange(n), turn)]  # each row gets the blocks that another had
        at, k = np.zeros(n, int), [heads(g, 160, kv, D) for _ in range(n)]
        stop = np.array([47, 90, 160]) - turn
        while (at < stop).any():
            m = np.minimum([new, 1 + new // 2, 33], stop - at)
            x = np.concatenate([k[i][at[i]:at[i] + m[i]] for i in range(n)])
            at += m
            c.append(dev(x), dev(x), s.batch(at, m))
        ctx.sync()
        for i in range(n):
            a, b = read(c, s.slots(i, 0, stop[i]))
            assert same(a, ref.values(k[i][:stop[i]])) and same(b, a), (turn, i)
    c.free()


def test_gpu_a_block_begun_anew_in_the_same_row(ctx):
    """The tokens of a row's last sequence are not held any more once their block is begun anew, even where the new
    sequence's last block has no place."""
    print("append: a block begun anew in its row", flush=True)
    g, kv, D = gen(33), 2, 64
    s = Seqs(g, [96])
    old, new = heads(g, 20, kv, D), heads(g, 71, kv, D)
    c = ctx.kv_cache(s.pool, kv, D, 1)
    c.append(dev(old), dev(old), s.batch([20], [20]))
    good, s.table = s.table, s.table.copy()
    s.table[0, 2] = ref.NONE
    c.append(dev(new[:70]), dev(new[:70]), s.batch([70], [70]))
    with pytest.raises(DeviceError, match="sequence 0: the table has no block"):
        ctx.sync()
    s.table = good
    assert same(read(c, s.slots(0, 0, 64))[0], ref.values(new[:64]))
    c.append(dev(new[20:21]), dev(new[20:21]), s.batch([21], [1]))
    with pytest.raises(DeviceError, match="sequence 0: append: the block's earlier tokens are not held"):
        ctx.sync()
    assert np.isnan(read(c, s.slots(0, 0, 21))[0]).all()
    c.append(dev(new), dev(new), s.batch([71], [71]))
    ctx.sync()
    assert same(read(c, s.slots(0, 0, 71))[0], ref.values(new))
    c.free()


@pytest.mark.parametrize("D", [64, 192])
@pytest.mark.parametrize("wrong,tokens", [(10, 3), (10, 40), (1, 90)])
def test_gpu_a_refused_append_spoils_no_held_tokens(ctx, D, wrong, tokens):
    """A length set back too far is told; set right, the sequence goes on with the tokens that it held."""
    print(f"append: set back too far {D} {wrong} {tokens}", flush=True)
    g, kv, n = gen(28, D, tokens), 2, 64 + 20
    s = Seqs(g, [n + 10])
    k = heads(g, n + 10, kv, D)
    c = ctx.kv_cache(s.pool, kv, D, 1)
    c.append(dev(k[:n]), dev(k[:n]), s.batch([n], [n]))
    if tokens == 3:
        x = heads(g, tokens, kv, D)
        c.append(dev(x), dev(x), s.batch([wrong + tokens], [tokens]))
        with pytest.raises(DeviceError, match="sequence 0: append: the block's earlier tokens are not held"):
            ctx.sync()
        c.append(dev(k[n:n + 1]), dev(k[n:n + 1]), s.batch([n + 1], [1]))
        ctx.sync()
        assert same(read(c, s.slots(0, 64, n + 1))[0], ref.values(k[64:n + 1]))
    else:  # later blocks were begun anew: those are held
        x = heads(g, tokens, kv, D)
        c.append(dev(x), dev(x), s.batch([wrong + tokens], [tokens]))
        with pytest.raises(DeviceError, match="sequence 0: append: the block's earlier tokens are not held"):
            ctx.sync()
        end = wrong + tokens
        more = heads(g, 2, kv, D)
        c.append(dev(more), dev(more), s.batch([end + 2], [2]))
        ctx.sync()
        a, _ = read(c, s.slots(0, 0, end + 2))
        assert np.isnan(a[:32]).all()
        assert same(a[32:], ref.values(np.concatenate([x[32 - wrong:], more])))
    c.free()


def test_gpu_a_block_that_is_not_there_leaves_the_held_tokens(ctx):
    print("append: no block for a token, then one", flush=True)
    g, kv, D = gen(29), 1, 128
    s = Seqs(g, [70])
    k = heads(g, 70, kv, D)
    c = ctx.kv_cache(s.pool, kv, D, 1)
    c.append(dev(k[:60]), dev(k[:60]), s.batch([60], [60]))
    good, s.table = s.table, s.table.copy()
    s.table[0, 1] = ref.NONE
    x = heads(g, 1, kv, D)
    c.append(dev(x), dev(x), s.batch([61], [1]))
    with pytest.raises(DeviceError, match="sequence 0: the table has no block"):
        ctx.sync()
    s.table = good
    c.append(dev(k[60:]), dev(k[60:]), s.batch([70], [10]))
    ctx.sync()
    assert same(read(c, s.slots(0, 0, 70))[0], ref.values(k))
    c.free()


@pytest.mark.parametrize("n,each", [(2, 3), (70, 2), (3, 200)])
def test_gpu_sequences_wholly_behind_the_batch_are_told(ctx, n, each):
    print(f"sequences behind n_tokens {n} {each}", flush=True)
    D, KV, G = 64, 1, 4
    g, s, k, v, c, q, total, scale = _attend(ctx, D, KV, G, [40] * n, [each] * n, 0, seed=30)
    room = each * (n - 1)  # the last one has no place
    want, bound = _expect(k, v, q, total, [each] * n, scale, 0)
    b = s.batch(total, [each] * n, room=room)
    c.free()
    c = ctx.kv_cache(s.pool, KV, D, n)
    first = [np.concatenate([x[:40] for x in a]) for a in (k, v)]
    c.append(dev(first[0]), dev(first[1]), s.batch([40] * n, [40] * n))
    c.append(dev(np.concatenate([x[40:] for x in k])[:room]), dev(np.concatenate([x[40:] for x in v])[:room]), b)
    with pytest.raises(DeviceError, match=f"sequence {n - 1}: the batch contradicts itself"):
        ctx.sync()
    out = DeviceArray((room, *q.shape[1:]))
    ctx.attention(out, dev(q[:room]), c, b, scale)
    with pytest.raises(DeviceError, match=f"sequence {n - 1}: the batch contradicts itself"):
        ctx.sync()
    close(out.numpy(), want[:room], bound[:room])
    # an idle one behind is nobody's fault
    start = np.minimum(np.arange(n + 1) * each, room)
    idle = lt.KvBatch(dev(start, np.uint32), dev(total, np.uint32), dev(s.table), room)
    ctx.attention(out, dev(q[:room]), c, idle, scale)
    ctx.sync()
    close(out.numpy(), want[:room], bound[:room])
    c.free()


def _short_plan(c):
    """A plan that finds no block (device arrays: nothing is told yet)."""
    z = lambda *s: dev(np.zeros(s), np.uint32)  # noqa: E731
    c.kv_plan(lt.KvBatch(z(2), z(1), z(1, 2), 1), z(1), dev([1], np.uint32), z(0), z(1), z(1), z(1), z(1))


def test_gpu_every_synchronising_call_tells(ctx):
    """What was found wrong on the device comes with the next lt_sync or LT_HOST_IO call, whichever that is, once, and the
    call's own results are there."""
    print("reports of host calls", flush=True)
    g = gen(31)
    D = 256
    w = g.standard_normal((D, D)).astype(np.float32)
    x = g.standard_normal(D).astype(np.float32)
    t = ctx.upload(w, ggml.F32, D, D)
    mx = ctx.create(ggml.MXFP4, 4, D)
    y = np.zeros(D, np.float32)
    rope = ctx.rope(64)
    h, pos = g.standard_normal((3, 2, 64)).astype(np.float32), np.zeros(3, np.uint32)
    calls = {
        "matvec": lambda: ctx.quant_matvec(y, t, x),
        "rmsnorm": lambda: rmsnorm(ctx, y[None], x[None]),
        "quantize": lambda: ctx.quantize(mx, np.zeros((4, D), np.float32)),
        "rotation": lambda: ctx.qk_norm_rope(np.zeros_like(h), None, h, None, None, None, pos, rope),
        "sync": ctx.sync,
    }
    for name, call in calls.items():
        _short_plan(ctx)
        y[:] = 0
        with pytest.raises(DeviceError, match="sequence 0: plan: no blocks left"):
            call()
        call()  # (told once)
        if name == "matvec":
            assert np.linalg.norm(y - w @ x) < 1e-4 * np.linalg.norm(y)
    ctx.sync()
    for a in (t, mx, rope):
        a.free()


def test_gpu_two_kinds_of_reports_at_once(ctx, monkeypatch):
    print("a wait that ran out and a plan that found no blocks", flush=True)
    from test_gpu_mxfp4_layer import layer
    g = gen(32)
    E, D, F, k = 128, 2048, 768, 8
    x = g.standard_normal(D).astype(np.float32)
    monkeypatch.setenv("LT_MX_WAIT_TICKS", "0")
    with lt.Context(0) as c:
        ts = layer(c, g, E, D, F)
        out, ids, w = DeviceArray((D,)), DeviceArray((k,), np.uint32), DeviceArray((k,))
        with pytest.raises(DeviceError, match="wait timed out"):  # (the hand-over memory's first call)
            c.moe_forward(np.zeros(D, np.float32), x, *ts, k, F)
        c.moe_forward(out, dev(x), *ts, k, F, out_ids=ids, out_w=w)
        _short_plan(c)
        with pytest.raises(DeviceError, match="(?s)wait timed out.*sequence 0: plan: no blocks left"):
            c.sync()
        c.sync()
        # an attention call on host arrays tells of a layer's wait too
        c.moe_forward(out, dev(x), *ts, k, F, out_ids=ids, out_w=w)
        rope = c.rope(64)
        h = g.standard_normal((1, 2, 64)).astype(np.float32)
        with pytest.raises(DeviceError, match="wait timed out"):
            c.qk_norm_rope(np.zeros_like(h), None, h, None, None, None, np.zeros(1, np.uint32), rope)
        c.sync()
        for t in (*ts, rope):
            t.free()


@pytest.mark.parametrize("D,KV,G,window,seed", [(64, 2, 2, 0, 1), (128, 1, 4, 50, 2), (64, 1, 8, 0, 3)])
def test_gpu_serving_with_rows_and_blocks_used_again(ctx, D, KV, G, window, seed):
    """Sequences that come, go on by tokens and by parts of prompts, are taken back and end, over a small pool: plan,
    append and attention at every step, the cache bit for bit and the outputs against 64 bits."""
    print(f"serving {D} {KV}x{G} {window} {seed}", flush=True)
    g = gen(D, seed, 34)
    n, width, pool, steps = 6, 5, 22, 60
    c = ctx.kv_cache(pool, KV, D, n)
    table = np.full((n, width), ref.NONE, np.uint32)
    free = list(g.permutation(pool))
    k, v = ([np.zeros((0, KV, D), np.float32) for _ in range(n)] for _ in range(2))
    held = [[None, None] for _ in range(n)]  # the blocks whose tokens a row has in fp32, by their parity

    def cut(i, length):
        """Sequence i keeps `length` tokens; blocks behind them go back."""
        keep = -(-length // 32)
        free.extend(int(b) for b in table[i, keep:] if b != ref.NONE)
        table[i, keep:] = ref.NONE
        k[i], v[i] = k[i][:length], v[i][:length]

    for step in range(steps):
        new = np.zeros(n, int)
        for i in range(n):
            what = g.random()
            if what < 0.06:
                cut(i, 0)
                held[i] = [None, None]
            elif what < 0.2 and len(k[i]):
                to = len(k[i]) - int(g.integers(1, min(32, len(k[i])) + 1))
                if to % 32 == 0 or held[i][to // 32 % 2] == to // 32:
                    cut(i, to)
            new[i] = int(g.choice([0, 1, 1, 1, 2, 3, 33, 70])) if len(k[i]) else int(g.integers(0, 70))
            new[i] = min(new[i], width * 32 - len(k[i]))
        past = np.array([len(x) for x in k])
        need = -(-(past + new) // 32) - -(-past // 32)
        for i in range(n):
            if need[:i + 1].sum() > len(free):
                new[i] = need[i] = 0
        free = [int(b) for b in g.permutation(free)]
        T = int(new.sum())
        room = T + 2
        b = lt.KvBatch(DeviceArray((n + 1,), np.uint32), DeviceArray((n,), np.uint32), dev(table), room, int(new.max()))
        used, pos, slots = dev([0], np.uint32), DeviceArray((room,), np.uint32), DeviceArray((room,), np.uint32)
        ctx.kv_plan(b, dev(past, np.uint32), dev(new, np.uint32), dev(free, np.uint32), used, used, pos, slots)
        x, y = heads(g, room, KV, D), heads(g, room, KV, D)
        q = g.standard_normal((room, KV * G, D)).astype(np.float32)
        out = dev(np.full(q.shape, 5, np.float32))
        c.append(dev(x), dev(y), b)
        ctx.attention(out, dev(q), c, b, D ** -0.5, window)
        ctx.sync()
        table = b.table.numpy()
        free = free[int(used.numpy()[0]):]
        t, got = 0, out.numpy()
        for i in range(n):
            k[i], v[i] = (np.concatenate([o, e[t:t + new[i]]]) for o, e in ((k[i], x), (v[i], y)))
            if new[i]:
                for j in range(max(past[i] // 32, (len(k[i]) - 1) // 32 - 1), (len(k[i]) - 1) // 32 + 1):
                    held[i][j % 2] = j
                at = np.arange(len(k[i]))
                a, w = read(c, u32(table[i, at // 32].astype(np.int64) * 32 + at % 32))
                assert same(a, ref.values(k[i])) and same(w, ref.values(v[i])), (step, i)
                close(got[t:t + new[i]], *ref.attention(q[t:t + new[i]], a, w, np.arange(past[i], len(k[i])), D ** -0.5, window))
            t += new[i]
        assert (got[T:] == 5).all()
        taken = table[table != ref.NONE]
        assert len(set(taken.tolist())) == len(taken) and len(taken) + len(free) == pool
    c.free()
