"""The MXFP4 operators on the GPU against 64-bit references (mx_reference.py):
quantisation byte for byte, products within bounds derived there."""
import numpy as np
import pytest

import llmtoy_amd as lt
import mx_reference as mx
from llmtoy_amd import ggml, synth
from llmtoy_amd import lib as ltlib
from llmtoy_amd.hip import DeviceArray, DeviceView, Graph

pytestmark = pytest.mark.gpu

MX = ggml.MXFP4


def gen(*seed):
    return np.random.default_rng([77, *seed])


def acts(g, *shape):
    """Normal values with a few channels ten times larger."""
    x = g.standard_normal(shape).astype(np.float32)
    x[..., g.random(shape[-1]) < 0.01] *= 10
    return x


def close(got, ref, bound):
    err = np.abs(np.asarray(got, np.float64) - ref)
    assert np.isfinite(got).all()
    worst = float((err / bound).max())
    assert worst <= 1.0, worst


# ------------------------------------------------------------------ tensors
@pytest.mark.parametrize("rows,cols,E", [(1, 32, 1), (17, 160, 1), (16, 512, 1), (5, 96, 3), (40, 544, 7), (3, 16384, 2)])
def test_gpu_mx_upload_read_clone(ctx, rows, cols, E):
    print(f"upload {rows}x{cols} x{E}", flush=True)
    m = gen(rows, cols, E).integers(0, 256, (E * rows, cols // 32 * 17), dtype=np.uint8)
    t = ctx.upload(m, MX, rows, cols, E)
    c = t.clone()
    assert t.nbytes == m.size
    t.free()
    assert np.array_equal(c.read(), m.reshape(-1))
    c.free()


def test_gpu_mx_upload_of_many_pieces(ctx):
    m = gen(1).integers(0, 256, (9000, 2816 // 32 * 17), dtype=np.uint8)  # over 8 pieces of 4 MiB
    t = ctx.upload(m, MX, 900, 2816, 10)
    assert np.array_equal(t.read(), m.reshape(-1))
    t.free()


SPECIAL = np.zeros((12, 32), np.float32)
SPECIAL[0, :8] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5]
SPECIAL[1, :8] = [-7.9, 6.1, 5.0000005, 4.9999995, -.25, -.2500001, 0.2, -0.0]
SPECIAL[2] = 3.4e38
SPECIAL[3, :4] = [1e-45, -3e-45, 1e-40, 2e-39]
SPECIAL[4, :4] = [2 ** -125, 2 ** -126, -2 ** -127, 2 ** -128]
SPECIAL[5, 31] = np.inf
SPECIAL[6, 0] = np.nan
SPECIAL[7, 16] = -np.inf
SPECIAL[8] = np.float32(1) + np.arange(32, dtype=np.float32) * 2 ** -23
SPECIAL[9, 5] = -2 ** -149
SPECIAL[10] = np.linspace(-6, 6, 32)


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 2816), (5, 96), (16, 128), (17, 160), (33, 4096), (300, 32), (20, 1056)])
@pytest.mark.parametrize("scale", [1.0, 3e-39, 1e36])
def test_gpu_mx_quantize(ctx, rows, cols, scale):
    print(f"quantize {rows}x{cols} scale {scale}", flush=True)
    x = acts(gen(rows, cols), rows, cols) * np.float32(scale)
    t = ctx.create(MX, rows, cols)
    ctx.quantize(t, x)
    want = mx.quantize(x)
    assert np.array_equal(t.read(), want.reshape(-1))
    out = np.empty_like(x)
    ctx.dequantize(out, t)
    assert np.array_equal(out, mx.decode(want, cols).astype(np.float32))
    t.free()


def test_gpu_mx_quantize_special_values(ctx):
    x = SPECIAL.reshape(4, 96)
    t = ctx.create(MX, 4, 96)
    ctx.quantize(t, x)
    want = mx.quantize(x)
    assert np.array_equal(t.read().reshape(-1, 17), want.reshape(-1, 17))
    out = np.empty_like(x)
    ctx.dequantize(out, t)
    assert np.array_equal(out, mx.decode(want, 96).astype(np.float32), equal_nan=True)
    t.free()


def test_gpu_mx_dequantize_every_scale_and_code(ctx):
    b = np.zeros((256, 17), np.uint8)
    b[:, 0] = np.arange(256)
    b[:, 1:] = np.arange(16) | (15 - np.arange(16)) << 4
    t = ctx.upload(b, MX, 256, 32)
    out = np.empty((256, 32), np.float32)
    ctx.dequantize(out, t)
    with np.errstate(over="ignore"):
        want = mx.decode(b, 32).astype(np.float32)  # 6 * 2^127 is beyond fp32
    assert np.array_equal(out, want, equal_nan=True)
    t.free()


def test_gpu_mx_rows_in_part(ctx):
    # rows 3..7 of three experts of 10: the others as they were
    g = gen(2)
    m = synth.quant_matrix(g, MX, 30, 96)
    t = ctx.upload(m, MX, 10, 96, 3)
    x = acts(g, 15, 96)
    ctx.quantize(t, x, row0=8)  # across the first expert's end
    want = m.copy()
    want[8:23] = mx.quantize(x)
    assert np.array_equal(t.read(), want.reshape(-1))
    out = np.full((6, 96), 7.0, np.float32)
    ctx.dequantize(out[1:5], t, row0=26)
    assert (out[[0, 5]] == 7).all() and np.array_equal(out[1:5], mx.decode(want[26:], 96).astype(np.float32))
    ctx.quantize(t, x[:0], row0=30)
    ctx.dequantize(out[:0], t, row0=30)
    assert np.array_equal(t.read(), want.reshape(-1))
    t.free()


# ------------------------------------------------------------------ one vector
SHAPES = [(1, 32), (15, 64), (16, 128), (17, 160), (64, 512), (33, 544), (100, 896), (64, 2816), (5, 4096), (3, 16384),
          (4865, 896), (1000, 2080), (20000, 256)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_gpu_mx_matvec(ctx, rows, cols):
    print(f"matvec {rows}x{cols}", flush=True)
    g = gen(rows, cols, 3)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, cols)
    t = ctx.upload(m, MX, rows, cols)
    y = np.empty(rows, np.float32)
    ctx.quant_matvec(y, t, x)
    close(y, *mx.product(mx.decode(m, cols), x))
    dx, dy = DeviceArray.from_numpy(x), DeviceArray.from_numpy(np.full(rows + 9, 5.0, np.float32))
    ctx.quant_matvec(dy, t, dx)
    ctx.sync()
    got = dy.numpy()
    assert np.array_equal(got[:rows], y) and (got[rows:] == 5).all()
    t.free(), dx.free(), dy.free()


@pytest.mark.parametrize("xs", [1e-30, 1e30, 2e-38])
def test_gpu_mx_matvec_magnitudes(ctx, xs):
    g = gen(4)
    m = synth.quant_matrix(g, MX, 40, 320)
    m.reshape(40, 10, 17)[..., 0] = g.integers(110, 140, (40, 10))
    x = acts(g, 320) * np.float32(xs)
    t = ctx.upload(m, MX, 40, 320)
    y = np.empty(40, np.float32)
    ctx.quant_matvec(y, t, x)
    ref, bound = mx.product(mx.decode(m, 320), x)
    close(y, ref, bound + np.abs(mx.decode(m, 320)).sum(1) * 2.0 ** -130 + 2.0 ** -126)  # (the least limb; subnormal sums)
    t.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("at", [0, 31, 100, 319])
def test_gpu_mx_matvec_not_finite(ctx, bad, at):
    g = gen(5)
    m, x = synth.quant_matrix(g, MX, 35, 320), acts(g, 320)
    x[at] = bad
    m[7] = 0  # a row of zeros too
    t = ctx.upload(m, MX, 35, 320)
    y = np.empty(35, np.float32)
    ctx.quant_matvec(y, t, x)
    assert np.isnan(y).all()
    t.free()


def test_gpu_mx_matvec_nan_blocks_and_expert_rows(ctx):
    g = gen(6)
    m, x = synth.quant_matrix(g, MX, 30, 320), acts(g, 320)
    m.reshape(30, 10, 17)[[4, 29], [9, 3], 0] = 255
    t = ctx.upload(m, MX, 10, 320, 3)
    y = np.empty(30, np.float32)
    ctx.quant_matvec(y, t, x)
    ref, bound = mx.product(mx.decode(m, 320), x)
    assert np.isnan(y[[4, 29]]).all()
    keep = np.setdiff1d(np.arange(30), [4, 29])
    close(y[keep], ref[keep], bound[keep])
    t.free()


@pytest.mark.parametrize("D,F,act", [(128, 96, 0), (320, 544, 1), (896, 4864, 0)])
def test_gpu_mx_ffn_dense(ctx, D, F, act):
    print(f"ffn {D} {F}", flush=True)
    g = gen(D, F)
    mats = [synth.quant_matrix(g, MX, r, c) for r, c in ((F, D), (F, D), (D, F))]
    x = acts(g, D)
    ts = [ctx.upload(m, MX, r, c) for m, (r, c) in zip(mats, ((F, D), (F, D), (D, F)))]
    y = np.empty(D, np.float32)
    ctx.ffn_dense(y, *ts, x, act=act)
    gate, up, dn = mx.decode(mats[0], D), mx.decode(mats[1], D), mx.decode(mats[2], F)
    close(y, *mx.down(dn, *mx.gated(gate, up, x, act)))
    for t in ts:
        t.free()


# ------------------------------------------------------------------ many vectors
MATS = [(1, 32), (16, 128), (17, 96), (100, 160), (33, 544), (130, 1024), (260, 2080)]


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 33, 64, 129])
@pytest.mark.parametrize("rows,cols", MATS)
def test_gpu_mx_matmul(ctx, T, rows, cols):
    print(f"matmul T {T} {rows}x{cols}", flush=True)
    g = gen(T, rows, cols)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, T, cols)
    t = ctx.upload(m, MX, rows, cols)
    y = np.full((T + 1, rows), 5.0, np.float32)
    ctx.quant_matmul(y[:T], t, x)
    close(y[:T], *mx.product(mx.decode(m, cols), x))
    assert (y[T] == 5).all()
    xq = ctx.create(MX, T + 3, cols)
    ctx.quantize(xq, x)
    z = np.full((T + 1, rows), 5.0, np.float32)
    ctx.quant_matmul(z[:T], t, xq)
    close(z[:T], *mx.product(mx.decode(m, cols), mx.decode(mx.quantize(x), cols)))
    assert (z[T] == 5).all()
    xq.free(), t.free()


# a few vectors beside each other in the matvec's instructions, up to what the LDS holds
@pytest.mark.parametrize("T", [2, 3, 4, 5])
@pytest.mark.parametrize("rows,cols", [(1, 32), (33, 544), (5000, 96), (17000, 64), (4099, 2048), (700, 4096), (300, 4384),
                                       (100, 10912), (50, 16384), (9000, 512)])
def test_gpu_mx_matmul_few(ctx, T, rows, cols):
    print(f"few T {T} {rows}x{cols}", flush=True)
    g = gen(T, rows, cols, 25)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, T, cols)
    t = ctx.upload(m, MX, rows, cols)
    buf = DeviceArray.from_numpy(np.full(T * rows + 16, 5.0, np.float32))
    dx = DeviceArray.from_numpy(x)
    ctx.quant_matmul(DeviceView(buf.ptr, (T, rows), np.float32), t, dx)
    ctx.sync()
    got = buf.numpy()
    assert (got[T * rows:] == 5).all()
    w = mx.decode(m, cols)
    close(got[:T * rows].reshape(T, rows), *mx.product(w, x))
    x[T - 2, cols // 2] = np.inf  # in one vector: the others keep theirs
    y = np.empty((T, rows), np.float32)
    ctx.quant_matmul(y, t, x)
    assert np.isnan(y[T - 2]).all()
    keep = [n for n in range(T) if n != T - 2]
    close(y[keep], *mx.product(w, x[keep]))
    for a in (buf, dx, t):
        a.free()


# past the thin kernel's range: each of the tiles, ragged on every side
@pytest.mark.parametrize("T,rows,cols", [(300, 700, 640), (1000, 300, 4096), (1100, 1030, 288), (1300, 1000, 1056),
                                         (130, 9001, 96), (9, 9001, 160), (2001, 8003, 96), (65536, 9, 32),
                                         (65536, 40, 64)])
def test_gpu_mx_matmul_larger(ctx, T, rows, cols):
    test_gpu_mx_matmul(ctx, T, rows, cols)


# more sums than are stored from registers, rows that begin anywhere in a line
@pytest.mark.parametrize("T,rows,cols,shift", [(2001, 8403, 32, 0), (1601, 8002, 64, 4), (3002, 4200, 32, 8), (1700, 8192, 64, 4),
                                               (1537, 8193, 32, 12)])
def test_gpu_mx_matmul_large_output(ctx, T, rows, cols, shift):
    print(f"matmul T {T} {rows}x{cols} out + {shift}", flush=True)
    g = gen(T, rows, cols, shift)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, T, cols)
    t = ctx.upload(m, MX, rows, cols)
    xq = ctx.create(MX, T, cols)
    ctx.quantize(xq, x)
    dx = DeviceArray.from_numpy(x)
    for X, xs in ((dx, x), (xq, mx.decode(mx.quantize(x), cols))):
        buf = DeviceArray.from_numpy(np.full(T * rows + 64, 5.0, np.float32))
        ctx.quant_matmul(DeviceView(buf.ptr + 4 * shift, (T, rows), np.float32), t, X)
        ctx.sync()
        got = buf.numpy()
        assert (got[:shift] == 5).all() and (got[shift + T * rows:] == 5).all()
        close(got[shift:shift + T * rows].reshape(T, rows), *mx.product(mx.decode(m, cols), xs))
        buf.free()
    for a in (dx, xq, t):
        a.free()


def test_gpu_mx_matmul_more_vectors_than_the_workspace_holds(ctx):
    # vectors in several batches: each gives what it gives alone
    T, rows, cols = 2600, 48, 16384
    g = gen(8)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, T, cols)
    t = ctx.upload(m, MX, rows, cols)
    y = np.empty((T, rows), np.float32)
    ctx.quant_matmul(y, t, x)
    close(y, *mx.product(mx.decode(m, cols), x))
    t.free()


@pytest.mark.parametrize("T,rows", [(40, 50), (1100, 1000)])
def test_gpu_mx_matmul_not_finite_stays_in_its_row(ctx, T, rows):
    g = gen(9)
    m, x = synth.quant_matrix(g, MX, rows, 352), acts(g, T, 352)
    x[3, 0], x[17, 351], x[39, 100] = np.nan, np.inf, -np.inf
    m.reshape(rows, 11, 17)[20, 10, 0] = 255
    bad_t, bad_r = [3, 17, 39], [20]
    t = ctx.upload(m, MX, rows, 352)
    y, z = np.empty((T, rows), np.float32), np.empty((T, rows), np.float32)
    ctx.quant_matmul(y, t, x)
    xq = ctx.create(MX, T, 352)
    ctx.quantize(xq, x)
    ctx.quant_matmul(z, t, xq)
    keep_t, keep_r = np.setdiff1d(np.arange(T), bad_t), np.setdiff1d(np.arange(rows), bad_r)
    w = mx.decode(m, 352)[keep_r]
    for got, xs in ((y, x[keep_t]), (z, mx.decode(mx.quantize(x), 352)[keep_t])):
        assert np.isnan(got[bad_t]).all() and np.isnan(got[:, bad_r]).all()
        close(got[np.ix_(keep_t, keep_r)], *mx.product(w, xs))
    xq.free(), t.free()


def test_gpu_mx_matmul_of_a_tensor_with_itself(ctx):
    g = gen(10)
    m = synth.quant_matrix(g, MX, 70, 224)
    t = ctx.upload(m, MX, 70, 224)
    y = np.empty((70, 70), np.float32)
    ctx.quant_matmul(y, t, t)
    w = mx.decode(m, 224)
    close(y, *mx.product(w, w))
    t.free()


def test_gpu_mx_offsets_past_32_bits(ctx):
    # codes of 4.3 GB: the last rows filled, all others zero
    g = gen(17)
    rows, cols, n, T = (1 << 19) + 32, 16384, 37, 20
    t = ctx.create(MX, rows, cols)
    w, x = g.standard_normal((n, cols)).astype(np.float32), acts(g, T, cols)
    ctx.quantize(t, w, row0=rows - n)
    m = mx.decode(mx.quantize(w), cols)
    back = np.empty((n, cols), np.float32)
    ctx.dequantize(back, t, row0=rows - n)
    assert np.array_equal(back, m)
    y, z = np.empty(rows, np.float32), np.empty((T, rows), np.float32)
    ctx.quant_matvec(y, t, x[0])
    ctx.quant_matmul(z, t, x)
    for got, ref in ((y, x[0]), (z, x)):
        assert not got[..., :rows - n].any()
        close(got[..., rows - n:], *mx.product(m, ref))
    t.free()


def test_gpu_mx_more_tiles_than_a_grid_holds(ctx):
    # 68,750 tiles of 16 rows, from a row inside one on
    rows, row0 = 1100000, 5
    x = np.tile(acts(gen(19), 1000, 32), (rows // 1000, 1))
    want = np.tile(mx.quantize(x[:1000]), (rows // 1000, 1))
    t = ctx.create(MX, rows + 20, 32)
    ctx.quantize(t, x, row0=row0)
    got = t.read().reshape(-1, 17)
    assert np.array_equal(got[row0:row0 + rows], want)
    assert not got[:row0].any() and not got[row0 + rows:].any()
    back = np.empty_like(x)
    ctx.dequantize(back, t, row0=row0)
    assert np.array_equal(back, np.tile(mx.decode(want[:1000], 32).astype(np.float32), (rows // 1000, 1)))
    t.free()


def test_gpu_mx_clone_behind_a_quantisation(ctx):
    # the copy is made of what the call before it has on its way
    x = DeviceArray.from_numpy(acts(gen(18), 4096, 4096))
    want = mx.quantize(x.numpy())
    t = ctx.create(MX, 4096, 4096)
    ctx.quantize(t, x)
    c = t.clone()
    assert np.array_equal(c.read().reshape(want.shape), want)
    for a in (x, t, c):
        a.free()


# ------------------------------------------------------------------ experts
def experts(ctx, g, E, D, F, Kd=None):
    Kd = Kd or F
    gu = synth.quant_matrix(g, MX, E * 2 * F, D)
    dn = synth.quant_matrix(g, MX, E * D, Kd)
    if Kd > F:  # the columns past the experts' width are zero
        full = mx.decode(dn, Kd)
        full[:, F:] = 0
        dn = mx.quantize(full.astype(np.float32))
    w = dict(gu=mx.decode(gu, D).reshape(E, 2 * F, D), dn=mx.decode(dn, Kd).reshape(E, D, Kd)[..., :F])
    return ctx.upload(gu, MX, 2 * F, D, E), ctx.upload(dn, MX, D, Kd, E), w


def expert_ref(w, x, ids, wts, F, act):
    hs = [mx.gated(w["gu"][e][:F], w["gu"][e][F:], x, act) for e in ids]
    ys = [mx.down(w["dn"][e], *h) for e, h in zip(ids, hs)]
    y = sum(p * v[0] for p, v in zip(wts, ys))
    # 2^-22: the weighting and adding of up to 16 slots in fp32
    b = sum(abs(p) * (v[1] + 2.0 ** -22 * np.abs(v[0])) for p, v in zip(wts, ys))
    return hs, y, b + 2.0 ** -22 * sum(abs(p) * np.abs(v[0]) for p, v in zip(wts, ys))


@pytest.mark.parametrize("E,D,F,Kd,k,act", [(4, 128, 64, 64, 1, 0), (8, 320, 96, 96, 3, 1), (6, 896, 40, 64, 4, 0),
                                            (32, 2048, 768, 768, 8, 0), (5, 2816, 2112, 2112, 4, 1),
                                            (16, 256, 1056, 2048, 16, 0)])
def test_gpu_mx_experts_by_id(ctx, E, D, F, Kd, k, act):
    print(f"experts E {E} D {D} F {F} Kd {Kd} k {k}", flush=True)
    g = gen(E, D, F, k)
    GU, DN, w = experts(ctx, g, E, D, F, Kd)
    x = acts(g, D)
    ids = g.integers(0, E, k).astype(np.uint32)  # the same expert twice among them
    ids[-1] = ids[0]
    p = g.random(k).astype(np.float32)
    h = np.full((k, Kd), 9.0, np.float32)
    ctx.expert_gate_up_id(GU, x, ids, k, F, Kd, h, act=act)
    hs, ref, bound = expert_ref(w, x, ids, p.astype(np.float64), F, act)
    for s in range(k):
        close(h[s, :F], *hs[s])
        assert (h[s, F:] == 0).all()
    out = g.standard_normal(D).astype(np.float32)
    before = out.astype(np.float64)
    ctx.expert_down_id(DN, h, ids, p, k, out, accumulate=True)
    close(out, before + ref, bound + 2.0 ** -23 * (np.abs(before) + np.abs(ref)))
    ctx.expert_down_id(DN, h, ids, p, k, out)
    close(out, ref, bound)
    again = np.empty_like(out)
    ctx.expert_down_id(DN, h, ids, p, k, again)
    assert np.array_equal(out, again)
    GU.free(), DN.free()


def route(logits, k, norm):
    p = np.exp(logits - logits.max())
    ids = np.argsort(-logits, kind="stable")[:k]
    return ids, p[ids] / (p[ids].sum() if norm else p.sum())


@pytest.mark.parametrize("E,D,F,k,norm,router", [(8, 256, 64, 2, True, ggml.F32), (128, 2048, 768, 8, True, ggml.F32),
                                                 (60, 2816, 704, 4, False, ggml.Q8_0), (300, 512, 64, 6, True, ggml.F32),
                                                 (256, 1056, 96, 16, False, ggml.F32)])
def test_gpu_mx_moe_forward(ctx, E, D, F, k, norm, router):
    print(f"moe E {E} D {D} F {F} k {k}", flush=True)
    g = gen(E, D, F, k, 2)
    GU, DN, w = experts(ctx, g, E, D, F)
    x, bias = acts(g, D), g.standard_normal(E).astype(np.float32)
    if router == ggml.F32:
        r = (g.standard_normal((E, D)) * 0.05).astype(np.float32)
        R, r64 = ctx.upload(r, ggml.F32, E, D), r.astype(np.float64)
    else:
        rb = synth.quant_matrix(g, ggml.Q8_0, E, D)
        blk = rb.reshape(E, D // 32, 34)
        d = blk[..., :2].copy().view(np.float16).astype(np.float64)
        R, r64 = ctx.upload(rb, ggml.Q8_0, E, D), (blk[..., 2:].view(np.int8) * d).reshape(E, D)
    ids, p = route(r64 @ x.astype(np.float64) + bias, k, norm)
    _, ref, bound = expert_ref(w, x, ids, p, F, 0)
    out, got_ids, got_p = np.empty(D, np.float32), np.empty(k, np.uint32), np.empty(k, np.float32)
    for unfused in (False, True):
        ctx.moe_forward(out, x, R, GU, DN, k, F, norm_topk=norm, bias=bias, out_ids=got_ids, out_w=got_p, unfused=unfused)
        assert got_ids.tolist() == ids.tolist()
        # the weights: logits exact to D 2^-24 of their terms' sum, exp and the division a few ulp
        slack = 2 * (D * 2.0 ** -24 * (np.abs(r64) @ np.abs(x)).max() + 2.0 ** -20)
        assert (np.abs(got_p - p) <= slack * p).all()
        close(out, ref, bound + slack * np.abs(ref) + slack * sum(q * np.abs(w["dn"][e]).sum(1) for e, q in zip(ids, p)))
    for t in (R, GU, DN):
        t.free()


# the layer in one launch: slots for every XCD or nearly, rows and experts of every kind
@pytest.mark.parametrize("E,D,F,Kd,k,act", [(6, 256, 40, 64, 6, 0), (7, 512, 32, 32, 7, 1), (128, 2048, 96, 96, 8, 0),
                                            (256, 256, 160, 160, 8, 0), (40, 768, 80, 544, 14, 1), (255, 256, 64, 64, 15, 0),
                                            (16, 1280, 48, 64, 16, 0), (9, 16384, 16, 32, 6, 0), (9, 256, 4100, 4128, 8, 0),
                                            (8, 2880, 96, 96, 8, 1), (7, 96, 32, 32, 7, 0), (20, 32, 64, 64, 3, 0),
                                            (60, 1056, 64, 64, 6, 0), (33, 544, 64, 64, 9, 0), (4, 224, 32, 32, 1, 0)])
def test_gpu_mx_moe_one_launch(ctx, E, D, F, Kd, k, act):
    print(f"one launch E {E} D {D} F {F} Kd {Kd} k {k}", flush=True)
    g = gen(E, D, F, k, 21)
    GU, DN, w = experts(ctx, g, E, D, F, Kd)
    r, bias = (g.standard_normal((E, D)) * 0.05).astype(np.float32), g.standard_normal(E).astype(np.float32)
    R, r64 = ctx.upload(r, ggml.F32, E, D), r.astype(np.float64)
    for seed in range(3):
        x, out = acts(gen(22, seed), D), g.standard_normal(D).astype(np.float32)
        before, norm = out.astype(np.float64), seed % 2 == 0
        ids, p = route(r64 @ x.astype(np.float64) + bias, k, norm)
        _, ref, bound = expert_ref(w, x, ids, p, F, act)
        got_ids, got_p = np.empty(k, np.uint32), np.empty(k, np.float32)
        ctx.moe_forward(out, x, R, GU, DN, k, F, act=act, norm_topk=norm, accumulate=True, bias=bias, out_ids=got_ids, out_w=got_p)
        assert got_ids.tolist() == ids.tolist()
        slack = 2 * (D * 2.0 ** -24 * (np.abs(r64) @ np.abs(x)).max() + 2.0 ** -20)  # as above
        assert (np.abs(got_p - p) <= slack * p).all()
        more = slack * np.abs(ref) + slack * sum(q * np.abs(w["dn"][e]).sum(1) for e, q in zip(ids, p))
        close(out, before + ref, bound + more + 2.0 ** -23 * (np.abs(before) + np.abs(ref)))
        first = np.empty(D, np.float32)
        for again in range(3):  # in the slots' order: the same bits
            y = np.empty(D, np.float32)
            ctx.moe_forward(y, x, R, GU, DN, k, F, act=act, norm_topk=norm, bias=bias)
            if again == 0:
                first = y
            assert np.array_equal(first, y)
        y = np.empty(D, np.float32)
        ctx.moe_forward(y, x, R, GU, DN, k, F, act=act, norm_topk=norm, bias=bias, unfused=True)
        assert np.linalg.norm(y - first) <= 2.0 ** -18 * np.linalg.norm(first)
    for t in (R, GU, DN):
        t.free()


def test_gpu_mx_moe_one_launch_in_graphs(ctx, monkeypatch):
    # two layers of different shapes and one of another k, eager and replayed in turn,
    # h handed over inside an XCD and (the second context) past the L2s: the same bits
    g = gen(23)
    shapes = [(32, 512, 64, 8), (32, 512, 64, 7), (64, 256, 96, 16)]
    layers, xs = [], [acts(g, 4, 512) for _ in range(3)]
    for E, D, F, k in shapes:
        layers.append(((g.standard_normal((E, D)) * 0.05).astype(np.float32), synth.quant_matrix(g, MX, E * 2 * F, D),
                       synth.quant_matrix(g, MX, E * D, F)))
    results = []
    monkeypatch.setenv("LT_FUSED_AGENT_HANDOVER", "1")
    with lt.Context(0) as other:
        for c in (ctx, other):
            ts = [(c.upload(r, ggml.F32, E, D), c.upload(a, MX, 2 * F, D, E), c.upload(b, MX, D, F, E))
                  for (r, a, b), (E, D, F, k) in zip(layers, shapes)]
            X = [DeviceArray((4, 512)) for _ in shapes]
            outs = [DeviceArray((4, 512)) for _ in shapes]

            def step():
                for i in range(4):
                    for (R, GU, DN), (E, D, F, k), x, o in zip(ts, shapes, X, outs):
                        c.moe_forward(o.row(i), x.row(i), R, GU, DN, k, F, norm_topk=True)

            def fill(seed):
                import ctypes
                from llmtoy_amd.hip import H2D, check, hip
                for i, x in enumerate(X):
                    v = xs[(i + seed) % 3]
                    check(hip().hipMemcpy(x.ptr, v.ctypes.data_as(ctypes.c_void_p), v.nbytes, H2D))

            fill(0)
            step()
            c.sync()
            graph, got = Graph(c.stream, step), []
            for seed in range(1, 4):
                fill(seed)
                step()
                c.sync()
                eager = [o.numpy()[:, :D] for o, (E, D, F, k) in zip(outs, shapes)]
                fill(seed + 1)
                graph.launch()
                step()
                c.sync()
                fill(seed)
                graph.launch()
                graph.launch()
                c.sync()
                for a, o, (E, D, F, k) in zip(eager, outs, shapes):
                    assert np.isfinite(a).all() and np.array_equal(a, o.numpy()[:, :D])
                got += eager
            results.append(got)
            graph.destroy()
            for t in (*[t for q in ts for t in q], *X, *outs):
                t.free()
    for a, b in zip(*results):
        assert np.array_equal(a, b)


def test_gpu_mx_moe_one_launch_first_call_in_a_capture(ctx):
    g = gen(24)
    E, D, F, k = 24, 256, 32, 7
    GU, DN, _ = experts(ctx, g, E, D, F)
    R = ctx.upload((g.standard_normal((E, D)) * 0.05).astype(np.float32), ggml.F32, E, D)
    x, y = DeviceArray.from_numpy(acts(g, D)), DeviceArray((D,))
    with lt.Context(0) as other:
        tensors = [other.upload(t.read(), t.type, t.rows, t.cols, t.n_experts) for t in (R, GU, DN)]

        def first():
            with pytest.raises(ltlib.InvalidError):
                other.moe_forward(y, x, *tensors, k, F)

        Graph(other.stream, first).destroy()
        other.moe_forward(y, x, *tensors, k, F)
        other.sync()
        want = y.numpy()
        graph = Graph(other.stream, lambda: other.moe_forward(y, x, *tensors, k, F))
        graph.launch()
        other.sync()
        assert np.array_equal(want, y.numpy())
        graph.destroy()
        for t in tensors:
            t.free()
    for t in (R, GU, DN, x, y):
        t.free()


def test_gpu_mx_experts_beside_other_formats(ctx):
    # gate/up in one format, down in another, a dense FFN of MXFP4 beside them
    g = gen(11)
    E, D, F, k = 6, 512, 256, 3
    GU, DN, w = experts(ctx, g, E, D, F)
    q4 = synth.quant_matrix(g, ggml.Q4_K, E * D, F)
    DQ = ctx.upload(q4, ggml.Q4_K, D, F, E)
    g4 = synth.quant_matrix(g, ggml.Q4_K, E * 2 * F, D)
    GQ = ctx.upload(g4, ggml.Q4_K, 2 * F, D, E)
    R = ctx.upload((g.standard_normal((E, D)) * 0.05).astype(np.float32), ggml.F32, E, D)
    x = acts(g, D)
    ids, p = np.empty(k, np.uint32), np.empty(k, np.float32)
    ctx.router_topk(R, x, k, ids, p)
    sh = [ctx.upload(synth.quant_matrix(g, MX, r, c), MX, r, c) for r, c in ((F, D), (F, D), (D, F))]
    dense = np.empty(D, np.float32)
    ctx.ffn_dense(dense, *sh, x)
    for gu, dn in ((GU, DQ), (GQ, DN), (GU, DN)):
        h, parts, whole = np.empty((k, F), np.float32), np.empty(D, np.float32), np.empty(D, np.float32)
        ctx.expert_gate_up_id(gu, x, ids, k, F, F, h)
        ctx.expert_down_id(dn, h, ids, p, k, parts)
        ctx.moe_forward(whole, x, R, gu, dn, k, F)
        assert np.linalg.norm(whole - parts) <= 1e-5 * np.linalg.norm(parts)
        ctx.moe_forward(whole, x, R, gu, dn, k, F, shared=tuple(sh), accumulate=False)
        assert np.linalg.norm(whole - (parts + dense)) <= 1e-5 * np.linalg.norm(parts + dense)
    for t in (GU, DN, DQ, GQ, R, *sh):
        t.free()


@pytest.mark.parametrize("precise", [False, True])
def test_gpu_mx_gemma4_block(ctx, precise):
    g = gen(12)
    E, D, F, k = 16, 512, 96, 4
    GU, DN, w = experts(ctx, g, E, D, F)
    r = (g.standard_normal((E, D)) * 0.3).astype(np.float32)
    R = ctx.upload(r, ggml.F32, E, D)
    x, dense = acts(g, D), acts(g, D)
    nm = {n: (1 + 0.2 * g.standard_normal(m)).astype(np.float32) for n, m in
          (("pre_ffw_norm_2", D), ("router_scale", D), ("down_exps_scale", E), ("post_ffw_norm_2", D), ("post_ffw_norm", D))}
    rms = lambda v, s: v / np.sqrt((v * v).mean() + 1e-6) * s  # noqa: E731
    x64 = x.astype(np.float64)
    ids, p = route(r.astype(np.float64) @ (rms(x64, nm["router_scale"]) / np.sqrt(D)), k, False)
    _, moe, _ = expert_ref(w, rms(x64, nm["pre_ffw_norm_2"]), ids, p * nm["down_exps_scale"][ids], F, 1)
    ref = (x64 + rms(dense + rms(moe, nm["post_ffw_norm_2"]), nm["post_ffw_norm"])) * 0.75
    got_ids = np.empty(k, np.uint32)
    got = ltlib.gemma4_moe_block(ctx, x.copy(), dense, R, GU, DN, k, F, nm, 0.75, 1e-6, precise=precise, out_ids=got_ids)
    assert got_ids.tolist() == ids.tolist()
    # the experts' sum to 2^-20 of its terms (about sqrt(D) of its size), the norms to a few ulp
    assert np.linalg.norm(got - ref) <= 2.0 ** -14 * np.linalg.norm(ref)
    for t in (R, GU, DN):
        t.free()


# ------------------------------------------------------------------ graphs, streams, refusals
def test_gpu_mx_decode_and_prompt_in_one_graph(ctx):
    # quantise, the product of it, the fp32 product, a layer: replayed with eager work between
    g = gen(13)
    T, D, F, E, k = 37, 512, 320, 8, 2
    GU, DN, _ = experts(ctx, g, E, D, F)
    W = ctx.upload(synth.quant_matrix(g, MX, 200, D), MX, 200, D)
    R = ctx.upload((g.standard_normal((E, D)) * 0.05).astype(np.float32), ggml.F32, E, D)
    xq = ctx.create(MX, T, D)
    X = DeviceArray((T, D))
    outs = [DeviceArray((T, 200)), DeviceArray((T, 200)), DeviceArray((D,)), DeviceArray((200,)), DeviceArray((T, D))]

    def step():
        ctx.quantize(xq, X)
        ctx.quant_matmul(outs[0], W, xq)
        ctx.quant_matmul(outs[1], W, X)
        ctx.moe_forward(outs[2], X.row(0), R, GU, DN, k, F)
        ctx.quant_matvec(outs[3], W, X.row(T - 1))
        ctx.dequantize(outs[4], xq)

    def fill(seed):
        import ctypes
        from llmtoy_amd.hip import H2D, check, hip
        x = acts(gen(13, seed), T, D)
        check(hip().hipMemcpy(X.ptr, x.ctypes.data_as(ctypes.c_void_p), x.nbytes, H2D))

    fill(0)
    step()
    ctx.sync()
    graph = Graph(ctx.stream, step)
    for seed in range(1, 5):
        fill(seed)
        step()
        ctx.sync()
        eager = [o.numpy() for o in outs]
        big = np.empty((T + 30, 200), np.float32)  # a larger call between replays: its scratch is another
        ctx.quant_matmul(big, W, acts(gen(14), T + 30, D))
        fill(seed + 10)
        step()
        ctx.sync()
        fill(seed)
        graph.launch()
        ctx.sync()
        for a, o in zip(eager, outs):
            assert np.array_equal(a, o.numpy())
    graph.destroy()
    for t in (GU, DN, W, R, xq, X, *outs):
        t.free()


def test_gpu_mx_two_graphs_of_one_context(ctx):
    # they share the context's workspace: replayed in turn, each with inputs of its own
    g = gen(20)
    W = ctx.upload(synth.quant_matrix(g, MX, 333, 640), MX, 333, 640)
    Ts, xs, outs, want, graphs = (37, 90), [], [], [], []
    for T in Ts:
        x = acts(g, T, 640)
        xs.append(DeviceArray.from_numpy(x))
        outs.append(DeviceArray((T, 333)))
        want.append(ctx.quant_matmul(np.empty((T, 333), np.float32), W, x).copy())
        ctx.quant_matmul(outs[-1], W, xs[-1])
        ctx.sync()
        graphs.append(Graph(ctx.stream, lambda o=outs[-1], d=xs[-1]: ctx.quant_matmul(o, W, d)))
    for i in (0, 1, 1, 0, 1, 0, 0):
        graphs[i].launch()
        graphs[1 - i].launch()
        ctx.sync()
        for w, o in zip(want, outs):
            assert np.array_equal(w, o.numpy())
    for a in (*graphs,):
        a.destroy()
    for a in (W, *xs, *outs):
        a.free()


def test_gpu_mx_two_contexts_side_by_side(ctx):
    g = gen(15)
    m, xs = synth.quant_matrix(g, MX, 300, 640), [acts(g, 50, 640) for _ in range(2)]
    want = []
    with lt.Context(0) as other:
        cs, sides = (ctx, other), []
        for c, x in zip(cs, xs):
            W = c.upload(m, MX, 300, 640)
            want.append(mx.product(mx.decode(m, 640), x))
            sides.append((c, W, DeviceArray.from_numpy(x), DeviceArray((50, 300))))
        for _ in range(3):
            for c, W, x, y in sides:
                c.quant_matmul(y, W, x)
        for (c, W, x, y), ref in zip(sides, want):
            c.sync()
            close(y.numpy(), *ref)
            W.free(), x.free(), y.free()


def test_gpu_mx_refusals(ctx):
    t, e = ctx.create(MX, 20, 64), ctx.create(MX, 20, 64, 2)
    q = ctx.upload(synth.quant_matrix(gen(16), ggml.Q8_0, 20, 64), ggml.Q8_0, 20, 64)
    wide = ctx.create(MX, 4, 16384 + 32)
    x, y = np.zeros((2, 64), np.float32), np.zeros((2, 20), np.float32)
    d = DeviceArray((4096,))

    class Shifted:
        def __init__(self, shape):
            self.ptr, self.shape, self.dtype = d.ptr + 4, shape, np.dtype(np.float32)

    def refused(kind, fn):
        with pytest.raises(kind):
            fn()

    I, U = ltlib.InvalidError, ltlib.UnsupportedError
    refused(U, lambda: ctx.create(ggml.Q8_0, 4, 64))
    refused(U, lambda: ctx.create(MX, 4, 48))
    refused(U, lambda: ctx.create(MX, 1 << 31, 32))
    refused(U, lambda: ctx.create(MX, 1 << 20, 32, 1 << 11))
    refused(I, lambda: ctx.create(MX, 0, 64))
    refused(I, lambda: ctx.create(MX, 1 << 40, 64, 1 << 40))
    refused(I, lambda: ctx.upload(np.zeros(33, np.uint8), MX, 1, 64))
    refused(I, lambda: ctx.quantize(t, x, row0=19))
    refused(I, lambda: ctx.quantize(t, x, row0=(1 << 64) - 1))
    refused(U, lambda: ctx.quantize(q, x))
    refused(U, lambda: ctx.dequantize(x, q))
    refused(I, lambda: ctx.dequantize(Shifted((2, 64)), t))
    refused(I, lambda: ctx.quantize(t, Shifted((2, 64))))
    refused(U, lambda: ctx.quant_matmul(y, q, x))
    refused(U, lambda: ctx.quant_matmul(y, t, q))
    refused(I, lambda: ctx.quant_matmul(y, e, x))
    refused(I, lambda: ctx.quant_matmul(y, t, e))
    refused(I, lambda: ctx.quant_matmul(np.zeros((21, 20), np.float32), t, t))
    refused(I, lambda: ctx.quant_matmul(y, t, wide))
    refused(U, lambda: ctx.quant_matmul(np.zeros((2, 4), np.float32), wide, np.zeros((2, 16416), np.float32)))
    refused(I, lambda: ctx.quant_matmul(Shifted((2, 20)), t, DeviceArray((2, 64))))
    refused(I, lambda: ctx.quant_matmul(DeviceArray((2, 20)), t, Shifted((2, 64))))
    refused(U, lambda: ctx.quant_matvec(np.zeros(4, np.float32), wide, np.zeros(16416, np.float32)))
    lib = ctx.lib
    assert lib.lt_matmul(ctx.ptr, y.ctypes.data, t.handle, x.ctypes.data, 65537, 1) == ltlib.LT_ERR_INVALID
    assert lib.lt_matmul(ctx.ptr, y.ctypes.data, t.handle, x.ctypes.data, 2, 3) == ltlib.LT_ERR_INVALID
    assert lib.lt_quantize(ctx.ptr, t.handle, x.ctypes.data, 0, 2, 5) == ltlib.LT_ERR_INVALID
    ctx.quant_matmul(y[:0], t, x[:0])
    ctx.quant_matmul(y[:0], t, t)
    assert lib.lt_matmul(ctx.ptr, None, t.handle, None, 0, 0) == lib.lt_matmul_quantized(ctx.ptr, None, t.handle, t.handle, 0, 0) == 0
    assert lib.lt_quantize(ctx.ptr, t.handle, None, 20, 0, 0) == lib.lt_dequantize(ctx.ptr, None, t.handle, 0, 0, 0) == 0
    for rc in (lib.lt_matmul(ctx.ptr, None, t.handle, x.ctypes.data, 2, 1), lib.lt_matmul(ctx.ptr, y.ctypes.data, t.handle, None, 2, 1),
               lib.lt_quantize(ctx.ptr, t.handle, None, 0, 1, 1), lib.lt_dequantize(ctx.ptr, None, t.handle, 0, 1, 1)):
        assert rc == ltlib.LT_ERR_INVALID
    refused(U, lambda: ctx.moe_forward_noalloc(DeviceArray((64,)), DeviceArray((64,)), ctx.upload(
        np.zeros((2, 64), np.float32), ggml.F32, 2, 64), ctx.create(MX, 64, 64, 2), ctx.create(MX, 64, 32, 2), 1, 32))
    for a in (t, e, q, wide, d):
        a.free()
