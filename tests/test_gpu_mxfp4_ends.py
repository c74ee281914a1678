"""MXFP4 products at the ends of the numbers' ranges: every scale byte, activations
from the least to the largest."""
import numpy as np
import pytest

import mx_accuracy as acc
import mx_reference as mx
from llmtoy_amd import ggml, synth
from llmtoy_amd import lib as ltlib
from llmtoy_amd.hip import DeviceArray, DeviceView
from test_gpu_mxfp4 import acts, close, gen, route

pytestmark = pytest.mark.gpu

MX = ggml.MXFP4
# the bytes, and what brings their products to the middle of fp32's range
LOW, HIGH = (np.arange(0, 5), 2.0 ** 40), (np.arange(250, 255), 2.0 ** -40)
HIGH_BF16 = (np.arange(248, 253), 2.0 ** -40)  # what the experts' kernels take


def weights(g, rows, cols, scales, ordinary=True):
    """Blocks of these scale bytes, each 16 rows one of them and the rest a mix; in the mix
    also a block of ordinary weights and one of zeros."""
    m = synth.quant_matrix(g, MX, rows, cols)
    b = m.reshape(rows, cols // 32, 17)
    b[..., 0] = g.choice(scales, (rows, cols // 32))
    for i, s in enumerate(scales):
        b[16 * i:16 * i + 16, :, 0] = s
    b[16 * len(scales):, 2, 1:] = 0
    if ordinary:
        b[16 * len(scales):, 1, 0] = 127
    return m


# one vector, a few, the thin product, the tiles, 4-bit vectors of both
@pytest.mark.parametrize("T,rows,cols", [(1, 130, 160), (1, 4100, 544), (3, 130, 160), (5, 90, 2080), (15, 130, 160), (40, 130, 544),
                                         (1100, 1030, 160), (2001, 8003, 96)])
@pytest.mark.parametrize("end", [LOW, HIGH], ids=["low", "high"])
def test_gpu_mx_products_of_every_scale(ctx, end, T, rows, cols):
    print(f"scales {end[0]} T {T} {rows}x{cols}", flush=True)
    g = gen(T, rows, cols, 41)
    m, x = weights(g, rows, cols, end[0]), acts(g, T, cols) * np.float32(end[1])
    t, w = ctx.upload(m, MX, rows, cols), mx.decode(m, cols)
    y = np.empty((T, rows), np.float32)
    if T == 1:
        ctx.quant_matvec(y[0], t, x[0])
    else:
        ctx.quant_matmul(y, t, x)
    close(y, *mx.product(w, x))
    q = ctx.quantize(ctx.create(MX, T, cols), x)
    ctx.quant_matmul(y, t, q)
    close(y, *mx.product(w, mx.decode(mx.quantize(x), cols)))
    q.free(), t.free()


@pytest.mark.parametrize("end", [LOW, HIGH_BF16], ids=["low", "high"])
def test_gpu_mx_experts_of_every_scale(ctx, end):
    g = gen(42)
    E, D, F, k = 9, 160, 96, 8
    print(f"experts of scales {end[0]}", flush=True)
    x = acts(g, D) * np.float32(end[1])
    gu, dn = weights(g, E * 2 * F, D, end[0], ordinary=False), weights(g, E * D, F, end[0])
    plain = synth.quant_matrix(g, MX, E * D, F)
    GU, DN, P = ctx.upload(gu, MX, 2 * F, D, E), ctx.upload(dn, MX, D, F, E), ctx.upload(plain, MX, D, F, E)
    wg, wd, wp = mx.decode(gu, D).reshape(E, 2 * F, D), mx.decode(dn, F).reshape(E, D, F), mx.decode(plain, F).reshape(E, D, F)
    # gate and up would be 2^-80 and below or 2^80 and above: brought near 1 by x (an
    # ordinary block among them would be beyond fp32 then)
    x = x * np.float32(2.0 ** (80 if end is LOW else -80))
    ids, p = g.permutation(E)[:k].astype(np.uint32), g.random(k).astype(np.float32)
    h = np.empty((k, F), np.float32)
    ctx.expert_gate_up_id(GU, x, ids, k, F, F, h)
    hs = [mx.gated(wg[e][:F], wg[e][F:], x, 0) for e in ids]
    for s in range(k):
        close(h[s], *hs[s])
    hd, out = acts(g, k, F) * np.float32(end[1]), np.empty(D, np.float32)
    ctx.expert_down_id(DN, hd, ids, p, k, out)
    ys = [mx.product(wd[e], v) for e, v in zip(ids, hd)]
    slots = sum(q * np.abs(y) for q, (y, _) in zip(p.astype(np.float64), ys)) * 2.0 ** -21  # (the slots' weighting and adding)
    close(out, sum(q * y for q, (y, _) in zip(p.astype(np.float64), ys)), sum(q * b for q, (_, b) in zip(p, ys)) + slots)
    # the layer, in one launch and in three: gate/up of these scales, down of ordinary ones
    r = (g.standard_normal((E, D)) * 0.05 / (x.astype(np.float64) ** 2).mean() ** 0.5).astype(np.float32)
    R = ctx.upload(r, ggml.F32, E, D)
    ids, p = route(r.astype(np.float64) @ x.astype(np.float64), k, True)
    ref, cut = np.zeros(D), np.zeros(D)
    for e, q in zip(ids, p):
        gate, up = wg[e][:F], wg[e][F:]
        ref += q * (wp[e] @ mx.gated(gate, up, x, 0)[0])
        # an activation's third bf16 part ends at 2^-133, the least subnormal; high: x is about
        # 2^-120, so that this is 2^-13 of it (as in gated, for an error of g and u)
        dg, du = np.abs(gate).sum(1) * 2.0 ** -133, np.abs(up).sum(1) * 2.0 ** -133
        a, u = mx.act(0, gate @ x.astype(np.float64)), up @ x.astype(np.float64)
        cut += q * (np.abs(wp[e]) @ (1.13 * dg * (np.abs(u) + du) + np.abs(a) * du))
    for unfused in (False, True):
        got = np.empty(k, np.uint32)
        ctx.moe_forward(out, x, R, GU, P, k, F, norm_topk=True, out_ids=got, unfused=unfused)
        assert got.tolist() == ids.tolist()
        # the routing's weights to 2^-17 of themselves (logits of 160 terms), the products as above
        assert np.linalg.norm(out - ref) <= 2.0 ** -16 * np.linalg.norm(ref) + np.linalg.norm(cut)
    for t in (GU, DN, P, R):
        t.free()


def test_gpu_mx_weights_beyond_bf16(ctx):
    # one block of 2^128 and more: the dense FFN takes it, the experts' calls say so; a clone
    # is as its source, rows quantised over it are ordinary ones
    g = gen(44)
    D, F, E, k = 96, 160, 4, 2
    mats = [synth.quant_matrix(g, MX, r, c) for r, c in ((F, D), (F, D), (D, F))]
    for m, (row, b) in zip(mats, ((5, 2), (159, 0), (95, 4))):
        m.reshape(m.shape[0], -1, 17)[row, b, 0] = 254
    ts = [ctx.upload(m, MX, r, c) for m, (r, c) in zip(mats, ((F, D), (F, D), (D, F)))]
    x, y = acts(g, D) * np.float32(2.0 ** -70), np.empty(D, np.float32)  # (row 159 of h: 2^57 * 2^-70)
    gate, up, dn = mx.decode(mats[0], D), mx.decode(mats[1], D), mx.decode(mats[2], F)
    ref = mx.gated(gate, up, x, 0)
    ctx.ffn_dense(y, *ts, x)
    want, bound = mx.down(dn, *ref)
    assert np.isfinite(want).all() and np.abs(want).max() < 3e38
    close(y, want, bound)
    c, one = ts[0].clone(), np.empty(F, np.float32)
    ctx.quant_matvec(one, c, x)
    close(one, *mx.product(gate, x))
    rows = acts(g, F, D)
    ctx.quantize(c, rows)
    ctx.quant_matvec(one, c, x)
    close(one, *mx.product(mx.decode(mx.quantize(rows), D), x))
    gu, de = synth.quant_matrix(g, MX, E * 2 * F, D), synth.quant_matrix(g, MX, E * D, F)
    R = ctx.upload(acts(g, E, D), ggml.F32, E, D)
    GU, DE = ctx.upload(gu, MX, 2 * F, D, E), ctx.upload(de, MX, D, F, E)
    gu.reshape(E * 2 * F, -1, 17)[7, 1, 0], de.reshape(E * D, -1, 17)[7, 1, 0] = 253, 253
    GB, DB = ctx.upload(gu, MX, 2 * F, D, E), ctx.upload(de, MX, D, F, E)
    ids, h, p = np.arange(k, dtype=np.uint32), np.zeros((k, F), np.float32), np.ones(k, np.float32)
    for call in (lambda: ctx.expert_gate_up_id(GB, x, ids, k, F, F, h), lambda: ctx.expert_down_id(DB, h, ids, p, k, y),
                 lambda: ctx.moe_forward(y, x, R, GB, DE, k, F), lambda: ctx.moe_forward(y, x, R, GU, DB, k, F, unfused=True),
                 lambda: ctx.quant_matvec(np.empty(E * 2 * F, np.float32), GB, x)):
        with pytest.raises(ltlib.UnsupportedError):
            call()
    ctx.moe_forward(y, x, R, GU, DE, k, F)
    assert np.isfinite(y).all()
    for t in (*ts, c, R, GU, DE, GB, DB):
        t.free()


@pytest.mark.parametrize("xs", [1e-30, 1e30, 2e-38, 3e38])
@pytest.mark.parametrize("T,rows", [(4, 40), (17, 40), (1100, 1030)])
def test_gpu_mx_matmul_magnitudes(ctx, T, rows, xs):
    print(f"magnitudes {xs} T {T} rows {rows}", flush=True)
    g = gen(T, rows, 43)
    m = synth.quant_matrix(g, MX, rows, 320)
    m.reshape(rows, 10, 17)[..., 0] = g.integers(110, 120 if xs > 1e35 else 140, (rows, 10))
    x = acts(g, T, 320)
    x = (x / np.abs(x).max() if xs > 1e35 else x) * np.float32(xs)
    t = ctx.upload(m, MX, rows, 320)
    y = np.empty((T, rows), np.float32)
    ctx.quant_matmul(y, t, x)
    w = mx.decode(m, 320)
    ref, bound = mx.product(w, x)
    # the last limb's remainder of the least scale is 2^-129, a vector's third part is cut at 2^-133; subnormal sums
    close(y, ref, bound + np.abs(w).sum(1) * 2.0 ** -129 + 2.0 ** -126)
    t.free()


@pytest.mark.parametrize("T,rows,least", [(1, 130, -109), (4, 130, -109), (17, 130, -104), (1100, 1030, -104)])
def test_gpu_mx_least_activations_in_full(ctx, T, rows, least):
    # the smallest that are taken in full: the elements themselves for a vector's parts, the
    # blocks' largest for limbs; a step below, no more than the documented remainder is lost
    print(f"least T {T} rows {rows}", flush=True)
    g = gen(T, rows, 45)
    m, x = synth.quant_matrix(g, MX, rows, 320), acts(g, T, 320)
    m.reshape(rows, 10, 17)[..., 0] = g.integers(130, 134, (rows, 10))
    x = np.copysign(1 + np.abs(x), x).astype(np.float32)  # no element and no block below 1
    t, w = ctx.upload(m, MX, rows, 320), mx.decode(m, 320)
    for e in (least, least - 12):
        xs, y = x * np.float32(2.0 ** e), np.empty((T, rows), np.float32)
        if T == 1:
            ctx.quant_matvec(y[0], t, xs[0])
        else:
            ctx.quant_matmul(y, t, xs)
        if e == least:
            assert acc.within_l2(y, w, xs).max() <= 1
        ref, _ = mx.product(w, xs)
        lost = np.abs(w).sum(1) * 2.0 ** (-133 if T < 6 else -129) if e < least else 0
        assert (np.linalg.norm(y - ref, axis=-1) <= acc.l2_limit(w, xs) + np.linalg.norm(lost)).all()
    t.free()


@pytest.mark.parametrize("rows", [130, 70001])
def test_gpu_mx_matvec_beyond_bf16_to_any_address(ctx, rows):
    # lt_matvec asks nothing of out's address: through the thin product and the tiles
    g = gen(rows, 46)
    m, x = synth.quant_matrix(g, MX, rows, 160), acts(g, 160) * np.float32(2.0 ** -40)
    m.reshape(rows, 5, 17)[[3, rows - 1], [0, 4], 0] = 254
    t, dx = ctx.upload(m, MX, rows, 160), DeviceArray.from_numpy(x)
    for shift in (1, 2, 3):
        buf = DeviceArray.from_numpy(np.full(rows + 8, 5.0, np.float32))
        ctx.quant_matvec(DeviceView(buf.ptr + 4 * shift, (rows,), np.float32), t, dx)
        ctx.sync()
        got = buf.numpy()
        assert (got[:shift] == 5).all() and (got[shift + rows:] == 5).all()
        close(got[shift:shift + rows], *mx.product(mx.decode(m, 160), x))
        buf.free()
    t.free(), dx.free()
