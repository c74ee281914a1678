"""What the MXFP4 products keep of their activations (mx_accuracy.py): in L2, and where all of
the answer lies in the activations' last bits."""
import numpy as np
import pytest

import mx_accuracy as acc
import mx_reference as mx
from llmtoy_amd import ggml, synth
from test_gpu_mxfp4 import acts, close, experts, gen, route

pytestmark = pytest.mark.gpu

MX = ggml.MXFP4
# one vector (rows in part of a tile, in many tiles), a few beside each other, few by way of limbs (more
# than fit the LDS together have longer rows), the thin product's two shapes, both tiles
CALLS = [(1, 130, 1024), (1, 4100, 544), (1, 4865, 896), (1, 17000, 64), (2, 300, 2080), (3, 130, 1024), (5, 4100, 544), (6, 130, 1024),
         (15, 300, 2080), (40, 130, 544), (9, 9001, 160), (300, 700, 640), (1100, 1030, 544), (130, 9001, 96), (2001, 8003, 512)]


def product(ctx, t, x, rows):
    y = np.empty((len(x), rows), np.float32)
    if len(x) == 1:
        ctx.quant_matvec(y[0], t, x[0])
    else:
        ctx.quant_matmul(y, t, x)
    return y


@pytest.mark.parametrize("T,rows,cols", CALLS)
def test_gpu_mx_products_in_l2(ctx, T, rows, cols):
    print(f"l2 T {T} {rows}x{cols}", flush=True)
    g = gen(T, rows, cols, 61)
    m, x = synth.quant_matrix(g, MX, rows, cols), acts(g, T, cols)
    t, w = ctx.upload(m, MX, rows, cols), mx.decode(m, cols)
    worst = acc.within_l2(product(ctx, t, x, rows), w, x).max()
    print(f"worst {worst:.3f} of the limit", flush=True)
    assert worst <= 1
    q = ctx.quantize(ctx.create(MX, T, cols), x)
    y = np.empty((T, rows), np.float32)
    ctx.quant_matmul(y, t, q)
    assert acc.within_l2(y, w, mx.decode(mx.quantize(x), cols)).max() <= 1
    q.free(), t.free()


@pytest.mark.parametrize("T,rows,cols", CALLS)
def test_gpu_mx_products_of_the_last_bits(ctx, T, rows, cols):
    print(f"last bits T {T} {rows}x{cols}", flush=True)
    g = gen(T, rows, cols, 62)
    m, x = acc.low_bits(g, rows, cols, lambda r, c: synth.quant_matrix(g, MX, r, c), T)
    t, w = ctx.upload(m, MX, rows, cols), mx.decode(m, cols)
    close(product(ctx, t, x, rows), x.astype(np.float64) @ w.T, acc.low_bits_limit(w, x))
    t.free()


@pytest.mark.parametrize("E,D,F,k,act", [(8, 1024, 544, 8, 0), (128, 2048, 768, 8, 0), (12, 2080, 256, 4, 1), (300, 512, 64, 6, 0)])
def test_gpu_mx_experts_in_l2(ctx, E, D, F, k, act):
    # by id and as a layer, in one launch and in three.  g and u are within 2^-22 s of themselves, s
    # about twice their size; h changes by 1.13 (act') and 1 times that, its own roundings are 2^-20;
    # down adds the same again: 2^-17 is above, a bf16 part that both products lost is 2^-15
    print(f"experts E {E} D {D} F {F} k {k}", flush=True)
    g = gen(E, D, F, k, 63)
    GU, DN, w = experts(ctx, g, E, D, F)
    x, r = acts(g, D), (g.standard_normal((E, D)) * 0.05).astype(np.float32)
    R, x64 = ctx.upload(r, ggml.F32, E, D), x.astype(np.float64)
    ids, p = route(r.astype(np.float64) @ x64, k, True)
    hs = np.stack([mx.act(act, w["gu"][e][:F] @ x64) * (w["gu"][e][F:] @ x64) for e in ids])
    ref = sum(q * (w["dn"][e] @ h) for e, q, h in zip(ids, p, hs))
    ids32, h, out = ids.astype(np.uint32), np.empty((k, F), np.float32), np.empty(D, np.float32)
    ctx.expert_gate_up_id(GU, x, ids32, k, F, F, h, act=act)
    for a, b in zip(h, hs):
        assert np.linalg.norm(a - b) <= 2.0 ** -17 * np.linalg.norm(b)
    ctx.expert_down_id(DN, hs.astype(np.float32), ids32, p.astype(np.float32), k, out)
    assert np.linalg.norm(out - ref) <= 2.0 ** -17 * np.linalg.norm(ref)
    for unfused in (False, True):
        got = np.empty(k, np.uint32)
        ctx.moe_forward(out, x, R, GU, DN, k, F, act=act, norm_topk=True, out_ids=got, unfused=unfused)
        assert got.tolist() == ids.tolist()
        assert np.linalg.norm(out - ref) <= 2.0 ** -17 * np.linalg.norm(ref)
    for t in (GU, DN, R):
        t.free()
