"""The MXFP4 layer: which shapes are one launch, routing and activations that are not finite,
waits that end at their limit."""
import re

import numpy as np
import pytest

import llmtoy_amd as lt
from llmtoy_amd import ggml, synth
from llmtoy_amd import lib as ltlib
from llmtoy_amd.hip import DeviceArray, Graph
from test_gpu_mxfp4 import acts, close, expert_ref, experts, gen, route

pytestmark = pytest.mark.gpu

MX = ggml.MXFP4


def layer(c, g, E, D, F):
    r = (g.standard_normal((E, D)) * 0.05).astype(np.float32)
    return (c.upload(r, ggml.F32, E, D), c.upload(synth.quant_matrix(g, MX, E * 2 * F, D), MX, 2 * F, D, E),
            c.upload(synth.quant_matrix(g, MX, E * D, F), MX, D, F, E))


def test_gpu_mx_layer_names_the_waits_that_ran_out(ctx, monkeypatch):
    # every wait ends at its first look: 128 rows of the router take 2 us, which the gate/up and the
    # down workgroups, 84 of them to an XCD and so all there at once, look for within the first
    E, D, F, k = 128, 2048, 768, 8
    x = acts(gen(51), D)
    monkeypatch.setenv("LT_MX_WAIT_TICKS", "0")
    with lt.Context(0) as c:
        ts, out, ids, w = layer(c, gen(52), E, D, F), np.zeros(D, np.float32), np.zeros(k, np.uint32), np.zeros(k, np.float32)
        for _ in range(3):  # the error is cleared, and comes again
            with pytest.raises(ltlib.DeviceError) as e:
                c.moe_forward(out, x, *ts, k, F)
            text = str(e.value)
            code = int(re.search(r"code 0x([0-9a-f]+):", text).group(1), 16)
            site = int(re.search(r"site 0x([0-9a-f]+), word and tag not recorded,", text).group(1), 16)
            # 1 logits for gate/up, 2 logits for down, 4 h, 8 the other slots' rows
            assert code & 3 == 3 and code & ~15 == 0, text
            assert site and site & code == site, text
            assert np.isnan(out).all()
        c.moe_forward(out, x, *ts, k, F, unfused=True)
        want = out.copy()
        for t in ts:
            t.free()
    monkeypatch.delenv("LT_MX_WAIT_TICKS")
    ts = layer(ctx, gen(52), E, D, F)
    ctx.moe_forward(out, x, *ts, k, F)
    assert np.linalg.norm(out - want) <= 2.0 ** -18 * np.linalg.norm(want)
    for t in ts:
        t.free()


# (E, D, F, Kd, k): those that test_gpu_mx_moe_one_launch computes, and larger ones
ONE = [(6, 256, 40, 64, 6), (7, 512, 32, 32, 7), (128, 2048, 96, 96, 8), (256, 256, 160, 160, 8), (40, 768, 80, 544, 14), (255, 256, 64, 64, 15),
       (16, 1280, 48, 64, 16), (9, 16384, 16, 32, 6), (9, 256, 4100, 4128, 8), (8, 2880, 96, 96, 8), (7, 96, 32, 32, 7), (20, 32, 64, 64, 3),
       (60, 1056, 64, 64, 6), (33, 544, 64, 64, 9), (4, 224, 32, 32, 1), (16, 2048, 768, 768, 8), (8, 2816, 2112, 2112, 8)]
THREE = [(8, 2816, 2112, 2112, 4), (16, 2048, 768, 768, 10), (300, 256, 64, 64, 8), (8, 2880, 1024, 1024, 6)]


def test_gpu_mx_layer_one_launch_or_three(ctx):
    # the hand-over memory of a shape's single launch is set up by its first call, which therefore
    # cannot be captured; three launches can be
    x, y = DeviceArray((16384,)), DeviceArray((16384,))
    with lt.Context(0) as c:
        for shapes, refused in ((ONE, True), (THREE, False)):
            for E, D, F, Kd, k in shapes:
                ts = (c.upload(np.zeros((E, D), np.float32), ggml.F32, E, D), c.create(MX, 2 * F, D, E), c.create(MX, D, Kd, E))
                seen = []

                def first():
                    try:
                        c.moe_forward(y, x, *ts, k, F)
                        seen.append(False)
                    except ltlib.InvalidError:
                        seen.append(True)

                Graph(c.stream, first).destroy()
                assert seen == [refused], (E, D, F, Kd, k)
                for t in ts:
                    t.free()
    x.free(), y.free()


@pytest.mark.parametrize("unfused", [False, True])
@pytest.mark.parametrize("E,k", [(9, 8), (200, 8), (300, 6)])
def test_gpu_mx_layer_not_finite(ctx, E, k, unfused):
    print(f"not finite E {E} k {k} unfused {unfused}", flush=True)
    D, F = 256, 64
    g = gen(E, k, 53)
    GU, DN, w = experts(ctx, g, E, D, F)
    r, x = (g.standard_normal((E, D)) * 0.05).astype(np.float32), acts(g, D)
    x[7] = 1.0
    out, ids, p = np.empty(D, np.float32), np.empty(k, np.uint32), np.empty(k, np.float32)

    def call(r, x):
        R = ctx.upload(r, ggml.F32, E, D)
        ctx.moe_forward(out, x, R, GU, DN, k, F, norm_topk=True, out_ids=ids, out_w=p, unfused=unfused)
        R.free()
        assert len(set(ids.tolist())) == k and (ids < E).all()

    def finite(r, x, logits):
        call(r, x)
        want, wts = route(logits, k, True)
        assert ids.tolist() == want.tolist()
        _, ref, bound = expert_ref(w, x, want, wts, F, 0)
        slack = 2 * (D * 2.0 ** -24 * (np.abs(r[want].astype(np.float64)) @ np.abs(x)).max() + 2.0 ** -20)  # the weights', as in the layer's tests
        close(out, ref, bound + slack * np.abs(ref) + slack * sum(q * np.abs(w["dn"][e]).sum(1) for e, q in zip(want, wts)))

    logits = r.astype(np.float64) @ x
    finite(r, x, logits)
    for bad in (np.nan, np.inf, -np.inf):
        b = x.copy()
        b[100] = bad
        call(r, b)
        assert np.isnan(out).all()
    every = np.full_like(r, np.nan)  # all logits rank as -inf: the lowest indices
    call(every, x)
    assert ids.tolist() == list(range(k)) and np.isnan(p).all() and np.isnan(out).all()
    for bad in (np.nan, -np.inf):  # one expert's logit: it is not selected, the others as ever
        b, best = r.copy(), int(np.argmax(logits))
        b[best, 7] = bad
        rest = logits.copy()
        rest[best] = -np.inf
        finite(b, x, rest)
    b = r.copy()  # +inf: it is selected first, and no weight is a number
    b[E - 1, 7] = np.inf
    call(b, x)
    assert ids[0] == E - 1 and np.isnan(out).all()
    finite(r, x, logits)
    GU.free(), DN.free()


@pytest.mark.parametrize("unfused", [False, True])
@pytest.mark.parametrize("E,D,F,Kd,k", [(1, 96, 1, 32, 1), (8, 64, 5, 64, 8), (9, 512, 33, 64, 7), (16, 2048, 96, 96, 16)])
def test_gpu_mx_layer_into_its_own_input(ctx, E, D, F, Kd, k, unfused):
    # x += layer(x) on the device, experts of one row and of odd numbers of them, one expert
    print(f"in place E {E} D {D} F {F} Kd {Kd} k {k} unfused {unfused}", flush=True)
    g = gen(E, D, F, k, 54)
    GU, DN, w = experts(ctx, g, E, D, F, Kd)
    r, x = (g.standard_normal((E, D)) * 0.05).astype(np.float32), acts(g, D)
    R, d = ctx.upload(r, ggml.F32, E, D), DeviceArray.from_numpy(x)
    for accumulate in (True, False):
        now = d.numpy()
        ids, p = route(r.astype(np.float64) @ now.astype(np.float64), k, True)
        _, ref, bound = expert_ref(w, now, ids, p, F, 0)
        ctx.moe_forward(d, d, R, GU, DN, k, F, norm_topk=True, accumulate=accumulate, unfused=unfused)
        ctx.sync()
        want = ref + now if accumulate else ref
        slack = 2 * (D * 2.0 ** -24 * (np.abs(r.astype(np.float64)) @ np.abs(now)).max() + 2.0 ** -20)  # the weights', as in the layer's tests
        close(d.numpy(), want, bound + slack * np.abs(ref) + slack * sum(q * np.abs(w["dn"][e]).sum(1) for e, q in zip(ids, p))
              + 2.0 ** -23 * (np.abs(now) + np.abs(ref)))
    for t in (GU, DN, R, d):
        t.free()
