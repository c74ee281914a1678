"""The MXFP4 layer in one launch: waits that end at their limit."""
import re

import numpy as np
import pytest

import llmtoy_amd as lt
from llmtoy_amd import ggml, synth
from llmtoy_amd import lib as ltlib
from test_gpu_mxfp4 import acts, gen

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
            site, index, saw, epoch = re.search(r"site 0x([0-9a-f]+), index (\d+), saw (\d+), expected epoch or count (\d+)", text).groups()
            # 1 logits for gate/up, 2 logits for down, 4 h, 8 the other slots' rows
            assert code & 3 == 3 and code & ~15 == 0, text
            site, index, saw, epoch = int(site, 16), int(index), int(saw), int(epoch)
            assert site in (1, 2, 4, 8) and site & code and saw != epoch, text
            assert index < {1: E, 2: E, 4: k * F, 8: k * D}[site], text
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
