"""The accuracy checks of the MXFP4 products reject activations that lost a part."""
import numpy as np
import pytest

import mx_accuracy as acc
import mx_reference as mx
from llmtoy_amd import ggml, synth


def inputs(rows, cols, T, seed):
    g = np.random.default_rng([80, rows, cols, T, seed])
    x = g.standard_normal((T, cols)).astype(np.float32)
    x[:, g.random(cols) < 0.01] *= 10
    return mx.decode(synth.quant_matrix(g, ggml.MXFP4, rows, cols), cols), x


@pytest.mark.parametrize("rows,cols,T", [(130, 1024, 15), (130, 544, 64), (300, 2080, 1), (1030, 288, 40)])
@pytest.mark.parametrize("seed", [0, 1])
def test_l2_limit_needs_every_part(rows, cols, T, seed):
    w, x = inputs(rows, cols, T, seed)
    assert (acc.within_l2(x.astype(np.float64) @ w.T, w, x) == 0).all()
    assert (acc.within_l2(acc.fp6_limbs(x, 5) @ w.T, w, x) < 0.3).all()
    assert (acc.within_l2(acc.fp6_limbs(x, 4) @ w.T, w, x) > 1).all()
    assert (acc.within_l2(acc.bf16_parts(x, 3) @ w.T, w, x) == 0).all()
    assert (acc.within_l2(acc.bf16_parts(x, 2) @ w.T, w, x) > 1).all()


def test_models_keep_what_is_promised():
    x = np.random.default_rng(81).standard_normal((50, 320)).astype(np.float32)
    x64 = x.astype(np.float64)
    assert (acc.bf16_parts(x, 3) == x64).all()
    assert (np.abs(acc.fp6_limbs(x, 5) - x64) <= 2.0 ** -24 * acc.block_tops(x)).all()
    assert (np.abs(acc.fp6_limbs(x, 4) - x64) > 2.0 ** -24 * acc.block_tops(x)).any()


def test_low_bits_need_every_part():
    g = np.random.default_rng(82)
    m, x = acc.low_bits(g, 64, 544, lambda r, c: synth.quant_matrix(g, ggml.MXFP4, r, c), 8)
    w, x64 = mx.decode(m, 544), x.astype(np.float64)
    y, limit = x64 @ w.T, acc.low_bits_limit(w, x)
    assert (np.abs(acc.fp6_limbs(x, 5) @ w.T - y) <= limit).all()
    for lost in (acc.fp6_limbs(x, 4), acc.bf16_parts(x, 1)):
        assert (np.abs(lost @ w.T - y) > limit).mean() > 0.5
