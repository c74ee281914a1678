"""MXFP4 without a GPU: the numpy reference against the format's definition,
sizes, the binding's own checks, and null arguments at the C entries."""
import ctypes as C

import numpy as np
import pytest

import llmtoy_amd as lt
import mx_reference as mx
from llmtoy_amd import ggml, gguf, synth
from llmtoy_amd import lib as ltlib


def test_block_known_answer():
    b = np.zeros(17, np.uint8)
    b[0] = 128  # 2^1
    b[1] = 0x17  # element 0: code 7 (6), element 16: code 1 (.5)
    b[16] = 0xFA  # element 15: code 10 (-1), element 31: code 15 (-6)
    v = mx.decode(b, 32)
    assert (v[0], v[16], v[15], v[31]) == (12.0, 1.0, -2.0, -12.0)
    assert np.count_nonzero(v) == 4
    b[0] = 255
    assert np.isnan(mx.decode(b, 32)).all()


def test_reference_quantisation_ties_and_ends():
    x = np.zeros(32, np.float32)
    # the largest is 4: scale 1; ties go to the even code
    x[:12] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, -.25, -1.75, .2500001, .7499999, -3.5]
    v = mx.decode(mx.quantize(x), 32)
    assert v[:12].tolist() == [4, 0, 1, 1, 2, 2, 4, 0, -2, .5, .5, -4]
    x[0] = 7.9  # beyond 6
    assert mx.decode(mx.quantize(x), 32)[0] == 6
    assert mx.quantize(np.zeros(32, np.float32)).tolist() == [0] * 17
    x[3] = np.inf
    assert mx.quantize(x).tolist() == [255] + [0] * 16


def test_reference_quantisation_is_the_nearest_value():
    x = synth.normal(synth.stream(91, 1), (64, 96))
    b = mx.quantize(x)
    v, x64 = mx.decode(b, 96).reshape(-1, 32), x.astype(np.float64).reshape(-1, 32)
    unit = np.ldexp(1.0, b.reshape(-1, 17)[:, :1].astype(np.int32) - 127)
    grid = np.concatenate([mx.MAGNITUDES, -mx.MAGNITUDES])
    best = np.abs(x64[..., None] - grid * unit[..., None]).min(-1)
    assert (np.abs(v - x64) == best).all()


def test_row_bytes_and_gguf_size():
    assert ggml.row_bytes(ggml.MXFP4, 2816) == 88 * 17
    m = synth.quant_matrix(synth.stream(91, 2), ggml.MXFP4, 3, 64)
    assert m.shape == (3, 34) and m.dtype == np.uint8


def bare_context():
    c = lt.Context.__new__(lt.Context)
    c.lib, c.ptr = lt.load_library(), None
    return c


def tensor(ctx, rows, cols):
    return lt.Tensor(ctx, None, ggml.MXFP4, rows, cols, 1)


@pytest.mark.parametrize("call", [
    lambda c, t: c.quantize(t, np.zeros((2, 32), np.float32)),           # rows of another length
    lambda c, t: c.quantize(t, np.zeros((2, 64), np.float64)),           # another type
    lambda c, t: c.quantize(t, np.zeros((2, 2, 64), np.float32)),        # another rank
    lambda c, t: c.quantize(t, np.zeros((64, 2), np.float32).T),         # not contiguous
    lambda c, t: c.dequantize(np.zeros((2, 65), np.float32), t),
    lambda c, t: c.quant_matmul(np.zeros((2, 8), np.float32), t, np.zeros((3, 64), np.float32)),
    lambda c, t: c.quant_matmul(np.zeros((2, 9), np.float32), t, np.zeros((2, 64), np.float32)),
    lambda c, t: c.quant_matmul(np.zeros((2, 8), np.float16), t, np.zeros((2, 64), np.float32)),
    lambda c, t: c.quant_matmul(np.zeros((2, 16), np.float32)[:, ::2], t, np.zeros((2, 64), np.float32)),
])
def test_binding_refuses_before_the_library_is_called(call):
    c = bare_context()
    with pytest.raises(ltlib.InvalidError):
        call(c, tensor(c, 8, 64))


def test_null_arguments_are_invalid():
    L, out = lt.load_library(), C.c_void_p()
    assert L.lt_tensor_create(None, ggml.MXFP4, 1, 32, 1, C.byref(out)) == ltlib.LT_ERR_INVALID
    assert L.lt_quantize(None, None, None, 0, 1, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_dequantize(None, None, None, 0, 1, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_matmul(None, None, None, None, 1, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_matmul_quantized(None, None, None, None, 1, 0) == ltlib.LT_ERR_INVALID


def test_gguf_reader_knows_the_type(tmp_path):
    m = synth.quant_matrix(synth.stream(91, 3), ggml.MXFP4, 5, 96)
    path = str(tmp_path / "m.gguf")
    w = gguf.GgufWriter()
    w.add_tensor("blk.0.w", (96, 5), ggml.MXFP4, m)
    w.write(path)
    r = gguf.GgufReader(path)
    got = r.raw_matrix("blk.0.w", 5, 96)
    assert got.type == ggml.MXFP4 and np.array_equal(np.asarray(got.data).reshape(-1), m.reshape(-1))
