"""Clones of tensors: whole when the call returns, refused while the stream is captured."""
import numpy as np
import pytest

from llmtoy_amd import ggml, synth
from llmtoy_amd import lib as ltlib
from llmtoy_amd.hip import DeviceArray, Graph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [ggml.MXFP4, ggml.Q8_0])
def test_gpu_clone_is_read_at_once(ctx, kind):
    # hundreds of MB, of which the read takes the first 4 MiB first
    rows, cols = 100000, 4096
    part = synth.quant_matrix(np.random.default_rng([78, kind]), kind, 1000, cols)
    m = np.tile(part, (rows // 1000, 1))
    t = ctx.upload(m, kind, rows, cols)
    for _ in range(2):
        c = t.clone()
        assert np.array_equal(c.read(), m.reshape(-1))
        c.free()
    t.free()


def test_gpu_clone_in_a_capture_is_refused(ctx):
    t = ctx.upload(synth.quant_matrix(np.random.default_rng(79), ggml.MXFP4, 64, 256), ggml.MXFP4, 64, 256)
    x, y = DeviceArray.from_numpy(np.ones(256, np.float32)), DeviceArray((64,))
    ctx.quant_matvec(y, t, x)
    ctx.sync()
    want = y.numpy()

    def step():
        with pytest.raises(ltlib.InvalidError):
            t.clone()
        ctx.quant_matvec(y, t, x)

    graph = Graph(ctx.stream, step)
    for _ in range(3):
        graph.launch()
        ctx.sync()
        assert np.array_equal(y.numpy(), want)
    graph.destroy()
    for a in (t, x, y):
        a.free()
