"""What the binding refuses before a device is asked."""
import numpy as np
import pytest
import torch

from llmtoy_amd import lib as ltlib
from llmtoy_amd.lib import InvalidError


def test_tokens_a_stride_of_no_whole_floats_apart():
    rec = np.zeros(5, [("heads", np.float32, (2, 64)), ("mark", np.uint8, 2)])
    assert rec["heads"].strides[0] == 514
    with pytest.raises(InvalidError, match="in a row"):
        ltlib._heads(rec["heads"], "a")
    one = np.zeros(5, [("heads", np.float32, (2, 64)), ("mark", np.float32, 3)])["heads"]
    assert ltlib._heads(one, "a")[2:] == (5, 2, 64, 131)
    assert ltlib._heads(rec["heads"][:1], "a")[2:] == (1, 2, 64, 128)  # (a single token has no stride)


class _Elsewhere:
    """A torch tensor's face, on another device."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device = shape, dtype, device
        self.is_cuda = device >= 0

    def numel(self):
        return int(np.prod(self.shape))

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    is_contiguous = lambda self: True  # noqa: E731
    data_ptr = lambda self: 64  # noqa: E731
    get_device = lambda self: self.device  # noqa: E731


_Elsewhere.__module__ = "torch"


def test_arrays_on_another_device_or_on_none():
    f32, i32 = torch.float32, torch.int32
    c = ltlib.Context.__new__(ltlib.Context)  # (no device is asked: every call is refused before)
    c.ptr, c.lib, c.device = None, None, 0
    cache, rope = ltlib.KvCache(c, None, 4, 2, 64, 3), ltlib.Rope(c, None, 64)
    t = _Elsewhere
    batch = lambda d: ltlib.KvBatch(t((4,), i32, d), t((3,), i32, d), t((3, 2), i32, d), 5)  # noqa: E731
    h = lambda n, d: t((5, n, 64), f32, d)  # noqa: E731
    w = lambda n, d: t((n,), i32, d)  # noqa: E731
    for at, other, what in ((1, 0, "an array on device 1"), (0, 1, "an array on device 1"), (1, 1, "an array on device 1"),
                            (-1, 0, "mix of host"), (0, -1, "mix of host"), (-1, 1, "mix of host")):
        for call in (lambda: c.attention(h(4, at), h(4, other), cache, batch(other), 1.0),
                     lambda: c.attention(h(4, other), h(4, other), cache, batch(at), 1.0),
                     lambda: cache.append(h(2, other), h(2, at), batch(other)),
                     lambda: cache.read(h(2, other), h(2, at), w(5, other)),
                     lambda: cache.read(h(2, other), h(2, other), w(5, at)),
                     lambda: c.qk_norm_rope(h(4, other), h(2, at), h(4, other), h(2, other), None, None, w(5, other), rope),
                     lambda: c.qk_norm_rope(h(4, other), None, h(4, other), None, t((64,), f32, at), None, w(5, other), rope),
                     lambda: c.qk_norm_rope(h(4, other), None, h(4, other), None, None, None, w(5, at), rope),
                     lambda: c.kv_plan(batch(other), *[w(n, other) for n in (3, 3, 9, 1, 1, 5)], w(5, at)),
                     lambda: c.kv_plan(batch(at), *[w(n, other) for n in (3, 3, 9, 1, 1, 5, 5)])):
            with pytest.raises(InvalidError, match=what):
                call()
