"""What the binding refuses before a device is asked."""
import numpy as np
import pytest

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
