"""The attention operators without a GPU: the reference against itself, the
binding's refusals, and the counting rules that the kernels' grids and
workspaces rest on."""
import ctypes as C
import math
import random

import numpy as np
import pytest

import attn_reference as ref
import llmtoy_amd as lt
from llmtoy_amd import lib as ltlib
from llmtoy_amd.lib import InvalidError


# ------------------------------------------------------------------ the reference
def test_codes_of_ties_and_special_blocks():
    x = np.zeros((2, 4), np.float32)
    x[0] = [127, 0.5, 1.5, -2.5]
    c, s = ref.codes(x)
    assert s == 1 and c[0].tolist() == [127, 0, 2, -2]
    assert ref.codes(np.zeros((3, 4)))[1] == 0
    x[1, 1] = np.inf
    assert np.isnan(ref.codes(x)[1])
    tiny = np.full((1, 4), 1e-45, np.float32)  # the scale rounds to nothing
    assert ref.codes(tiny)[1] == 0


@pytest.mark.parametrize("style", ["neox", "pairs"])
def test_rotation_keeps_lengths_and_depends_on_differences(style):
    g = np.random.default_rng(3)
    q, k = g.standard_normal((2, 1, 1, 64)).astype(np.float32)
    dots = []
    for p in (0, 5, 70000):
        a, _ = ref.rope(q, None, [p + 9], 64, 1e4, style, norm=False)
        b, _ = ref.rope(k, None, [p], 64, 1e4, style, norm=False)
        assert math.isclose((a * a).sum(), (q.astype(np.float64) ** 2).sum(), rel_tol=1e-12)
        dots.append((a * b).sum())
    assert np.allclose(dots, dots[0], rtol=1e-9)


def test_attention_of_one_key_is_its_value():
    g = np.random.default_rng(4)
    q, k, v = g.standard_normal((1, 4, 64)), g.standard_normal((3, 2, 64)), g.standard_normal((3, 2, 64))
    out, _ = ref.attention(q, k, v, [2], 0.1, window=1)
    assert np.allclose(out[0], np.repeat(v[2], 2, 0))


# ------------------------------------------------------------------ counting rules
def _row(bases, u):
    """kv_row's answer: the last row whose base is at most u."""
    return max((i for i, b in enumerate(bases) if b <= u), default=0)


def test_append_units_reach_every_block():
    r = random.Random(5)
    for _ in range(400):
        n = r.randint(1, 9)
        new = [r.choice([0, 1, 2, 31, 32, 33, r.randint(0, 200)]) for _ in range(n)]
        past = [r.randint(0, 100) for _ in range(n)]
        start = [sum(new[:i]) for i in range(n + 1)]
        bases = [start[i] // 32 + 2 * i for i in range(n)]
        units = (start[n] + r.randint(0, 40)) // 32 + 2 * n
        got = set()
        for u in range(units):
            i = _row(bases, u)
            if not new[i]:
                continue
            j = u - bases[i] + past[i] // 32
            if past[i] // 32 <= j <= (past[i] + new[i] - 1) // 32:
                assert (i, j) not in got
                got.add((i, j))
        want = {(i, p // 32) for i in range(n) for p in range(past[i], past[i] + new[i])}
        assert got == want


def test_parts_of_split_rows_fit_their_workspace():
    r = random.Random(6)
    target = 512
    for _ in range(300):
        heads = r.choice([1, 2, 3, 4, 8, 64, 256])
        rows = [(r.randint(0, 5), r.choice([1, 2, 40, r.randint(1, 5000)])) for _ in range(r.randint(1, 80))]
        total = sum(t * b for t, b in rows)
        share = max(4, math.ceil(total * heads / target))
        splits = [-(-b // share) for _, b in rows]
        parts = sum(t * s for (t, _), s in zip(rows, splits) if s > 1)
        assert parts <= 2 * (target // heads + 1) + 2
        # workgroups of a head: the tiles and the target's share
        assert sum(t * s for (t, _), s in zip(rows, splits)) <= sum(t for t, _ in rows) + target // heads + 1


# ------------------------------------------------------------------ refusals
def test_null_arguments_are_invalid_without_a_device():
    L = lt.load_library()
    p = C.c_void_p()
    b = ltlib.KvBatchStruct()
    assert L.lt_rope_create(None, 64, 64, 1e4, None, 0, C.byref(p)) == ltlib.LT_ERR_INVALID
    assert L.lt_kv_create(None, 1, 1, 64, 1, C.byref(p)) == ltlib.LT_ERR_INVALID
    assert L.lt_kv_plan(None, C.byref(b), *[None] * 3, 0, *[None] * 4, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_kv_append(None, None, None, None, 0, 0, C.byref(b), 0) == ltlib.LT_ERR_INVALID
    assert L.lt_kv_read(None, None, None, None, None, 0, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_attention(None, None, None, None, C.byref(b), 1, 0, 1.0, 0, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_qk_norm_rope(None, *[None] * 8, 0, 0, 0, 0, 0, 0, 0, 0.0, 0) == ltlib.LT_ERR_INVALID
    assert L.lt_rope_free(None, None) == ltlib.LT_OK and L.lt_kv_free(None, None) == ltlib.LT_OK
    assert L.lt_kv_bytes(None) == 0


def test_batches_of_the_wrong_shape_or_type():
    u = lambda *s: np.zeros(s, np.uint32)  # noqa: E731
    lt.KvBatch(u(4), u(3), u(3, 5), 10)
    with pytest.raises(InvalidError, match="start"):
        lt.KvBatch(u(3), u(3), u(3, 5), 10)
    with pytest.raises(InvalidError, match="table"):
        lt.KvBatch(u(4), u(3), u(2, 5), 10)
    with pytest.raises(InvalidError, match="whole numbers"):
        lt.KvBatch(u(4), u(3).astype(np.int64), u(3, 5), 10)


def test_heads_that_do_not_lie_in_a_row():
    a = np.zeros((5, 4, 64), np.float32)
    assert ltlib._heads(a[:, :2], "a")[2:] == (5, 2, 64, 256)  # a fused projection's part
    with pytest.raises(InvalidError, match="in a row"):
        ltlib._heads(a[:, ::2], "a")
    with pytest.raises(InvalidError, match="in a row"):
        ltlib._heads(a[:, :, ::2], "a")
    with pytest.raises(InvalidError, match="float32"):
        ltlib._heads(a.astype(np.float16), "a")
