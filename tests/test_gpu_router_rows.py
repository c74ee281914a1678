"""The F32 router's row pairs at rows of 32 elements a stride, not only of 256:
dotf32's chains end inside a load's 16 strides."""
import pytest

import test_gpu_parity as parity

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,D", [(1, 32), (3, 96), (64, 1056), (130, 2880), (33, 480), (7, 544), (20, 2784), (9, 16352),
                                 (257, 2080), (1024, 224)])
def test_gpu_router_rows_of_32_bit_exact(ctx, E, D):
    parity.test_gpu_router_row_pairs_bit_exact(ctx, E, D)
