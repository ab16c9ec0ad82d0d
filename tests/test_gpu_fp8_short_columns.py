"""8-bit products whose columns end inside the first blocks that a workgroup loads at a time, one weight row left in the
last tile: the loads of the blocks behind lie outside the weights' buffer and give zeros."""
import pytest

from test_gpu_fp8_matmul import dense, grouped

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [16, 112, 144, 272, 400, 528, 656, 784, 912, 1040])
@pytest.mark.parametrize("T,rows", [(3, 33), (40, 4129), (130, 1505), (300, 2049), (700, 801)])
def test_one_matrix(T, rows, cols):
    dense(T, rows, cols, "f32", residual=True, seed=cols)


@pytest.mark.parametrize("cols", [16, 144, 272, 400, 912])
@pytest.mark.parametrize("T,rows,y", [(2, 16, "e4m3"), (60, 272, "e4m3"), (40, 2065, "f32"), (300, 2049, "bf16")])
def test_gated(T, rows, y, cols):
    dense(T, rows, cols, y, "silu", glu=True, seed=cols)


@pytest.mark.parametrize("cols", [16, 144, 400, 912])
@pytest.mark.parametrize("G,n,rows,y,glu", [(20, 60, 33, "f32", False), (24, 900, 529, "f32", True), (12, 300, 272, "e4m3", True),
                                            (8, 540, 513, "f16", False)])
def test_groups(G, n, rows, y, glu, cols):
    grouped(G, n, rows, cols, y, glu, "gather", seed=cols)
