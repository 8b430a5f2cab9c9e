"""Rows that end inside a piece of 16 bytes, on the GPU: every number of values
in the last piece and rows of less than one, with NaN between the rows."""
import pytest

import test_gpu_compute as G
import test_gpu_gated as F
import test_gpu_gated_backward as B
import test_gpu_norm as N

pytestmark = pytest.mark.gpu
ENDS = list(range(1, 18)) + list(range(61, 69)) + list(range(121, 129))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norms(dtype):
    for n in ENDS + [505, 509, 1019, 1021]:
        N.check(5, n, dtype, ["same", "f32", None][n % 3], n % 3 != 2, ["layer", "rms"][n % 2], pad=1 + n % 4)


@pytest.mark.parametrize("dtype", G.DT)
def test_products(dtype):
    for k in ENDS:
        G.check_linear(70 + k % 3, 65 + k % 5, k, dtype, pad=1 + k % 2, bias=True)
        F.check(70 + k % 3, 33 + k % 5, k, dtype, pad=1 + k % 2)


@pytest.mark.parametrize("dtype", G.DT)
def test_products_of_int4_weights(dtype):
    for m, n, k in ((67, 65, 32), (129, 31, 96), (70, 250, 160)):
        G.check_linear(m, n, k, dtype, "int4", pad=3)
        F.check(m, n, k, dtype, "int4", pad=3)


@pytest.mark.parametrize("dtype", G.DT)
def test_gated_gradients(dtype):
    for i in ENDS:
        B.check(3, 5, i, dtype, "silu", pad=1 + i % 2)
        B.check(67, i, 9 + i % 5, dtype, "gelu", pad=1 + i % 2)
        B.check(i, 67, 70 + i % 4, dtype, "silu", pad=1 + i % 2)
