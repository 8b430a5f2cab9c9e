"""Rows that differential attention has no tokens for are zeros, whatever the
norm's weight is."""
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_zeros(bad, rows):
    t = G.T()
    c = G.new_cache(3, 16, 1, 64, 0)[0]
    q, lam = t.ones(rows, 2, 64, dtype=t.bfloat16, device="cuda"), t.ones(2, device="cuda")
    for eps in (0.0, 1e-5):
        o = c.diff_attention(q, lam, G.i32([[-1, -1]]), G.i32([0, rows]), G.i32([30]), norm_weight=t.full((64,), bad, device="cuda"),
                             eps=eps)
        assert (o == 0).all()


def test_zeros_where_chunks_are_joined():
    t = G.T()
    c = G.new_cache(3, 16, 1, 64, 0)[0]
    q, lam = t.ones(1, 2, 64, dtype=t.bfloat16, device="cuda"), t.ones(2, device="cuda")
    o = c.diff_attention(q, lam, t.full((1, 300), -1, dtype=t.int32, device="cuda"), G.i32([0, 1]), G.i32([4800]),
                         norm_weight=t.full((64,), float("nan"), device="cuda"))
    assert (o == 0).all()
