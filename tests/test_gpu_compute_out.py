"""Outputs that a caller gives: rows in other orders, rows that overlap."""
import numpy as np
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def case(rows):
    t = G.T()
    c = G.new_cache(12, 16, 2, 64, 0)[0]
    q = t.randn(2 * rows, 4, 64, device="cuda").bfloat16()
    return c, (q, G.i32(np.arange(12).reshape(2, 6)), G.i32([0, rows, 2 * rows]), G.i32([90, 81]))


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_into_heads_first_and_parts(rows):
    t = G.T()
    c, args = case(rows)
    want = c.attention(*args)
    for out in (t.empty(4, 2 * rows, 64, dtype=t.bfloat16, device="cuda").transpose(0, 1),
                t.empty(2 * rows, 9, 80, dtype=t.bfloat16, device="cuda")[:, 1:8:2, 5:69]):
        assert c.attention(*args, out=out) is out and t.equal(out, want)


def test_attention_refuses_rows_that_overlap():
    t, H = G.T(), __import__("haagenti_amd")
    c, args = case(3)
    flat = t.zeros(6 * 4 * 64, dtype=t.bfloat16, device="cuda")
    for strides in ((0, 64, 1), (256, 0, 1), (256, 63, 1), (128, 64, 1), (64, 64, 1)):
        with pytest.raises(H.HaagentiError) as e:
            c.attention(*args, out=flat.as_strided((6, 4, 64), strides))
        assert e.value.code == H.INVALID_ARGUMENT
    assert (flat == 0).all()
