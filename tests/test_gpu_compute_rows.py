"""Attention's rows that no request computes: outputs that held something
else are zeros afterwards."""
import numpy as np
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def filled(rows, heads, dim, pad=0):
    t = G.T()
    return t.full((rows, heads, dim + pad), float("nan"), dtype=t.bfloat16, device="cuda")[:, :, :dim]


@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("rows", [1, 7, 5000])
def test_no_requests(rows, dim):
    t = G.T()
    c = G.new_cache(3, 16, 2, dim, 0)[0]
    q, out = t.randn(rows, 4, dim, device="cuda").bfloat16(), filled(rows, 4, dim, 3)
    o = c.attention(q, G.i32(np.zeros((0, 2))), G.i32([0]), G.i32([]), out=out)
    assert o is out and (o == 0).all()
    o = c.attention(q, G.i32(np.zeros((0, 0))), G.i32([0]), G.i32([]))
    assert (o == 0).all()


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("bound", [0, 1, 3, 20])
def test_rows_beyond_the_bound(bound, pad):
    t = G.T()
    c = G.new_cache(12, 16, 2, 64, 0)[0]
    table, start, lens = G.i32(np.arange(12).reshape(3, 4)), [0, 2, 32, 36], G.i32([50, 60, 4])
    q = t.randn(36, 8, 64, device="cuda").bfloat16()
    whole = c.attention(q, table, G.i32(start), lens)
    o = c.attention(q, table, G.i32(start), lens, max_q=bound, out=filled(36, 8, 64, pad))
    for a, b in zip(start, start[1:]):
        n = min(b - a, bound)
        # another bound may take other tiles; each row's error is that of one rounding more
        assert t.allclose(o[a:a + n].float(), whole[a:a + n].float(), rtol=2.0 ** -7, atol=2.0 ** -9)
        assert (o[a + n:b] == 0).all()


def test_rows_before_the_first_request_and_past_the_last():
    t = G.T()
    c = G.new_cache(6, 16, 2, 64, 0)[0]
    table, lens = G.i32([[0, 1, 2], [3, 4, 5]]), G.i32([40, 33])
    q = t.randn(50, 4, 64, device="cuda").half()
    out = t.full((50, 4, 64), float("nan"), dtype=t.float16, device="cuda")
    o = c.attention(q, table, G.i32([5, 6, 39]), lens, out=out)
    want = c.attention(q[5:39], table, G.i32([0, 1, 34]), lens)
    assert (o[:5] == 0).all() and (o[39:] == 0).all() and t.equal(o[5:39], want)
