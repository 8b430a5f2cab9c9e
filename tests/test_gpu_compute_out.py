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


def test_linear_refuses_outputs_over_its_inputs():
    t, H, k = G.T(), __import__("haagenti_amd"), G.K()
    buf = t.randn(70, 400, device="cuda").bfloat16()
    x, w, kept = buf[:64, :64], t.randn(64, 64, device="cuda").bfloat16(), buf.clone()
    bias, wide = t.randn(64, device="cuda").bfloat16(), t.randn(64, 128, device="cuda").bfloat16()
    int4 = k.Int4Weight(t.zeros(64 * 36, dtype=t.uint8, device="cuda"), 64, 64)
    bad = [
        dict(out=x), dict(out=buf[:1, :64].expand(64, 64)), dict(out=buf[:64, 63:127]), dict(out=buf[1:65, :64]), dict(w=w, out=w),
        dict(bias=w[3], out=w), dict(residual=wide[:, :64], out=wide[:, 1:65]),
        dict(mul=wide[:, :64], out=wide.view(128, 64)[:64]),
        dict(w=int4, out=int4.data.view(t.bfloat16)[:1024].as_strided((16, 64), (64, 1)), m=16),
    ]
    for a in bad:
        a = dict(a)
        m = a.pop("m", 64)
        with pytest.raises(H.HaagentiError) as e:
            k.linear(G.ctx(), x[:m], a.pop("w", w), **a)
        assert e.value.code == H.INVALID_ARGUMENT
    assert t.equal(buf, kept)


@pytest.mark.parametrize("m", [1, 5, 64])
def test_linear_beside_its_inputs_and_into_what_it_adds(m):
    t, k = G.T(), G.K()
    buf = t.randn(64, 400, device="cuda").bfloat16()
    w, kept = t.randn(64, 64, device="cuda").bfloat16(), buf.clone()
    for at in (64, 200, 336):
        x, out = buf[:m, :64], buf[:m, at:at + 64]
        want = k.linear(G.ctx(), x, w, residual=out)
        assert t.equal(k.linear(G.ctx(), x, w, residual=out, out=out), want)
        want = k.linear(G.ctx(), x, w, mul=out)
        assert t.equal(k.linear(G.ctx(), x, w, mul=out, out=out), want)
        assert t.equal(buf[:, :64], kept[:, :64])
    full = t.randn(80, 64, device="cuda").bfloat16()
    want = k.linear(G.ctx(), full[:8], w)
    assert t.equal(k.linear(G.ctx(), full[:8], w, out=full[8:16]), want)
