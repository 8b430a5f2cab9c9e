"""Differential attention where the two maps nearly cancel, so that what their
probabilities are off by is a large part of the output: against the 64-bit
form with 22 bits a probability, for few and for many rows."""
import numpy as np
import pytest

import compute_ref as R
import test_gpu_compute as G
from test_gpu_diff_attention import differ

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,tokens,q_heads,heads", [(1, 40, 4, 2), (4, 40, 2, 1), (9, 9, 1, 1), (40, 40, 4, 2), (60, 200, 4, 1),
                                                       (150, 150, 2, 2)])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,norm", [("f16", False), ("f16", True), ("bf16", False)])
def test_maps_that_nearly_cancel(dtype, norm, dim, rows, tokens, q_heads, heads):
    t, rng = G.T(), np.random.default_rng(rows + dim)
    bs = 32
    blocks, half = (tokens + bs - 1) // bs, dim // 2
    c, kq, vq, ks, vs = G.new_cache(blocks, bs, heads, dim, rows + dim)
    # the second map's keys are the first's but for one code in 16, the queries of both alike
    kq[..., half:] = kq[..., :half]
    change = rng.random(kq[..., half:].shape) < 1 / 16
    kq[..., half:] = np.clip(kq[..., half:] + change * rng.integers(-8, 9, change.shape), -127, 127)
    c.k.copy_(t.from_numpy((kq + 128).astype(np.uint8)))
    q = rng.normal(0, 1, (rows, q_heads, dim))
    q[..., half:] = q[..., :half]
    qt, qv = G.dev(q, dtype)
    lt, lv = G.dev(np.ones(q_heads), "f32")
    wt, wv = G.dev(1 + 0.3 * rng.normal(size=dim), "f32") if norm else (None, None)
    print(f"diff bits {rows} of {tokens} {q_heads}/{heads}x{dim} {dtype}", flush=True)
    o = c.diff_attention(qt, lt, G.i32(np.arange(blocks)[None]), G.i32([0, rows]), G.i32([tokens]), norm_weight=wt, eps=1e-5,
                         gain=0.7)
    key = (kq * ks[:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:tokens]
    val = (vq * vs[:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:tokens]
    want, err = differ(qv, key, val, tokens, half ** -0.5, lv, wv, 1e-5, 0.7, 22, 127 * float(vs.max()))
    off = np.abs(G.f64(o) - want)
    assert (off <= err + R.half_ulp(np.abs(want) + err, dtype)).all(), float((off - err).max())
