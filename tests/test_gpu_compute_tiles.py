"""hh_linear through every one of its kernels, tile shapes and splits of k
(test_host_compute_shapes.py asserts which shape takes which), with the whole
epilogue, against its plain form in 64 bits."""
import numpy as np
import pytest

import compute_ref as R
import test_gpu_compute as G
from compute_shapes import cases

pytestmark = pytest.mark.gpu


def act(z, name):
    t = G.T()
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + t.erf(z / 2 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + t.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + t.exp(-z))
    return z


def rows_of(shape, dtype, gen, pad, size=1.0):
    """Random rows, `pad` values apart that are no part of them."""
    t = G.T()
    wide = t.full((shape[0], shape[1] + pad), float("nan"), dtype=G.tdt(dtype), device="cuda")
    wide[:, :shape[1]] = (t.randn(shape, generator=gen, device="cuda") * size).to(G.tdt(dtype))
    return wide[:, :shape[1]]


def check(m, n, k, weight, dtype, out, name, epilogue=True, pad=0):
    import haagenti_amd as H
    t, K = G.T(), G.K()
    gen = t.Generator("cuda").manual_seed(m + 3 * n + 7 * k)
    x = rows_of((m, k), dtype, gen, pad)
    if weight == "int4":
        w0 = t.randn((n, k), generator=gen, device="cuda").mul(0.05).cpu().numpy()
        buf = H.quantize_int4(w0.reshape(-1))
        q, s = (t.from_numpy(a).cuda() for a in R.int4_parts(buf, n, k))
        w, wv, mag = K.Int4Weight(t.from_numpy(buf.copy()).cuda(), n, k), q * s, 55.0 * s  # 16 + nibble and 24 summed apart
    else:
        w = rows_of((n, k), dtype, gen, pad, 0.05)
        wv = w.double()
        mag = wv.abs()
    b = c = d = None
    if epilogue:
        b = rows_of((1, n), dtype, gen, 0)[0]
        c, d = rows_of((m, n), dtype, gen, pad), rows_of((m, n), dtype, gen, pad)
    print(f"linear {m}x{n}x{k} {dtype} {weight} {name} to {out}", flush=True)
    y = K.linear(G.ctx(), x, w, bias=b, act=name, mul=c, residual=d, out_dtype=G.tdt(out))
    xv = x.double()
    bv, cv, dv = (0.0 if b is None else b.double(), 1.0 if c is None else c.double(), 0.0 if d is None else d.double())
    z = xv @ wv.t().contiguous() + bv
    want = act(z, name) * cv + dv
    # f32 sums of k terms and the bias; activations have slopes below 1.13 and are computed to 2^-20; then the
    # epilogue's roundings and half a unit of the output
    sums = (k + 40) * 2.0 ** -24 * (xv.abs() @ mag.t().contiguous() + (0.0 if b is None else bv.abs()))
    err = 1.13 * sums + 2.0 ** -20 * z.abs()
    if epilogue:
        err = err * cv.abs() + 2.0 ** -22 * (want.abs() + dv.abs())
    else:
        err = err + 2.0 ** -22 * want.abs()
    bits, least = {"f16": (10, -24), "bf16": (7, -133), "f32": (23, -149)}[out]
    e = t.floor(t.log2((want.abs() + err).clamp(min=1e-300)))
    half = t.exp2((e - bits).clamp(min=least) - 1)
    off = (y.double() - want).abs()
    assert y.shape == (m, n) and y.dtype == G.tdt(out)
    assert bool((off <= err + half).all()), float((off - err - half).max())


@pytest.mark.parametrize("m,n,k,weight", [c[:4] for c in cases()])
def test_every_kernel(m, n, k, weight):
    check(m, n, k, weight, "bf16", "bf16", "silu")
    check(m, n, k, weight, "f16", "f32", "gelu")


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,n,k", [(35, 44, 192), (34, 40, 2240), (150, 1132, 192), (300, 520, 64)])
def test_aligned_epilogues(m, n, k, name):
    check(m, n, k, "same", "bf16", "f32", name)
    check(m, n, k, "same", "f16", "f16", name)
    check(m, n, k, "same", "bf16", "bf16", name, epilogue=False)


@pytest.mark.parametrize("m,n,k", [(35, 44, 192), (34, 41, 2176), (129, 967, 192)])
@pytest.mark.parametrize("pad", [1, 4, 8, 24])
def test_aligned_and_other_strides(m, n, k, pad):
    check(m, n, k, "same", "bf16", "bf16", "none", pad=pad)


@pytest.mark.parametrize("k", [64, 128, 192, 256, 320])
@pytest.mark.parametrize("m,n", [(33, 128), (64, 300), (257, 256)])
def test_steps_of_aligned_tiles(m, n, k):
    check(m, n, k, "same", "f16", "f16", "none", epilogue=False)
