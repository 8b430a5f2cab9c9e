"""The gated feed-forward's two projections with their activation and product,
on the GPU against their 64-bit form: every kernel, tile shape and split of k,
odd sizes and strides, what is kept for the backward pass, and refusals."""
import numpy as np
import pytest

import compute_ref as R
import gated_shapes
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def weight(rng, n, k, kind, pad, dtype):
    """(what the call takes, its values, the magnitudes that its sums are off by)."""
    import haagenti_amd as H
    w0 = rng.normal(0, 0.05, (n, k))
    if kind == "int4":
        buf = H.quantize_int4(w0.astype(np.float32).reshape(-1)) if n * k else np.zeros(1, np.uint8)
        q, s = R.int4_parts(buf, n, k)
        return G.K().Int4Weight(G.T().from_numpy(buf.copy()).cuda(), n, k), q * s, 55.0 * s
    w, wv = G.padded(w0, pad, dtype)
    return w, wv, np.abs(wv)


def check(m, n, k, dtype="bf16", kind="same", act="silu", bias=True, out=None, pad=0, save=True, seed=0):
    rng = np.random.default_rng(seed + 7 * m + 3 * n + k)
    x, xv = G.padded(rng.normal(0, 1, (m, k)), pad, dtype)
    g, gv, gm = weight(rng, n, k, kind, pad, dtype)
    u, uv, um = weight(rng, n, k, kind, 2 * pad, dtype)
    bg, bgv = G.dev(rng.normal(0, 1, n), dtype) if bias else (None, 0.0)
    bu, buv = G.dev(rng.normal(0, 1, n), dtype) if bias else (None, 0.0)
    od = out or dtype
    print(f"gated {m}x{n}x{k} {dtype} {kind} {act} pad {pad}", flush=True)
    y = G.K().gated_linear(G.ctx(), x, g, u, bg, bu, act=act, save=save, out_dtype=G.tdt(od))
    y, saved = y if save else (y, None)
    zg, zu = xv @ gv.T + bgv, xv @ uv.T + buv
    a = R.act(zg, act)
    # f32 sums of k terms and the bias; activations have slopes below 1.13 and are computed to 2^-20; the product and the
    # output's rounding
    mag = np.abs(xv)
    eg = (k + 40) * 2.0 ** -24 * (mag @ gm.T + np.abs(bgv))
    eu = (k + 40) * 2.0 ** -24 * (mag @ um.T + np.abs(buv))
    ea = 1.13 * eg + 2.0 ** -20 * np.abs(zg)
    err = ea * (np.abs(zu) + eu) + np.abs(a) * eu + 2.0 ** -23 * np.abs(a * zu)
    assert y.shape == (m, n) and y.dtype == G.tdt(od)
    off = np.abs(G.f64(y) - a * zu)
    assert (off <= err + R.half_ulp(np.abs(a * zu) + err, od)).all(), float((off - err).max())
    if save:
        assert saved.shape == (m, 2 * n) and saved.dtype == G.T().float32
        s = G.f64(saved)
        assert (np.abs(s[:, :n] - zg) <= eg + 2.0 ** -23 * np.abs(zg)).all()
        assert (np.abs(s[:, n:] - zu) <= eu + 2.0 ** -23 * np.abs(zu)).all()


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("kind", ["same", "int4"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (1, 1, 1), (3, 17, 33), (16, 128, 128), (17, 100, 96), (33, 65, 1000),
                                   (64, 256, 160), (65, 129, 64), (130, 200, 257), (257, 300, 352), (200, 64, 31), (40, 16, 64)])
def test_shapes(m, n, k, kind, dtype):
    check(m, n, k, dtype, kind)


@pytest.mark.parametrize("m,n,k,kind", [c[:4] for c in gated_shapes.cases()])
def test_every_kernel(m, n, k, kind):
    check(m, n, k, "bf16", kind, bias=n % 2 == 0, seed=1)
    check(m, n, k, "f16", kind, "gelu", out="f32", bias=n % 2 == 1, save=False, seed=2)


@pytest.mark.parametrize("m,n,k", [c[:3] for c in gated_shapes.TWO])
def test_whole_rounds_and_the_rest(m, n, k):
    check(m, n, k, seed=3)
    check(m, n, k, "f16", act="relu", out="f32", bias=False, pad=8, seed=4)


@pytest.mark.parametrize("m", [1, 5, 40, 150])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_activations(m, act):
    check(m, 132, 96, "bf16", act=act)
    check(m, 131, 64, "f16", "int4", act=act, out="f32", pad=3)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("m", [2, 20, 140])
def test_strides(m, pad):
    check(m, 150, 136, "bf16", pad=pad)
    check(m, 150, 128, "f16", bias=False, pad=pad)


@pytest.mark.parametrize("m", [1, 100])
@pytest.mark.parametrize("kind", ["same", "int4"])
def test_no_columns(m, kind):
    check(m, 40, 0, "bf16", kind)


def test_no_rows_and_no_outputs():
    t, k = G.T(), G.K()
    e = lambda *s: t.empty(*s, dtype=t.bfloat16, device="cuda")  # noqa: E731
    y, s = k.gated_linear(G.ctx(), e(0, 64), e(32, 64), e(32, 64), save=True)
    assert y.shape == (0, 32) and s.shape == (0, 64)
    y, s = k.gated_linear(G.ctx(), e(5, 64), e(0, 64), e(0, 64), save=True)
    assert y.shape == (5, 0) and s.shape == (5, 0)


@pytest.mark.parametrize("m,n", [(3, 96), (200, 96), (200, 95)])
def test_into_a_wider_buffer_and_one_bias(m, n):
    t, k = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(m)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    x, wg, wu, b = r(m, 192), r(n, 192) * 0.05, r(n, 192) * 0.05, r(n)
    zero = t.zeros_like(b)
    for biases in ((b, None), (None, b)):
        want = k.gated_linear(G.ctx(), x, wg, wu, *[zero if q is None else q for q in biases])
        wide = t.full((m, n + 7), 3.0, dtype=t.half, device="cuda")
        k.gated_linear(G.ctx(), x, wg, wu, *biases, out=wide[:, 2:n + 2])
        assert t.equal(wide[:, 2:n + 2], want) and (wide[:, :2] == 3).all() and (wide[:, n + 2:] == 3).all()
    shared = k.gated_linear(G.ctx(), x, wg, wg)       # one weight for both
    z = G.f64(x) @ G.f64(wg).T
    assert np.abs(G.f64(shared) - z * z / (1 + np.exp(-z))).max() < 2.0 ** -9 * np.abs(z * z).max()


def test_what_is_not_finite_stays_in_its_row():
    t, k = G.T(), G.K()
    for m in (4, 100):
        x = t.randn(m, 128, device="cuda").to(t.bfloat16)
        w = [t.randn(80, 128, device="cuda").to(t.bfloat16) for _ in range(2)]
        x[1, 5], x[2, 7] = float("nan"), float("inf")
        y = k.gated_linear(G.ctx(), x, *w, act="none")
        assert y[1].isnan().all() and not t.isfinite(y[2]).any()
        assert t.isfinite(y[[i for i in range(m) if i not in (1, 2)]]).all()


def test_streams_and_graphs():
    t, k = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(5)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    sets = [(r(34, 2240), r(20 + i, 2240) * 0.02, r(20 + i, 2240) * 0.02) for i in range(2)]    # k is split
    call = lambda s: k.gated_linear(G.ctx(), *s, save=True)  # noqa: E731
    want = [[y.clone() for y in call(s)] for s in sets]
    streams, got = [t.cuda.Stream(), t.cuda.Stream()], []
    t.cuda.synchronize()
    for _ in range(10):
        for s, st in zip(sets, streams):
            with t.cuda.stream(st):
                got.append(call(s))
    t.cuda.synchronize()
    assert all(t.equal(p, q) for i, y in enumerate(got) for p, q in zip(y, want[i % 2]))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        held = call(sets[0])
    for _ in range(4):
        for y in held:
            y.zero_()
        call(sets[1])
        graph.replay()
        t.cuda.synchronize()
        assert all(t.equal(p, q) for p, q in zip(held, want[0]))


def test_refusals():
    t, k, H, c = G.T(), G.K(), __import__("haagenti_amd"), G.ctx()
    x = t.zeros(4, 64, dtype=t.bfloat16, device="cuda")
    w = t.zeros(32, 64, dtype=t.bfloat16, device="cuda")
    q = k.Int4Weight(t.zeros(32 * 64 // 32 * 18, dtype=t.uint8, device="cuda"), 32, 64)
    short = k.Int4Weight(t.zeros(100, dtype=t.uint8, device="cuda"), 32, 64)
    bad = [
        (lambda: k.gated_linear(c, x.float(), w, w), H.UNSUPPORTED), (lambda: k.gated_linear(c, x, w.half(), w), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, w, w.half()), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x, w, w[:31]), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, w, w[:, :63]), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x, w, q), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, q, w), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x[:, :32], q, q), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, q, k.Int4Weight(q.data, 31, 64)), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, short, q), H.UNEXPECTED_EOF), (lambda: k.gated_linear(c, x, q, short), H.UNEXPECTED_EOF),
        (lambda: k.gated_linear(c, x, w, w, act="swish"), H.UNSUPPORTED),
        (lambda: k.gated_linear(c, x, w, w, gate_bias=x[0, :31]), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, w, w, up_bias=x[0, :32].float()), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, w, w, out_dtype=t.float16), H.UNSUPPORTED),
        (lambda: k.gated_linear(c, x, w, w, out=x), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x, w, w, out=x[:, :32]), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x.cpu(), w, w), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x, w.cpu(), w), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x, w, w.cpu()), H.INVALID_ARGUMENT), (lambda: k.gated_linear(c, x[0], w, w), H.INVALID_ARGUMENT),
        (lambda: k.gated_linear(c, x.clone().requires_grad_(), w, w), H.UNSUPPORTED),
        (lambda: k.gated_linear(c, x, w.clone().requires_grad_(), w), H.UNSUPPORTED),
        (lambda: k.gated_linear(c, x, w, w.clone().requires_grad_()), H.UNSUPPORTED),
    ]
    for i, (call, code) in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            call()
        assert e.value.code == code, i
