"""The gradients of the gated feed-forward's projections on the GPU: whole
numbers through every kernel, tile shape and split (every bit), activations
and biases against their 64-bit forms and against differences, strides,
streams, graphs and refusals."""
import numpy as np
import pytest

import compute_ref as R
import gated_back_shapes
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def slope(z, act):
    """act'(z), 64 bits."""
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "gelu":
        return R.act(z, act) / np.where(z == 0, 1, z) + (z == 0) * 0.5 + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if act == "gelu_tanh":
        c = np.sqrt(2 / np.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        with np.errstate(over="ignore"):
            p = 1 / (1 + np.exp(-z))
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def whole(g, low, high, *shape):
    return G.T().randint(low, high + 1, shape, generator=g, device="cuda").float()


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("m,n,k", gated_back_shapes.SHAPES)
def test_whole_numbers_are_exact(m, n, k, dtype):
    """Every product, sum and dg, du up to 6 is exact, so the outputs are the rounded sums."""
    t, K = G.T(), G.K()
    g, dt = t.Generator("cuda").manual_seed(m + n + k), G.tdt(dtype)
    pad = 8 if k % 8 == 0 else 1
    x, wg, wu = (whole(g, -2, 2, r, k + pad).to(dt)[:, :k] for r in (m, n, n))
    dy, saved = whole(g, -2, 2, m, n + 3).to(dt)[:, :n], whole(g, -3, 3, m, 2 * n)
    print(f"gated backward {m}x{n}x{k} {dtype}", flush=True)
    d = K.gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, act="none", bias=True)
    du, dg = dy.double() * saved[:, :n].double(), dy.double() * saved[:, n:].double()
    dx = dg @ wg.double().contiguous() + du @ wu.double().contiguous()
    assert t.equal(d.dx, dx.to(dt))
    xd = x.double().contiguous()
    assert t.equal(d.dgate, (dg.t().contiguous() @ xd).to(dt)) and t.equal(d.dup, (du.t().contiguous() @ xd).to(dt))
    assert t.equal(d.dgate_bias, dg.sum(0).float()) and t.equal(d.dup_bias, du.sum(0).float())


def check(m, n, k, dtype, act, pad=0, seed=0):
    rng = np.random.default_rng(seed + 7 * m + 3 * n + k)
    x, xv = G.padded(rng.normal(0, 1, (m, k)), pad, dtype)
    wg, gv = G.padded(rng.normal(0, 0.1, (n, k)), pad, dtype)
    wu, uv = G.padded(rng.normal(0, 0.1, (n, k)), 2 * pad, dtype)
    dy, dv = G.padded(rng.normal(0, 1, (m, n)), pad, dtype)
    biases = [G.dev(rng.normal(0, 1, n), dtype)[0] for _ in range(2)]
    y, saved = G.K().gated_linear(G.ctx(), x, wg, wu, *biases, act=act, save=True)
    d = G.K().gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, act=act, bias=True)
    s = G.f64(saved)
    z, u = s[:, :n], s[:, n:]
    a, sl = R.act(z, act), slope(z, act)
    du, dg = dv * a, dv * u * sl
    # activations are computed to 2^-20 |z|, their slopes to 2^-19 (1 + |z|); two products of f32; then D's rounding
    eu = np.abs(dv) * 2.0 ** -20 * np.abs(z) + 2.0 ** -23 * np.abs(du)
    eg = np.abs(dv * u) * 2.0 ** -19 * (1 + np.abs(z)) + 2.0 ** -22 * np.abs(dg)
    ru, rg = eu + R.half_ulp(np.abs(du) + eu, dtype), eg + R.half_ulp(np.abs(dg) + eg, dtype)

    def near(got, want, err, kind):
        off = np.abs(G.f64(got) - want)
        assert (off <= err + R.half_ulp(np.abs(want) + err, kind)).all(), float((off - err).max())

    f32 = lambda terms: (terms + 40) * 2.0 ** -24  # noqa: E731
    sums = (np.abs(dg) + rg) @ np.abs(gv) + (np.abs(du) + ru) @ np.abs(uv)
    near(d.dx, dg @ gv + du @ uv, rg @ np.abs(gv) + ru @ np.abs(uv) + f32(2 * n) * sums, dtype)
    near(d.dgate, dg.T @ xv, rg.T @ np.abs(xv) + f32(m) * ((np.abs(dg) + rg).T @ np.abs(xv)), dtype)
    near(d.dup, du.T @ xv, ru.T @ np.abs(xv) + f32(m) * ((np.abs(du) + ru).T @ np.abs(xv)), dtype)
    near(d.dgate_bias, dg.sum(0), eg.sum(0) + f32(m) * np.abs(dg).sum(0), "f32")
    near(d.dup_bias, du.sum(0), eu.sum(0) + f32(m) * np.abs(du).sum(0), "f32")
    return d, (x, wg, wu, dy, saved), (xv, gv, uv, dv, [G.f64(b) for b in biases])


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_activations(act, dtype):
    check(70, 100, 72, dtype, act)
    check(3, 37, 65, dtype, act, pad=1)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (64, 1, 8), (2, 3, 300), (257, 130, 136), (130, 257, 131)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_sizes_and_strides(m, n, k, pad):
    check(m, n, k, "bf16", "silu", pad)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_against_differences(act):
    """What the products would give with dg and du unrounded, along a direction v: the difference's own error (h^2) and
    f16's roundings are far below a hundredth of the sum of magnitudes."""
    d, (x, wg, wu, dy, _), (xv, gv, uv, dv, (bg, bu)) = check(20, 40, 48, "f16", act)
    rng = np.random.default_rng(1)
    L = lambda x, g, u: np.sum(dv * R.act(x @ g.T + bg, act) * (x @ u.T + bu))  # noqa: E731
    for i, grad in enumerate((d.dx, d.dgate, d.dup)):
        at = [xv, gv, uv]
        v, h = rng.normal(size=at[i].shape), 1e-4
        up, down = (L(*[w + s * h * v if j == i else w for j, w in enumerate(at)]) for s in (1, -1))
        want, got = (up - down) / (2 * h), np.sum(G.f64(grad) * v)
        assert abs(want - got) < 0.01 * np.sqrt(np.sum((G.f64(grad) * v) ** 2)), (i, want, got)


def test_large_and_unusual_sums():
    """Far out, where exponentials overflow and vanish, and at 0: slopes of 1, 0 and their like, nothing that isn't finite."""
    t, K = G.T(), G.K()
    z = t.tensor([0.0, -0.0, 1e-30, 80.0, -80.0, 100.0, -100.0, 1e4, -1e4, 1e20, -1e20, 3e38, -3e38], device="cuda")
    n = z.numel()
    saved = t.cat([z, t.ones(n, device="cuda")])[None].contiguous()
    one = t.ones(1, n, dtype=t.bfloat16, device="cuda")
    x, w = t.ones(1, 8, dtype=t.bfloat16, device="cuda"), t.ones(n, 8, dtype=t.bfloat16, device="cuda")
    for act, at0 in (("relu", 0.0), ("gelu", 0.5), ("gelu_tanh", 0.5), ("silu", 0.5), ("none", 1.0)):
        d = K.gated_linear_backward(G.ctx(), one, x, w, w, saved, act=act, dx=False, bias=True)
        s, a = d.dgate_bias, d.dup_bias
        assert (s[:2] == at0).all() and abs(float(s[2]) - (1.0 if act == "relu" else at0)) < 1e-6, (act, s)  # relu'(1e-30) = 1
        far = [1.0, 0.0] if act != "none" else [1.0, 1.0]
        assert t.allclose(s[3:], t.tensor(far * 5, device="cuda"), atol=1e-6), (act, s)
        assert t.allclose(a[3::2], z[3::2], rtol=1e-6) and (act == "none" or (a[4::2].abs() < 1e-6).all()), (act, a)


def test_what_is_not_finite_stays_in_its_row_and_column():
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(3)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    for m, n, k in ((70, 100, 64), (70, 100, 63)):
        x, wg, wu, dy = r(m, k), r(n, k), r(n, k), r(m, n)
        dy[5, 7], x[m - 1, 3], wg[n - 1, 9] = float("nan"), float("inf"), float("inf")
        saved = t.randn(m, 2 * n, generator=g, device="cuda")
        d = K.gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, act="none", bias=True)
        bad = ~t.isfinite(d.dx)
        assert bad[5].all() and bad[:, 9].all()
        bad[5], bad[:, 9] = False, False
        assert not bad.any()
        for w, b in ((d.dgate, d.dgate_bias), (d.dup, d.dup_bias)):
            bad = ~t.isfinite(w)
            assert bad[7].all() and bad[:, 3].all() and bool(b[7].isnan())
            bad[7], bad[:, 3] = False, False
            assert not bad.any() and int(t.isnan(b).sum()) == 1


def test_outputs_that_are_not_asked_for():
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(4)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    x, wg, wu, dy = r(70, 64), r(90, 64), r(90, 64), r(70, 90)
    saved = t.randn(70, 180, generator=g, device="cuda")
    back = lambda **a: K.gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, **a)  # noqa: E731
    whole_ = back(bias=True)
    for a in (dict(), dict(dx=False), dict(dw=False), dict(dx=False, dw=False, bias=True), dict(dx=False, dw=False)):
        d = back(**a)
        for name, on in (("dx", a.get("dx", True)), ("dgate", a.get("dw", True)), ("dup", a.get("dw", True)),
                         ("dgate_bias", a.get("bias")), ("dup_bias", a.get("bias"))):
            got = getattr(d, name)
            assert t.equal(got, getattr(whole_, name)) if on else got is None


def test_nothing_to_sum():
    t, K = G.T(), G.K()
    e = lambda *s: t.ones(*s, dtype=t.bfloat16, device="cuda")  # noqa: E731
    f = lambda *s: t.ones(*s, device="cuda")  # noqa: E731
    d = K.gated_linear_backward(G.ctx(), e(0, 9), e(0, 5), e(9, 5), e(9, 5), f(0, 18), bias=True)
    assert d.dx.shape == (0, 5) and not d.dgate.any() and not d.dup.any() and not d.dgate_bias.any() and not d.dup_bias.any()
    d = K.gated_linear_backward(G.ctx(), e(6, 0), e(6, 5), e(0, 5), e(0, 5), f(6, 0), bias=True)
    assert d.dx.shape == (6, 5) and not d.dx.any() and d.dgate.shape == (0, 5) and d.dgate_bias.shape == (0,)
    d = K.gated_linear_backward(G.ctx(), e(6, 9), e(6, 0), e(9, 0), e(9, 0), f(6, 18), act="none", bias=True)
    assert d.dx.shape == (6, 0) and d.dgate.shape == (9, 0) and (d.dgate_bias == 6).all()


def test_streams_and_graphs():
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(5)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    sets = [(r(645, 321), r(645, 16), r(321, 16), r(321, 16), t.randn(645, 642, generator=g, device="cuda")),
            (r(402, 230), r(402, 24), r(230, 24), r(230, 24), t.randn(402, 460, generator=g, device="cuda"))]
    out = lambda d: [getattr(d, n) for n in d.__slots__]  # noqa: E731
    call = lambda s: out(K.gated_linear_backward(G.ctx(), *s, bias=True))  # noqa: E731
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
    t, K, H, c = G.T(), G.K(), __import__("haagenti_amd"), G.ctx()
    z = lambda *s: t.zeros(*s, dtype=t.bfloat16, device="cuda")  # noqa: E731
    x, w, dy, saved = z(4, 64), z(32, 64), z(4, 32), t.zeros(4, 64, device="cuda")
    q = K.Int4Weight(t.zeros(32 * 64 // 32 * 18, dtype=t.uint8, device="cuda"), 32, 64)
    base = dict(dy=dy, x=x, gate=w, up=w, saved=saved)
    bad = [
        (dict(gate=q, up=q), H.UNSUPPORTED), (dict(x=x.float()), H.UNSUPPORTED), (dict(act="swish"), H.UNSUPPORTED),
        (dict(dy=dy.half()), H.INVALID_ARGUMENT), (dict(dy=dy[:3]), H.INVALID_ARGUMENT), (dict(dy=dy.cpu()), H.INVALID_ARGUMENT),
        (dict(dy=dy.t().contiguous().t()), H.INVALID_ARGUMENT), (dict(dy=dy[:1].expand(4, 32)), H.INVALID_ARGUMENT),
        (dict(saved=saved.half()), H.INVALID_ARGUMENT), (dict(saved=saved[:, :63]), H.INVALID_ARGUMENT),
        (dict(saved=saved.cpu()), H.INVALID_ARGUMENT), (dict(saved=t.zeros(4, 65, device="cuda")[:, :64]), H.INVALID_ARGUMENT),
        (dict(up=w[:31]), H.INVALID_ARGUMENT), (dict(gate=w.half()), H.INVALID_ARGUMENT),
        (dict(dy=dy.clone().requires_grad_()), H.UNSUPPORTED), (dict(saved=saved.clone().requires_grad_()), H.UNSUPPORTED),
        (dict(x=x.clone().requires_grad_()), H.UNSUPPORTED),
    ]
    for i, (a, code) in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            K.gated_linear_backward(c, **{**base, **a})
        assert e.value.code == code, i
