"""The gated gradients of float16 calls whose dg and du lie beyond float16's
range, on either side, though the outputs don't: against 64-bit forms, rows
and columns of very different sizes, through every kernel."""
import numpy as np
import pytest

import compute_ref as R
import gated_back_shapes
import test_gpu_compute as G
from test_gpu_gated_backward import slope

pytestmark = pytest.mark.gpu


def check(m, n, k, dy, gate, up, act="none", w=1.0, x=1.0, pad=0, seed=0):
    """dy (m x n), gate and up (m x n: what the forward pass saved) as given; weights and x of sizes w and x (numbers,
    or arrays of their shapes)."""
    t, rng = G.T(), np.random.default_rng(seed)
    xt, xv = G.padded(x * rng.normal(0, 1, (m, k)), pad, "f16")
    wg, gv = G.padded(w * rng.normal(0, 1, (n, k)), pad, "f16")
    wu, uv = G.padded(w * rng.normal(0, 1, (n, k)), pad, "f16")
    dyt, dv = G.padded(dy, 0, "f16")
    saved = t.from_numpy(np.concatenate([gate, up], 1).astype(np.float32)).cuda()
    z, u = G.f64(saved[:, :n]), G.f64(saved[:, n:])
    print(f"gated range {m}x{n}x{k} {act} pad {pad}", flush=True)
    d = G.K().gated_linear_backward(G.ctx(), dyt, xt, wg, wu, saved, act=act, bias=True)
    a, sl = R.act(z, act), slope(z, act)
    dg, du = dv * u * sl, dv * a
    # activations to 2^-20 |z|, their slopes to 2^-19 (1 + |z|), two products of f32 (as for ordinary sizes)
    exact = act in ("none", "relu")
    eg = (0 if exact else np.abs(dv * u) * 2.0 ** -19 * (1 + np.abs(z))) + 2.0 ** -22 * np.abs(dg)
    eu = (0 if exact else np.abs(dv) * 2.0 ** -20 * np.abs(z)) + 2.0 ** -23 * np.abs(du)

    def rounded(v, e, top):
        """To half a step of 11 bits; a largest of 2^14 or more beside steps of 2^-24: at least to 2^-39 of the largest."""
        return e + 2.0 ** -11 * (np.abs(v) + e) + 2.0 ** -39 * top

    rows = np.maximum((np.abs(dg) + eg).max(1), (np.abs(du) + eu).max(1))[:, None]
    f32 = lambda terms: (terms + 40) * 2.0 ** -24  # noqa: E731

    def near(got, want, err, kind="f16"):
        got = G.f64(got)
        with np.errstate(over="ignore"):
            fits = np.abs(want) + err < 65504.0
        off = np.abs(np.where(fits, got - want, 0.0))
        assert (off <= err + R.half_ulp(np.abs(want) + err, kind)).all(), float((off - err).max())
        assert fits.mean() > 0.5 and np.isfinite(got[fits]).all()

    rg, ru = rounded(dg, eg, rows), rounded(du, eu, rows)
    sums = (np.abs(dg) + rg) @ np.abs(gv) + (np.abs(du) + ru) @ np.abs(uv)
    near(d.dx, dg @ gv + du @ uv, rg @ np.abs(gv) + ru @ np.abs(uv) + f32(2 * n) * sums)
    for got, v, e in ((d.dgate, dg, eg), (d.dup, du, eu)):
        r = rounded(v, e, (np.abs(v) + e).max(0)[None])
        near(got, v.T @ xv, r.T @ np.abs(xv) + f32(m) * ((np.abs(v) + r).T @ np.abs(xv)))
    for got, v, e in ((d.dgate_bias, dg, eg), (d.dup_bias, du, eu)):
        off = np.abs(G.f64(got) - v.sum(0))
        assert (off <= e.sum(0) + f32(m) * np.abs(v).sum(0)).all()
    return d


SIZES = [(70, 100, 72, 0), (70, 100, 65, 1), (3, 37, 65, 0), (300, 260, 264, 8), (1, 513, 64, 0), (257, 1, 8, 0)]


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("m,n,k,pad", SIZES)
def test_above_the_largest_float16(m, n, k, pad, act):
    rng = np.random.default_rng(m + n)
    dy, gate, up = (s * rng.normal(0, 1, (m, n)) for s in (300, 300, 300))
    check(m, n, k, dy, gate, up, act, w=2.0 ** -9, x=2.0 ** -9, pad=pad)


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("m,n,k,pad", SIZES)
def test_below_the_least_float16(m, n, k, pad, act):
    rng = np.random.default_rng(m + n)
    dy, gate, up = (s * rng.normal(0, 1, (m, n)) for s in (1e-4, 1e-4, 1e-4))
    check(m, n, k, dy, gate, up, act, w=3e3, x=3e3, pad=pad)


@pytest.mark.parametrize("m,n,k,pad", SIZES)
def test_rows_and_columns_of_very_different_sizes(m, n, k, pad):
    """Rows of dy and columns of the sums from 2^-12 to 2^15: each row of dx and of the weights' gradients keeps its own
    largest's precision."""
    rng = np.random.default_rng(m + 5 * n)
    tall = np.exp2(rng.integers(-12, 6, (m, 1)))
    wide = np.exp2(rng.integers(-12, 16, (1, n)))
    dy = tall * rng.uniform(1, 2, (m, n))
    check(m, n, k, dy, rng.normal(0, 1, (m, n)) * wide, rng.normal(0, 1, (m, n)) * wide, w=2.0 ** -11, x=2.0 ** -13, pad=pad)
    # a row (a column) of zeros beside large ones
    dy[m // 2] = 0
    up = rng.normal(0, 300, (m, n))
    up[:, n // 2] = 0
    d = check(m, n, k, dy, up, up, w=2.0 ** -9, x=2.0 ** -9, pad=pad)
    assert not d.dx[m // 2].any() and not d.dgate[n // 2].any() and not d.dup[n // 2].any()


def test_small_values_beside_large_ones_that_meet_zeros():
    """The largest of a row of dg meets zeros of the weights, of a column zeros of x: what is 2^-20 to 2^-28 of it remains."""
    rng = np.random.default_rng(3)
    for k, pad in ((64, 0), (63, 1)):
        m, n = 130, 200
        dy, up = np.full((m, n), 2.0 ** -10), rng.normal(0, 1, (m, n)) * np.exp2(rng.integers(-10, -2, (1, n)))
        up[:, 0], dy[0] = 2.0 ** 18, 2.0 ** 15
        w, x = np.full((n, 1), 500.0), np.full((m, 1), 500.0)
        w[0], x[0] = 0, 0
        check(m, n, k, dy, up, up, w=w, x=x, pad=pad)


@pytest.mark.parametrize("m,n,k", gated_back_shapes.SHAPES)
def test_whole_numbers_of_any_size_are_exact(m, n, k):
    """dg and du are whole numbers up to 6 times a power of two of their row, far above float16: every product and sum is
    exact, and so are dx (the power undone by a weight's) and, rows being alike, the weights' gradients."""
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(m + n + k)
    whole = lambda low, high, *s: t.randint(low, high + 1, s, generator=g, device="cuda").float()  # noqa: E731
    x, wg, wu = ((whole(-2, 2, r, k) * 2.0 ** -12).half() for r in (m, n, n))
    dy = (whole(-2, 2, m, n) * 2.0 ** 10).half()
    saved = whole(-3, 3, m, 2 * n) * 2.0 ** 9
    print(f"gated range {m}x{n}x{k}", flush=True)
    d = K.gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, act="none", bias=True)
    du, dg = dy.double() * saved[:, :n].double(), dy.double() * saved[:, n:].double()
    assert t.equal(d.dx, (dg @ wg.double() + du @ wu.double()).half())
    assert t.equal(d.dgate, (dg.t().contiguous() @ x.double()).half()) and t.equal(d.dup, (du.t().contiguous() @ x.double()).half())
    assert t.equal(d.dgate_bias, dg.sum(0).float()) and t.equal(d.dup_bias, du.sum(0).float())


def test_what_is_not_finite_stays_in_its_row_and_column():
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(3)
    r = lambda *s: t.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    for m, n, k in ((70, 100, 64), (70, 100, 63)):
        for bad_dy in (float("nan"), float("inf")):
            x, wg, wu, dy = r(m, k), r(n, k), r(n, k), r(m, n) * 200
            dy[5, 7], x[m - 1, 3], wg[n - 1, 9] = bad_dy, float("inf"), float("inf")
            saved = t.randn(m, 2 * n, generator=g, device="cuda")
            d = K.gated_linear_backward(G.ctx(), dy, x, wg, wu, saved, act="none", bias=True)
            bad = ~t.isfinite(d.dx)
            assert bad[5].all() and bad[:, 9].all()
            bad[5], bad[:, 9] = False, False
            assert not bad.any()
            for w in (d.dgate, d.dup):
                bad = ~t.isfinite(w)
                assert bad[7].all() and bad[:, 3].all()
                bad[7], bad[:, 3] = False, False
                assert not bad.any()


def test_replayed_graphs_and_parts_of_the_outputs():
    t, K = G.T(), G.K()
    g = t.Generator("cuda").manual_seed(5)
    r = lambda s, *shape: (s * t.randn(*shape, generator=g, device="cuda")).half()  # noqa: E731
    m, n, k = 130, 200, 72
    args = [r(300, m, n), r(2e-3, m, k), r(2e-3, n, k), r(2e-3, n, k), 300 * t.randn(m, 2 * n, generator=g, device="cuda")]
    other = [a * 2.0 ** -9 for a in args]
    out = lambda d: [getattr(d, s) for s in d.__slots__]  # noqa: E731
    call = lambda a, **o: out(K.gated_linear_backward(G.ctx(), *a, act="none", **o))  # noqa: E731
    want, less = [[y.clone() for y in call(a, bias=True)] for a in (args, other)]
    assert all(y.isfinite().all() for y in want)
    for o in (dict(), dict(dx=False), dict(dw=False), dict(dx=False, dw=False, bias=True)):
        assert all(a is None or t.equal(a, b) for a, b in zip(call(args, **o), want))
    graph, held = t.cuda.CUDAGraph(), None
    with t.cuda.graph(graph):
        held = call(args, bias=True)
    for _ in range(4):
        for y in held:
            y.zero_()
        assert all(t.equal(a, b) for a, b in zip(call(other, bias=True), less))
        graph.replay()
        t.cuda.synchronize()
        assert all(t.equal(a, b) for a, b in zip(held, want))
