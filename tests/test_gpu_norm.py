"""Layer norm and root mean square norm with their gradients, on the GPU
against their 64-bit forms, at the widths, rows and strides where they can go
wrong."""
import numpy as np
import pytest

import norm_ref as R
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def inputs(rows, n, dtype, weight, bias, pad, seed, scale=1.0, shift=0.5):
    rng = np.random.default_rng(seed)
    x = (rng.normal(size=(rows, n)) + shift * rng.normal(size=(rows, 1))) * scale
    wt = {"same": dtype, "f32": "f32", None: None}[weight]
    x, xv = G.padded(x, pad, dtype)
    w, wv = (None, None) if wt is None else G.dev(1 + 0.3 * rng.normal(size=n), wt)
    b, bv = (None, None) if not bias else G.dev(rng.normal(size=n), wt or dtype)
    return x, xv, w, wv, b, bv, rng


def near(got, want, bound, dtype):
    got = G.f64(got)
    off = np.abs(got - want) - (bound + R.half_step(np.abs(want) + bound, dtype))
    assert not (off > 0).any(), (dtype, float(np.nanmax(off)), np.argwhere(off > 0)[:4])
    assert np.isfinite(got).all()


def check(rows, n, dtype="bf16", weight="f32", bias=True, kind="layer", pad=0, eps=1e-5, seed=0, **more):
    x, xv, w, wv, b, bv, rng = inputs(rows, n, dtype, weight, bias, pad, seed, **more)
    want, bound = R.norm(xv, wv, bv, kind, eps)[:2]
    near(G.K().norm(G.ctx(), x, w, b, kind=kind, eps=eps), want, bound, dtype)
    dy, dyv = G.padded(rng.normal(size=(rows, n)), pad, dtype)
    for add in (False, True):
        at, av = G.padded(rng.normal(size=(rows, n)), pad, dtype) if add else (None, None)
        want = R.norm_backward(dyv, xv, wv, kind, eps, av)
        got = G.K().norm_backward(G.ctx(), dy, x, w, bias=bias, kind=kind, eps=eps, add=at)
        near(got[0], *want[0], dtype)
        if w is not None:
            assert got[1].dtype == G.T().float32
            near(got[1], *want[1], "f32")
        else:
            assert got[1] is None
        if bias:
            near(got[2], *want[2], "f32")
        else:
            assert got[2] is None


# one wave, 4 and 16 of them to a row; pieces of 1, 2, 4 and 8 to a lane; rows that end inside a piece
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 64, 65, 513, 1003, 1024, 1025, 2047, 4096, 4097, 8191, 16384, 16385, 32767])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_widths(n, rows):
    check(rows, n, pad=n % 3, kind=["layer", "rms"][n % 2])


@pytest.mark.parametrize("n", [1, 5, 64, 255, 512, 1001, 2048, 4096, 4100])
def test_many_rows(n):
    check(1500 if n < 4096 else 1100, n, pad=n % 3, kind=["rms", "layer"][n % 2])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("weight", ["same", "f32", None])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_types(dtype, weight, kind):
    check(33, 1000, dtype, weight, weight is not None, kind, pad=1)
    check(1200, 257, dtype, weight, False, kind, pad=5)


@pytest.mark.parametrize("n", [1, 3, 2049, 8193, 16384])
def test_f32_widths(n):
    check(5, n, "f32", "same", True)
    check(1100, min(n, 2049), "f32", "same", True)


def test_values():
    """Rows far from 0 beside their spread, large and tiny ones, zeros, a single outlier; eps of 0 and a large one."""
    check(20, 500, "f32", shift=1000.0)
    check(20, 500, "f32", scale=1e15)
    check(20, 500, "bf16", scale=1e-12)
    check(20, 500, "f16", scale=1e-4, eps=0.0)
    check(20, 500, "bf16", eps=3.0)
    t, k = G.T(), G.K()
    zero = t.zeros(3, 100, dtype=t.bfloat16, device="cuda")
    b = t.arange(100, device="cuda").float()
    for kind in ("layer", "rms"):
        assert t.equal(k.norm(G.ctx(), zero, None, b, kind=kind).float(), b.bfloat16().float().expand(3, 100))
        dx, dw, db = k.norm_backward(G.ctx(), zero + 1, zero, b, bias=True, kind=kind)
        assert (dw == 0).all() and (db == 3).all() and dx.isfinite().all()
    x = t.zeros(2, 300, device="cuda")
    x[:, 7] = 1e4
    want = R.norm(G.f64(x), None, None, "layer", 1e-5)
    near(k.norm(G.ctx(), x), *want[:2], "f32")


def test_what_is_not_finite_stays_in_its_row():
    t, k = G.T(), G.K()
    x = t.randn(5, 700, generator=t.Generator("cuda").manual_seed(1), device="cuda")
    want, dwant = k.norm(G.ctx(), x), k.norm_backward(G.ctx(), x, x)[0]
    bad = x.clone()
    bad[1, 3], bad[3, 699] = float("inf"), float("nan")
    y, dx = k.norm(G.ctx(), bad), k.norm_backward(G.ctx(), x, bad)[0]
    for got, w in ((y, want), (dx, dwant)):
        assert t.equal(got[[0, 2, 4]], w[[0, 2, 4]])
        assert got[1].isnan().any() and got[3].isnan().all()


def test_no_rows_and_no_columns():
    t, k, c = G.T(), G.K(), G.ctx()
    w = t.ones(40, device="cuda")
    x = t.ones(0, 40, device="cuda")
    assert k.norm(c, x, w).shape == (0, 40)
    dx, dw, db = k.norm_backward(c, x, x, w, bias=True)
    assert dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all()
    x = t.ones(4, 0, device="cuda")
    assert k.norm(c, x).shape == (4, 0)
    dx, dw, db = k.norm_backward(c, x, x, t.ones(0, device="cuda"), bias=True)
    assert dx.shape == (4, 0) and dw.numel() == 0 and db.numel() == 0


@pytest.mark.parametrize("rows,n", [(6, 900), (1500, 900)])
def test_in_place_and_wider_outputs(rows, n):
    t, k, c = G.T(), G.K(), G.ctx()
    g = t.Generator("cuda").manual_seed(2)
    x, dy, add = (t.randn(rows, n, generator=g, device="cuda").half() for _ in range(3))
    w = t.randn(n, generator=g, device="cuda").half()
    want = k.norm(c, x, w)
    wide = t.full((rows, n + 9), 7.0, dtype=t.half, device="cuda")
    assert k.norm(c, x, w, out=wide[:, 3:n + 3]).data_ptr() == wide.data_ptr() + 6
    assert t.equal(wide[:, 3:n + 3], want) and (wide[:, :3] == 7).all() and (wide[:, n + 3:] == 7).all()
    y = x.clone()
    assert t.equal(k.norm(c, y, w, out=y), want)
    dwant = k.norm_backward(c, dy, x, w, bias=True, add=add)
    for i in range(3):
        a = [dy.clone(), x.clone(), add.clone()]
        got = k.norm_backward(c, a[0], a[1], w, bias=True, add=a[2], out=a[i])
        assert all(t.equal(p, q) for p, q in zip(got, dwant))


def test_gradients_against_differences():
    """(L(x + h v) - L(x - h v)) / 2 h in 64 bits against the gradient's product with v: off by h^2 of the third derivative."""
    x, xv, w, wv, b, bv, rng = inputs(7, 130, "f32", "f32", True, 0, 3)
    c, v = rng.normal(size=(7, 130)), rng.normal(size=(7, 130))
    dy, cv = G.dev(c, "f32")
    for kind in ("layer", "rms"):
        dx = G.f64(G.K().norm_backward(G.ctx(), dy, x, w, kind=kind)[0])
        h = 1e-5
        up, down = (np.sum(cv * R.norm(xv + s * h * v, wv, bv, kind, 1e-5)[0]) for s in (1, -1))
        assert abs((up - down) / (2 * h) - np.sum(dx * v)) < 1e-4 * np.sum(np.abs(dx * v))


def test_same_bits_again_on_streams_and_in_graphs():
    t, k, c = G.T(), G.K(), G.ctx()
    g = t.Generator("cuda").manual_seed(4)
    sets = [[t.randn(r, 1000, generator=g, device="cuda").bfloat16() for _ in range(2)] for r in (3000, 1700)]
    w = t.randn(1000, generator=g, device="cuda")
    call = lambda s: [k.norm(c, s[0], w), *k.norm_backward(c, s[1], s[0], w, bias=True)]  # noqa: E731
    want = [[y.clone() for y in call(s)] for s in sets]
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    t.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, st in zip(sets, streams):
            with t.cuda.stream(st):
                got.append(call(s))
    t.cuda.synchronize()
    for i, y in enumerate(got):
        assert all(t.equal(p, q) for p, q in zip(y, want[i % 2])), i
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
    t, k, c, H = G.T(), G.K(), G.ctx(), __import__("haagenti_amd")
    x = t.zeros(4, 64, dtype=t.bfloat16, device="cuda")
    w = t.ones(64, device="cuda")
    bad = [
        (lambda: k.norm(c, x.double()), H.UNSUPPORTED), (lambda: k.norm(c, x, kind="batch"), H.UNSUPPORTED),
        (lambda: k.norm(c, x[0]), H.INVALID_ARGUMENT), (lambda: k.norm(c, x.t()), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x, w[:63]), H.INVALID_ARGUMENT), (lambda: k.norm(c, x, w.half()), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x, w, w.bfloat16()), H.INVALID_ARGUMENT), (lambda: k.norm(c, x, w.cpu()), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x.cpu()), H.INVALID_ARGUMENT), (lambda: k.norm(c, x, eps=-1.0), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x, eps=float("nan")), H.INVALID_ARGUMENT), (lambda: k.norm(c, x, eps="a"), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x[:1].expand(4, 64)), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, t.zeros(1, 32769, dtype=t.half, device="cuda")), H.UNSUPPORTED),
        (lambda: k.norm(c, t.zeros(1, 16385, device="cuda")), H.UNSUPPORTED),
        (lambda: k.norm(c, x, out=x.float()), H.INVALID_ARGUMENT), (lambda: k.norm(c, x, out=x[:3]), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x[1:], out=x[:3]), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x, out=x[:1].expand(4, 64)), H.INVALID_ARGUMENT),
        (lambda: k.norm_backward(c, x.half(), x), H.INVALID_ARGUMENT),
        (lambda: k.norm_backward(c, x[:3], x), H.INVALID_ARGUMENT),
        (lambda: k.norm_backward(c, x, x, add=x.float()), H.INVALID_ARGUMENT),
        (lambda: k.norm_backward(c, x, x, add=x[:, :63]), H.INVALID_ARGUMENT),
        (lambda: k.norm(c, x.float().requires_grad_()), H.UNSUPPORTED),
        (lambda: k.norm(c, x, w.clone().requires_grad_()), H.UNSUPPORTED),
        (lambda: k.norm_backward(c, x.float().requires_grad_(), x.float()), H.UNSUPPORTED),
    ]
    for i, (call, code) in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            call()
        assert e.value.code == code, i
