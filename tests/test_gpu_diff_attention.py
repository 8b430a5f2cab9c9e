"""Differential attention over the paged 8-bit cache on the GPU against its
64-bit form: steps, prompts and mixed batches, splits over tokens, masks that
leave rows empty, strides, the norm, streams, graphs and refusals."""
import numpy as np
import pytest

import compute_ref as R
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def one_map(q, k, v, kv_len, scale, bits, top):
    """softmax(scale q k^T) v of rows that are the last of kv_len tokens, and what it may be off by."""
    rows, heads, half = q.shape
    group = heads // k.shape[1]
    out, err = np.zeros((rows, heads, v.shape[2])), np.zeros((rows, heads, v.shape[2]))
    for i in range(rows):
        n = min(max(kv_len - rows + i + 1, 0), len(k))
        if n == 0:
            continue
        for h in range(heads):
            kk, vv = k[:n, h // group], v[:n, h // group]
            z = kk @ q[i, h] * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i, h] = p @ vv
            # scores: f32 sums of the dimensions, and queries of bf16 to 2^-25 of their row's largest; an error d of a
            # score changes p and the sum by d each; p is rounded to `bits` bits, or to 2^-25 of the largest value scale
            # where it is small; exp and the sums to 2^-18
            d = float((np.abs(kk) @ np.abs(q[i, h])).max() * scale) * ((2 * half + 8) * 2.0 ** -24 + 2 * half * 2.0 ** -25)
            err[i, h] = p @ np.abs(vv) * (2 * d + 2.0 ** -bits + 2.0 ** -18) + top * 2.0 ** -25
    return out, err


def differ(q, k, v, kv_len, scale, lam, weight, eps, gain, bits, top):
    """The operator for one request, and what it may be off by."""
    half = q.shape[2] // 2
    a, ea = one_map(q[..., :half], k[..., :half], v, kv_len, scale, bits, top)
    b, eb = one_map(q[..., half:], k[..., half:], v, kv_len, scale, bits, top)
    lam = lam[None, :, None]
    o, e = a - lam * b, ea + np.abs(lam) * eb + 2.0 ** -22 * (np.abs(a) + np.abs(lam * b))
    if weight is None:
        return o * gain, (e + 2.0 ** -23 * np.abs(o)) * abs(gain)
    r = lambda x: 1 / np.sqrt(np.square(x).mean(-1, keepdims=True) + eps)  # noqa: E731
    with np.errstate(divide="ignore"):
        mid, high, low = r(o), r(np.maximum(np.abs(o) - e, 0)), r(np.abs(o) + e)
    seen = (kv_len - len(q) + 1 + np.arange(len(q)) > 0)[:, None, None]   # rows that see nothing are zeros, not 0 / 0
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(seen, o * mid * weight * gain, 0.0)
        off = np.where(seen, e * high + np.abs(o) * np.maximum(high - mid, mid - low), 0.0)
    return y, off * np.abs(weight * gain) + 2.0 ** -20 * np.abs(y)


def check(lens, rows, q_heads, heads, dim, bs, dtype, seed=0, pad=0, extra=0, size=1.0, norm=True, max_q=None, max_kv=None,
          drop=(), lam=None, scales=None, q_change=None, eps=1e-5):
    rng = np.random.default_rng(seed)
    counts = [(n + bs - 1) // bs for n in lens]
    blocks = sum(counts) + 2
    c, kq, vq, ks, vs = G.new_cache(blocks, bs, heads, dim, seed)
    if scales is not None:
        vs = R.up8(vs * scales(rng, blocks)[:, None])
        c.v_scale.copy_(G.T().from_numpy(vs))
        vs = G.f64(c.v_scale)
    ids = rng.permutation(blocks)
    table = np.full((len(lens), max(counts + [1]) + 1), -1, np.int64)
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1]) + extra
    wide = rng.normal(0, size, (total, q_heads * (dim + pad)))
    if q_change:
        q_change(wide)
    qt, qv = G.dev(wide, dtype)
    qt = qt.view(total, q_heads, dim + pad)[:, :, :dim]
    qv = qv.reshape(total, q_heads, dim + pad)[:, :, :dim]
    lt, lv = G.dev(rng.uniform(0.1, 0.9, q_heads) if lam is None else np.full(q_heads, lam), "f32")
    wt, wv = G.dev(1 + 0.3 * rng.normal(size=dim), "f32") if norm else (None, None)
    lost = table.copy()
    for r, col in drop:
        lost[r, col] = blocks + 3 * r
    print(f"diff attention {lens} {rows} {q_heads}/{heads}x{dim} bs {bs} {dtype}", flush=True)
    o = c.diff_attention(qt, lt, G.i32(lost), G.i32(start), G.i32(lens), max_q=max_q, max_kv=max_kv, norm_weight=wt, eps=eps,
                         gain=0.7)
    got = G.f64(o)
    assert o.shape == (total, q_heads, dim) and o.dtype == G.tdt(dtype)
    for r, n in enumerate(lens):
        if rows[r] == 0:
            continue
        b = table[r, :counts[r]]
        key = (kq[b] * ks[b][:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:max(n, 0)]
        val = (vq[b] * vs[b][:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:max(n, 0)]
        gone = [x for (rr, col) in drop if rr == r for x in range(col * bs, min((col + 1) * bs, n))]
        assert not gone or rows[r] == 1
        keep = np.setdiff1d(np.arange(n), gone)
        bits = 22 if rows[r] * (q_heads // heads) <= 8 else 11
        top = 127 * float(vs[b].max()) if len(b) else 0.0
        want, err = differ(qv[start[r]:start[r + 1]], key[keep], val[keep], len(keep), (dim // 2) ** -0.5, lv, wv, eps, 0.7, bits,
                           top)
        off = np.abs(got[start[r]:start[r + 1]] - want)
        assert (off <= err + R.half_ulp(np.abs(want) + err, dtype)).all(), (r, float((off - err).max()))
    assert (got[start[-1]:] == 0).all()
    return o


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_step(bs, dim, dtype):
    check([1, 15, 64, 65, 257, 700], [1] * 6, 8, 2, dim, bs, dtype, seed=bs + dim, norm=bs != 32)


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (6, 2), (10, 2), (8, 1), (7, 7), (24, 1), (40, 2)])
@pytest.mark.parametrize("rows", [1, 3])
def test_groups(q_heads, heads, rows):
    check([5, 300, 129], [rows] * 3, q_heads, heads, 64, 32, "bf16", seed=q_heads + rows, norm=rows == 1)


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("bs", [16, 128])
def test_prompt(bs, dim, dtype):
    check([90, 200, 33], [90, 70, 17], 4, 2, dim, bs, dtype, seed=bs + dim, norm=bs == 16)


def test_mixed():
    check([700, 150, 1, 64, 300], [1, 150, 1, 64, 5], 8, 2, 64, 32, "bf16", extra=3)
    check([40, 31], [0, 31], 4, 4, 64, 16, "f16", extra=1)


def test_long_splits_join():
    check([9000, 17, 2500], [1, 1, 1], 8, 1, 64, 64, "bf16")
    check([9000], [2], 4, 1, 128, 128, "f16", norm=False)
    check([5000], [1], 3, 1, 96, 16, "f16", max_kv=5000, max_q=1)
    check([4000, 4100], [1, 1], 5, 1, 256, 32, "bf16", max_q=1)


def test_empty_rows():
    # requests without tokens, more rows than tokens: rows that see nothing are zeros, whatever eps is
    for eps in (1e-5, 0.0):
        o = check([0, 10, 3], [2, 1, 7], 4, 2, 64, 16, "bf16", eps=eps)
        assert (o[:2] == 0).all() and (o[3:7] == 0).all() and (o[7:] != 0).any()
        o = check([0, 20], [40, 60], 4, 1, 64, 16, "f16", eps=eps)
        assert (o[:80] == 0).all()
    t = G.T()
    c = G.new_cache(3, 16, 1, 64, 0)[0]
    q = t.ones(3, 2, 64, dtype=t.bfloat16, device="cuda")
    for bad in (float("inf"), float("nan")):
        o = c.diff_attention(q, t.full((2,), bad, device="cuda"), G.i32([[-1, -1]]), G.i32([0, 3]), G.i32([20]))
        assert (o == 0).all()
    # without requests
    o = c.diff_attention(q, t.ones(2, device="cuda"), t.zeros(0, 2, dtype=t.int32, device="cuda"), G.i32([0]), G.i32([]))
    assert (o == 0).all()


def test_strides_and_lost_blocks():
    check([70, 33], [1, 33], 4, 2, 64, 16, "bf16", pad=3)
    check([70, 33], [1, 33], 4, 2, 64, 16, "f16", pad=8, norm=False)
    check([70, 133], [1, 1], 4, 2, 64, 16, "bf16", drop=[(0, 1), (1, 8)])
    check([1900], [1], 4, 2, 64, 16, "f16", drop=[(0, 0), (0, 50), (0, 118)])


def test_scales_far_apart_and_large_queries():
    far = lambda rng, n: 2.0 ** rng.integers(-12, 12, n)  # noqa: E731
    check([300, 128], [1, 1], 4, 1, 64, 16, "bf16", scales=far)
    check([300, 128], [60, 20], 4, 1, 64, 16, "bf16", scales=far)
    check([100, 40], [1, 40], 4, 2, 64, 16, "bf16", size=40.0)
    check([1, 30], [1, 30], 4, 2, 64, 16, "bf16", q_change=lambda w: w.__imul__(1e-30))


def test_lambda_of_zero_is_one_map_and_equal_maps_vanish():
    t = G.T()
    for rows in (1, 40):
        c = G.new_cache(8, 16, 2, 64, 1)[0]
        g = t.Generator("cuda").manual_seed(rows)
        q = t.randn(rows, 4, 64, generator=g, device="cuda").bfloat16()
        table, start, lens = G.i32([[3, 1, 5, 0]]), G.i32([0, rows]), G.i32([57])
        zero, one = t.zeros(4, device="cuda"), t.ones(4, device="cuda")
        first = q.clone()
        first[..., 32:] = 0
        want = c.attention(first, table, start, lens, scale=32 ** -0.5)
        # the same map twice: each is off by half a step of its output, and by 2^-11 of its terms
        got = c.diff_attention(q, zero, table, start, lens)
        assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs().amax()).all()
        c.k[..., 32:] = c.k[..., :32]
        q[..., 32:] = q[..., :32]
        assert (c.diff_attention(q, one, table, start, lens) == 0).all()


def test_bounds_leave_rows_and_tokens_out():
    t = G.T()
    c = G.new_cache(8, 16, 1, 64, 2)[0]
    q = t.randn(30, 2, 64, generator=t.Generator("cuda").manual_seed(1), device="cuda").half()
    lam, table = t.full((2,), 0.5, device="cuda"), G.i32([[3, 1, 5, 0]])
    whole = c.diff_attention(q, lam, table, G.i32([0, 30]), G.i32([60]))
    for most in (2, 20):
        o = c.diff_attention(q, lam, table, G.i32([0, 30]), G.i32([60]), max_q=most)
        assert (o[most:] == 0).all() and t.allclose(o[:most].float(), whole[:most].float(), atol=2e-3)


def test_nan_query_stays_in_its_row():
    t = G.T()
    c = G.new_cache(8, 16, 1, 64, 3)[0]
    lam = t.full((2,), 0.5, device="cuda")
    for rows in (3, 40):
        q = t.randn(rows, 2, 64, device="cuda").bfloat16()
        q[1, 0, 40], q[2, 1, 3] = float("nan"), float("nan")
        o = c.diff_attention(q, lam, G.i32([[3, 1, 5, 0]]), G.i32([0, rows]), G.i32([60]), norm_weight=t.ones(64, device="cuda"))
        assert o[1, 0].isnan().all() and o[2, 1].isnan().all()
        o[1, 0], o[2, 1] = 0, 0
        assert o.isfinite().all()


def test_streams_and_graphs():
    t = G.T()

    def call(seed, tokens, rows):
        n = (tokens + 15) // 16
        c = G.new_cache(n, 16, 2, 64, seed)[0]
        g = t.Generator("cuda").manual_seed(seed)
        q = t.randn(rows, 8, 64, generator=g, device="cuda").bfloat16()
        lam, w = t.rand(8, generator=g, device="cuda"), t.rand(64, generator=g, device="cuda")
        table, start, lens = G.i32(np.random.default_rng(seed).permutation(n)[None]), G.i32([0, rows]), G.i32([tokens])
        out = t.empty_like(q)
        return (lambda: c.diff_attention(q, lam, table, start, lens, max_q=rows, max_kv=tokens, norm_weight=w, out=out)), out

    sides = [[call(1, 30000, 1), call(2, 500, 60)], [call(3, 20000, 2), call(4, 700, 30)]]
    want = [[f().clone() for f, _ in side] for side in sides]
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    for _ in range(10):
        for side in sides:
            for _, out in side:
                out.zero_()
        t.cuda.synchronize()
        for i in range(2):
            for st, side in zip(streams, sides):
                with t.cuda.stream(st):
                    side[i][0]()
        t.cuda.synchronize()
        assert all(t.equal(out, w) for side, ws in zip(sides, want) for (_, out), w in zip(side, ws))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        for f, _ in sides[0]:
            f()
    for _ in range(4):
        for _, out in sides[0]:
            out.zero_()
        for f, _ in sides[1]:
            f()
        graph.replay()
        t.cuda.synchronize()
        assert all(t.equal(out, w) for (_, out), w in zip(sides[0], want[0]))


def test_refusals():
    t, H = G.T(), __import__("haagenti_amd")
    c = G.new_cache(3, 16, 2, 64, 0)[0]
    q, lam = t.zeros(2, 4, 64, dtype=t.float16, device="cuda"), t.zeros(4, device="cuda")
    base = dict(q=q, lam=lam, table=G.i32([[0, 1]]), start=G.i32([0, 2]), kv_len=G.i32([2]))
    bad = [
        (dict(q=q.float()), H.UNSUPPORTED), (dict(q=q[0]), H.INVALID_ARGUMENT), (dict(q=q[:, :3], lam=lam[:3]), H.INVALID_ARGUMENT),
        (dict(q=q.cpu()), H.INVALID_ARGUMENT), (dict(lam=lam[:3]), H.INVALID_ARGUMENT), (dict(lam=lam.half()), H.INVALID_ARGUMENT),
        (dict(lam=lam.cpu()), H.INVALID_ARGUMENT), (dict(lam=t.zeros(8, device="cuda")[::2]), H.INVALID_ARGUMENT),
        (dict(norm_weight=t.ones(63, device="cuda")), H.INVALID_ARGUMENT),
        (dict(norm_weight=t.ones(64, device="cuda").half()), H.INVALID_ARGUMENT),
        (dict(norm_weight=t.ones(64)), H.INVALID_ARGUMENT), (dict(eps=-1.0), H.INVALID_ARGUMENT),
        (dict(eps=float("nan")), H.INVALID_ARGUMENT), (dict(eps="a"), H.INVALID_ARGUMENT),
        (dict(start=G.i32([0])), H.INVALID_ARGUMENT), (dict(table=G.i32([0, 1])), H.INVALID_ARGUMENT),
        (dict(out=q.float()), H.INVALID_ARGUMENT), (dict(out=q), H.INVALID_ARGUMENT),
        (dict(out=t.zeros(1, 4, 64, dtype=t.half, device="cuda").expand(2, 4, 64)), H.INVALID_ARGUMENT),
        (dict(q=q.clone().requires_grad_()), H.UNSUPPORTED), (dict(lam=lam.clone().requires_grad_()), H.UNSUPPORTED),
        (dict(norm_weight=t.ones(64, device="cuda").requires_grad_()), H.UNSUPPORTED),
    ]
    for i, (a, code) in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            c.diff_attention(**{**base, **a})
        assert e.value.code == code, i
