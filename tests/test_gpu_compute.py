"""The decoder-layer operators on the GPU against their plain 64-bit forms:
matrix products with their epilogue, and the paged 8-bit cache's plan, append,
read and attention, at the sizes, strides and masks where they can go wrong,
and their refusals."""
import numpy as np
import pytest

import compute_ref as R

pytestmark = pytest.mark.gpu

DT = ["bf16", "f16"]


def T():
    import torch
    return torch


def K():
    import haagenti_amd.compute as k
    return k


def ctx():
    import gpu_util as G
    return G.ctx()


def tdt(name):
    t = T()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[name]


def dev(a, dtype):
    """float64 values, rounded once to the type, on the device, and as they are there."""
    t = T().from_numpy(np.ascontiguousarray(a)).to(tdt(dtype))
    return t.cuda(), t.double().numpy()


def i32(a):
    return T().from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- linear

def padded(a, pad, dtype):
    """a's rows in a wider buffer."""
    wide = np.full((a.shape[0], a.shape[1] + pad), np.nan)
    wide[:, :a.shape[1]] = a
    t, v = dev(wide, dtype)
    return t[:, :a.shape[1]], v[:, :a.shape[1]]


def check_linear(m, n, k, dtype, weight="same", act="none", bias=False, mul=False, res=False, out=None, pad=0, seed=0):
    import haagenti_amd as H
    rng = np.random.default_rng(seed + 7 * m + 3 * n + k)
    x, xv = padded(rng.normal(0, 1, (m, k)), pad, dtype)
    w0 = rng.normal(0, 0.05, (n, k))
    if weight == "int4":
        buf = H.quantize_int4(w0.astype(np.float32).reshape(-1)) if n * k else np.zeros(1, np.uint8)
        q, s = R.int4_parts(buf, n, k)
        wv, mag = q * s, 55.0 * s        # (16 + nibble) and -24 are summed apart: at most 31 + 24 times the scale
        w = K().Int4Weight(T().from_numpy(buf.copy()).cuda(), n, k)
    else:
        w, wv = padded(w0, pad, dtype)
        mag = np.abs(wv)
    b, bv = dev(rng.normal(0, 1, n), dtype) if bias else (None, 0.0)
    c, cv = padded(rng.normal(0, 1, (m, n)), pad, dtype) if mul else (None, 1.0)
    d, dv = padded(rng.normal(0, 1, (m, n)), pad, dtype) if res else (None, 0.0)
    od = out or dtype
    print(f"linear {m}x{n}x{k} {dtype} {weight} {act} pad {pad}", flush=True)
    y = K().linear(ctx(), x, w, bias=b, act=act, mul=c, residual=d, out_dtype=tdt(od))
    z = xv @ wv.T + bv
    want = R.act(z, act) * cv + dv
    # f32 sums of k terms and the bias; activations have slopes below 1.13 and
    # are computed to 2^-20; then the epilogue's roundings and the output's
    sums = (k + 40) * 2.0 ** -24 * (np.abs(xv) @ mag.T + np.abs(bv))
    err = (1.13 * sums + 2.0 ** -20 * np.abs(z)) * np.abs(cv) + 2.0 ** -22 * (np.abs(want) + np.abs(dv))
    assert y.shape == (m, n) and y.dtype == tdt(od)
    off = np.abs(f64(y) - want)
    assert (off <= err + R.half_ulp(np.abs(want) + err, od)).all(), float((off - err).max())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("weight", ["same", "int4"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (1, 1, 1), (3, 17, 33), (16, 128, 128), (17, 100, 96), (33, 65, 1000),
                                   (64, 256, 160), (65, 129, 64), (130, 200, 257), (257, 300, 352), (200, 64, 31)])
def test_linear_shapes(m, n, k, weight, dtype):
    check_linear(m, n, k, dtype, weight)


@pytest.mark.parametrize("m", [1, 5, 40, 150])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_linear_epilogue(m, act):
    check_linear(m, 132, 96, "bf16", act=act, bias=True, mul=True, res=True)
    check_linear(m, 131, 64, "f16", "int4", act=act, bias=True, mul=True, res=True, out="f32", pad=3)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("m", [2, 20, 140])
def test_linear_strides(m, pad):
    check_linear(m, 150, 136, "bf16", bias=True, mul=True, res=True, pad=pad)
    check_linear(m, 150, 160, "f16", "int4", res=True, pad=pad)


@pytest.mark.parametrize("m", [1, 100])
@pytest.mark.parametrize("weight", ["same", "int4"])
def test_linear_no_columns(m, weight):
    check_linear(m, 40, 0, "bf16", weight, act="silu", bias=True, res=True)


def test_linear_no_rows():
    t = T()
    y = K().linear(ctx(), t.empty(0, 64, dtype=t.bfloat16, device="cuda"), t.empty(32, 64, dtype=t.bfloat16, device="cuda"))
    assert y.shape == (0, 32)


@pytest.mark.parametrize("m", [3, 200])
def test_linear_into_its_residual_and_on_a_stream(m):
    t = T()
    rng = np.random.default_rng(5)
    x, xv = dev(rng.normal(0, 1, (m, 192)), "bf16")
    w, wv = dev(rng.normal(0, 0.05, (96, 192)), "bf16")
    r, rv = dev(rng.normal(0, 1, (m, 96)), "bf16")
    s = t.cuda.Stream()
    s.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(s):
        y = K().linear(ctx(), x, w, residual=r, out=r)
    s.synchronize()
    assert y is r
    want = xv @ wv.T + rv
    err = 240 * 2.0 ** -24 * (np.abs(xv) @ np.abs(wv).T) + 2.0 ** -22 * (np.abs(want) + np.abs(rv))
    assert (np.abs(f64(y) - want) <= err + R.half_ulp(np.abs(want) + err, "bf16")).all()


@pytest.mark.parametrize("m", [4, 100])
def test_linear_nonfinite_stays_in_its_row(m):
    t = T()
    x = t.randn(m, 128, device="cuda").to(t.bfloat16)
    w = t.randn(80, 128, device="cuda").to(t.bfloat16)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    y = K().linear(ctx(), x, w)
    fine = t.isfinite(y)
    assert t.isnan(y[1]).all() and not fine[2].any()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert fine[keep].all()


def test_linear_refusals():
    t, k, H = T(), K(), __import__("haagenti_amd")
    x = t.zeros(4, 64, dtype=t.bfloat16, device="cuda")
    w = t.zeros(32, 64, dtype=t.bfloat16, device="cuda")
    bad = [
        (lambda: k.linear(ctx(), x.float(), w), H.UNSUPPORTED),
        (lambda: k.linear(ctx(), x, w.half()), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x, w[:, :32]), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x.t().contiguous().t(), w), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x, w, act="swish"), H.UNSUPPORTED),
        (lambda: k.linear(ctx(), x, w, bias=x[0, :31]), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x, w, residual=x), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x, w, out_dtype=t.float16), H.UNSUPPORTED),
        (lambda: k.linear(ctx(), x.cpu(), w), H.INVALID_ARGUMENT),
        (lambda: k.linear(ctx(), x, k.Int4Weight(t.zeros(100, dtype=t.uint8, device="cuda"), 32, 64)), H.UNEXPECTED_EOF),
    ]
    for call, code in bad:
        with pytest.raises(H.HaagentiError) as e:
            call()
        assert e.value.code == code


# ---------------------------------------------------------------- plan

def check_plan(lens, new, bs, width, free, tokens=None, head=0, spare=3, seed=0):
    rng = np.random.default_rng(seed)
    held = [min(max((max(n, 0) + bs - 1) // bs, 0), width) for n in lens]
    ids = rng.permutation(sum(held) + free)
    table = np.full((len(lens), width), -1, np.int64)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = ids[at:at + n]
        at += n
    cap = len(ids) + spare
    ring = np.full(cap, -5, np.int64)
    for j in range(free):
        ring[(head + j) % cap] = ids[at + j]
    tokens = sum(max(a, 0) for a in new) + 4 if tokens is None else tokens
    want = R.plan(lens, new, table, ring, (head, free), bs, tokens)
    dt, dr, ds = i32(table), i32(ring), i32([head, free])
    p = K().kv_plan(ctx(), i32(lens), i32(new), dt, dr, ds, bs, tokens)
    got = dict(start=p.start, kv_len=p.kv_len, status=p.status, slots=p.slots, table=dt, ring=dr, state=p.state)
    for key, v in got.items():
        assert (v.cpu().numpy() == np.asarray(want[key])).all(), key
    assert ds.cpu().tolist() == [head, free]
    return want


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 7, 300, 1024, 1025, 3000])
def test_plan_ragged(n, bs):
    rng = np.random.default_rng(n + bs)
    lens = rng.integers(0, 500, n)
    new = np.where(rng.random(n) < 0.1, -1, rng.integers(0, 3, n) * rng.integers(0, 60, n))
    check_plan(lens, new, bs, 48, 20 * n, head=17 * n, seed=n)


def test_plan_edges():
    check_plan([0], [0], 16, 4, 2)
    check_plan([0, 16, 15, 17], [1, 1, 1, 1], 16, 4, 5, head=6)
    check_plan([16, 0], [0, 5000], 16, 320, 400)                       # a long prompt
    # blocks run out: later requests that need none are served
    w = check_plan([16, 3, 16, 5, 40], [16, 2, 17, 1, 100], 16, 10, 2)
    assert w["status"] == [0, 0, 8, 0, 8]
    # rows too wide for the table, too many for the slots, negative lengths
    w = check_plan([30, 60, 4, -2], [2, 20, 3, 1], 16, 4, 9, tokens=30)
    assert w["status"] == [0, 2, 0, 7]
    w = check_plan([0, 0, 0], [5, 6, 0], 16, 4, 9, tokens=9)
    assert w["status"] == [0, 2, 0]
    # everything ends; a full ring
    check_plan([33, 1, 0], [-1, -1, -1], 16, 4, 3, head=2, spare=0)


def test_plan_no_requests():
    t = T()
    e = t.empty(0, dtype=t.int32, device="cuda")
    p = K().kv_plan(ctx(), e, e, t.empty(0, 4, dtype=t.int32, device="cuda"), i32([3, 4]), i32([1, 1]), 16, 5)
    assert p.start.cpu().tolist() == [0] and p.slots.cpu().tolist() == [-1] * 5 and p.state.cpu().tolist() == [1, 1]


def test_plan_refusals():
    t, k, H = T(), K(), __import__("haagenti_amd")
    a = dict(lens=i32([1]), new=i32([1]), table=i32([[0]]), ring=i32([1, 2]), state=i32([0, 2]), block_size=16, tokens=3)
    for change, code in [(dict(block_size=24), H.UNSUPPORTED), (dict(lens=i32([1, 2])), H.INVALID_ARGUMENT),
                         (dict(state=i32([1])), H.INVALID_ARGUMENT), (dict(new=t.ones(1, device="cuda")), H.INVALID_ARGUMENT),
                         (dict(ring=t.arange(4, dtype=t.int32)), H.INVALID_ARGUMENT)]:
        with pytest.raises(H.HaagentiError) as e:
            k.kv_plan(ctx(), **{**a, **change})
        assert e.value.code == code


# ---------------------------------------------------------------- cache

def new_cache(blocks, bs, heads, dim, seed):
    """A cache with something in every block; (cache, key integers, value integers by token, scales)."""
    rng = np.random.default_rng(seed)
    k = rng.integers(1, 256, (blocks, heads, bs, dim)).astype(np.uint8)
    v = rng.integers(1, 256, (blocks, heads, bs, dim)).astype(np.uint8)
    ks = R.up8(rng.uniform(0.005, 0.03, (blocks, heads)))
    vs = R.up8(rng.uniform(0.005, 0.03, (blocks, heads)))
    t = T()
    c = K().KvCache(ctx(), t.from_numpy(k).cuda(), t.from_numpy(np.swapaxes(v, 2, 3).copy()).cuda(),
                    t.from_numpy(ks.astype(np.float32)).cuda(), t.from_numpy(vs.astype(np.float32)).cuda())
    return c, k.astype(np.float64) - 128, v.astype(np.float64) - 128, ks, vs


def run_slots(bs, blocks, runs):
    """Slots of runs (block, first token, rows); a run may go on into the blocks listed after it."""
    out = []
    for ids, first, n in runs:
        out += [ids[(first + i) // bs] * bs + (first + i) % bs for i in range(n)]
    return out


def check_append(bs, heads, dim, dtype, runs, blocks=9, pad=0, seed=0, change=None):
    rng = np.random.default_rng(seed)
    c, kq, vq, ks, vs = new_cache(blocks, bs, heads, dim, seed)
    slots = run_slots(bs, blocks, runs)
    slots = slots + [-1, blocks * bs, -7]
    n = len(slots)
    wide = rng.normal(0, 1, (n, 3 * heads * dim + pad)) * rng.choice([0.2, 1.0, 4.0], (n, 1))
    if change:
        change(wide, heads, dim)
    qkv, v = dev(wide, dtype)
    k_rows, v_rows = (qkv[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in (1, 2))
    kv, vv = (v[:, i * heads * dim:(i + 1) * heads * dim].reshape(n, heads, dim) for i in (1, 2))
    c.append(k_rows, v_rows, i32(slots))
    for codes, scale, q0, s0, rows, last in ((c.k, c.k_scale, kq, ks, kv, False), (c.v, c.v_scale, vq, vs, vv, True)):
        q, s = R.append(q0, s0, rows, slots, bs)
        got = codes.cpu().numpy().astype(np.float64) - 128
        got = np.swapaxes(got, 2, 3) if last else got
        assert (f64(scale) == s).all()
        assert (got == q).all()
    return c


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_append_runs(bs, dim, dtype):
    check_append(bs, 3, dim, dtype, [((4,), 0, 1), ((2,), bs - 1, 1), ((7,), 3, bs - 5), ((1, 0), 5, bs + 2), ((8,), 0, bs)],
                 seed=bs + dim)


@pytest.mark.parametrize("pad", [1, 2, 8])
def test_append_strides(pad):
    check_append(32, 2, 64, "bf16", [((3, 1), 9, 40), ((0,), 4, 2)], pad=pad)


def test_append_nonfinite_and_zeros():
    def change(w, heads, dim):
        w[0, :] = 0.0
        w[3, heads * dim:] = np.inf
        w[4, heads * dim + 3::7] = -np.inf
        w[5, heads * dim + 2::5] = np.nan
        w[6, :] *= 1e-30
    check_append(16, 2, 64, "bf16", [((3,), 0, 1), ((4,), 7, 3), ((5,), 2, 3)], change=change)


def test_append_row_by_row_and_all_at_once_read_alike():
    """Rows of falling size leave a scale set by the first: one call or many, the same codes."""
    t = T()
    rng = np.random.default_rng(3)
    rows = rng.normal(0, 1, (40, 2, 64)) * np.geomspace(4, 0.1, 40)[:, None, None]
    rows[[0, 16, 32], :, 0] = 30.0
    x, _ = dev(rows, "f16")
    slots = i32(run_slots(16, 9, [((5, 2, 8), 0, 40)]))
    a = new_cache(9, 16, 2, 64, 1)[0]
    b = new_cache(9, 16, 2, 64, 1)[0]
    a.append(x, x, slots)
    for i in range(40):
        b.append(x[i:i + 1], x[i:i + 1], slots[i:i + 1])
    assert all(t.equal(p, q) for p, q in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bs,dim", [(16, 64), (32, 96), (64, 128), (128, 256), (16, 192)])
def test_read(bs, dim, dtype):
    t = T()
    c, kq, vq, ks, vs = new_cache(6, bs, 3, dim, 2)
    ids = [4, 0, 5, 4, 6, -1]
    k, v = c.read(i32(ids), dtype=tdt(dtype))
    for got, q, s in ((k, kq, ks), (v, vq, vs)):
        want = np.swapaxes(q * s[:, :, None, None], 1, 2)
        want = np.concatenate([want[[4, 0, 5, 4]], np.zeros((2,) + want.shape[1:])])
        assert t.equal(got.cpu(), t.from_numpy(want).to(tdt(dtype)))


def test_cache_refusals():
    t, k, H = T(), K(), __import__("haagenti_amd")
    c = new_cache(3, 16, 2, 64, 0)[0]
    x = t.zeros(2, 2, 64, dtype=t.float16, device="cuda")
    s = i32([0, 1])
    q = t.zeros(2, 4, 64, dtype=t.float16, device="cuda")
    table, start, kv = i32([[0, 1]]), i32([0, 2]), i32([2])
    odd = k.KvCache(ctx(), t.zeros(3, 2, 24, 64, dtype=t.uint8, device="cuda"),
                    t.zeros(3, 2, 64, 24, dtype=t.uint8, device="cuda"), c.k_scale, c.v_scale)
    dim = k.KvCache(ctx(), t.zeros(3, 2, 16, 80, dtype=t.uint8, device="cuda"),
                    t.zeros(3, 2, 80, 16, dtype=t.uint8, device="cuda"), c.k_scale, c.v_scale)
    bad = [
        (lambda: odd.append(x, x, s), H.UNSUPPORTED),
        (lambda: dim.read(s), H.UNSUPPORTED),
        (lambda: c.append(x.float(), x.float(), s), H.UNSUPPORTED),
        (lambda: c.append(x, x.bfloat16(), s), H.INVALID_ARGUMENT),
        (lambda: c.append(x, x, s[:1]), H.INVALID_ARGUMENT),
        (lambda: c.append(x[:, :1], x, s), H.INVALID_ARGUMENT),
        (lambda: c.append(x, x, s.long()), H.INVALID_ARGUMENT),
        (lambda: c.read(s, dtype=t.int8), H.UNSUPPORTED),
        (lambda: c.attention(q[:, :3], table, start, kv), H.INVALID_ARGUMENT),
        (lambda: c.attention(q.float(), table, start, kv), H.UNSUPPORTED),
        (lambda: c.attention(q, table, start[:1], kv), H.INVALID_ARGUMENT),
        (lambda: c.attention(q.cpu(), table, start, kv), H.INVALID_ARGUMENT),
        (lambda: k.KvCache(ctx(), c.k, c.k, c.k_scale, c.v_scale), H.INVALID_ARGUMENT),
    ]
    for call, code in bad:
        with pytest.raises(H.HaagentiError) as e:
            call()
        assert e.value.code == code


# ---------------------------------------------------------------- attention

def check_attention(lens, rows, q_heads, heads, dim, bs, dtype, seed=0, pad=0, scales=None, extra=0, size=1.0, max_q=None,
                    max_kv=None, drop=(), q_change=None):
    """Requests of lens cached tokens (rows of them new), blocks dealt out unordered; drop: (request, column)
    entries of the table replaced by ids that are no blocks."""
    rng = np.random.default_rng(seed)
    counts = [(n + bs - 1) // bs for n in lens]
    blocks = sum(counts) + 2
    c, kq, vq, ks, vs = new_cache(blocks, bs, heads, dim, seed)
    if scales is not None:
        ks, vs = scales(rng, ks, vs)
        c.k_scale.copy_(T().from_numpy(ks)), c.v_scale.copy_(T().from_numpy(vs))
        ks, vs = f64(c.k_scale), f64(c.v_scale)
    ids = rng.permutation(blocks)
    width = max(counts + [1]) + 1
    table = np.full((len(lens), width), -1, np.int64)
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1]) + extra
    wide = rng.normal(0, size, (total, q_heads * (dim + pad)))
    if q_change:
        q_change(wide)
    qt, qv = dev(wide, dtype)
    qt = qt.view(total, q_heads, dim + pad)[:, :, :dim]
    qv = qv.reshape(total, q_heads, dim + pad)[:, :, :dim]
    lost = table.copy()
    for r, col in drop:
        lost[r, col] = blocks + 3 * r
    print(f"attention {lens} {rows} {q_heads}/{heads}x{dim} bs {bs} {dtype}", flush=True)
    o = K().KvCache.attention(c, qt, i32(lost), i32(start), i32(lens), max_q=max_q, max_kv=max_kv)
    got = f64(o)
    assert o.shape == (total, q_heads, dim) and o.dtype == tdt(dtype)
    for r, n in enumerate(lens):
        if rows[r] == 0:
            continue
        b = table[r, :counts[r]]
        key = (kq[b] * ks[b][:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:max(n, 0)]
        val = (vq[b] * vs[b][:, :, None, None]).swapaxes(1, 2).reshape(-1, heads, dim)[:max(n, 0)]
        gone = [x for (rr, col) in drop if rr == r for x in range(col * bs, min((col + 1) * bs, n))]
        assert not gone or rows[r] == 1
        keep = np.setdiff1d(np.arange(n), gone)
        want, mass, most = R.attention(qv[start[r]:start[r + 1]], key[keep], val[keep], len(keep), dim ** -0.5)
        # scores: f32 sums of dim terms, and queries of bf16 to 2^-25 of their row's largest; an error d of a
        # score changes p and the sum by d each; p is rounded to 11 bits, or to 2^-25 of the largest value scale
        # where it is small; exp and the sums to 2^-18; then the output
        d = most * ((dim + 8) * 2.0 ** -24 + dim * 2.0 ** -25)
        top = 127 * float(vs[b].max()) if len(b) else 0.0
        err = mass * (2 * d + 2.0 ** -11 + 2.0 ** -18) + top * 2.0 ** -25
        off = np.abs(got[start[r]:start[r + 1]] - want)
        assert (off <= err + R.half_ulp(np.abs(want) + err, dtype)).all(), (r, float((off - err).max()))
    assert (got[start[-1]:] == 0).all()
    return o


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_attention_step(bs, dim, dtype):
    check_attention([1, 15, 64, 65, 257, 700], [1] * 6, 8, 2, dim, bs, dtype, seed=bs + dim)


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (6, 2), (10, 2), (16, 1), (7, 7), (24, 1), (40, 2)])
@pytest.mark.parametrize("rows", [1, 3])
def test_attention_groups(q_heads, heads, rows):
    check_attention([5, 300, 129], [rows] * 3, q_heads, heads, 64, 32, "bf16", seed=q_heads + rows)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("bs", [16, 128])
def test_attention_prompt(bs, dim, dtype):
    check_attention([90, 200, 33], [90, 70, 17], 4, 2, dim, bs, dtype, seed=bs + dim)


def test_attention_mixed():
    check_attention([700, 150, 1, 64, 300], [1, 150, 1, 64, 5], 8, 2, 64, 32, "bf16", extra=3)
    check_attention([40, 31], [0, 31], 4, 4, 64, 16, "f16", extra=1)


def test_attention_long_splits_join():
    check_attention([9000, 17, 2500], [1, 1, 1], 8, 1, 64, 64, "bf16")
    check_attention([9000], [2], 4, 1, 128, 128, "f16")
    check_attention([5000], [1], 4, 1, 96, 16, "f16", max_kv=5000, max_q=1)


def test_attention_empty_rows():
    # left out by the plan (nothing seen), and prompts longer than what is held
    o = check_attention([0, 10, 3], [2, 1, 7], 4, 2, 64, 16, "bf16")
    assert (o[:2] == 0).all() and (o[3:7] == 0).all() and (o[7:] != 0).any()
    o = check_attention([0, 20], [40, 60], 4, 1, 64, 16, "f16")
    assert (o[:80] == 0).all()


def test_attention_strides():
    check_attention([70, 33], [1, 33], 4, 2, 64, 16, "bf16", pad=3)
    check_attention([70, 33], [1, 33], 4, 2, 64, 16, "f16", pad=8)


def test_attention_scales_far_apart():
    def far(rng, ks, vs):
        return ks, R.up8(vs * 10.0 ** rng.integers(-4, 4, vs.shape))
    check_attention([300, 128], [1, 1], 4, 1, 64, 16, "bf16", scales=far)
    check_attention([300, 128], [60, 20], 4, 1, 64, 16, "bf16", scales=far)

    def none(rng, ks, vs):
        return ks * 0, vs * 0
    o = check_attention([300, 70], [1, 70], 4, 1, 64, 16, "bf16", scales=none)
    assert (o == 0).all()


def test_attention_scales_of_unseen_blocks():
    """Blocks that no request holds may be scaled by anything."""
    t = T()
    c = new_cache(6, 16, 2, 64, 0)[0]
    for s in (c.k_scale, c.v_scale):
        s[0], s[5] = float("nan"), float("inf")
    q = t.randn(42, 4, 64, device="cuda").half()
    o = c.attention(q, i32([[1, 0, 5], [3, 2, 4]]), i32([0, 1, 42]), i32([16, 48]))
    assert t.isfinite(o).all()


def test_attention_large_queries():
    check_attention([100, 40], [1, 40], 4, 2, 64, 16, "bf16", size=40.0)

    t = T()
    o = check_attention([1, 30], [1, 30], 4, 2, 64, 16, "bf16", q_change=lambda w: w.__imul__(1e-30))
    assert t.isfinite(o).all()
    # far beyond f16: the largest score takes all
    c = new_cache(2, 16, 1, 64, 1)[0]
    q = t.randn(1, 1, 64, device="cuda").mul(1e30).bfloat16()
    o = c.attention(q, i32([[1]]), i32([0, 1]), i32([16]))
    assert t.isfinite(o).all()


def test_attention_nan_query_stays_in_its_row():
    t = T()
    c = new_cache(9, 16, 2, 64, 0)[0]
    for rows in ([1, 1, 1], [20, 30, 10]):
        n = sum(rows)
        q = t.randn(n, 4, 64, device="cuda").bfloat16()
        q[1, 2, 3] = float("nan")
        start = np.concatenate([[0], np.cumsum(rows)])
        o = c.attention(q, i32(np.arange(9).reshape(3, 3)), i32(start), i32([40, 30, 45]))
        bad = t.isnan(o).any(2)
        assert bad[1, 2] and int(bad.sum()) == 1


def test_attention_ids_that_are_no_blocks():
    check_attention([100, 60], [1, 1], 4, 2, 64, 16, "bf16", drop=[(0, 2), (0, 6), (1, 0)])


def test_attention_bounds_that_are_tight():
    check_attention([333, 20], [1, 1], 4, 2, 64, 32, "bf16", max_q=1, max_kv=333)
    check_attention([333, 120], [80, 120], 4, 2, 64, 32, "bf16", max_q=120, max_kv=333)


def test_offsets_past_32_bits():
    """The last blocks of a cache of more than 4 GiB a side."""
    t = T()
    blocks, bs, heads, dim = (1 << 32) // (64 * 8 * 128) + 40, 64, 8, 128
    if t.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB of device memory")
    c = K().KvCache.create(ctx(), blocks, bs, heads, dim)
    small = new_cache(3, bs, heads, dim, 4)[0]
    table = i32([[blocks - 1, blocks - 30, 2]])
    rows = t.randn(2, 150, heads, dim, device="cuda").bfloat16()
    slots = [(blocks - 1) * bs + i for i in range(64)] + [(blocks - 30) * bs + i for i in range(64)] + [2 * bs + i for i in range(22)]
    c.append(rows[0], rows[1], i32(slots))
    small.append(rows[0], rows[1], i32(list(range(150))))
    q = t.randn(9, 16, dim, device="cuda").bfloat16()
    for n in (1, 9):
        a = c.attention(q[:n], table, i32([0, n]), i32([150]))
        b = small.attention(q[:n], i32([[0, 1, 2]]), i32([0, n]), i32([150]))
        assert t.equal(a, b)
    for x, y in zip(c.read(table.view(-1)[:2]), small.read(i32([0, 1]))):
        assert t.equal(x, y)


def test_a_step_replayed_from_a_graph():
    """Plan, append and attention captured once and replayed on other lengths and rows."""
    t = T()
    bs, heads, dim, n = 16, 2, 64, 3
    k = K()
    ring, state = k.free_ring(40)
    cache = k.KvCache.create(ctx(), 40, bs, heads, dim)
    lens, new = i32([0] * n), i32([1] * n)
    table = t.full((n, 12), -1, dtype=t.int32, device="cuda")
    q = t.zeros(n, 4, dim, dtype=t.bfloat16, device="cuda")
    kv = t.zeros(2, n, heads, dim, dtype=t.bfloat16, device="cuda")

    def step():
        p = k.kv_plan(ctx(), lens, new, table, ring, state, bs, n)
        cache.append(kv[0], kv[1], p.slots)
        o = cache.attention(q, table, p.start, p.kv_len, max_q=1, max_kv=600)
        state.copy_(p.state)
        lens.copy_(p.kv_len)
        return o

    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        step()                 # sizes the context's scratch
    t.cuda.current_stream().wait_stream(side)
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        out = step()
    hist = [(kv.clone(), 1)]   # the first, eager step
    plain = k.KvCache.create(ctx(), 40, bs, heads, dim)
    plain_table = i32(np.arange(36).reshape(n, 12))
    for i in range(20):
        kv.normal_()
        q.normal_()
        g.replay()
        t.cuda.synchronize()
        hist.append((kv.clone(), 1))
        # the same rows appended row by row elsewhere
        for j, (rows, _) in enumerate(hist if i == 0 else hist[-1:]):
            at = (0 if i == 0 else i + 1) + j
            plain.append(rows[0], rows[1], i32([(r * 12 + at // bs) * bs + at % bs for r in range(n)]))
        want = plain.attention(q, plain_table, i32([0, 1, 2, 3]), i32([i + 2] * n), max_q=1, max_kv=600)
        assert t.equal(out, want), i
    assert lens.cpu().tolist() == [21] * n
