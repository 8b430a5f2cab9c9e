"""Attention over values whose scales lie far apart: what a row gets depends
on the tokens that it sees and on no others, to f16's 11 bits of each
probability whatever the scales are."""
import numpy as np
import pytest

import compute_ref as R
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def attention(q, kq, ks, vq, vs, rows, scale, lost=2.0 ** -25, bits=11):
    """One request, its blocks in order: q (rows, heads, dim), integers of keys and values (blocks, kv heads, tokens,
    dim) with their scales; the output, and what its f16 probabilities and its scores may cost."""
    group = q.shape[1] // kq.shape[1]
    bs = kq.shape[2]
    n = kq.shape[0] * bs
    key = (kq * ks[:, :, None, None]).swapaxes(1, 2).reshape(n, -1, q.shape[2])
    vi = np.abs(vq).swapaxes(1, 2).reshape(n, -1, q.shape[2])
    val = (vq * vs[:, :, None, None]).swapaxes(1, 2).reshape(n, -1, q.shape[2])
    out, err = np.zeros_like(q), np.zeros_like(q)
    for i in range(q.shape[0]):
        seen = rows[i]
        for h in range(q.shape[1]):
            j = h // group
            z = key[:seen, j] @ q[i, h] * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i, h] = p @ val[:seen, j]
            # a score of f32 sums, and of bf16 queries to `lost` of the row's largest: its error d changes p and the sum
            # by d each; p is rounded to `bits` bits, or to 2^-25 of the row's largest probability times scale where it is
            # small; exp and the sums to 2^-18
            dim = q.shape[2]
            d = (np.abs(key[:seen, j]) @ np.abs(q[i, h])).max() * scale * (dim + 8) * 2.0 ** -24
            d += np.abs(key[:seen, j]).sum(1).max() * np.abs(q[i, h]).max() * scale * lost
            d += np.abs(z).max() * 2.0 ** -22
            s = np.repeat(vs[:, j], bs)[:seen]
            err[i, h] = p @ np.abs(val[:seen, j]) * (2 * d + 2.0 ** -bits + 2.0 ** -18) + vi[:seen, j].sum(0) * (p * s).max() * 2.0 ** -25
    return out, err


def close(o, want, err, dtype):
    """Within err and the output's rounding; what lies beyond f16's range is an infinity of its sign."""
    got = G.f64(o)
    with np.errstate(invalid="ignore"):
        fine = np.abs(got - want) <= err + R.half_ulp(np.abs(want) + err, dtype)
    if dtype == "f16":
        fine |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + err >= 65520)
    assert fine.all(), (int((~fine).sum()), float(np.abs(got - want)[~fine].max()))


def check(kv_len, rows, q_heads, heads, dim, bs, dtype, scales, keys=None, seed=0, size=1.0):
    rng = np.random.default_rng(seed)
    blocks = (kv_len + bs - 1) // bs
    c, kq, vq, ks, vs = G.new_cache(blocks, bs, heads, dim, seed)
    t = G.T()
    vs = R.up8(vs * scales(rng, blocks)[:, None])
    c.v_scale.copy_(t.from_numpy(vs))
    vs = G.f64(c.v_scale)
    if keys:
        kq = keys(rng, kq)
        c.k.copy_(t.from_numpy((kq + 128).astype(np.uint8)))
    q, qv = G.dev(rng.normal(0, size, (rows, q_heads, dim)), dtype)
    print(f"attention {kv_len} {rows} {q_heads}/{heads}x{dim} bs {bs} {dtype}", flush=True)
    o = c.attention(q, G.i32(np.arange(blocks)[None]), G.i32([0, rows]), G.i32([kv_len]), max_q=rows, max_kv=kv_len)
    want, err = attention(qv, kq, ks, vq, vs, kv_len - rows + 1 + np.arange(rows), dim ** -0.5)
    close(o, want, err, dtype)


HIDDEN = [
    (17, 2, 4, 2, 64, 16),        # the first row sees one block, the second a token of the next
    (70, 8, 2, 1, 128, 64),
    (33, 3, 4, 1, 96, 32),
    (64, 48, 4, 2, 64, 16),       # tiles: rows that see 17 to 64 tokens of one tile
    (300, 260, 4, 1, 128, 16),
    (130, 70, 1, 1, 256, 32),
    (1100, 3, 4, 1, 64, 16),      # several chunks, hidden ones in the last
]


@pytest.mark.parametrize("power", [12, 20, 30])
@pytest.mark.parametrize("kv_len,rows,q_heads,heads,dim,bs", HIDDEN)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_hidden_blocks_of_large_scale(kv_len, rows, q_heads, heads, dim, bs, dtype, power):
    """The last rows' own blocks are scaled up: rows before them don't see these."""
    check(kv_len, rows, q_heads, heads, dim, bs, dtype,
          lambda rng, n: 2.0 ** np.where(np.arange(n) >= (kv_len - rows) // bs + 1, power if dtype == "bf16" else power - 12, 0))


@pytest.mark.parametrize("gap", [10.0, 30.0, 200.0])
@pytest.mark.parametrize("kv_len,rows", [(64, 1), (200, 2), (1500, 1), (1500, 60), (64, 64)])
def test_visible_blocks_of_large_scale_and_small_probability(kv_len, rows, gap):
    """Every other block's keys lie `gap` below in score, their values are 2^30 larger."""
    def keys(rng, kq):
        kq = kq.copy()
        kq[:, :, :, 0] = np.where(np.arange(kq.shape[0]) % 2, -127, 127)[:, None, None]
        return kq

    rng = np.random.default_rng(1)
    c, kq, vq, ks, vs = G.new_cache((kv_len + 15) // 16, 16, 1, 64, 0)
    del c
    n = len(ks)
    ks[:] = R.up8(np.asarray([0.01]))
    vs = R.up8(vs * np.where(np.arange(n) % 2, 2.0 ** 30, 1.0)[:, None])
    kq = keys(rng, kq)
    t = G.T()
    q = rng.normal(0, 0.01, (rows, 2, 64))
    q[:, :, 0] = gap * 8 / (254 * ks[0, 0])
    q, qv = G.dev(q, "bf16")
    c = G.K().KvCache(G.ctx(), t.from_numpy((kq + 128).astype(np.uint8)).cuda(),
                      t.from_numpy((np.swapaxes(vq, 2, 3) + 128).astype(np.uint8).copy()).cuda(),
                      t.from_numpy(ks.astype(np.float32)).cuda(), t.from_numpy(vs.astype(np.float32)).cuda())
    o = c.attention(q, G.i32(np.arange(n)[None]), G.i32([0, rows]), G.i32([kv_len]), max_q=rows, max_kv=kv_len)
    want, err = attention(qv, kq, ks, vq, vs, kv_len - rows + 1 + np.arange(rows), 0.125)
    close(o, want, err, "bf16")


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("power", [-110, -60, 100])
def test_all_scales_far_from_one(rows, power):
    check(90, rows, 2, 1, 64, 16, "bf16", lambda rng, n: np.full(n, 2.0 ** power))
    check(700, rows, 2, 1, 64, 16, "bf16", lambda rng, n: 2.0 ** (power + rng.integers(-8, 9, n)))


@pytest.mark.parametrize("rows", [1, 40])
def test_scales_of_zero_beside_others(rows):
    check(128, rows, 2, 1, 64, 16, "bf16", lambda rng, n: np.where(np.arange(n) % 3, 0.0, 1.0))
    check(128, rows, 2, 1, 64, 16, "bf16", lambda rng, n: np.where(np.arange(n) < n - 1, 0.0, 2.0 ** 20))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("power", [-8, -17, -24, -30])
def test_small_parts_of_queries_beside_a_large_one(rows, power):
    """A dimension of the query far larger than the others meets keys of 0: the others' scores keep their bits."""
    t = G.T()
    c, kq, vq, ks, vs = G.new_cache(6, 16, 2, 64, 5)
    kq[:, :, :, 7] = 0
    c.k.copy_(t.from_numpy((kq + 128).astype(np.uint8)))
    for size in (1.0, 2.0 ** 30, 2.0 ** -60):
        q = np.random.default_rng(rows).normal(0, 1, (rows, 4, 64))
        q[:, :, 7] = 2.0 ** -power * np.where(np.arange(rows) % 2, -1.5, 1.0)[:, None]
        q, qv = G.dev(q * size, "bf16")
        o = c.attention(q, G.i32(np.arange(6)[None]), G.i32([0, rows]), G.i32([90]), scale=0.125 / size)
        want, err = attention(qv / size, kq, ks, vq, vs, 90 - rows + 1 + np.arange(rows), 0.125, lost=2.0 ** -39)
        close(o, want, err, "bf16")


@pytest.mark.parametrize("rows", [1, 40])
def test_queries_of_any_size(rows):
    t = G.T()
    c, kq, vq, ks, vs = G.new_cache(6, 16, 2, 64, 5)
    for power in (-133, -126, -120, -113, -100, 100, 120):
        q = np.random.default_rng(3).normal(0, 1, (rows, 4, 64)).clip(-3, 3)
        if power < -120:
            q = np.rint(q * 8) / 8 if power == -126 else np.rint(q)
        q, qv = G.dev(q * 2.0 ** power, "bf16")
        scale = 2.0 ** min(-power, 126) * 0.125
        o = c.attention(q, G.i32(np.arange(6)[None]), G.i32([0, rows]), G.i32([90]), scale=scale)
        want, err = attention(qv * scale, kq, ks, vq, vs, 90 - rows + 1 + np.arange(rows), 1.0)
        close(o, want, err, "bf16")


@pytest.mark.parametrize("kv_len", [2, 3, 5, 17, 40, 700])
@pytest.mark.parametrize("q_heads,heads,dim,bs", [(32, 2, 64, 16), (24, 8, 128, 32), (6, 3, 96, 64), (8, 8, 256, 128), (16, 1, 192, 16)])
def test_few_columns_keep_22_bits(kv_len, q_heads, heads, dim, bs):
    t = G.T()
    blocks = (kv_len + bs - 1) // bs
    c, kq, vq, ks, vs = G.new_cache(blocks, bs, heads, dim, kv_len)
    vq = np.abs(vq) * np.where(np.arange(bs) % 2, -1, 1)[:, None]  # sums that cancel
    c.v.copy_(t.from_numpy((np.swapaxes(vq, 2, 3) + 128).astype(np.uint8)))
    q, qv = G.dev(np.random.default_rng(kv_len).normal(0, 0.3, (1, q_heads, dim)), "f16")
    o = c.attention(q, G.i32(np.arange(blocks)[None]), G.i32([0, 1]), G.i32([kv_len]), max_q=1, max_kv=kv_len)
    want, err = attention(qv, kq, ks, vq, vs, [kv_len], dim ** -0.5, lost=0.0, bits=21)
    close(o, want, err, "f16")


@pytest.mark.parametrize("rows", [2, 50])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 0.0])
def test_hidden_blocks_of_any_scale(rows, bad):
    """Rows don't take part in what later tokens' blocks are scaled by, whatever that is."""
    t = G.T()
    outs = []
    for worst in (0.01, bad):
        c = G.new_cache(4, 16, 1, 64, 3)[0]
        c.v_scale[1:], c.k_scale[1:] = worst, worst
        q = t.randn(rows, 4, 64, generator=t.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
        outs.append(c.attention(q, G.i32([[0, 1, 2, 3]]), G.i32([0, rows]), G.i32([17 if rows == 2 else 64])))
    seen = 17 - 1 if rows == 2 else 64 - rows + 1
    first = 17 - seen if rows == 2 else 16 - seen + 1
    assert first >= 1 and t.isfinite(outs[1][:first]).all() and t.equal(outs[0][:first], outs[1][:first])


def test_a_request_is_the_same_beside_tokens_that_it_does_not_see():
    """A prompt's first rows get bit for bit what they get where the later tokens' values are small."""
    t = G.T()
    for rows in (3, 64):
        outs = []
        for power in (0, 25):
            c = G.new_cache(4, 16, 1, 64, 3)[0]
            c.v_scale[1:] *= 2.0 ** power
            q = t.randn(rows, 4, 64, generator=t.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
            kv = 16 + rows - 2 if rows < 64 else 64
            outs.append(c.attention(q, G.i32([[0, 1, 2, 3]]), G.i32([0, rows]), G.i32([kv])))
        first = 2 if rows < 64 else 16
        assert t.equal(outs[0][:first], outs[1][:first])
        assert not t.equal(outs[0][first:], outs[1][first:])
