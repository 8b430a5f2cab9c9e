"""Rotary positions on the GPU against their 64-bit form: axes, pairings,
sizes, strides, far positions, in place, and back again."""
import numpy as np
import pytest

import norm_ref as R
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def check(tokens, heads, dim, sections, dtype="bf16", interleaved=False, inverse=False, far=1000, extra=0, in_place=False,
          seed=0, base=10000.0):
    t, rng = G.T(), np.random.default_rng(seed)
    pairs = sum(sections)
    whole, wv = G.dev(rng.normal(size=(tokens, heads + extra, dim)), dtype)
    x, xv = whole[:, extra // 2:extra // 2 + heads], wv[:, extra // 2:extra // 2 + heads]
    pos = rng.integers(-far, far + 1, size=(len(sections), tokens)).astype(np.int32)
    freq = (base ** (-np.arange(pairs) / max(pairs, 1))).astype(np.float32)
    want, bound = R.rotary(xv, pos, freq, sections, interleaved, inverse)
    p, f = t.from_numpy(pos).cuda(), t.from_numpy(freq).cuda()
    before = whole.clone()
    y = G.K().rotary(G.ctx(), x, p if len(sections) > 1 or seed % 2 else p[0], f,
                     sections=sections if len(sections) > 1 else None, interleaved=interleaved, inverse=inverse,
                     out=x if in_place else None)
    if not in_place:
        assert t.equal(whole, before)
    else:
        assert y.data_ptr() == x.data_ptr()
        a, b = extra // 2, extra // 2 + heads
        assert t.equal(whole[:, :a], before[:, :a]) and t.equal(whole[:, b:], before[:, b:])
    off = np.abs(G.f64(y) - want) - bound - np.where(bound > 0, R.half_step(np.abs(want) + bound, dtype), 0)
    assert not (off > 0).any(), (float(off.max()), np.argwhere(off > 0)[:4])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,sections", [
    (64, [32]), (128, [64]), (128, [16, 24, 24]), (80, [20, 20]), (96, [48]), (256, [128]), (128, [32]), (2, [1]), (3, [1]),
    (30, [1, 5, 2, 7]), (130, [3, 0, 62]), (1024, [512]), (70, [9, 4]), (17, [8]), (48, [0, 24])])
def test_dimensions_and_axes(dim, sections, interleaved):
    for dtype in ("bf16", "f16", "f32"):
        check(5, 3, dim, sections, dtype, interleaved, inverse=dim % 4 == 0, extra=dim % 3, seed=dim)
        check(5, 3, dim, sections, dtype, interleaved, in_place=True, extra=2, seed=dim + 1)


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 72), (2, 513), (7, 40), (511, 5), (513, 1), (2500, 3), (9000, 2)])
def test_tokens_and_heads(tokens, heads):
    check(tokens, heads, 64, [32], extra=1, seed=tokens)
    check(tokens, heads, 64, [10, 11, 11], "f32", True, extra=1, seed=tokens)


def test_far_positions():
    for dtype in ("bf16", "f32"):
        check(64, 2, 128, [64], dtype, far=1000000, seed=3)
        check(64, 2, 128, [64], dtype, far=2 ** 31 - 1, seed=4)
        check(64, 2, 128, [64], dtype, far=2 ** 31 - 1, seed=5, base=0.001)  # frequencies above 1


def test_the_inverse_is_the_gradient():
    """sum(dy R x) = sum(R^-1 dy x): what the gradient has to be, for a map that is linear; and there and back."""
    t, k, c = G.T(), G.K(), G.ctx()
    g = t.Generator("cuda").manual_seed(1)
    x, dy = (t.randn(50, 4, 96, generator=g, device="cuda") for _ in range(2))
    pos = t.randint(0, 100000, (2, 50), generator=g, device="cuda").int()
    f = 10000.0 ** -(t.arange(48, device="cuda") / 48.0)
    for inter in (False, True):
        y = k.rotary(c, x, pos, f, sections=(20, 28), interleaved=inter)
        dx = k.rotary(c, dy, pos, f, sections=(20, 28), interleaved=inter, inverse=True)
        a, b = (dy.double() * y.double()).sum(), (dx.double() * x.double()).sum()
        # each of the 19200 terms is off by at most 2^-21 of its pair's magnitudes
        assert abs(float(a - b)) < 2.0 ** -21 * 2 * float((dy.double().abs() * x.double().abs()).sum() + 19200)
        back = k.rotary(c, y, pos, f, sections=(20, 28), interleaved=inter, inverse=True)
        assert float((back - x).abs().max()) < 2.0 ** -20 * float(x.abs().max())


def test_one_row_of_positions_for_all_axes_and_other_strides():
    t, k, c = G.T(), G.K(), G.ctx()
    g = t.Generator("cuda").manual_seed(2)
    x = t.randn(33, 6, 64, generator=g, device="cuda").bfloat16()
    pos = t.arange(33, device="cuda").int()
    f = 100.0 ** -(t.arange(32, device="cuda") / 32.0)
    want = k.rotary(c, x, pos, f)
    assert t.equal(k.rotary(c, x, pos.expand(3, 33), f, sections=[8, 20, 4]), want)
    wide = t.cat([pos[None], pos[None] + 5, pos[None]]).contiguous()
    assert t.equal(k.rotary(c, x, wide[::2], f, sections=[30, 2]), want)
    heads_first = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert t.equal(k.rotary(c, heads_first, pos, f), want)
    out = t.zeros(6, 33, 64, dtype=t.bfloat16, device="cuda").transpose(0, 1)
    assert t.equal(k.rotary(c, x, pos, f, out=out), want)
    one = x[:1].expand(33, 6, 64)     # one row read by all tokens
    assert t.equal(k.rotary(c, one, pos, f), k.rotary(c, one.contiguous(), pos, f))


def test_nothing_to_turn():
    t, k, c = G.T(), G.K(), G.ctx()
    f, none = t.ones(4, device="cuda"), t.ones(0, device="cuda")
    for shape in ((0, 3, 8), (3, 0, 8)):
        x = t.ones(shape, device="cuda")
        assert k.rotary(c, x, t.zeros(shape[0], dtype=t.int32, device="cuda"), f).shape == shape
    x = t.randn(3, 2, 9, device="cuda")
    assert t.equal(k.rotary(c, x, G.i32([1, 2, 3]), none), x)
    assert t.equal(k.rotary(c, x, G.i32([1, 2, 3]), none, out=x), x)
    assert t.equal(k.rotary(c, x, G.i32([0, 0, 0]), f), x)


def test_captured_and_replayed():
    t, k, c = G.T(), G.K(), G.ctx()
    x = t.randn(300, 10, 128, device="cuda").bfloat16()
    pos, f = t.zeros(300, dtype=t.int32, device="cuda"), 100.0 ** -(t.arange(64, device="cuda") / 64.0)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        y = k.rotary(c, x, pos, f)
    for i in range(4):
        pos.copy_(t.arange(300, device="cuda") * i)
        graph.replay()
        assert t.equal(y, k.rotary(c, x, pos, f))


def test_refusals():
    t, k, c, H = G.T(), G.K(), G.ctx(), __import__("haagenti_amd")
    x = t.zeros(4, 2, 64, device="cuda")
    p, f = G.i32([0, 1, 2, 3]), t.ones(32, device="cuda")
    bad = [
        (dict(x=x.double()), H.UNSUPPORTED), (dict(x=x[0]), H.INVALID_ARGUMENT), (dict(x=x.cpu()), H.INVALID_ARGUMENT),
        (dict(x=x.transpose(1, 2)), H.INVALID_ARGUMENT), (dict(positions=p.long()), H.INVALID_ARGUMENT),
        (dict(positions=p[:3]), H.INVALID_ARGUMENT), (dict(positions=p.cpu()), H.INVALID_ARGUMENT),
        (dict(positions=p.expand(2, 4)), H.INVALID_ARGUMENT), (dict(inv_freq=f.half()), H.INVALID_ARGUMENT),
        (dict(inv_freq=t.ones(33, device="cuda")), H.INVALID_ARGUMENT), (dict(sections=[31]), H.INVALID_ARGUMENT),
        (dict(positions=p.expand(2, 4), sections=[40, -8]), H.INVALID_ARGUMENT),
        (dict(positions=p.expand(5, 4), sections=[8, 8, 8, 8, 0]), H.INVALID_ARGUMENT),
        (dict(out=x.half()), H.INVALID_ARGUMENT), (dict(out=x[:3]), H.INVALID_ARGUMENT),
        (dict(out=t.zeros(1, 2, 64, device="cuda").expand(4, 2, 64)), H.INVALID_ARGUMENT),
        (dict(x=x[:3], out=x[1:], positions=p[:3]), H.INVALID_ARGUMENT),
        (dict(x=t.zeros(1, 1, 1200, device="cuda"), positions=p[:1], inv_freq=t.ones(513, device="cuda")), H.UNSUPPORTED),
        (dict(x=x.clone().requires_grad_()), H.UNSUPPORTED), (dict(inv_freq=f.clone().requires_grad_()), H.UNSUPPORTED),
    ]
    for i, (args, code) in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            k.rotary(c, **{**dict(x=x, positions=p, inv_freq=f), **args})
        assert e.value.code == code, i
